// Shared pieces of the serving kernels: 16-bit activations, packed batches, 8-bit cache codes.
#pragma once

#include <cuda_fp16.h>
#include <float.h>

#include "common.cuh"

namespace qmoe {

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32(float v) { return v; }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }

// Rows [begin, end) of sequence s of a packed batch, clamped to the tensor's `total` rows.
__device__ __forceinline__ int2 packed_rows(const int32_t *__restrict__ cu, int s, long long total) {
  const int lim = (int)(total > 0x7fffffffLL ? 0x7fffffffLL : total);
  const int b = min(max(cu[s], 0), lim);
  return make_int2(b, min(max(cu[s + 1], b), lim));
}

// Sequence that owns `row`: the last s with cu[s] <= row; -1 when the row lies before the first or
// behind the last sequence.
__device__ __forceinline__ int packed_seq(const int32_t *__restrict__ cu, int n_seqs, int row) {
  if (row < cu[0] || row >= cu[n_seqs]) return -1;
  int lo = 0, hi = n_seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu[mid] <= row) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Two fp32 values in one 64-bit register: one instruction works on both.
using pair_t = unsigned long long;
__device__ __forceinline__ pair_t pair_of(float lo, float hi) {
  pair_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
  return v;
}
__device__ __forceinline__ void pair_split(pair_t v, float &lo, float &hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ pair_t pair_fma(pair_t a, pair_t b, pair_t c) {
  pair_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ pair_t pair_add(pair_t a, pair_t b) {
  pair_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ pair_t pair_mul(pair_t a, pair_t b) {
  pair_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// Lets a kernel use `bytes` of dynamic shared memory on a device; remembered, as the attribute call costs a
// microsecond.  `regs` > 0: fails unless the kernel was built with that many registers a thread.
int allow_shared(const void *kernel, int bytes, int device, int regs = 0);

__host__ __device__ constexpr int cache_row_bytes(int head_dim) { return (head_dim + 15) & ~15; }

}  // namespace qmoe
