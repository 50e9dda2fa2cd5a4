// Sampling of one token per row of logits (qmoe_sample).
#include <math.h>

#include "serving.cuh"

namespace qmoe {

constexpr int kMaxVocab = 262144;
constexpr int kSampleThreads = 1024;
constexpr double kMassUnit = 35184372088832.0;  // 2^45

struct SampleArgs {
  const void *logits;
  long long row_stride;
  int vocab;
  const float *temperature, *top_p, *min_p, *uniform;
  const int32_t *top_k;
  long long *tokens;
  float *logprob;
};

// Unsigned key in the order of the logits; both zeros have the same key.
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t b = __float_as_uint(v == 0.f ? 0.f : v);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// exp((l - max) / temperature) in 64 bits, and as a multiple of 2^-45: at most 2^18 of them, each at
// most 1, fit 64 bits, and integer sums are the same in every order.
__device__ __forceinline__ double weight_of(float l, double top, double inv_t) { return exp(((double)l - top) * inv_t); }
__device__ __forceinline__ unsigned long long mass_of(double w) { return __double2ull_rn(w * kMassUnit); }

template <typename V>
__device__ __forceinline__ V block_total(V v, V *scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  V t = 0;
  for (int w = 0; w < kSampleThreads / 32; w++) t += scratch[w];
  return t;
}

// One CTA per row; the row is read again from L2 for every step.
//   1. largest logit;  2. key of the k-th largest by radix selection on counts;  3. key at which the
//   mass from the top reaches top_p by radix selection on masses;  4. per-warp segments: kept mass,
//   then the segment and the token that the uniform number falls into.
template <typename T>
__global__ void __launch_bounds__(kSampleThreads) k_sample(const SampleArgs a) {
  __shared__ unsigned long long s_sum[32], s_hist[256];
  __shared__ uint32_t s_key[32];
  __shared__ int s_cnt[32];
  __shared__ uint32_t s_prefix;
  __shared__ unsigned long long s_left;
  __shared__ int s_found;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = blockIdx.x, n = a.vocab;
  const T *logits = reinterpret_cast<const T *>(a.logits) + row * a.row_stride;
  const float t = a.temperature != nullptr ? a.temperature[row] : 1.f;

  bool bad = false;
  uint32_t top_key = 0;
  for (int i = tid; i < n; i += kSampleThreads) {
    const float l = to_f32(logits[i]);
    bad = bad || !(l <= FLT_MAX);
    top_key = max(top_key, order_key(l));
  }
  top_key = __reduce_max_sync(0xffffffffu, top_key);
  if (lane == 0) s_key[warp] = top_key;
  bad = __syncthreads_or(bad);
  for (int w = 0; w < kSampleThreads / 32; w++) top_key = max(top_key, s_key[w]);
  const float top = key_value(top_key);
  if (bad || top == -INFINITY || !(t >= 0.f) || t > FLT_MAX) {
    if (tid == 0) {
      a.tokens[row] = -1;
      if (a.logprob != nullptr) a.logprob[row] = __int_as_float(0x7fffffff);
    }
    return;
  }
  if (t == 0.f) {
    int first = n;
    for (int i = tid; i < n; i += kSampleThreads)
      if (order_key(to_f32(logits[i])) == top_key) {
        first = i;
        break;
      }
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0) s_cnt[warp] = first;
    __syncthreads();
    if (tid == 0) {
      for (int w = 0; w < kSampleThreads / 32; w++) first = min(first, s_cnt[w]);
      a.tokens[row] = first;
      if (a.logprob != nullptr) a.logprob[row] = 0.f;
    }
    return;
  }
  const double dtop = (double)top, inv_t = 1.0 / (double)t;

  // kept: keys above `edge`, and the first `edge_count` (by index) of those equal to it
  uint32_t edge = 0;
  int edge_count = n;
  const int k = a.top_k != nullptr ? a.top_k[row] : 0;
  const bool cut_k = k > 0 && k < n;
  if (cut_k) {
    uint32_t prefix = 0;
    int left = k;
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) s_hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += kSampleThreads) {
        const uint32_t key = order_key(to_f32(logits[i]));
        if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&s_hist[(key >> shift) & 255], 1ull);
      }
      __syncthreads();
      if (tid == 0) {
        int b = 255;
        while (b > 0 && s_hist[b] < (unsigned long long)left) left -= (int)s_hist[b--];
        s_prefix = prefix | ((uint32_t)b << shift);
        s_found = left;
      }
      __syncthreads();
      prefix = s_prefix;
      left = s_found;
    }
    edge = prefix;
    edge_count = left;
  }
  const float p = a.top_p != nullptr ? a.top_p[row] : 1.f;
  if (p < 1.f) {
    unsigned long long z = 0;
    for (int i = tid; i < n; i += kSampleThreads) {
      const float l = to_f32(logits[i]);
      const uint32_t key = order_key(l);
      if (key > edge || (!cut_k && key == edge)) z += mass_of(weight_of(l, dtop, inv_t));
    }
    z = block_total(z, s_sum);
    const unsigned long long edge_mass = cut_k ? mass_of(weight_of(key_value(edge), dtop, inv_t)) : 0ull;
    z += edge_mass * (unsigned long long)(cut_k ? edge_count : 0);
    // tokens before which less than `goal` lies: integers below p * z
    const unsigned long long goal = p > 0.f ? (unsigned long long)ceil((double)p * (double)z) : 0ull;
    uint32_t prefix = 0;
    unsigned long long above = 0;  // mass of the keys above the prefix's range
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) s_hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += kSampleThreads) {
        const float l = to_f32(logits[i]);
        const uint32_t key = order_key(l);
        if ((key > edge || (!cut_k && key == edge)) && (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))))
          atomicAdd(&s_hist[(key >> shift) & 255], mass_of(weight_of(l, dtop, inv_t)));
      }
      if (tid == 0 && cut_k && (shift == 24 || (edge >> (shift + 8)) == (prefix >> (shift + 8))))
        atomicAdd(&s_hist[(edge >> shift) & 255], edge_mass * (unsigned long long)edge_count);
      __syncthreads();
      if (tid == 0) {
        // the first digit, from the top, with which the mass reaches the goal (the largest logit's at least)
        int b = 255;
        unsigned long long sum = above;
        while (b > 0 && sum + s_hist[b] < max(goal, 1ull)) sum += s_hist[b--];
        s_prefix = prefix | ((uint32_t)b << shift);
        s_left = sum;
      }
      __syncthreads();
      prefix = s_prefix;
      above = s_left;
    }
    const unsigned long long w = mass_of(weight_of(key_value(prefix), dtop, inv_t));
    const unsigned long long need = max(goal, 1ull) - above;  // > 0
    const unsigned long long count = w > 0 ? (need + w - 1) / w : (unsigned long long)n;
    const int limit = prefix == edge && cut_k ? edge_count : n;
    edge = prefix;
    edge_count = (int)min(count, (unsigned long long)limit);
  }
  const float least = a.min_p != nullptr ? a.min_p[row] : 0.f;
  const double min_w = least > 0.f ? fmin((double)least, 1.0) : 0.0;

  // segments of 32-element strides, one per warp: tokens equal to the edge, then kept mass
  const int per_warp = ((n + kSampleThreads - 1) / kSampleThreads) * 32;
  const int begin = min(n, warp * per_warp), end = min(n, begin + per_warp);
  int ties = 0;
  for (int i = begin + lane; i < end; i += 32) ties += order_key(to_f32(logits[i])) == edge;
  ties = __reduce_add_sync(0xffffffffu, ties);
  if (lane == 0) s_cnt[warp] = ties;
  __syncthreads();
  int ties_before = 0;
  for (int w = 0; w < warp; w++) ties_before += s_cnt[w];
  auto kept_mass = [&](int i, int &seen, double &w) {
    const float l = i < end ? to_f32(logits[i]) : -INFINITY;
    const uint32_t key = i < end ? order_key(l) : 0u;
    const unsigned tied = __ballot_sync(0xffffffffu, i < end && key == edge);
    const int rank = seen + __popc(tied & ((1u << lane) - 1u));
    seen += __popc(tied);
    w = 0.0;
    if (i < end && (key > edge || (key == edge && rank < edge_count))) w = weight_of(l, dtop, inv_t);
    if (!(w >= min_w)) w = 0.0;
    return mass_of(w);
  };
  unsigned long long mine = 0;
  int seen = ties_before;
  double w;
  for (int i = begin; i < end; i += 32) mine += kept_mass(i + lane, seen, w);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  __syncthreads();
  if (lane == 0) s_sum[warp] = mine;
  __syncthreads();
  unsigned long long total = 0, before = 0;
  for (int v = 0; v < kSampleThreads / 32; v++) {
    if (v == warp) before = total;
    total += s_sum[v];
  }
  const float u = a.uniform[row];
  const double at = (u > 0.f ? (double)u : 0.0) * (double)total;
  unsigned long long target = at >= (double)total ? total - 1 : (unsigned long long)at;
  if (target >= total) target = total - 1;
  if (target < before || target >= before + mine) return;
  seen = ties_before;
  for (int i = begin; i < end; i += 32) {
    const unsigned long long m = kept_mass(i + lane, seen, w);
    unsigned long long upto = m;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + upto > target);
    if (hit != 0) {
      if (lane == __ffs(hit) - 1) {
        a.tokens[row] = i + lane;
        if (a.logprob != nullptr) a.logprob[row] = (float)log(w * kMassUnit / (double)total);
      }
      return;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
}

}  // namespace qmoe

using namespace qmoe;

extern "C" int qmoe_sample(const void *logits_dev, int64_t row_stride, int rows, int vocab, int dtype,
                           const float *temperature_dev, const int32_t *top_k_dev, const float *top_p_dev,
                           const float *min_p_dev, const float *uniform_dev, int64_t *tokens_dev, float *logprob_dev,
                           int device, void *stream) {
  QMOE_REQUIRE(rows >= 0 && vocab >= 1 && row_stride >= 0, "bad shape");
  QMOE_REQUIRE(dtype == QMOE_FP32 || dtype == QMOE_BF16 || dtype == QMOE_FP16, "logits are fp32, bf16 or fp16");
  if (rows == 0) return QMOE_OK;
  QMOE_REQUIRE(logits_dev && uniform_dev && tokens_dev, "null device pointer");
  if (vocab > kMaxVocab) {
    set_error("%s: at most %d logits a row are supported", __func__, kMaxVocab);
    return QMOE_ERR_UNSUPPORTED;
  }
  const SampleArgs a{logits_dev, row_stride, vocab, temperature_dev, top_p_dev, min_p_dev, uniform_dev, top_k_dev,
                     reinterpret_cast<long long *>(tokens_dev), logprob_dev};
  DeviceGuard guard(device);
  if (!guard.ok) return cuda_fail(cudaGetLastError(), "cudaSetDevice");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == QMOE_FP32)
    QMOE_LAUNCH((k_sample<float>), (unsigned)rows, kSampleThreads, 0, st, a);
  else if (dtype == QMOE_BF16)
    QMOE_LAUNCH((k_sample<__nv_bfloat16>), (unsigned)rows, kSampleThreads, 0, st, a);
  else
    QMOE_LAUNCH((k_sample<__half>), (unsigned)rows, kSampleThreads, 0, st, a);
  QMOE_CUDA(cudaGetLastError());
  return QMOE_OK;
}
