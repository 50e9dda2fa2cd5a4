// Causal attention over a packed batch of prompts (qmoe_prompt_attention).
#include <math.h>

#include "serving.cuh"

namespace qmoe {

struct PromptArgs {
  const void *q, *k, *v;
  void *out;
  const int32_t *cu_q, *cu_k;
  const float *bias;
  qmoe_prompt_shape s;
};

// One warp per query row and head, keys one after another with a running maximum: 32 lanes share the
// head's values.
template <typename T, int J>  // J = ceil(head_dim / 32)
__global__ void __launch_bounds__(128) k_prompt_rows(const PromptArgs a) {
  const int lane = threadIdx.x & 31, head = blockIdx.x;
  const int row = blockIdx.y * 4 + (threadIdx.x >> 5);
  if (row >= a.s.total_q) return;
  const int seq = packed_seq(a.cu_q, a.s.n_seqs, row);
  if (seq < 0) return;
  const int2 rq = packed_rows(a.cu_q, seq, a.s.total_q), rk = packed_rows(a.cu_k, seq, a.s.total_k);
  const int last = row - rq.x + (rk.y - rk.x) - (rq.y - rq.x);  // last key that the query sees
  const int kv = head / (a.s.heads / a.s.kv_heads), d = a.s.head_dim;
  const T *q = reinterpret_cast<const T *>(a.q) + row * a.s.q_row + head * a.s.q_head;
  const float *bias = a.bias != nullptr ? a.bias + (size_t)head * a.s.n_dist : nullptr;
  float qv[J], acc[J];
#pragma unroll
  for (int j = 0; j < J; j++) {
    qv[j] = lane + 32 * j < d ? to_f32(q[lane + 32 * j]) : 0.f;
    acc[j] = 0.f;
  }
  float m = -INFINITY, sum = 0.f;
  for (int t = 0; t <= last; t++) {
    const T *k = reinterpret_cast<const T *>(a.k) + (rk.x + (long long)t) * a.s.k_row + kv * a.s.k_head;
    const T *v = reinterpret_cast<const T *>(a.v) + (rk.x + (long long)t) * a.s.v_row + kv * a.s.v_head;
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < J; j++)
      if (lane + 32 * j < d) dot += qv[j] * to_f32(k[lane + 32 * j]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    const float s = dot * a.s.scale + (bias != nullptr ? bias[min(last - t, a.s.n_dist - 1)] : 0.f);
    const float m_new = fmaxf(m, s);
    const float base = m_new == -INFINITY ? 0.f : m_new;  // scores of -inf only so far
    const float keep = expf(m - base), p = expf(s - base);
    m = m_new;
    sum = sum * keep + p;
#pragma unroll
    for (int j = 0; j < J; j++)
      if (lane + 32 * j < d) acc[j] = acc[j] * keep + (p != 0.f ? p * to_f32(v[lane + 32 * j]) : 0.f);  // weight 0: whatever is there
  }
  T *out = reinterpret_cast<T *>(a.out) + row * a.s.out_row + head * a.s.out_head;
#pragma unroll
  for (int j = 0; j < J; j++)
    if (lane + 32 * j < d) out[lane + 32 * j] = from_f32<T>(sum == 0.f ? 0.f : acc[j] / sum);
}

template <typename T>
static int run_prompt(const PromptArgs &a, cudaStream_t stream) {
  const dim3 grid((unsigned)a.s.heads, (unsigned)((a.s.total_q + 3) / 4));
  if (a.s.head_dim <= 64)
    QMOE_LAUNCH((k_prompt_rows<T, 2>), grid, 128, 0, stream, a);
  else if (a.s.head_dim <= 128)
    QMOE_LAUNCH((k_prompt_rows<T, 4>), grid, 128, 0, stream, a);
  else
    QMOE_LAUNCH((k_prompt_rows<T, 8>), grid, 128, 0, stream, a);
  QMOE_CUDA(cudaGetLastError());
  return QMOE_OK;
}

}  // namespace qmoe

using namespace qmoe;

extern "C" int qmoe_prompt_attention(const void *q_dev, const void *k_dev, const void *v_dev, void *out_dev,
                                     const int32_t *cu_q_dev, const int32_t *cu_k_dev, const float *rel_bias_dev,
                                     const qmoe_prompt_shape *shape, int device, void *stream) {
  QMOE_REQUIRE(shape != nullptr && cu_q_dev && cu_k_dev, "null pointer");
  PromptArgs a{q_dev, k_dev, v_dev, out_dev, cu_q_dev, cu_k_dev, rel_bias_dev, *shape};
  QMOE_REQUIRE(a.s.n_seqs >= 0 && a.s.total_q >= 0 && a.s.total_k >= 0, "negative size");
  QMOE_REQUIRE(a.s.heads >= 1 && a.s.kv_heads >= 1 && a.s.heads % a.s.kv_heads == 0 && a.s.head_dim >= 1,
               "heads must be a positive multiple of kv_heads");
  QMOE_REQUIRE(a.s.dtype == QMOE_BF16 || a.s.dtype == QMOE_FP16, "q, k and v are bf16 or fp16");
  QMOE_REQUIRE((rel_bias_dev == nullptr) == (a.s.n_dist == 0) && a.s.n_dist >= 0, "bias and n_dist do not agree");
  QMOE_REQUIRE(isfinite(a.s.scale), "scale is not finite");
  if (a.s.n_seqs == 0 || a.s.total_q == 0) return QMOE_OK;
  QMOE_REQUIRE(q_dev && out_dev && (a.s.total_k == 0 || (k_dev && v_dev)), "null device pointer");
  if (a.s.head_dim > 256 || a.s.total_q > (1 << 18) - 4 || a.s.total_k > 0x7fffffffLL) {
    set_error("%s: head_dim <= 256, 262140 query rows and 2^31 - 1 key rows are supported", __func__);
    return QMOE_ERR_UNSUPPORTED;
  }
  if (a.s.scale <= 0.f) a.s.scale = 1.f / sqrtf((float)a.s.head_dim);
  DeviceGuard guard(device);
  if (!guard.ok) return cuda_fail(cudaGetLastError(), "cudaSetDevice");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return a.s.dtype == QMOE_BF16 ? run_prompt<__nv_bfloat16>(a, st) : run_prompt<__half>(a, st);
}
