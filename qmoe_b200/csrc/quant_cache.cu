// A paged key/value cache in 8 bits: append, read back, and the attention of single tokens over it.
#include <math.h>

#include "serving.cuh"

namespace qmoe {

constexpr float kScaleFloor = 1.17549435e-38f;  // 2^-126: a row of zeros still has a scale to divide by

struct CacheView {
  uint8_t *k_codes, *v_codes;
  float *k_scale, *v_scale;
  const int32_t *table;
  int32_t *status;
  int n_pages, page_shift, kv_heads, head_dim, max_pages;
};

// Index of (page, head, place) in the scale arrays for a position of a sequence, head 0; -1 when the
// position has no valid page.
__device__ __forceinline__ long long cache_slot(const CacheView &c, int seq, long long pos) {
  if (pos < 0 || pos >= ((long long)c.max_pages << c.page_shift)) return -1;
  const int page = c.table[(long long)seq * c.max_pages + (pos >> c.page_shift)];
  if (page < 0 || page >= c.n_pages) return -1;
  return (((long long)page * c.kv_heads) << c.page_shift) + (pos & ((1 << c.page_shift) - 1));
}

__device__ __forceinline__ uint8_t to_e4m3(float v) { return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3); }
__device__ __forceinline__ float from_e4m3(uint8_t c) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
}

// Code nearest to x / s, ties to the even code.  x * (1 / s) is within 2^-23 of the quotient, so it
// decides unless a rounding border lies that near; then the sign of x - border * s, which one fused
// multiply-add gives exactly, does.  (The border has 5 bits, s 24: both operands are scaled up where
// their difference could leave the normal range.)
__device__ __forceinline__ float beyond_border(float x, float s, float border) {
  const float up = s < 1e-25f ? 1.8446744e19f : 1.f;  // 2^64
  return fmaf(-border, s * up, x * up);
}
template <int FMT>
__device__ __forceinline__ uint8_t quantise(float x, float s, float inv) {
  const float q = x * inv;
  if (FMT == QMOE_CACHE_E4M3) {
    const uint8_t lo = to_e4m3(q * (1.f - 0x1p-21f)), hi = to_e4m3(q * (1.f + 0x1p-21f));
    if (lo == hi) return lo;
    const float r = beyond_border(x, s, 0.5f * (from_e4m3(lo) + from_e4m3(hi))) * copysignf(1.f, q);
    return r > 0.f ? hi : (r < 0.f ? lo : ((lo & 1) ? hi : lo));
  } else {
    const float n = rintf(q);
    int code = (int)n;
    if (fabsf(fabsf(q - n) - 0.5f) < 0x1p-14f) {
      const float f = floorf(q), r = beyond_border(x, s, f + 0.5f);
      code = (int)f;
      if (r > 0.f || (r == 0.f && (code & 1))) code++;
    }
    return (uint8_t)(int8_t)code;
  }
}
template <int FMT>
__device__ __forceinline__ float code_value(uint8_t c) {
  return FMT == QMOE_CACHE_E4M3 ? from_e4m3(c) : (float)(int8_t)c;
}

struct RowsArgs {
  CacheView c;
  const void *k, *v;     // append: sources
  void *k_out, *v_out;   // read: destinations
  long long k_row, k_head, v_row, v_head;
  const int32_t *cu, *start;
  int n_seqs;
  long long n_rows;
};

// One warp per row, head and tensor: four values per lane and step.
template <typename T, int FMT>
__global__ void __launch_bounds__(256) k_cache_append(const RowsArgs a) {
  const int lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int which = (int)(item & 1);
  const int head = (int)((item >> 1) % a.c.kv_heads);
  const long long row = (item >> 1) / a.c.kv_heads;
  if (row >= a.n_rows) return;
  const int seq = packed_seq(a.cu, a.n_seqs, (int)row);
  if (seq < 0) return;
  const long long slot0 = cache_slot(a.c, seq, (long long)a.start[seq] + (row - a.cu[seq]));
  if (slot0 < 0) {
    if (head == 0 && which == 0 && lane == 0) atomicAdd(a.c.status, 1);
    return;
  }
  const long long slot = slot0 + ((long long)head << a.c.page_shift);
  const T *src = which ? reinterpret_cast<const T *>(a.v) + row * a.v_row + head * a.v_head
                       : reinterpret_cast<const T *>(a.k) + row * a.k_row + head * a.k_head;
  const int d = a.c.head_dim, width = cache_row_bytes(d);
  float x[2][4], amax = 0.f;
  bool finite = true;
#pragma unroll
  for (int j = 0; j < 2; j++)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int at = 128 * j + 4 * lane + i;
      x[j][i] = at < d ? to_f32(src[at]) : 0.f;
      finite = finite && fabsf(x[j][i]) <= FLT_MAX;
      amax = fmaxf(amax, fabsf(x[j][i]));
    }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  finite = __all_sync(0xffffffffu, finite);
  const float s = fmaxf(__fdiv_rn(amax, FMT == QMOE_CACHE_E4M3 ? 448.f : 127.f), kScaleFloor);
  const float inv = __fdiv_rn(1.f, s);
  uint8_t *dst = (which ? a.c.v_codes : a.c.k_codes) + slot * width;
#pragma unroll
  for (int j = 0; j < 2; j++) {
    if (128 * j + 4 * lane >= width) break;
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) word |= (uint32_t)(finite ? quantise<FMT>(x[j][i], s, inv) : 0) << (8 * i);
    *reinterpret_cast<uint32_t *>(dst + 128 * j + 4 * lane) = word;
  }
  if (lane == 0) (which ? a.c.v_scale : a.c.k_scale)[slot] = finite ? s : __int_as_float(0x7fffffff);
}

template <typename T, int FMT>
__global__ void __launch_bounds__(256) k_cache_read(const RowsArgs a) {
  const int lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int which = (int)(item & 1);
  const int head = (int)((item >> 1) % a.c.kv_heads);
  const long long row = (item >> 1) / a.c.kv_heads;
  if (row >= a.n_rows) return;
  const int seq = packed_seq(a.cu, a.n_seqs, (int)row);
  if (seq < 0) return;
  const long long slot0 = cache_slot(a.c, seq, (long long)a.start[seq] + (row - a.cu[seq]));
  if (slot0 < 0 && head == 0 && which == 0 && lane == 0) atomicAdd(a.c.status, 1);
  const long long slot = slot0 + ((long long)head << a.c.page_shift);
  const int d = a.c.head_dim, width = cache_row_bytes(d);
  const uint8_t *src = (which ? a.c.v_codes : a.c.k_codes) + slot * width;
  const float s = slot0 < 0 ? 0.f : (which ? a.c.v_scale : a.c.k_scale)[slot];
  T *dst = reinterpret_cast<T *>(which ? a.v_out : a.k_out) + (row * a.c.kv_heads + head) * d;
  for (int at = 4 * lane; at < d; at += 128) {
    const uint32_t word = slot0 < 0 ? 0u : *reinterpret_cast<const uint32_t *>(src + at);
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (at + i < d) dst[at + i] = from_f32<T>(code_value<FMT>((uint8_t)(word >> (8 * i))) * s);
  }
}

struct PagedArgs {
  CacheView c;
  const void *q;
  void *out;
  long long q_row, q_head;
  const int32_t *lengths;
  const float *bias;
  int n_dist, heads;
  float scale;
};

// One CTA per sequence and query head: every warp runs a running-maximum softmax over its share of the
// positions, the warps' partial results are merged at the end.
constexpr int kPagedWarps = 8;
template <typename T, int FMT>
__global__ void __launch_bounds__(32 * kPagedWarps) k_decode_paged(const PagedArgs a) {
  __shared__ float s_acc[kPagedWarps][256], s_m[kPagedWarps], s_sum[kPagedWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, head = blockIdx.x, seq = blockIdx.y;
  const int d = a.c.head_dim, width = cache_row_bytes(d), kv = head / (a.heads / a.c.kv_heads);
  const int len = a.lengths[seq];
  const int seen = (int)min((long long)len, (long long)a.c.max_pages << a.c.page_shift);  // positions that the table can hold
  if (seen < len && head % (a.heads / a.c.kv_heads) == 0 && threadIdx.x == 0) atomicAdd(a.c.status, 1);
  const T *q = reinterpret_cast<const T *>(a.q) + seq * a.q_row + head * a.q_head;
  float qv[8], acc[8];
#pragma unroll
  for (int j = 0; j < 8; j++) {
    qv[j] = lane + 32 * j < d ? to_f32(q[lane + 32 * j]) : 0.f;
    acc[j] = 0.f;
  }
  float m = -INFINITY, sum = 0.f;
  for (int t = warp; t < seen; t += kPagedWarps) {
    const long long slot0 = cache_slot(a.c, seq, t);
    if (slot0 < 0) {
      if (lane == 0 && head % (a.heads / a.c.kv_heads) == 0 && (t & 15) == 0) atomicAdd(a.c.status, 1);
      continue;
    }
    const long long slot = slot0 + ((long long)kv << a.c.page_shift);
    const uint8_t *k = a.c.k_codes + slot * width, *v = a.c.v_codes + slot * width;
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (lane + 32 * j < d) dot += qv[j] * code_value<FMT>(k[lane + 32 * j]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    float s = dot * a.c.k_scale[slot] * a.scale;
    if (a.bias != nullptr) s += a.bias[(size_t)head * a.n_dist + min(len - 1 - t, a.n_dist - 1)];
    const float m_new = fmaxf(m, s), base = m_new == -INFINITY ? 0.f : m_new;
    const float keep = expf(m - base), p = expf(s - base), pv = p != 0.f ? p * a.c.v_scale[slot] : 0.f;
    m = m_new;
    sum = sum * keep + p;
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (lane + 32 * j < d) acc[j] = acc[j] * keep + pv * code_value<FMT>(v[lane + 32 * j]);
  }
#pragma unroll
  for (int j = 0; j < 8; j++)
    if (lane + 32 * j < d) s_acc[warp][lane + 32 * j] = acc[j];
  if (lane == 0) {
    s_m[warp] = m;
    s_sum[warp] = sum;
  }
  __syncthreads();
  float top = -INFINITY, total = 0.f;
  for (int w = 0; w < kPagedWarps; w++) top = fmaxf(top, s_m[w]);
  if (top == -INFINITY) top = 0.f;
  for (int w = 0; w < kPagedWarps; w++) total += s_sum[w] * expf(s_m[w] - top);
  T *out = reinterpret_cast<T *>(a.out) + ((long long)seq * a.heads + head) * d;
  for (int i = threadIdx.x; i < d; i += blockDim.x) {
    float o = 0.f;
    for (int w = 0; w < kPagedWarps; w++) o += s_acc[w][i] * expf(s_m[w] - top);
    out[i] = from_f32<T>(total == 0.f ? 0.f : o / total);
  }
}

static int cache_view(const char *fn, const qmoe_quant_cache *cache, const int32_t *table, int32_t *status, int n_seqs,
                      int max_pages, int dtype, CacheView *view) {
  if (cache == nullptr || n_seqs < 0 || max_pages < 0 || cache->n_pages < 0 || cache->kv_heads < 1 || cache->head_dim < 1) {
    set_error("%s: null cache or bad shape", fn);
    return QMOE_ERR_INVALID_ARG;
  }
  if (dtype != QMOE_BF16 && dtype != QMOE_FP16) {
    set_error("%s: activations are bf16 or fp16", fn);
    return QMOE_ERR_INVALID_ARG;
  }
  if (cache->format != QMOE_CACHE_E4M3 && cache->format != QMOE_CACHE_INT8) {
    set_error("%s: unknown cache format", fn);
    return QMOE_ERR_INVALID_ARG;
  }
  const int page = cache->page_size;
  if (page < 16 || page > 1024 || (page & (page - 1)) != 0 || cache->head_dim > 256) {
    set_error("%s: page_size is a power of two in [16, 1024], head_dim at most 256", fn);
    return QMOE_ERR_UNSUPPORTED;
  }
  if (n_seqs > 0 && (status == nullptr || (max_pages > 0 && table == nullptr))) {
    set_error("%s: null device pointer", fn);
    return QMOE_ERR_INVALID_ARG;
  }
  if (cache->n_pages > 0 && (!cache->k_codes || !cache->v_codes || !cache->k_scale || !cache->v_scale)) {
    set_error("%s: null cache pointer", fn);
    return QMOE_ERR_INVALID_ARG;
  }
  if (((reinterpret_cast<uintptr_t>(cache->k_codes) | reinterpret_cast<uintptr_t>(cache->v_codes)) & 15u) != 0) {
    set_error("%s: codes must be 16-byte aligned", fn);
    return QMOE_ERR_INVALID_ARG;
  }
  int shift = 4;
  while ((1 << shift) < page) shift++;
  *view = CacheView{reinterpret_cast<uint8_t *>(cache->k_codes), reinterpret_cast<uint8_t *>(cache->v_codes),
                    cache->k_scale, cache->v_scale, table, status, cache->n_pages, shift, cache->kv_heads,
                    cache->head_dim, max_pages};
  return QMOE_OK;
}

}  // namespace qmoe

using namespace qmoe;

#define QMOE_CACHE_DISPATCH(kernel, dtype, format, grid, block, stream, args)                                  \
  do {                                                                                                         \
    if ((dtype) == QMOE_BF16 && (format) == QMOE_CACHE_E4M3)                                                   \
      QMOE_LAUNCH((kernel<__nv_bfloat16, QMOE_CACHE_E4M3>), grid, block, 0, stream, args);                     \
    else if ((dtype) == QMOE_BF16)                                                                             \
      QMOE_LAUNCH((kernel<__nv_bfloat16, QMOE_CACHE_INT8>), grid, block, 0, stream, args);                     \
    else if ((format) == QMOE_CACHE_E4M3)                                                                      \
      QMOE_LAUNCH((kernel<__half, QMOE_CACHE_E4M3>), grid, block, 0, stream, args);                            \
    else                                                                                                       \
      QMOE_LAUNCH((kernel<__half, QMOE_CACHE_INT8>), grid, block, 0, stream, args);                            \
    QMOE_CUDA(cudaGetLastError());                                                                             \
  } while (0)

extern "C" {

int qmoe_cache_append(const qmoe_quant_cache *cache, const void *k_dev, const void *v_dev, int64_t k_row,
                      int64_t k_head, int64_t v_row, int64_t v_head, const int32_t *cu_dev,
                      const int32_t *start_dev, const int32_t *page_table_dev, int32_t *status_dev, int n_seqs,
                      int max_pages, int64_t n_rows, int dtype, int device, void *stream) {
  RowsArgs a{};
  const int rc = cache_view(__func__, cache, page_table_dev, status_dev, n_seqs, max_pages, dtype, &a.c);
  if (rc != QMOE_OK) return rc;
  QMOE_REQUIRE(n_rows >= 0 && n_rows <= 0x7fffffffLL, "bad number of rows");
  if (n_rows == 0 || n_seqs == 0) return QMOE_OK;
  QMOE_REQUIRE(k_dev && v_dev && cu_dev && start_dev, "null device pointer");
  a.k = k_dev;
  a.v = v_dev;
  a.k_row = k_row;
  a.k_head = k_head;
  a.v_row = v_row;
  a.v_head = v_head;
  a.cu = cu_dev;
  a.start = start_dev;
  a.n_seqs = n_seqs;
  a.n_rows = n_rows;
  const int64_t items = 2 * n_rows * cache->kv_heads;
  QMOE_REQUIRE(items <= 8LL * 0x7fffffffLL, "too many rows");
  DeviceGuard guard(device);
  if (!guard.ok) return cuda_fail(cudaGetLastError(), "cudaSetDevice");
  QMOE_CACHE_DISPATCH(k_cache_append, dtype, cache->format, (unsigned)((items + 7) / 8), 256,
                      reinterpret_cast<cudaStream_t>(stream), a);
  return QMOE_OK;
}

int qmoe_cache_read(const qmoe_quant_cache *cache, void *k_out_dev, void *v_out_dev, const int32_t *cu_dev,
                    const int32_t *start_dev, const int32_t *page_table_dev, int32_t *status_dev, int n_seqs,
                    int max_pages, int64_t n_rows, int dtype, int device, void *stream) {
  RowsArgs a{};
  const int rc = cache_view(__func__, cache, page_table_dev, status_dev, n_seqs, max_pages, dtype, &a.c);
  if (rc != QMOE_OK) return rc;
  QMOE_REQUIRE(n_rows >= 0 && n_rows <= 0x7fffffffLL, "bad number of rows");
  if (n_rows == 0 || n_seqs == 0) return QMOE_OK;
  QMOE_REQUIRE(k_out_dev && v_out_dev && cu_dev && start_dev, "null device pointer");
  a.k_out = k_out_dev;
  a.v_out = v_out_dev;
  a.cu = cu_dev;
  a.start = start_dev;
  a.n_seqs = n_seqs;
  a.n_rows = n_rows;
  const int64_t items = 2 * n_rows * cache->kv_heads;
  QMOE_REQUIRE(items <= 8LL * 0x7fffffffLL, "too many rows");
  DeviceGuard guard(device);
  if (!guard.ok) return cuda_fail(cudaGetLastError(), "cudaSetDevice");
  QMOE_CACHE_DISPATCH(k_cache_read, dtype, cache->format, (unsigned)((items + 7) / 8), 256,
                      reinterpret_cast<cudaStream_t>(stream), a);
  return QMOE_OK;
}

int64_t qmoe_decode_paged_work_bytes(int n_seqs, int heads, int kv_heads, int head_dim, int max_pages, int page_size,
                                     int device) {
  (void)n_seqs, (void)heads, (void)kv_heads, (void)head_dim, (void)max_pages, (void)page_size, (void)device;
  return 0;
}

int qmoe_decode_attention_paged(const qmoe_quant_cache *cache, const void *q_dev, int64_t q_row, int64_t q_head,
                                void *out_dev, const int32_t *page_table_dev, const int32_t *lengths_dev,
                                const float *rel_bias_dev, int n_dist, int32_t *status_dev, void *work_dev, int n_seqs,
                                int heads, int max_pages, float scale, int dtype, int device, void *stream) {
  PagedArgs a{};
  const int rc = cache_view(__func__, cache, page_table_dev, status_dev, n_seqs, max_pages, dtype, &a.c);
  if (rc != QMOE_OK) return rc;
  QMOE_REQUIRE(heads >= 1 && heads % cache->kv_heads == 0, "heads must be a positive multiple of kv_heads");
  QMOE_REQUIRE((rel_bias_dev == nullptr) == (n_dist == 0) && n_dist >= 0, "bias and n_dist do not agree");
  QMOE_REQUIRE(isfinite(scale), "scale is not finite");
  if (n_seqs == 0) return QMOE_OK;
  QMOE_REQUIRE(q_dev && out_dev && lengths_dev, "null device pointer");
  if (n_seqs > 65535) {
    set_error("%s: at most 65535 sequences", __func__);
    return QMOE_ERR_UNSUPPORTED;
  }
  (void)work_dev;
  a.q = q_dev;
  a.out = out_dev;
  a.q_row = q_row;
  a.q_head = q_head;
  a.lengths = lengths_dev;
  a.bias = rel_bias_dev;
  a.n_dist = n_dist;
  a.heads = heads;
  a.scale = scale > 0.f ? scale : 1.f / sqrtf((float)cache->head_dim);
  DeviceGuard guard(device);
  if (!guard.ok) return cuda_fail(cudaGetLastError(), "cudaSetDevice");
  const dim3 grid((unsigned)heads, (unsigned)n_seqs);
  QMOE_CACHE_DISPATCH(k_decode_paged, dtype, cache->format, grid, 32 * kPagedWarps, reinterpret_cast<cudaStream_t>(stream), a);
  return QMOE_OK;
}

}  // extern "C"
