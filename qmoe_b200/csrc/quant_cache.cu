// A paged key/value cache in 8 bits: append, read back, and the attention of single tokens over it.
#include <math.h>

#include <type_traits>

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

// ---- attention of single tokens ---------------------------------------------------------------------
// The cache is read once, at 8 bits a value; everything else is arranged so that nothing but that read
// takes time.
//
// Work: sequences x key heads x blocks of 16 query heads x tiles of 16 positions, counted through in that
// order and dealt out evenly to the warps of a fixed grid, whatever the lengths are.  A warp owns a
// contiguous run of tiles; what belongs to one (sequence, head block) is a segment.  A segment that lies
// wholly in one warp's run is written to the output at once, of the others each warp leaves its part
// (maximum, sum, quotient) in the workspace, and a second kernel joins the parts.  No warp waits for another.
//
// Tile: S[heads, 16 positions] = Q K^T and O[heads, columns] += W V by mma.sync m16n8k16 in fp16 with fp32
// sums; both code formats are exact in fp16.  The order of the K axis of a product is free, so every lane's
// operand comes straight from global memory in pieces of 16 bytes: lane (g, c) of the warp (g = lane / 4,
// c = lane % 4) holds bytes 16 c .. 16 c + 15 of every 64 of key g, and columns 16 g .. of values 2c, 2c + 1,
// 2c + 8, 2c + 9.  Q is brought to fp16 by a power of two per head.
// Weights: p = exp2(s - m), w = p * value scale / r with r the largest p * value scale so far, so that rows of
// small and large scale keep their accuracy in fp16.  m and r only move when p or w grew by more than 2^8 or
// 2^12.
struct PagedArgs {
  CacheView c;
  const void *q;
  void *out;
  long long q_row, q_head;
  const int32_t *lengths;
  const float *bias;
  long long *prefix;  // tiles before every sequence, n_seqs + 1 entries (workspace)
  float *parts;       // [warp][first, last segment][rows][columns + 2]
  int n_dist, heads, n_seqs, dtype, warps;
  float scale;
};

constexpr int kPagedThreads = 128;
constexpr int kPagedMaxSeqs = 4096;
constexpr int kPagedMinTiles = 2;  // per warp
__host__ __device__ constexpr int paged_ctas(int nb) { return nb <= 5 ? 4 : (nb <= 8 ? 3 : 2); }  // per SM

struct PagedShape {
  int group, blocks, rows, width;  // query heads per key head, blocks of 16 of them, rows of a part, padded columns
};
__host__ __device__ inline PagedShape paged_shape(int heads, int kv_heads, int head_dim) {
  const int group = heads / kv_heads;
  return {group, (group + 15) / 16, group < 16 ? group : 16, cache_row_bytes(head_dim)};
}

__device__ __forceinline__ long long paged_quota(long long total, int warps) {
  const long long q = (total + warps - 1) / warps;
  return q < kPagedMinTiles ? kPagedMinTiles : q;
}
// Positions of a sequence that its row of the page table can hold.
__device__ __forceinline__ int paged_seen(const PagedArgs &a, int seq) {
  return (int)max(0LL, min((long long)a.lengths[seq], (long long)a.c.max_pages << a.c.page_shift));
}

__device__ __forceinline__ float paged_log2(float b) {  // a bias in units of log 2; the lowest values stay finite
  return b == -INFINITY ? b : fmaxf(b * 1.4426950408889634f, -FLT_MAX);
}
__device__ __forceinline__ float paged_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Four codes to two pairs of fp16: (bytes 0, 1) and (bytes 2, 3).  int8: 0x6400 + (code + 128) is 1024 +
// code + 128 in fp16.
template <int FMT>
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t &lo, uint32_t &hi) {
  if (FMT == QMOE_CACHE_E4M3) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi) : "r"(w));
  } else {
    const uint32_t u = w ^ 0x80808080u;
    const __half2 off = __half2half2(__ushort_as_half(0x6480));  // 1152
    uint32_t x = __byte_perm(u, 0x64646464u, 0x4140), y = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 hx = __hsub2(*reinterpret_cast<__half2 *>(&x), off), hy = __hsub2(*reinterpret_cast<__half2 *>(&y), off);
    lo = *reinterpret_cast<const uint32_t *>(&hx);
    hi = *reinterpret_cast<const uint32_t *>(&hy);
  }
}

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 ld_codes16(const uint8_t *p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 ld_codes8(const uint8_t *p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t ld_codes4(const uint8_t *p) {
  uint32_t v;
  asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t ld_codes2(const uint8_t *p) {
  uint16_t v;
  asm volatile("ld.global.nc.L1::no_allocate.u16 %0, [%1];" : "=h"(v) : "l"(p));
  return v;
}

__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

// Registers of one tile: NB units of 16 columns.  Keys: blocks of 64 columns, then single units.  Values:
// blocks of 128, 64, 32 and 16 columns (16, 8, 4 and 2 bytes a lane) for each of the lane's four rows.
template <int NB>
struct CacheTile {
  static constexpr int KB = NB / 4, KR = NB % 4, V16 = NB / 8, V8 = NB % 8 / 4, V4 = NB % 4 / 2, V2 = NB % 2;
  static constexpr int kWords = 4 * V16 + 2 * V8 + V4 + V2;  // value words per row and lane
  uint32_t k[2][4 * KB + KR];
  uint32_t v[4][kWords];
  float2 ks[2], vs[2];
};

template <int NB>
__device__ __forceinline__ void load_cache_tile(CacheTile<NB> &t, const CacheView &c, long long slot, int width, int left, int g,
                                                int q) {
  using C = CacheTile<NB>;
  const int units = width >> 4;
#pragma unroll
  for (int n = 0; n < 2; n++) {
    const uint8_t *row = c.k_codes + (slot + 8 * n + g) * width;
#pragma unroll
    for (int b = 0; b < C::KB; b++) {
      uint4 x = make_uint4(0u, 0u, 0u, 0u);
      if (4 * b + q < units) x = ld_codes16(row + 64 * b + 16 * q);
      t.k[n][4 * b] = x.x;
      t.k[n][4 * b + 1] = x.y;
      t.k[n][4 * b + 2] = x.z;
      t.k[n][4 * b + 3] = x.w;
    }
#pragma unroll
    for (int r = 0; r < C::KR; r++) t.k[n][4 * C::KB + r] = 4 * C::KB + r < units ? ld_codes4(row + 64 * C::KB + 16 * r + 4 * q) : 0u;
    t.ks[n] = *reinterpret_cast<const float2 *>(c.k_scale + slot + 8 * n + 2 * q);
    t.vs[n] = *reinterpret_cast<const float2 *>(c.v_scale + slot + 8 * n + 2 * q);
  }
#pragma unroll
  for (int r = 0; r < 4; r++) {
    const int at = 8 * (r >> 1) + 2 * q + (r & 1);
    const uint8_t *row = c.v_codes + (slot + at) * width;
    const bool in = at < left;  // places behind the last position may hold anything: zeros instead
#pragma unroll
    for (int b = 0; b < C::V16; b++) {
      uint4 x = make_uint4(0u, 0u, 0u, 0u);
      if (in && 128 * b + 16 * g < width) x = ld_codes16(row + 128 * b + 16 * g);
      t.v[r][4 * b] = x.x;
      t.v[r][4 * b + 1] = x.y;
      t.v[r][4 * b + 2] = x.z;
      t.v[r][4 * b + 3] = x.w;
    }
    if (C::V8) {
      const int off = 128 * C::V16 + 8 * g;
      uint2 x = make_uint2(0u, 0u);
      if (in && off < width) x = ld_codes8(row + off);
      t.v[r][4 * C::V16] = x.x;
      t.v[r][4 * C::V16 + 1] = x.y;
    }
    if (C::V4) {
      const int off = 128 * C::V16 + 64 * C::V8 + 4 * g;
      t.v[r][4 * C::V16 + 2 * C::V8] = in && off < width ? ld_codes4(row + off) : 0u;
    }
    if (C::V2) {
      const int off = 128 * C::V16 + 64 * C::V8 + 32 * C::V4 + 2 * g;
      t.v[r][C::kWords - 1] = in && off < width ? ld_codes2(row + off) : 0u;
    }
  }
}

// Column of n-tile `n` (of 2 * NB) and its column index x (0 .. 7).
template <int NB>
__device__ __forceinline__ int value_column(int n, int x) {
  using C = CacheTile<NB>;
  if (n < 16 * C::V16) return 128 * (n / 16) + 16 * x + n % 16;
  n -= 16 * C::V16;
  if (C::V8 && n < 8) return 128 * C::V16 + 8 * x + n;
  n -= 8 * C::V8;
  if (C::V4 && n < 4) return 128 * C::V16 + 64 * C::V8 + 4 * x + n;
  n -= 4 * C::V4;
  return 128 * C::V16 + 64 * C::V8 + 32 * C::V4 + 2 * x + n;
}

template <int NB, int FMT, bool WIDE>  // WIDE: more than 8 query heads per key head
__global__ void __launch_bounds__(kPagedThreads, paged_ctas(NB)) k_decode_paged(const PagedArgs a) {
  extern __shared__ long long s_prefix[];  // n_seqs + 1
  __shared__ long long s_warp[kPagedThreads / 32];
  using C = CacheTile<NB>;
  constexpr int R = WIDE ? 2 : 1;  // rows of a lane: g and g + 8
  const int tid = threadIdx.x, lane = tid & 31, g = lane >> 2, q = lane & 3;
  const PagedShape shape = paged_shape(a.heads, a.c.kv_heads, a.c.head_dim);
  const int per_seq = a.c.kv_heads * shape.blocks, d = a.c.head_dim;

  // tiles before every sequence
  long long before = 0;
  for (int s0 = 0; s0 < a.n_seqs; s0 += kPagedThreads) {
    const int s = s0 + tid;
    long long upto = s < a.n_seqs ? (long long)((paged_seen(a, s) + 15) / 16) * per_seq : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    if (lane == 31) s_warp[tid >> 5] = upto;
    __syncthreads();
    long long all = 0;
    for (int w = 0; w < kPagedThreads / 32; w++) {
      if (w < (tid >> 5)) upto += s_warp[w];
      all += s_warp[w];
    }
    if (s < a.n_seqs) s_prefix[s + 1] = before + upto;
    before += all;
    __syncthreads();
  }
  if (tid == 0) s_prefix[0] = 0;
  __syncthreads();
  if (blockIdx.x == 0)
    for (int s = tid; s <= a.n_seqs; s += kPagedThreads) a.prefix[s] = s_prefix[s];

  const long long total = before, quota = paged_quota(total, a.warps);
  const int worker = blockIdx.x * (kPagedThreads / 32) + (tid >> 5);
  const long long run_begin = worker * quota, run_end = min(total, run_begin + quota);
  const int row_floats = shape.width + 2;

  for (long long x = run_begin; x < run_end;) {
    // ---- segment: sequence, key head, block of query heads
    int lo = 0, hi = a.n_seqs - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_prefix[mid] <= x) lo = mid;
      else hi = mid - 1;
    }
    const int seq = lo, seen = paged_seen(a, seq), length = a.lengths[seq], n_tiles = (seen + 15) / 16;
    const long long in_seq = x - s_prefix[seq];
    const int which = (int)(in_seq / n_tiles), tile0 = (int)(in_seq % n_tiles);
    const long long seg_begin = x - tile0;
    const int tile1 = (int)min((long long)n_tiles, run_end - seg_begin);
    const int kv = which / shape.blocks, block = which % shape.blocks;
    const int head0 = kv * shape.group + block * 16, n_heads = min(16, shape.group - block * 16);

    // ---- queries of the lane's rows in the order of the key bytes, brought to fp16
    uint32_t qa[NB][2 * R];
    float factor[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
      const bool live = g + 8 * r < n_heads;
      const long long at = seq * a.q_row + (long long)(head0 + (live ? g + 8 * r : 0)) * a.q_head;
      auto element = [&](int col) {
        if (!live || col >= d) return 0.f;
        return a.dtype == QMOE_BF16 ? to_f32(reinterpret_cast<const __nv_bfloat16 *>(a.q)[at + col])
                                    : to_f32(reinterpret_cast<const __half *>(a.q)[at + col]);
      };
      float v[NB][4], amax = 0.f;
#pragma unroll
      for (int n = 0; n < NB; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          v[n][i] = element(n < 4 * C::KB ? 64 * (n >> 2) + 16 * q + 4 * (n & 3) + i : 16 * n + 4 * q + i);
          amax = fmaxf(amax, fabsf(v[n][i]));
        }
      amax = quad_max(amax);
      const int e = amax > 0.f && amax <= FLT_MAX ? ilogbf(amax) : 0;
      factor[r] = scalbnf(a.scale * 1.4426950408889634f, e);
#pragma unroll
      for (int n = 0; n < NB; n++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const __half2 h = __floats2half2_rn(scalbnf(v[n][2 * i], -e), scalbnf(v[n][2 * i + 1], -e));
          qa[n][i * R + r] = *reinterpret_cast<const uint32_t *>(&h);
        }
    }

    float o[2 * NB][4];
#pragma unroll
    for (int n = 0; n < 2 * NB; n++)
#pragma unroll
      for (int i = 0; i < 4; i++) o[n][i] = 0.f;
    float m[R], sum[R], unit[R];  // maximum in units of log 2, sum of p, r
#pragma unroll
    for (int r = 0; r < R; r++) {
      m[r] = -INFINITY;
      sum[r] = 0.f;
      unit[r] = 0.f;
    }
    auto rescale = [&](int r, float by) {
#pragma unroll
      for (int n = 0; n < 2 * NB; n++) {
        o[n][2 * r] *= by;
        o[n][2 * r + 1] *= by;
      }
    };

    auto process = [&](const CacheTile<NB> &t, int tile) {
      const int pos0 = tile * 16;
      float c[2][4];
#pragma unroll
      for (int n = 0; n < 2; n++) {
#pragma unroll
        for (int i = 0; i < 4; i++) c[n][i] = 0.f;
#pragma unroll
        for (int s = 0; s < NB; s++) {
          uint32_t b0, b1;
          codes_to_half<FMT>(t.k[n][s], b0, b1);
          mma_16816(c[n], qa[s][0], WIDE ? qa[s][1] : 0u, qa[s][R], WIDE ? qa[s][2 * R - 1] : 0u, b0, b1);
        }
      }
      uint32_t w16[R][2];
#pragma unroll
      for (int r = 0; r < R; r++) {
        float s[4], vs[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int n = i >> 1, at = pos0 + 8 * n + 2 * q + (i & 1);
          const float ks = (i & 1) ? t.ks[n].y : t.ks[n].x;
          vs[i] = (i & 1) ? t.vs[n].y : t.vs[n].x;
          s[i] = c[n][2 * r + (i & 1)] * ks * factor[r];
          if (a.bias != nullptr && g + 8 * r < n_heads && at < seen)
            s[i] += paged_log2(__ldg(a.bias + (size_t)(head0 + g + 8 * r) * a.n_dist + min(length - 1 - at, a.n_dist - 1)));
          if (at >= seen) s[i] = -INFINITY;
        }
        const float top = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
        if (__any_sync(0xffffffffu, top > m[r] + 8.f)) {
          const float next = fmaxf(m[r], quad_max(top));
          const float keep = next == -INFINITY ? 1.f : paged_exp2(m[r] - next);
          m[r] = next;
          sum[r] *= keep;
          rescale(r, keep);
        }
        const float base = m[r] == -INFINITY ? 0.f : m[r];
        float u[4], largest = 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float p = paged_exp2(s[i] - base);
          sum[r] += p;
          u[i] = p != 0.f ? p * vs[i] : 0.f;  // weight 0: whatever the scale is
          largest = fmaxf(largest, u[i]);
        }
        if (__any_sync(0xffffffffu, largest > unit[r] * 4096.f)) {
          const float next = fmaxf(fmaxf(quad_max(largest), unit[r]), 0x1p-100f);
          rescale(r, unit[r] / next);
          unit[r] = next;
        }
        const float inv = unit[r] > 0.f ? 1.f / unit[r] : 0.f;
#pragma unroll
        for (int n = 0; n < 2; n++) {
          const __half2 h = __floats2half2_rn(u[2 * n] * inv, u[2 * n + 1] * inv);
          w16[r][n] = *reinterpret_cast<const uint32_t *>(&h);
        }
      }
      auto product = [&](int n, uint32_t b0, uint32_t b1) {
        mma_16816(o[n], w16[0][0], WIDE ? w16[R - 1][0] : 0u, w16[0][1], WIDE ? w16[R - 1][1] : 0u, b0, b1);
      };
#pragma unroll
      for (int w = 0; w < C::kWords; w++) {
        // bytes of rows 2c and 2c + 1 side by side: two columns per word
        uint32_t p0, p1, r0, r1;
        codes_to_half<FMT>(__byte_perm(t.v[0][w], t.v[1][w], 0x5140), p0, p1);
        codes_to_half<FMT>(__byte_perm(t.v[2][w], t.v[3][w], 0x5140), r0, r1);
        product(4 * w, p0, r0);
        product(4 * w + 1, p1, r1);
        if (!(C::V2 && w == C::kWords - 1)) {
          codes_to_half<FMT>(__byte_perm(t.v[0][w], t.v[1][w], 0x7362), p0, p1);
          codes_to_half<FMT>(__byte_perm(t.v[2][w], t.v[3][w], 0x7362), r0, r1);
          product(4 * w + 2, p0, r0);
          product(4 * w + 3, p1, r1);
        }
      }
    };

    // ---- tiles; the next one's loads are on their way while one is worked on
    int pages = 0;  // of lane l: page of tile (first of 32) + l
    auto load = [&](CacheTile<NB> &t, int tile) {
      const int in_window = (tile - tile0) & 31;
      if (in_window == 0) {
        const long long pos = (long long)(tile + lane) * 16;
        pages = tile + lane < tile1 ? __ldg(a.c.table + (long long)seq * a.c.max_pages + (pos >> a.c.page_shift)) : -1;
      }
      const int page = __shfl_sync(0xffffffffu, pages, in_window);
      const bool good = page >= 0 && page < a.c.n_pages;
      if (!good) {
        if (lane == 0 && block == 0) atomicAdd(a.c.status, 1);
        return false;
      }
      const long long slot = ((((long long)page * a.c.kv_heads + kv) << a.c.page_shift) + ((tile * 16) & ((1 << a.c.page_shift) - 1)));
      load_cache_tile<NB>(t, a.c, slot, shape.width, seen - tile * 16, g, q);
      return true;
    };
    if (NB <= 8) {
      CacheTile<NB> t0, t1;
      bool good0 = load(t0, tile0), good1 = false;
      for (int tile = tile0; tile < tile1; tile += 2) {
        if (tile + 1 < tile1) good1 = load(t1, tile + 1);
        if (good0) process(t0, tile);
        if (tile + 1 >= tile1) break;
        if (tile + 2 < tile1) good0 = load(t0, tile + 2);
        if (good1) process(t1, tile + 1);
      }
    } else {
      CacheTile<NB> t0;
      for (int tile = tile0; tile < tile1; tile++)
        if (load(t0, tile)) process(t0, tile);
    }

    // ---- result of the segment, or the warp's part of it
    const bool whole = tile0 == 0 && tile1 == n_tiles;
    float *part = a.parts + (size_t)(2 * worker + (tile0 == 0 ? 1 : 0)) * shape.rows * row_floats;
#pragma unroll
    for (int r = 0; r < R; r++) {
      const int row = g + 8 * r;
      const float l = quad_sum(sum[r]);
      const float by = l == 0.f ? 0.f : unit[r] / l;
      if (row >= n_heads) continue;
      if (whole) {
        const long long at = ((long long)seq * a.heads + head0 + row) * d;
#pragma unroll
        for (int n = 0; n < 2 * NB; n++)
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const int col = value_column<NB>(n, 2 * q + i);
            if (col >= d) continue;
            const float v = o[n][2 * r + i] * by;
            if (a.dtype == QMOE_BF16) reinterpret_cast<__nv_bfloat16 *>(a.out)[at + col] = from_f32<__nv_bfloat16>(v);
            else reinterpret_cast<__half *>(a.out)[at + col] = from_f32<__half>(v);
          }
      } else {
        float *p = part + (size_t)row * row_floats;
        if (q == 0) {
          p[0] = m[r];
          p[1] = l;
        }
#pragma unroll
        for (int n = 0; n < 2 * NB; n++)
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const int col = value_column<NB>(n, 2 * q + i);
            if (col < d) p[2 + col] = o[n][2 * r + i] * by;
          }
      }
    }
    x = seg_begin + tile1;
  }
}

// One CTA per sequence and block of query heads: joins the parts of the warps that share it, writes zeros
// for a sequence without positions, counts a length that its page table cannot hold.
__global__ void __launch_bounds__(kPagedThreads) k_decode_join(const PagedArgs a) {
  const PagedShape shape = paged_shape(a.heads, a.c.kv_heads, a.c.head_dim);
  const int per_seq = a.c.kv_heads * shape.blocks, seq = blockIdx.x / per_seq, which = blockIdx.x % per_seq;
  const int kv = which / shape.blocks, block = which % shape.blocks, d = a.c.head_dim, row_floats = shape.width + 2;
  const int head0 = kv * shape.group + block * 16, n_heads = min(16, shape.group - block * 16);
  const int seen = paged_seen(a, seq), n_tiles = (seen + 15) / 16;
  if (threadIdx.x == 0 && block == 0 && a.lengths[seq] > seen) atomicAdd(a.c.status, 1);
  const long long quota = paged_quota(a.prefix[a.n_seqs], a.warps);
  const long long begin = a.prefix[seq] + (long long)which * n_tiles, end = begin + n_tiles;
  const int w0 = (int)(begin / quota), w1 = n_tiles > 0 ? (int)((end - 1) / quota) : w0;
  if (n_tiles > 0 && w0 == w1) return;
  auto part = [&](int w, int row) {
    return a.parts + ((size_t)(2 * w + (w == w0 ? 1 : 0)) * shape.rows + row) * row_floats;
  };
  for (int at = threadIdx.x; at < n_heads * d; at += kPagedThreads) {
    const int row = at / d, col = at % d;
    float top = -INFINITY, sum = 0.f, o = 0.f;
    if (n_tiles > 0) {
      for (int w = w0; w <= w1; w++) top = fmaxf(top, part(w, row)[0]);
      const float base = top == -INFINITY ? 0.f : top;
      for (int w = w0; w <= w1; w++) {
        const float *p = part(w, row);
        const float l = p[1];
        const float weight = l == 0.f ? 0.f : l * paged_exp2(p[0] - base);
        sum += weight;
        if (weight != 0.f) o += weight * p[2 + col];
      }
    }
    const float v = sum == 0.f ? 0.f : o / sum;
    const long long to = ((long long)seq * a.heads + head0 + row) * d + col;
    if (a.dtype == QMOE_BF16) reinterpret_cast<__nv_bfloat16 *>(a.out)[to] = from_f32<__nv_bfloat16>(v);
    else reinterpret_cast<__half *>(a.out)[to] = from_f32<__half>(v);
  }
}

// Units of 16 columns that a kernel is built for: the smallest that holds the row.
static int paged_units(int width) {
  const int units = width / 16;
  for (int nb : {1, 2, 4, 5, 6, 8, 12, 16})
    if (units <= nb) return nb;
  return 16;
}
// Warps of the grid: what fits the SMs with the kernel's registers.
static int paged_warps(int width, int device) {
  return sm_count(device) * paged_ctas(paged_units(width)) * (kPagedThreads / 32);
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
  if (((reinterpret_cast<uintptr_t>(cache->k_codes) | reinterpret_cast<uintptr_t>(cache->v_codes) |
        reinterpret_cast<uintptr_t>(cache->k_scale) | reinterpret_cast<uintptr_t>(cache->v_scale)) & 15u) != 0) {
    set_error("%s: codes and scales must be 16-byte aligned", fn);
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

int64_t qmoe_decode_paged_work_bytes(int n_seqs, int heads, int kv_heads, int head_dim, int device) {
  if (n_seqs < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || head_dim < 1 || head_dim > 256) return 0;
  const PagedShape shape = paged_shape(heads, kv_heads, head_dim);
  const int64_t prefix = ((int64_t)(n_seqs + 1) * 8 + 15) / 16 * 16;
  return prefix + (int64_t)paged_warps(shape.width, device) * 2 * shape.rows * (shape.width + 2) * 4;
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
  QMOE_REQUIRE(q_dev && out_dev && lengths_dev && work_dev, "null device pointer");
  QMOE_REQUIRE((reinterpret_cast<uintptr_t>(work_dev) & 15u) == 0, "workspace must be 16-byte aligned");
  if (n_seqs > kPagedMaxSeqs) {
    set_error("%s: at most %d sequences", __func__, kPagedMaxSeqs);
    return QMOE_ERR_UNSUPPORTED;
  }
  const PagedShape shape = paged_shape(heads, cache->kv_heads, cache->head_dim);
  a.q = q_dev;
  a.out = out_dev;
  a.q_row = q_row;
  a.q_head = q_head;
  a.lengths = lengths_dev;
  a.bias = rel_bias_dev;
  a.n_dist = n_dist;
  a.heads = heads;
  a.n_seqs = n_seqs;
  a.dtype = dtype;
  a.warps = paged_warps(shape.width, device);
  a.prefix = reinterpret_cast<long long *>(work_dev);
  a.parts = reinterpret_cast<float *>(reinterpret_cast<uint8_t *>(work_dev) + ((int64_t)(n_seqs + 1) * 8 + 15) / 16 * 16);
  a.scale = scale > 0.f ? scale : 1.f / sqrtf((float)cache->head_dim);
  DeviceGuard guard(device);
  if (!guard.ok) return cuda_fail(cudaGetLastError(), "cudaSetDevice");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool wide = shape.group > 8, e4m3 = cache->format == QMOE_CACHE_E4M3;
  const size_t smem = sizeof(long long) * (size_t)(n_seqs + 1);
  const unsigned grid = (unsigned)(a.warps / (kPagedThreads / 32));
  auto run = [&](auto nb) {
    constexpr int NB = decltype(nb)::value;
    if (e4m3 && wide) QMOE_LAUNCH((k_decode_paged<NB, QMOE_CACHE_E4M3, true>), grid, kPagedThreads, smem, st, a);
    else if (e4m3) QMOE_LAUNCH((k_decode_paged<NB, QMOE_CACHE_E4M3, false>), grid, kPagedThreads, smem, st, a);
    else if (wide) QMOE_LAUNCH((k_decode_paged<NB, QMOE_CACHE_INT8, true>), grid, kPagedThreads, smem, st, a);
    else QMOE_LAUNCH((k_decode_paged<NB, QMOE_CACHE_INT8, false>), grid, kPagedThreads, smem, st, a);
  };
  switch (paged_units(shape.width)) {
    case 1: run(std::integral_constant<int, 1>()); break;
    case 2: run(std::integral_constant<int, 2>()); break;
    case 4: run(std::integral_constant<int, 4>()); break;
    case 5: run(std::integral_constant<int, 5>()); break;
    case 6: run(std::integral_constant<int, 6>()); break;
    case 8: run(std::integral_constant<int, 8>()); break;
    case 12: run(std::integral_constant<int, 12>()); break;
    default: run(std::integral_constant<int, 16>()); break;
  }
  QMOE_CUDA(cudaGetLastError());
  QMOE_LAUNCH(k_decode_join, (unsigned)(n_seqs * cache->kv_heads * shape.blocks), kPagedThreads, 0, st, a);
  QMOE_CUDA(cudaGetLastError());
  return QMOE_OK;
}

}  // extern "C"
