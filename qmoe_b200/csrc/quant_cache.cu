// A paged key/value cache in 8 bits: append, read back, and the attention of single tokens over it.
#include <math.h>

#include <type_traits>

#include "serving.cuh"
#include "tcgen05.cuh"

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

// Codes nearest to x / s, ties to the even code, of four values of a row at once; `inv` is 1 / s to 2^-23.
// Rounding the fp32 quotient would round twice, so the quotient is rounded to odd instead: q, one
// Newton step from x * inv, is within one unit of its last place of the quotient, x - q * s is exact in one
// fused multiply-add, and where it is not zero q is replaced by the neighbour with the last bit set on the
// quotient's side.  That is never a rounding border, and lies on the quotient's side of every border.
// (A branch for quotients that look like borders is taken by most warps: s is a rounded amax / 448, so that many
// quotients of 16-bit values lie within its rounding of a border.)
struct RowScale {
  float s, inv;
};
__device__ __forceinline__ uint32_t to_odd(float q, float rest, float x) {
  const uint32_t bits = __float_as_uint(q);
  const uint32_t moved = (bits + (uint32_t)((int)(__float_as_uint(rest) ^ __float_as_uint(x)) >> 31)) | 1u;  // 1 less: towards 0
  return rest != 0.f ? moved : bits;
}
template <int FMT>
__device__ __forceinline__ uint32_t quantise4(const float (&x)[4], const RowScale &r) {
  const pair_t s_minus = pair_of(-r.s, -r.s), inv = pair_of(r.inv, r.inv);
  float q[4], rest[4];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const pair_t x2 = pair_of(x[2 * i], x[2 * i + 1]), q0 = pair_mul(x2, inv);
    const pair_t q2 = pair_fma(pair_fma(q0, s_minus, x2), inv, q0);
    pair_split(q2, q[2 * i], q[2 * i + 1]);
    pair_split(pair_fma(q2, s_minus, x2), rest[2 * i], rest[2 * i + 1]);
  }
#pragma unroll
  for (int i = 0; i < 4; i++) q[i] = __uint_as_float(to_odd(q[i], rest[i], x[i]));
  if (FMT == QMOE_CACHE_E4M3) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(q[1]), "f"(q[0]));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(q[3]), "f"(q[2]));
    return __byte_perm(lo, hi, 0x5410);
  }
  // q + 1.5 * 2^23 holds the nearest integer in its low bits
  uint32_t n[4];
#pragma unroll
  for (int i = 0; i < 4; i++) n[i] = __float_as_uint(q[i] + 12582912.f);
  return __byte_perm(__byte_perm(n[0], n[1], 0x0040), __byte_perm(n[2], n[3], 0x0040), 0x5410);
}
template <typename T>
__device__ __forceinline__ uint32_t pack_values(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack_values<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack_values<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&v);
}

struct RowsArgs {
  CacheView c;
  const void *k, *v;     // append: sources
  void *k_out, *v_out;   // read: destinations
  long long k_row, k_head, v_row, v_head;
  const int32_t *cu, *start;
  int n_seqs, tokens;  // tokens of a CTA
  uint32_t per_token_inverse;  // 2^32 / (2 * kv_heads), rounded up
  long long n_rows;
};

// Both directions are bounded by memory: 2 bytes read or written per value of the 16-bit side, 1 of the codes,
// 4 per row for the scale; what is left to do is to spend few instructions on a value.  A CTA takes `tokens`
// tokens with all their heads, keys and values: their places in the cache are looked up once, one thread a
// token, then every thread moves pieces of 16 values.  A row of one head is shared by LANES neighbouring lanes,
// heads run fastest, so that 16-bit rows are read or written in order.  Rows of 3, 5 and 6 pieces have their own
// kernels with 30 of 32 lanes at work (17408 tokens of 12 heads of 80 enter the cache in 33 us, with the next power of
// two lanes a row in 54).
// Where the 16-bit tensors' rows do not begin on 16-byte boundaries (VEC false) they are read in words of 4 bytes
// (7680 tokens of 32 heads of 65: 52 us, value by value 93) and written value by value, neighbouring lanes neighbouring values, through shared memory:
// [row of the warp][16 * LANES values].
// 16384 tokens of 8 heads of 128 in bf16 enter an e4m3 cache in 33 us (3.1 TB/s): 15.5 us of memory at the copy rate and
// some 19 of issue (the rounding is about twenty instructions a value) that follow one another, as nothing is
// requested while a pair of pieces is rounded; 65536 of them come back in 75 us (5.4 TB/s).
constexpr int kRowsThreads = 256;
constexpr int kRowsPieces = 8;  // of a thread, at most
constexpr int kRowsTokens = 64;

__host__ __device__ constexpr int row_lanes(int width) { return width <= 96 ? (width + 15) / 16 : (width <= 128 ? 8 : 16); }

// Places of the CTA's tokens: index of (page, head 0, place); -1 without a valid page, -2 when nobody owns the
// row.
__device__ __forceinline__ void find_slots(const RowsArgs &a, long long *s_slot) {
  if (threadIdx.x < a.tokens) {
    const long long row = (long long)blockIdx.x * a.tokens + threadIdx.x;
    long long slot = -2;
    const int seq = row < a.n_rows ? packed_seq(a.cu, a.n_seqs, (int)row) : -1;
    if (seq >= 0) {
      slot = cache_slot(a.c, seq, (long long)a.start[seq] + (row - max(a.cu[seq], 0)));  // offsets are clamped to the tensor
      if (slot < 0) atomicAdd(a.c.status, 1);
    }
    s_slot[threadIdx.x] = slot;
  }
  __syncthreads();
}

// Row `r` of the CTA's (token, key or value, head) rows.
struct CacheRow {
  long long row, slot;
  int head;
  bool is_v;
};
template <int LANES>
__device__ __forceinline__ CacheRow cache_row(const RowsArgs &a, const long long *s_slot, int r) {
  CacheRow c;
  const int token = (int)__umulhi((uint32_t)r, a.per_token_inverse), in_token = r - token * 2 * a.c.kv_heads;
  c.is_v = in_token >= a.c.kv_heads;
  c.head = in_token - (c.is_v ? a.c.kv_heads : 0);
  c.row = (long long)blockIdx.x * a.tokens + token;
  const bool idle = (threadIdx.x & 31) >= 32 / LANES * LANES;  // lanes that are left over own no row
  c.slot = token < a.tokens && !idle ? s_slot[token] : -2;
  if (c.slot >= 0) c.slot += (long long)c.head << a.c.page_shift;
  return c;
}

__device__ __forceinline__ uint32_t abs_max2(uint32_t m, uint32_t v, __nv_bfloat16) {
  const uint32_t u = v & 0x7fff7fffu;
  const __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162 *>(&m), *reinterpret_cast<const __nv_bfloat162 *>(&u));
  return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t abs_max2(uint32_t m, uint32_t v, __half) {
  const uint32_t u = v & 0x7fff7fffu;
  const __half2 r = __hmax2_nan(*reinterpret_cast<const __half2 *>(&m), *reinterpret_cast<const __half2 *>(&u));
  return *reinterpret_cast<const uint32_t *>(&r);
}
template <typename T>
__device__ __forceinline__ float2 pair_values(uint32_t v);
template <>
__device__ __forceinline__ float2 pair_values<__nv_bfloat16>(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 pair_values<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2 *>(&v)); }

template <typename T, int FMT, int LANES, bool VEC>
__global__ void __launch_bounds__(kRowsThreads) k_cache_append(const RowsArgs a) {
  constexpr int kPerWarp = 32 / LANES, kStep = kRowsThreads / 32 * kPerWarp;
  __shared__ long long s_slot[kRowsTokens];
  const int lane = threadIdx.x & 31, at = 16 * (lane % LANES);
  const int d = a.c.head_dim, width = cache_row_bytes(d), rows = a.tokens * 2 * a.c.kv_heads;
  find_slots(a, s_slot);
  auto source = [&](const CacheRow &c) {
    return c.is_v ? reinterpret_cast<const T *>(a.v) + c.row * a.v_row + c.head * a.v_head
                  : reinterpret_cast<const T *>(a.k) + c.row * a.k_row + c.head * a.k_head;
  };
  auto finish = [&](const CacheRow &c, const uint4 (&v)[2]) {
    const uint32_t w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) m = abs_max2(m, w[i], T());
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1)  // of the row's lanes, taken round
      m = abs_max2(m, __shfl_sync(0xffffffffu, m, lane - lane % LANES + (lane % LANES + o) % LANES), T());
    const float2 m2 = pair_values<T>(m);
    const bool finite = m2.x <= FLT_MAX && m2.y <= FLT_MAX;  // NaN and infinity stay in the maximum
    if (c.slot < 0 || at >= width) return;
    RowScale r;
    r.s = fmaxf(__fdiv_rn(fmaxf(m2.x, m2.y), FMT == QMOE_CACHE_E4M3 ? 448.f : 127.f), kScaleFloor);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.inv) : "f"(r.s));  // s is a normal number, and so is 1 / s
    const float stored = r.s;
    const bool tiny = r.s < 1e-25f;  // remainders would leave the normal range: all of it 2^64 times as large
    if (tiny) {
      r.inv *= 0x1p-64f;
      r.s *= 0x1p64f;
    }
    uint32_t codes[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float2 p = pair_values<T>(w[2 * i]), q = pair_values<T>(w[2 * i + 1]);
      float x[4] = {p.x, p.y, q.x, q.y};
      if (tiny) {
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] *= 0x1p64f;
      }
      codes[i] = finite ? quantise4<FMT>(x, r) : 0u;
    }
    *reinterpret_cast<uint4 *>((c.is_v ? a.c.v_codes : a.c.k_codes) + c.slot * width + at) = make_uint4(codes[0], codes[1], codes[2], codes[3]);
    if (at == 0) (c.is_v ? a.c.v_scale : a.c.k_scale)[c.slot] = finite ? stored : __int_as_float(0x7fffffff);
  };
  auto load = [&](const CacheRow &c, uint4 (&v)[2]) {
    v[0] = v[1] = make_uint4(0u, 0u, 0u, 0u);
    if (c.slot < 0) return;
    const T *src = source(c) + at;
    if (VEC && at + 16 <= d) {
      v[0] = __ldg(reinterpret_cast<const uint4 *>(src));
      v[1] = __ldg(reinterpret_cast<const uint4 *>(src) + 1);
    } else if (VEC) {
      T *to = reinterpret_cast<T *>(v);
#pragma unroll
      for (int i = 0; i < 16; i++)
        if (at + i < d) to[i] = src[i];
    } else {
      // the nine 4-byte words that the 16 values lie in, shifted by half a word where they begin in its middle;
      // of words that reach over the row's ends only the row's half is read
      const int odd = (int)(reinterpret_cast<uintptr_t>(src) >> 1) & 1;
      const uint16_t *from = reinterpret_cast<const uint16_t *>(src) - odd;
      uint32_t w[9];
#pragma unroll
      for (int x = 0; x < 9; x++) {
        const int first = at + 2 * x - odd;
        const bool lo = first >= 0 && first < d && (x < 8 || odd), hi = first + 1 < d && x < 8;
        w[x] = 0u;
        if (lo && hi) w[x] = __ldg(reinterpret_cast<const uint32_t *>(from) + x);
        else if (lo) w[x] = __ldg(from + 2 * x);
        else if (hi) w[x] = (uint32_t)__ldg(from + 2 * x + 1) << 16;
      }
      uint32_t o[8];
#pragma unroll
      for (int x = 0; x < 8; x++) o[x] = odd ? __funnelshift_r(w[x], w[x + 1], 16) : w[x];
      v[0] = make_uint4(o[0], o[1], o[2], o[3]);
      v[1] = make_uint4(o[4], o[5], o[6], o[7]);
    }
  };
  // two pieces at a time: both loads are under way before the first is used
  for (int base = (threadIdx.x >> 5) * kPerWarp; base < rows; base += 2 * kStep) {
    const int r0 = base + lane / LANES;
    CacheRow c[2];
    uint4 v[2][2];
#pragma unroll
    for (int b = 0; b < 2; b++) {
      c[b] = cache_row<LANES>(a, s_slot, r0 + b * kStep);
      load(c[b], v[b]);
    }
#pragma unroll
    for (int b = 0; b < 2; b++) finish(c[b], v[b]);
  }
}

template <typename T, int FMT, int LANES, bool VEC>
__global__ void __launch_bounds__(kRowsThreads) k_cache_read(const RowsArgs a) {
  constexpr int kPerWarp = 32 / LANES, kStep = kRowsThreads / 32 * kPerWarp;
  __shared__ long long s_slot[kRowsTokens];
  __shared__ __align__(16) T s_rows[VEC ? 1 : kRowsThreads / 32][VEC ? 1 : 512];
  const int lane = threadIdx.x & 31, at = 16 * (lane % LANES);
  const int d = a.c.head_dim, width = cache_row_bytes(d), rows = a.tokens * 2 * a.c.kv_heads;
  find_slots(a, s_slot);
  for (int base = (threadIdx.x >> 5) * kPerWarp; base < rows; base += 2 * kStep) {  // uniform in a warp
    const int r0 = base + lane / LANES;
    CacheRow c[2];
    uint4 codes[2];
    float scale[2];
#pragma unroll
    for (int b = 0; b < 2; b++) {
      c[b] = cache_row<LANES>(a, s_slot, r0 + b * kStep);
      codes[b] = make_uint4(0u, 0u, 0u, 0u);
      scale[b] = 0.f;
      if (c[b].slot >= 0 && at < width) {
        codes[b] = __ldg(reinterpret_cast<const uint4 *>((c[b].is_v ? a.c.v_codes : a.c.k_codes) + c[b].slot * width + at));
        scale[b] = __ldg((c[b].is_v ? a.c.v_scale : a.c.k_scale) + c[b].slot);
      }
    }
#pragma unroll
    for (int b = 0; b < 2; b++) {
      const uint32_t w[4] = {codes[b].x, codes[b].y, codes[b].z, codes[b].w};
      T *dst = reinterpret_cast<T *>(c[b].is_v ? a.v_out : a.k_out) + (c[b].row * a.c.kv_heads + c[b].head) * d;
      uint32_t v[8];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        uint32_t lo, hi;
        codes_to_half<FMT>(w[i], lo, hi);
        const float2 x = pair_values<__half>(lo), y = pair_values<__half>(hi);
        v[2 * i] = pack_values<T>(x.x * scale[b], x.y * scale[b]);
        v[2 * i + 1] = pack_values<T>(y.x * scale[b], y.y * scale[b]);
      }
      if (!VEC) {
        T *stage = s_rows[threadIdx.x >> 5];
        uint4 *to = reinterpret_cast<uint4 *>(stage + (lane / LANES) * 16 * LANES + at);
        to[0] = make_uint4(v[0], v[1], v[2], v[3]);
        to[1] = make_uint4(v[4], v[5], v[6], v[7]);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kPerWarp; i++) {
          T *out = reinterpret_cast<T *>(__shfl_sync(0xffffffffu, (unsigned long long)dst, i * LANES));
          const bool owned = __shfl_sync(0xffffffffu, (int)(c[b].slot != -2), i * LANES);
          for (int col = lane; owned && col < d; col += 32) out[col] = stage[i * 16 * LANES + col];
        }
        __syncwarp();
      } else if (c[b].slot != -2) {  // d is a multiple of 8
        if (at + 8 <= d) *reinterpret_cast<uint4 *>(dst + at) = make_uint4(v[0], v[1], v[2], v[3]);
        if (at + 16 <= d) *reinterpret_cast<uint4 *>(dst + at + 8) = make_uint4(v[4], v[5], v[6], v[7]);
      }
    }
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
// (Two to four times as many, shorter runs, started as earlier ones end, even out the warps' speeds but cost
// more in starts and parts: 131 us became 135 to 148 on a batch of 64 sequences and 554 MB.)
//
// Tile: S[16 positions, 8 heads] = K Q^T and O[columns, 8 heads] += V^T W by mma.sync m16n8k16 in fp16 with
// fp32 sums; both code formats are exact in fp16.  The order of the K axis of a product and of the columns is
// free, so every lane's operand comes from the tile's rows in pieces of 16 bytes: lane (g, c) of the warp
// (g = lane / 4, c = lane % 4) holds bytes 16 c .. 16 c + 15 of every 64 of keys g and g + 8, and columns 16 g ..
// of values 2c, 2c + 1, 2c + 8, 2c + 9.  Q is brought to fp16 by a power of two per head.  W comes out of S with
// positions along g and heads along c and is turned by movmatrix.
// Weights: p = exp2(s - m), w = p * value scale / r in fp16, r being 2^-7 of the largest p * value scale so far, so
// that rows of small and large scale keep their accuracy: half a step of fp16, and where w is subnormal 2^-32 of that
// largest one (the sums are fp32, of which a product loses what lies 2^-24 below them).  m only moves when p grew by more than 2^8, and r moves with it: p and r are relative to the same m, so
// the sums stay as they are.  r grows, and the sums are taken down, when w would pass 2^15.  (r left behind when m
// moves would belong to weights that have just become small: a later row that has all the weight but a scale
// 2^-20 of an earlier one's would be rounded to a few bits, or to nothing.)
//
// Measured: 64 sequences, 32 query and 8 key heads of 128, 554 MB of e4m3 codes and scales in 130 us a call (4.3
// TB/s), 121 of them on the GPU (int8 codes, which take fewer conversion instructions, 115).  Bound by the warps' uneven
// speeds, a tenth of them ending before 83 us, half before 87 and the last at 111, and the join behind that; the
// conversions are the 6 us between the formats.  One sequence of 1000 positions takes 11 us on the GPU, two launches and
// one trip to memory each.  More than 16 query heads a key head read the cache once per 16 (32 heads on one: 76 us,
// 16 on one: 58).
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
constexpr float kUnitFloor = FLT_MIN;  // of r: 1 / r is finite
constexpr float kUnitShare = 0x1p-7f, kWeightLimit = 0x1p15f;
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
// Tiles of that many positions, which may be 2^31 - 1.
__device__ __forceinline__ int paged_tiles(int seen) { return (int)(((uint32_t)seen + 15u) / 16u); }

__device__ __forceinline__ float paged_log2(float b) {  // a bias in units of log 2; the lowest values stay finite
  return b == -INFINITY ? b : fmaxf(b * 1.4426950408889634f, -FLT_MAX);
}
__device__ __forceinline__ float paged_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float paged_inverse(float x) {  // to 2^-23; x and 1 / x are normal numbers
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Over the lanes of a quad (one g), and over those of one c.
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float column_max(float v) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float column_sum(float v) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {  // of 16-bit values, two of a row per lane
  uint32_t t;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(t) : "r"(v));
  return t;
}

// A tile in shared memory: 16 rows of key codes, 16 of value codes, 16 + 16 scales.  Rows are `pitch` bytes
// apart, pitch = 16 mod 64, so that the eight lanes that read together from four value rows meet different
// banks (and those that read from two key rows at most twice the same).  Every warp has its own ring of
// kPagedStages tiles, filled by asynchronous copies.
//
// A lane's columns of a value row: 16 bytes of every block of 128 columns, then 8, 4 and 2 bytes of blocks
// of 64, 32 and 16.
constexpr int kPagedStages = 3;
__host__ __device__ constexpr int paged_pitch(int nb) { return (16 * nb + 47) / 64 * 64 + 16; }
__host__ __device__ constexpr int paged_stage(int nb) { return 32 * paged_pitch(nb) + 128; }
template <int NB>
struct CacheCols {
  static constexpr int KB = NB / 4, KR = NB % 4, V16 = NB / 8, V8 = NB % 8 / 4, V4 = NB % 4 / 2, V2 = NB % 2;
};

// Column `n` (of 2 * NB) of lane g = x.
template <int NB>
__device__ __forceinline__ int value_column(int n, int x) {
  using C = CacheCols<NB>;
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
  extern __shared__ __align__(16) uint8_t paged_smem[];  // the warps' rings, n_seqs + 1 prefixes, n_seqs lengths
  __shared__ long long s_warp[kPagedThreads / 32];
  using C = CacheCols<NB>;
  constexpr int R = WIDE ? 2 : 1;  // blocks of 8 heads
  const int tid = threadIdx.x, lane = tid & 31, g = lane >> 2, q = lane & 3;
  const PagedShape shape = paged_shape(a.heads, a.c.kv_heads, a.c.head_dim);
  const int per_seq = a.c.kv_heads * shape.blocks, d = a.c.head_dim;
  constexpr int pitch = paged_pitch(NB), stage_bytes = paged_stage(NB);
  const int units = shape.width >> 4;
  uint8_t *ring = paged_smem + (tid >> 5) * kPagedStages * stage_bytes;
  long long *s_prefix = reinterpret_cast<long long *>(paged_smem + (kPagedThreads / 32) * kPagedStages * stage_bytes);
  int *s_seen = reinterpret_cast<int *>(s_prefix + a.n_seqs + 1);
  // copies of this lane: pieces lane, lane + 32, ... of 16 bytes of a tile's 16 rows
  int piece_at[(NB + 1) / 2], piece_row[(NB + 1) / 2];
#pragma unroll
  for (int i = 0; i < (NB + 1) / 2; i++) {
    const int piece = lane + 32 * i, row = piece / units;
    piece_row[i] = piece < 16 * units ? row : 16;
    piece_at[i] = row * pitch + (piece - row * units) * 16;
  }

  // a kernel may be built for more columns than the rows have: zeros there
  if (units < NB)
    for (int i = lane; i < kPagedStages * 32; i += 32)
      for (int u = units; u < NB; u++)
        *reinterpret_cast<uint4 *>(ring + (i >> 5) * stage_bytes + (i & 31) * pitch + 16 * u) = make_uint4(0u, 0u, 0u, 0u);

  // tiles before every sequence
  long long before = 0;
  for (int s0 = 0; s0 < a.n_seqs; s0 += kPagedThreads) {
    const int s = s0 + tid;
    const int seen = s < a.n_seqs ? paged_seen(a, s) : 0;
    if (s < a.n_seqs) s_seen[s] = seen;
    long long upto = (long long)paged_tiles(seen) * per_seq;
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
    const int seq = lo, seen = s_seen[seq], n_tiles = paged_tiles(seen);
    const long long in_seq = x - s_prefix[seq];
    const int which = in_seq <= 0x7fffffff ? (int)((uint32_t)in_seq / (uint32_t)n_tiles) : (int)(in_seq / n_tiles);
    const int tile0 = (int)(in_seq - (long long)which * n_tiles);
    const long long seg_begin = x - tile0;
    const int tile1 = (int)min((long long)n_tiles, run_end - seg_begin);
    const int kv = which / shape.blocks, block = which % shape.blocks;
    const int head0 = kv * shape.group + block * 16, n_heads = min(16, shape.group - block * 16);

    // ---- tiles, kPagedStages - 1 of them ahead on their way
    const int tiles_per_page = 1 << (a.c.page_shift - 4);
    const long long row_bytes = shape.width;
    int pages = 0, ahead = tile0, fill = 0;  // of lane l: page of tile l of a window of 32; next tile to load and its stage
    unsigned good = 0;                       // bit i: stage i holds a tile
    auto load = [&]() {
      good &= ~(1u << fill);
      if (ahead < tile1) {
        const int in_window = (ahead - tile0) & 31;
        if (in_window == 0) {
          const int at = ahead + lane;
          pages = at < tile1 ? __ldg(a.c.table + (long long)seq * a.c.max_pages + (at >> (a.c.page_shift - 4))) : -1;
        }
        const int page = __shfl_sync(0xffffffffu, pages, in_window);
        if (page >= 0 && page < a.c.n_pages) {
          good |= 1u << fill;
          const long long slot = (((long long)page * a.c.kv_heads + kv) << a.c.page_shift) + 16 * (ahead & (tiles_per_page - 1));
          const uint32_t to = smem_u32(ring) + fill * stage_bytes;
          const uint8_t *k = a.c.k_codes + slot * row_bytes + lane * 16, *v = a.c.v_codes + slot * row_bytes + lane * 16;
          const int left = seen - ahead * 16;
          if (left >= 16) {
#pragma unroll
            for (int i = 0; i < (NB + 1) / 2; i++) {
              if (piece_row[i] >= 16) continue;
              cp_async16(to + piece_at[i], k + 512 * i);
              cp_async16(to + 16 * pitch + piece_at[i], v + 512 * i);
            }
          } else {  // places behind the last position may hold anything: zeros instead
#pragma unroll
            for (int i = 0; i < (NB + 1) / 2; i++) {
              if (piece_row[i] >= 16) continue;
              const int bytes = piece_row[i] < left ? 16 : 0;
              cp_async16(to + piece_at[i], k + 512 * i, bytes);
              cp_async16(to + 16 * pitch + piece_at[i], v + 512 * i, bytes);
            }
          }
          if (lane < 8) cp_async16(to + 32 * pitch + lane * 16, (lane < 4 ? a.c.k_scale : a.c.v_scale) + slot + 4 * (lane & 3));
        } else if (lane == 0 && block == 0) {
          atomicAdd(a.c.status, 1);
        }
      }
      cp_async_commit();
      ahead++;
      fill = fill == kPagedStages - 1 ? 0 : fill + 1;
    };
#pragma unroll
    for (int i = 0; i < kPagedStages - 1; i++) load();

    // ---- queries of the lane's rows in the order of the key bytes, brought to fp16
    uint32_t qa[NB][2 * R];
    float factor[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
      const bool live = g + 8 * r < n_heads;
      const long long at = seq * a.q_row + (long long)(head0 + (live ? g + 8 * r : 0)) * a.q_head;
      float v[NB][4], amax = 0.f;
#pragma unroll
      for (int n = 0; n < NB; n++) {
        const int col = n < 4 * C::KB ? 64 * (n >> 2) + 16 * q + 4 * (n & 3) : 16 * n + 4 * q;
        if (a.dtype == QMOE_BF16) {
#pragma unroll
          for (int i = 0; i < 4; i++) v[n][i] = live && col + i < d ? to_f32(reinterpret_cast<const __nv_bfloat16 *>(a.q)[at + col + i]) : 0.f;
        } else {
#pragma unroll
          for (int i = 0; i < 4; i++) v[n][i] = live && col + i < d ? to_f32(reinterpret_cast<const __half *>(a.q)[at + col + i]) : 0.f;
        }
#pragma unroll
        for (int i = 0; i < 4; i++) amax = fmaxf(amax, fabsf(v[n][i]));
      }
      amax = quad_max(amax);
      // 2^-e in two factors, either of which is a normal number
      const int e = amax > 0.f && amax <= FLT_MAX ? ilogbf(amax) : 0;
      const float down0 = scalbnf(1.f, -(e / 2)), down1 = scalbnf(1.f, -(e - e / 2));
      factor[r] = scalbnf(a.scale * 1.4426950408889634f, e);
#pragma unroll
      for (int n = 0; n < NB; n++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const __half2 h = __floats2half2_rn(v[n][2 * i] * down0 * down1, v[n][2 * i + 1] * down0 * down1);
          qa[n][i * R + r] = *reinterpret_cast<const uint32_t *>(&h);
        }
    }

    // The lane's heads from here on: 2c and 2c + 1 of every block of 8.
    float o[NB][R][4];  // two columns by two heads
    float m[R][2], sum[R][2], unit[R][2], inv[R][2], by_head[R][2];  // maximum in units of log 2, sum of p, r, 1 / r
#pragma unroll
    for (int r = 0; r < R; r++) {
#pragma unroll
      for (int n = 0; n < NB; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) o[n][r][i] = 0.f;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        m[r][h] = -INFINITY;
        sum[r][h] = 0.f;
        unit[r][h] = kUnitFloor;
        inv[r][h] = 1.f / kUnitFloor;
        by_head[r][h] = __shfl_sync(0xffffffffu, factor[r], 4 * (2 * q + h));
      }
    }
    auto rescale = [&](int r, float by0, float by1) {
#pragma unroll
      for (int n = 0; n < NB; n++) {
        o[n][r][0] *= by0;
        o[n][r][1] *= by1;
        o[n][r][2] *= by0;
        o[n][r][3] *= by1;
      }
    };

    auto process = [&](const uint8_t *keys, int tile) {
      const uint8_t *values = keys + 16 * pitch;
      const float *scales = reinterpret_cast<const float *>(keys + 32 * pitch);
      const int pos0 = tile * 16;
      float c[R][4];
#pragma unroll
      for (int r = 0; r < R; r++)
#pragma unroll
        for (int i = 0; i < 4; i++) c[r][i] = 0.f;
      auto scores = [&](int s, uint32_t key0, uint32_t key8) {
        uint32_t a0, a1, a2, a3;
        codes_to_half<FMT>(key0, a0, a2);
        codes_to_half<FMT>(key8, a1, a3);
#pragma unroll
        for (int r = 0; r < R; r++) mma_16816(c[r], a0, a1, a2, a3, qa[s][r], qa[s][R + r]);
      };
#pragma unroll
      for (int b = 0; b < C::KB; b++) {
        const uint4 x = *reinterpret_cast<const uint4 *>(keys + g * pitch + 64 * b + 16 * q);
        const uint4 y = *reinterpret_cast<const uint4 *>(keys + (g + 8) * pitch + 64 * b + 16 * q);
        scores(4 * b, x.x, y.x);
        scores(4 * b + 1, x.y, y.y);
        scores(4 * b + 2, x.z, y.z);
        scores(4 * b + 3, x.w, y.w);
      }
#pragma unroll
      for (int i = 0; i < C::KR; i++) {
        const int off = 64 * C::KB + 16 * i + 4 * q;
        scores(4 * C::KB + i, *reinterpret_cast<const uint32_t *>(keys + g * pitch + off),
               *reinterpret_cast<const uint32_t *>(keys + (g + 8) * pitch + off));
      }
      const float ks0 = scales[g], ks8 = scales[g + 8], vs0 = scales[16 + g], vs8 = scales[24 + g];
      uint32_t w16[R][2];
#pragma unroll
      for (int r = 0; r < R; r++) {
        // [0] position g, head 2c  [1] position g, head 2c + 1  [2], [3] position g + 8
        float s[4];
        s[0] = c[r][0] * (ks0 * by_head[r][0]);
        s[1] = c[r][1] * (ks0 * by_head[r][1]);
        s[2] = c[r][2] * (ks8 * by_head[r][0]);
        s[3] = c[r][3] * (ks8 * by_head[r][1]);
        if (a.bias != nullptr) {
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int row = min(8 * r + 2 * q + (i & 1), n_heads - 1);
            const int far = a.lengths[seq] - 1 - (pos0 + 8 * (i >> 1) + g);
            const float b = paged_log2(__ldg(a.bias + (size_t)(head0 + row) * a.n_dist + max(0, min(far, a.n_dist - 1))));
            s[i] = b == -INFINITY ? b : s[i] + b;  // chosen, not added: a masked key may hold anything
          }
        }
        if (seen - pos0 < 16) {
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (pos0 + 8 * (i >> 1) + g >= seen) s[i] = -INFINITY;
        }
        const float top0 = fmaxf(s[0], s[2]), top1 = fmaxf(s[1], s[3]);
        if (__any_sync(0xffffffffu, top0 > m[r][0] + 8.f || top1 > m[r][1] + 8.f)) {
          const float next0 = fmaxf(m[r][0], column_max(top0)), next1 = fmaxf(m[r][1], column_max(top1));
          const float keep0 = next0 == -INFINITY ? 1.f : paged_exp2(m[r][0] - next0);
          const float keep1 = next1 == -INFINITY ? 1.f : paged_exp2(m[r][1] - next1);
          const float moved0 = unit[r][0] * keep0, moved1 = unit[r][1] * keep1;
          // below the least r the sums go down after all; without a maximum so far they are 0
          const bool low = (moved0 < kUnitFloor && m[r][0] != -INFINITY) || (moved1 < kUnitFloor && m[r][1] != -INFINITY);
          m[r][0] = next0;
          m[r][1] = next1;
          sum[r][0] *= keep0;
          sum[r][1] *= keep1;
          unit[r][0] = fmaxf(moved0, kUnitFloor);
          unit[r][1] = fmaxf(moved1, kUnitFloor);
          inv[r][0] = paged_inverse(unit[r][0]);
          inv[r][1] = paged_inverse(unit[r][1]);
          if (__any_sync(0xffffffffu, low)) rescale(r, moved0 * inv[r][0], moved1 * inv[r][1]);
        }
        const float base0 = m[r][0] == -INFINITY ? 0.f : m[r][0], base1 = m[r][1] == -INFINITY ? 0.f : m[r][1];
        const float p0 = paged_exp2(s[0] - base0), p1 = paged_exp2(s[1] - base1);
        const float p2 = paged_exp2(s[2] - base0), p3 = paged_exp2(s[3] - base1);
        sum[r][0] += p0 + p2;
        sum[r][1] += p1 + p3;
        // weight 0: whatever the scale is
        const float u0 = p0 != 0.f ? p0 * vs0 : 0.f, u1 = p1 != 0.f ? p1 * vs0 : 0.f;
        const float u2 = p2 != 0.f ? p2 * vs8 : 0.f, u3 = p3 != 0.f ? p3 * vs8 : 0.f;
        const float large0 = fmaxf(u0, u2), large1 = fmaxf(u1, u3);
        if (__any_sync(0xffffffffu, large0 > unit[r][0] * kWeightLimit || large1 > unit[r][1] * kWeightLimit)) {
          const float next0 = fmaxf(column_max(large0) * kUnitShare, unit[r][0]);
          const float next1 = fmaxf(column_max(large1) * kUnitShare, unit[r][1]);
          inv[r][0] = paged_inverse(next0);
          inv[r][1] = paged_inverse(next1);
          rescale(r, unit[r][0] * inv[r][0], unit[r][1] * inv[r][1]);
          unit[r][0] = next0;
          unit[r][1] = next1;
        }
        const __half2 h0 = __floats2half2_rn(u0 * inv[r][0], u1 * inv[r][1]);
        const __half2 h8 = __floats2half2_rn(u2 * inv[r][0], u3 * inv[r][1]);
        w16[r][0] = transpose_8x8(*reinterpret_cast<const uint32_t *>(&h0));
        w16[r][1] = transpose_8x8(*reinterpret_cast<const uint32_t *>(&h8));
      }
      // words of the lane's four rows (positions 2c, 2c + 1, 2c + 8, 2c + 9): bytes of two rows side by side;
      // two columns a product
      auto products = [&](int n, int count, uint32_t v0, uint32_t v1, uint32_t v2, uint32_t v3) {
        uint32_t a0, a1, a2, a3;
        codes_to_half<FMT>(__byte_perm(v0, v1, 0x5140), a0, a1);
        codes_to_half<FMT>(__byte_perm(v2, v3, 0x5140), a2, a3);
#pragma unroll
        for (int r = 0; r < R; r++) mma_16816(o[n][r], a0, a1, a2, a3, w16[r][0], w16[r][1]);
        if (count > 2) {
          codes_to_half<FMT>(__byte_perm(v0, v1, 0x7362), a0, a1);
          codes_to_half<FMT>(__byte_perm(v2, v3, 0x7362), a2, a3);
#pragma unroll
          for (int r = 0; r < R; r++) mma_16816(o[n + 1][r], a0, a1, a2, a3, w16[r][0], w16[r][1]);
        }
      };
      const uint8_t *row[4];
#pragma unroll
      for (int r = 0; r < 4; r++) row[r] = values + (8 * (r >> 1) + 2 * q + (r & 1)) * pitch;
#pragma unroll
      for (int b = 0; b < C::V16; b++) {
        uint4 v[4];
#pragma unroll
        for (int r = 0; r < 4; r++) v[r] = *reinterpret_cast<const uint4 *>(row[r] + 128 * b + 16 * g);
        products(8 * b, 4, v[0].x, v[1].x, v[2].x, v[3].x);
        products(8 * b + 2, 4, v[0].y, v[1].y, v[2].y, v[3].y);
        products(8 * b + 4, 4, v[0].z, v[1].z, v[2].z, v[3].z);
        products(8 * b + 6, 4, v[0].w, v[1].w, v[2].w, v[3].w);
      }
      if constexpr (C::V8 != 0) {
        uint2 v[4];
#pragma unroll
        for (int r = 0; r < 4; r++) v[r] = *reinterpret_cast<const uint2 *>(row[r] + 128 * C::V16 + 8 * g);
        products(8 * C::V16, 4, v[0].x, v[1].x, v[2].x, v[3].x);
        products(8 * C::V16 + 2, 4, v[0].y, v[1].y, v[2].y, v[3].y);
      }
      if constexpr (C::V4 != 0) {
        const int off = 128 * C::V16 + 64 * C::V8 + 4 * g;
        uint32_t v[4];
#pragma unroll
        for (int r = 0; r < 4; r++) v[r] = *reinterpret_cast<const uint32_t *>(row[r] + off);
        products(8 * C::V16 + 4 * C::V8, 4, v[0], v[1], v[2], v[3]);
      }
      if constexpr (C::V2 != 0) {
        const int off = 128 * C::V16 + 64 * C::V8 + 32 * C::V4 + 2 * g;
        uint32_t v[4];
#pragma unroll
        for (int r = 0; r < 4; r++) v[r] = *reinterpret_cast<const uint16_t *>(row[r] + off);
        products(NB - 1, 2, v[0], v[1], v[2], v[3]);
      }
    };

    int stage = 0;
    for (int tile = tile0; tile < tile1; tile++) {
      load();
      cp_async_wait<kPagedStages - 1>();
      __syncwarp();
      if (good >> stage & 1) process(ring + stage * stage_bytes, tile);
      __syncwarp();  // the stage is filled again next
      stage = stage == kPagedStages - 1 ? 0 : stage + 1;
    }
    cp_async_wait<0>();

    // ---- result of the segment, or the warp's part of it
    const bool whole = tile0 == 0 && tile1 == n_tiles;
    float *part = a.parts + (size_t)(2 * worker + (tile0 == 0 ? 1 : 0)) * shape.rows * row_floats;
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int row = 8 * r + 2 * q + h;
        const float l = column_sum(sum[r][h]);
        const float by = l == 0.f ? 0.f : 1.f / l, of = unit[r][h];  // of / l may be subnormal
        if (row >= n_heads) continue;
        const long long at = ((long long)seq * a.heads + head0 + row) * d;
        float *p = part + (size_t)row * row_floats;
        if (!whole && g == 0) {
          p[0] = m[r][h];
          p[1] = l;
        }
#pragma unroll
        for (int n = 0; n < 2 * NB; n++) {
          const int col = value_column<NB>(n, g);
          if (col >= d) continue;
          const float v = o[n >> 1][r][2 * (n & 1) + h] * by * of;
          if (!whole) p[2 + col] = v;
          else if (a.dtype == QMOE_BF16) reinterpret_cast<__nv_bfloat16 *>(a.out)[at + col] = from_f32<__nv_bfloat16>(v);
          else reinterpret_cast<__half *>(a.out)[at + col] = from_f32<__half>(v);
        }
      }
    x = seg_begin + tile1;
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// One CTA per sequence and query head: joins the parts of the warps that share it, writes zeros for a
// sequence without positions, counts a length that its page table cannot hold.  The parts' weights are found
// by all threads at once; then every warp sums its share of the parts, four at a time.
constexpr int kJoinThreads = 256;
__global__ void __launch_bounds__(kJoinThreads) k_decode_join(const PagedArgs a) {
  extern __shared__ float s_weight[];  // one per warp of the first kernel, then [warps of this CTA][columns]
  __shared__ float s_red[kJoinThreads / 32];
  const PagedShape shape = paged_shape(a.heads, a.c.kv_heads, a.c.head_dim);
  const int seq = blockIdx.x / a.heads, head = blockIdx.x % a.heads, d = a.c.head_dim, row_floats = shape.width + 2;
  const int kv = head / shape.group, block = head % shape.group / 16, row = head % shape.group % 16;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int seen = paged_seen(a, seq), n_tiles = paged_tiles(seen);
  asm volatile("griddepcontrol.wait;" ::: "memory");  // launched while the first kernel ends
  if (tid == 0 && head % shape.group == 0 && a.lengths[seq] > seen) atomicAdd(a.c.status, 1);
  auto store = [&](int col, float v) {
    const long long to = ((long long)seq * a.heads + head) * d + col;
    if (a.dtype == QMOE_BF16) reinterpret_cast<__nv_bfloat16 *>(a.out)[to] = from_f32<__nv_bfloat16>(v);
    else reinterpret_cast<__half *>(a.out)[to] = from_f32<__half>(v);
  };
  if (n_tiles == 0) {
    for (int col = tid; col < d; col += kJoinThreads) store(col, 0.f);
    return;
  }
  const long long quota = paged_quota(a.prefix[a.n_seqs], a.warps);
  const long long begin = a.prefix[seq] + (long long)(kv * shape.blocks + block) * n_tiles, end = begin + n_tiles;
  const int w0 = (int)(begin / quota), n_parts = (int)((end - 1) / quota) - w0 + 1;
  if (n_parts == 1) return;
  auto part = [&](int p) { return a.parts + ((size_t)(2 * (w0 + p) + (p == 0 ? 1 : 0)) * shape.rows + row) * row_floats; };
  float top = -INFINITY;
  for (int p = tid; p < n_parts; p += kJoinThreads) top = fmaxf(top, part(p)[0]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) s_red[warp] = top;
  __syncthreads();
  for (int w = 0; w < kJoinThreads / 32; w++) top = fmaxf(top, s_red[w]);
  const float base = top == -INFINITY ? 0.f : top;
  __syncthreads();
  float sum = 0.f;
  for (int p = tid; p < n_parts; p += kJoinThreads) {
    const float2 ml = make_float2(part(p)[0], part(p)[1]);
    const float weight = ml.y == 0.f ? 0.f : ml.y * paged_exp2(ml.x - base);
    s_weight[p] = weight;
    sum += weight;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) s_red[warp] = sum;
  __syncthreads();
  sum = 0.f;
  for (int w = 0; w < kJoinThreads / 32; w++) sum += s_red[w];
  float *s_acc = s_weight + a.warps + warp * 256;
  for (int c0 = 0; c0 < d; c0 += 128) {
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int p0 = warp; p0 < n_parts; p0 += 4 * (kJoinThreads / 32)) {
      float v[4][4], weight[4];
#pragma unroll
      for (int x = 0; x < 4; x++) {
        const int p = p0 + x * (kJoinThreads / 32);
        weight[x] = p < n_parts ? s_weight[p] : 0.f;
        const float *from = part(p < n_parts ? p : p0) + 2;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int col = c0 + lane + 32 * i;
          v[x][i] = col < d && weight[x] != 0.f ? from[col] : 0.f;
        }
      }
#pragma unroll
      for (int x = 0; x < 4; x++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[i] += weight[x] * v[x][i];
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (c0 + lane + 32 * i < d) s_acc[c0 + lane + 32 * i] = acc[i];
  }
  __syncthreads();
  for (int col = tid; col < d; col += kJoinThreads) {
    float o = 0.f;
    for (int w = 0; w < kJoinThreads / 32; w++) o += s_weight[a.warps + w * 256 + col];
    store(col, sum == 0.f ? 0.f : o / sum);
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

// Launches a row kernel for the activations' type, the code format, the lanes that share a row and the
// alignment of the 16-bit tensors.
#define QMOE_ROWS_KERNELS(kernel, T, FMT, vec)                                                                  \
  (lanes == 1   ? (vec ? kernel<T, FMT, 1, true> : kernel<T, FMT, 1, false>)                                    \
   : lanes == 2 ? (vec ? kernel<T, FMT, 2, true> : kernel<T, FMT, 2, false>)                                    \
   : lanes == 3 ? (vec ? kernel<T, FMT, 3, true> : kernel<T, FMT, 3, false>)                                    \
   : lanes == 5 ? (vec ? kernel<T, FMT, 5, true> : kernel<T, FMT, 5, false>)                                    \
   : lanes == 6 ? (vec ? kernel<T, FMT, 6, true> : kernel<T, FMT, 6, false>)                                    \
   : lanes == 4 ? (vec ? kernel<T, FMT, 4, true> : kernel<T, FMT, 4, false>)                                    \
   : lanes == 8 ? (vec ? kernel<T, FMT, 8, true> : kernel<T, FMT, 8, false>)                                    \
                : (vec ? kernel<T, FMT, 16, true> : kernel<T, FMT, 16, false>))
template <bool READ>
static int run_rows(RowsArgs a, int dtype, int format, bool vec, int device, cudaStream_t stream) {
  const int lanes = row_lanes(cache_row_bytes(a.c.head_dim));
  // tokens of a CTA: what gives its threads kRowsPieces pieces each, fewer where the GPU would not be filled
  const long long pieces = 2LL * a.c.kv_heads * lanes, fill = (a.n_rows + 8 * sm_count(device) - 1) / (8 * sm_count(device));
  long long tokens = kRowsPieces * kRowsThreads / pieces;
  tokens = tokens < fill ? tokens : fill;
  a.tokens = (int)(tokens < 1 ? 1 : (tokens > kRowsTokens ? kRowsTokens : tokens));
  a.per_token_inverse = (uint32_t)(((1ull << 32) + 2 * a.c.kv_heads - 1) / (2 * a.c.kv_heads));
  const dim3 grid((unsigned)((a.n_rows + a.tokens - 1) / a.tokens));
  void (*kernel)(RowsArgs);
  if (READ) {
    if (dtype == QMOE_BF16)
      kernel = format == QMOE_CACHE_E4M3 ? QMOE_ROWS_KERNELS(k_cache_read, __nv_bfloat16, QMOE_CACHE_E4M3, vec)
                                         : QMOE_ROWS_KERNELS(k_cache_read, __nv_bfloat16, QMOE_CACHE_INT8, vec);
    else
      kernel = format == QMOE_CACHE_E4M3 ? QMOE_ROWS_KERNELS(k_cache_read, __half, QMOE_CACHE_E4M3, vec)
                                         : QMOE_ROWS_KERNELS(k_cache_read, __half, QMOE_CACHE_INT8, vec);
  } else {
    if (dtype == QMOE_BF16)
      kernel = format == QMOE_CACHE_E4M3 ? QMOE_ROWS_KERNELS(k_cache_append, __nv_bfloat16, QMOE_CACHE_E4M3, vec)
                                         : QMOE_ROWS_KERNELS(k_cache_append, __nv_bfloat16, QMOE_CACHE_INT8, vec);
    else
      kernel = format == QMOE_CACHE_E4M3 ? QMOE_ROWS_KERNELS(k_cache_append, __half, QMOE_CACHE_E4M3, vec)
                                         : QMOE_ROWS_KERNELS(k_cache_append, __half, QMOE_CACHE_INT8, vec);
  }
  QMOE_LAUNCH(kernel, grid, kRowsThreads, 0, stream, a);
  QMOE_CUDA(cudaGetLastError());
  return QMOE_OK;
}

template <bool READ>
static int rows_entry(const char *fn, const qmoe_quant_cache *cache, const qmoe_cache_rows *rows, int device, void *stream) {
  if (rows == nullptr) {
    set_error("%s: null pointer", fn);
    return QMOE_ERR_INVALID_ARG;
  }
  RowsArgs a{};
  const int rc = cache_view(fn, cache, rows->page_table_dev, rows->status_dev, rows->n_seqs, rows->max_pages, rows->dtype, &a.c);
  if (rc != QMOE_OK) return rc;
  if (rows->n_rows < 0 || rows->n_rows > 0x7fffffffLL) {
    set_error("%s: bad number of rows", fn);
    return QMOE_ERR_INVALID_ARG;
  }
  if (rows->n_rows == 0 || rows->n_seqs == 0) return QMOE_OK;
  if (!rows->k_dev || !rows->v_dev || !rows->cu_dev || !rows->start_dev) {
    set_error("%s: null device pointer", fn);
    return QMOE_ERR_INVALID_ARG;
  }
  if (cache->kv_heads > 1024) {
    set_error("%s: at most 1024 key heads", fn);
    return QMOE_ERR_UNSUPPORTED;
  }
  a.k = a.k_out = rows->k_dev;
  a.v = a.v_out = rows->v_dev;
  a.k_row = rows->k_row;
  a.k_head = rows->k_head;
  a.v_row = rows->v_row;
  a.v_head = rows->v_head;
  a.cu = rows->cu_dev;
  a.start = rows->start_dev;
  a.n_seqs = rows->n_seqs;
  a.n_rows = rows->n_rows;
  // 16-byte accesses to the 16-bit tensors where every row begins on a 16-byte boundary
  uintptr_t bits = reinterpret_cast<uintptr_t>(rows->k_dev) | reinterpret_cast<uintptr_t>(rows->v_dev);
  bits |= READ ? (uintptr_t)(2 * cache->head_dim) : (uintptr_t)(2 * (a.k_row | a.k_head | a.v_row | a.v_head));
  DeviceGuard guard(device);
  if (!guard.ok) return cuda_fail(cudaGetLastError(), "cudaSetDevice");
  return run_rows<READ>(a, rows->dtype, cache->format, (bits & 15u) == 0, device, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" {

int qmoe_cache_append(const qmoe_quant_cache *cache, const qmoe_cache_rows *rows, int device, void *stream) {
  return rows_entry<false>(__func__, cache, rows, device, stream);
}

int qmoe_cache_read(const qmoe_quant_cache *cache, const qmoe_cache_rows *rows, int device, void *stream) {
  return rows_entry<true>(__func__, cache, rows, device, stream);
}

int64_t qmoe_decode_paged_work_bytes(int n_seqs, int heads, int kv_heads, int head_dim, int device) {
  if (n_seqs < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || head_dim < 1 || head_dim > 256) return 0;
  const PagedShape shape = paged_shape(heads, kv_heads, head_dim);
  const int64_t prefix = ((int64_t)(n_seqs + 1) * 8 + 15) / 16 * 16;
  return prefix + (int64_t)paged_warps(shape.width, device) * 2 * shape.rows * (shape.width + 2) * 4;
}

int qmoe_decode_attention_paged(const qmoe_quant_cache *cache, const qmoe_paged_args *args, int device, void *stream) {
  QMOE_REQUIRE(args != nullptr, "null pointer");
  const int n_seqs = args->n_seqs, heads = args->heads;
  PagedArgs a{};
  const int rc = cache_view(__func__, cache, args->page_table_dev, args->status_dev, n_seqs, args->max_pages, args->dtype, &a.c);
  if (rc != QMOE_OK) return rc;
  QMOE_REQUIRE(heads >= 1 && heads % cache->kv_heads == 0, "heads must be a positive multiple of kv_heads");
  QMOE_REQUIRE((args->rel_bias_dev == nullptr) == (args->n_dist == 0) && args->n_dist >= 0, "bias and n_dist do not agree");
  QMOE_REQUIRE(isfinite(args->scale), "scale is not finite");
  if (n_seqs == 0) return QMOE_OK;
  QMOE_REQUIRE(args->q_dev && args->out_dev && args->lengths_dev && args->work_dev, "null device pointer");
  QMOE_REQUIRE((reinterpret_cast<uintptr_t>(args->work_dev) & 15u) == 0, "workspace must be 16-byte aligned");
  if (n_seqs > kPagedMaxSeqs || (int64_t)n_seqs * heads > 0x7fffffffLL) {
    set_error("%s: at most %d sequences", __func__, kPagedMaxSeqs);
    return QMOE_ERR_UNSUPPORTED;
  }
  const PagedShape shape = paged_shape(heads, cache->kv_heads, cache->head_dim);
  a.q = args->q_dev;
  a.out = args->out_dev;
  a.q_row = args->q_row;
  a.q_head = args->q_head;
  a.lengths = args->lengths_dev;
  a.bias = args->rel_bias_dev;
  a.n_dist = args->n_dist;
  a.heads = heads;
  a.n_seqs = n_seqs;
  a.dtype = args->dtype;
  a.warps = paged_warps(shape.width, device);
  a.prefix = reinterpret_cast<long long *>(args->work_dev);
  a.parts = reinterpret_cast<float *>(reinterpret_cast<uint8_t *>(args->work_dev) + ((int64_t)(n_seqs + 1) * 8 + 15) / 16 * 16);
  a.scale = args->scale > 0.f ? args->scale : 1.f / sqrtf((float)cache->head_dim);
  DeviceGuard guard(device);
  if (!guard.ok) return cuda_fail(cudaGetLastError(), "cudaSetDevice");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool wide = shape.group > 8, e4m3 = cache->format == QMOE_CACHE_E4M3;
  const size_t smem = (size_t)(kPagedThreads / 32) * kPagedStages * paged_stage(paged_units(shape.width)) + 12 * (size_t)(n_seqs + 1);
  const unsigned grid = (unsigned)(a.warps / (kPagedThreads / 32));
  auto run = [&](auto nb) {
    constexpr int NB = decltype(nb)::value;
    auto kernel = e4m3 ? (wide ? k_decode_paged<NB, QMOE_CACHE_E4M3, true> : k_decode_paged<NB, QMOE_CACHE_E4M3, false>)
                       : (wide ? k_decode_paged<NB, QMOE_CACHE_INT8, true> : k_decode_paged<NB, QMOE_CACHE_INT8, false>);
    const int allowed = allow_shared(reinterpret_cast<const void *>(kernel), (int)smem, device);
    if (allowed != QMOE_OK) return allowed;
    QMOE_LAUNCH(kernel, grid, kPagedThreads, smem, st, a);
    QMOE_CUDA(cudaGetLastError());
    return QMOE_OK;
  };
  int done = QMOE_OK;
  switch (paged_units(shape.width)) {
    case 1: done = run(std::integral_constant<int, 1>()); break;
    case 2: done = run(std::integral_constant<int, 2>()); break;
    case 4: done = run(std::integral_constant<int, 4>()); break;
    case 5: done = run(std::integral_constant<int, 5>()); break;
    case 6: done = run(std::integral_constant<int, 6>()); break;
    case 8: done = run(std::integral_constant<int, 8>()); break;
    case 12: done = run(std::integral_constant<int, 12>()); break;
    default: done = run(std::integral_constant<int, 16>()); break;
  }
  if (done != QMOE_OK) return done;
  cudaLaunchAttribute overlap{};
  overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  overlap.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3((unsigned)(n_seqs * heads));
  config.blockDim = dim3(kJoinThreads);
  config.dynamicSmemBytes = (a.warps + 256 * (kJoinThreads / 32)) * sizeof(float);
  config.stream = st;
  config.attrs = &overlap;
  config.numAttrs = 1;
  QMOE_CUDA(cudaLaunchKernelEx(&config, k_decode_join, a));
  count_launch();
  QMOE_CUDA(cudaGetLastError());
  return QMOE_OK;
}

}  // extern "C"
