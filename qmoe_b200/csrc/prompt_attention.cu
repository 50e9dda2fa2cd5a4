// Causal attention over a packed batch of prompts (qmoe_prompt_attention).
#include <cuda.h>
#include <math.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "serving.cuh"
#include "tcgen05.cuh"

namespace qmoe {

struct PromptArgs {
  const void *q, *k, *v;
  void *out;
  const int32_t *cu_q, *cu_k;
  const float *bias;
  qmoe_prompt_args s;
  // split keys (n_parts > 1): every part's output rows and their (maximum in units of log 2, sum)
  float *part_out;    // [row][head][part][8 * chunks columns]
  float2 *part_stat;  // [row][head][part]
  int n_parts;
  int row_step, head_step;  // of an item's second query tile from its first: 128 rows further on, or the next head
  unsigned long long wait_ns;  // bound of the waits that decide to give up
};

// One query row of one head by one warp, a running maximum over the keys; 32 lanes share the head's values.  A key whose
// weight is 0 contributes nothing, whatever its value row holds.  Bound by the way from a key's load over five
// exchanges between the lanes and an exponential to its weight, so several keys are on that way at a time (2048 tokens,
// 8 heads of 256: 2.7 ms; one key at a time 8.8).
// `progress`, if given, moves at least every kProgressKeys keys: others of the CTA wait meanwhile.
constexpr int kProgressKeys = 1024;
template <typename T, int J>  // J >= ceil(head_dim / 32)
__device__ __forceinline__ void attend_row(const PromptArgs &a, int head, int row, int2 rq, int2 rk, int *progress = nullptr) {
  constexpr int kKeys = 32 / J;  // at a time
  const int lane = threadIdx.x & 31;
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
  for (int t0 = 0; t0 <= last; t0 += kKeys) {
    if (progress != nullptr && t0 % kProgressKeys == 0 && lane == 0) atomicAdd(progress, 1);
    T kk[kKeys][J], vv[kKeys][J];
#pragma unroll
    for (int x = 0; x < kKeys; x++) {
      const long long at = rk.x + (long long)min(t0 + x, last);
      const T *k = reinterpret_cast<const T *>(a.k) + at * a.s.k_row + kv * a.s.k_head;
      const T *v = reinterpret_cast<const T *>(a.v) + at * a.s.v_row + kv * a.s.v_head;
#pragma unroll
      for (int j = 0; j < J; j++) {
        kk[x][j] = lane + 32 * j < d ? k[lane + 32 * j] : from_f32<T>(0.f);
        vv[x][j] = lane + 32 * j < d ? v[lane + 32 * j] : from_f32<T>(0.f);
      }
    }
    float s[kKeys];
#pragma unroll
    for (int x = 0; x < kKeys; x++) {
      s[x] = 0.f;
#pragma unroll
      for (int j = 0; j < J; j++)
        if (lane + 32 * j < d) s[x] += qv[j] * to_f32(kk[x][j]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int x = 0; x < kKeys; x++) s[x] += __shfl_xor_sync(0xffffffffu, s[x], o);
    float m_new = m;
#pragma unroll
    for (int x = 0; x < kKeys; x++) {
      const float b = bias != nullptr ? bias[max(0, min(last - t0 - x, a.s.n_dist - 1))] : 0.f;
      s[x] = b == -INFINITY || t0 + x > last ? -INFINITY : s[x] * a.s.scale + b;  // masked, whatever the key holds
      m_new = fmaxf(m_new, s[x]);
    }
    const float base = m_new == -INFINITY ? 0.f : m_new;  // scores of -inf only so far
    const float keep = expf(m - base);
    m = m_new;
    sum *= keep;
#pragma unroll
    for (int j = 0; j < J; j++) acc[j] *= keep;
#pragma unroll
    for (int x = 0; x < kKeys; x++) {
      const float p = expf(s[x] - base);
      sum += p;
#pragma unroll
      for (int j = 0; j < J; j++) acc[j] += p != 0.f ? p * to_f32(vv[x][j]) : 0.f;
    }
  }
  T *out = reinterpret_cast<T *>(a.out) + row * a.s.out_row + head * a.s.out_head;
#pragma unroll
  for (int j = 0; j < J; j++)
    if (lane + 32 * j < d) out[lane + 32 * j] = from_f32<T>(sum == 0.f ? 0.f : acc[j] / sum);
}

template <typename T>
__global__ void __launch_bounds__(128) k_prompt_rows(const PromptArgs a) {
  const int row = blockIdx.y * 4 + (threadIdx.x >> 5);
  if (row >= a.s.total_q) return;
  const int seq = packed_seq(a.cu_q, a.s.n_seqs, row);
  if (seq < 0) return;
  attend_row<T, 8>(a, blockIdx.x, row, packed_rows(a.cu_q, seq, a.s.total_q), packed_rows(a.cu_k, seq, a.s.total_k));
}

// ---- tensor-core tiles ----------------------------------------------------------------------------
// One CTA per SM takes items of work one after another: two tiles of 128 queries, of one head or of two that share
// their keys (two_heads), the keys walked 128 at a time:
//   S[128 queries, 128 keys] = Q K^T        both from shared memory, fp32 in tensor memory
//   P = exp2(S * scale * log2 e - m)        by a warpgroup per query tile, one thread per query; P
//                                           replaces S in tensor memory as 16-bit values
//   O[128 queries, head_dim] += P V         P from tensor memory, V from shared memory
// Roles: warps 0-3 and 4-7 the two softmax warpgroups, which also write the output; warp 8 issues the matrix
// instructions; warp 9 finds out from the offsets what the items are; warps 12-15 copy queries, and keys and
// values into a ring of four buffers.  While one query tile's softmax runs, the tensor core works for the other,
// and the next item's tiles come in while this one's output is written (one CTA per item instead: 126 against
// 110 us for 16 uneven prompts of 8192 tokens together, 32 heads of 128; 105 with two heads an item, 93 with the items in order).
// Few items with many keys are split along the keys (key_parts): every part leaves its unfinished rows, maximum and
// sum in the workspace, and a second kernel joins them.
//
// Bound by the chain scores -> softmax -> product of each tile: a step of 2 x 128 queries by 128 keys takes 3200 clocks
// over one long prompt and 3700 over uneven ones, of which the tensor core works 2048 at head_dim 128 (in 900 to 1000
// of them a softmax warp waits for its scores).  The same warps rescale O, and write an item's output in another 4600
// clocks, in which the tensor core has nothing to do: a quarter of the time of 16 uneven prompts.  The exponentials are the softmax's
// largest part (a special function unit gives 16 results a clock and SM: 2048 clocks a step), so two pairs of
// eight are polynomials on the FMA units (1165 instead of 1143 TFLOP/s over one prompt of 8192 tokens).
// One prompt of 16384 tokens, 32 heads of 128: 1.96 to 2.01 ms, 1.10 to 1.12 PFLOP/s; 16 uneven prompts of 8192 tokens
// together 91 to 94 us.
//
// Every tile lies in shared memory as rows of 64 columns (128 bytes) under the 128-byte swizzle, one block
// of 128 rows per 64 columns: K-major for Q and K, and the same bytes with the head axis contiguous for V.
// Tiles come by bulk tensor copies, a sequence's last, partial key tile by the copying warps, which write zeros
// behind the last row.  Tensors that no tensor map describes are packed first.
// The running maximum is only moved when it grew by more than 2^8: O then stays as it is and P and the
// sum are taken relative to the older maximum, which is exact up to rounding since both are scaled alike.
// P is rounded to the type of the inputs for the second product (half a step of it relative to every
// weight); the sum is taken from the unrounded fp32 weights.
// A query that sees a score of NaN or +inf, which the tiles' maxima show, gets NaN, as the formula has it.
// A query row is computed again by a warp of its own where its result is not finite, as a value row that is not finite
// spoils queries that give it weight 0 too (0 * inf), and where its scores are so large (2^27 and more) that the rounded
// maximum lies some units of log 2 beside the largest score, by which all weights could underflow or overflow.
// That is some hundred times slower than the tiles: 4096 tokens, 32 heads of 128, take 120 us, and 42 ms with an
// infinite first value row, which every query sees.
// All waits are bounded (kPromptWait); when one runs out the CTA counts itself in d_prompt_timeouts, waits for its
// copies and products in flight, frees its tensor memory and returns.
constexpr int kPromptThreads = 512;
constexpr int kPromptRegs = 128;  // at launch; the softmax warps then hold 192 and the others 64
constexpr int kTileRows = 128;
constexpr int kStages = 4;
constexpr int kItems = 4;         // decided ahead
constexpr int kItemReaders = 10;  // arrivals that give an item back: eight softmax warps, one for products, one for copies
constexpr int kBlockBytes = kTileRows * 128;  // 64 columns of a tile
constexpr int kPolyPairs = 2;
constexpr int kWave = 148;      // CTAs at a time
constexpr int kMaxParts = 32;   // a warp's lanes look after one each when they are joined
constexpr unsigned long long kPromptWait = 4000000000ull;  // ns without progress
__device__ int d_prompt_timeouts;

struct PromptMaps {
  CUtensorMap q, k, v;
};

struct PromptBars {
  uint64_t q_full, q_empty, s_full[2], p_full[2][2], pv_done[2], kv_full[kStages], kv_empty[kStages];
  uint64_t item_full[kItems], item_empty[kItems], drain;
};

// The bound in use: tests lower it so that waits run out without anything hanging (1: give up without polling;
// 0: kPromptWait).  The clean-up waits before a block ends have their own, which stays.
static std::atomic<long long> g_prompt_wait_ns{0};

// Waits for a phase of a barrier for `limit` nanoseconds at most, or until another wait of the CTA ran out.
// `fail[1]` moves while rows are computed again key by key, which takes as long as it takes (up to some seconds for a
// row of 2^25 keys): when it has moved, the wait begins again.
__device__ __forceinline__ bool wait_until(uint32_t bar, uint32_t parity, volatile int *fail, unsigned long long limit) {
  if (limit != 1 && mbar_wait(bar, parity, 2)) return true;
  unsigned long long now, begin;
  int seen = fail[1];
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(begin));
  while (limit != 1) {
    if (mbar_wait(bar, parity, 2)) return true;
    if (*fail) return false;
    if (seen != fail[1]) {
      seen = fail[1];
      asm volatile("mov.u64 %0, %globaltimer;" : "=l"(begin));
    }
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now));
    if (now - begin >= limit) break;
  }
  *fail = 1;
  return false;
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A bias in units of log 2.  The lowest finite values stay finite: a row of them is a row of equal scores.
constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float in_log2(float b) { return b == -INFINITY ? b : fmaxf(b * kLog2e, -FLT_MAX); }

// NaN if one of them is.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max2(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// 2^x of a pair without the special function unit, which is what bounds the softmax (16 results a clock and
// SM).  x = n + f with n the nearest integer (adding 1.5 * 2^23 leaves it in the low bits), 2^f by the
// degree-4 polynomial of least relative error on [-1/2, 1/2] (2.6e-6, an order below the rounding of the
// weights to 16 bits, 2^-9 or 2^-11), n added to the exponent.  x below -126 gives about 2^-126.
__device__ __forceinline__ pair_t pair_exp2(pair_t x) {
  float lo, hi;
  pair_split(x, lo, hi);
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(lo) : "f"(-126.f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(hi) : "f"(-126.f));
  x = pair_of(lo, hi);
  const pair_t n = pair_add(x, pair_of(12582912.f, 12582912.f));
  const pair_t whole = pair_add(n, pair_of(-12582912.f, -12582912.f));
  const pair_t f = pair_fma(whole, pair_of(-1.f, -1.f), x);
  pair_t p = pair_fma(pair_of(0.009570102207362652f, 0.009570102207362652f), f, pair_of(0.05591785907745361f, 0.05591785907745361f));
  p = pair_fma(p, f, pair_of(0.240247443318367f, 0.240247443318367f));
  p = pair_fma(p, f, pair_of(0.6931217908859253f, 0.6931217908859253f));
  p = pair_fma(p, f, pair_of(0.9999992847442627f, 0.9999992847442627f));
  float n_lo, n_hi;
  pair_split(n, n_lo, n_hi);
  pair_split(p, lo, hi);
  return pair_of(__uint_as_float(__float_as_uint(lo) + (__float_as_uint(n_lo) << 23)),
                 __uint_as_float(__float_as_uint(hi) + (__float_as_uint(n_hi) << 23)));
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&v);
}

// Rows [0, rows) of a tile from global memory (`pitch` elements apart, on 16-byte boundaries), zeros behind them
// and behind the head's values up to 8 * chunks columns: asynchronous copies, to be waited for by the caller.
__device__ __forceinline__ uint32_t tile_offset(int row, int unit) {
  return (uint32_t)((unit >> 3) * kBlockBytes + row * 128 + (((unit & 7) ^ (row & 7)) << 4));
}
template <typename T, int THREADS>
__device__ __forceinline__ void load_tile(uint8_t *tile, const T *src, long long pitch, int rows, int d, int chunks, int tid) {
  const uint32_t base = smem_u32(tile);
  const int shift = chunks > 8 ? 4 : (chunks > 4 ? 3 : 2);
  const int c = tid & ((1 << shift) - 1);
  if (c >= chunks) return;
  const int bytes = max(min(16, 2 * (d - 8 * c)), 0);
#pragma unroll 8
  for (int r = tid >> shift; r < kTileRows; r += THREADS >> shift)
    cp_async16(base + tile_offset(r, c), r < rows ? src + r * pitch + 8 * c : src, r < rows ? bytes : 0);
}

// Copies of tensors whose rows do not begin on 16-byte boundaries, as [rows][heads][pitch] with pitch = head_dim
// rounded up to 8 (what stands behind the head's values is not read).  A pass over the inputs is little next to
// the attention itself; copying such rows value by value inside it was slower even for one tile of 128 queries
// (25 us against 13 us for 32 heads of 65).
struct PackArgs {
  const void *src[3];
  void *dst[3];
  long long row[3], head[3], rows[3];
  int heads[3], d, pitch;
};
template <typename T>
__global__ void __launch_bounds__(256) k_prompt_pack(const PackArgs a) {
  const int which = blockIdx.y, units = a.pitch / 8;
  if (a.dst[which] == nullptr) return;
  const long long n = a.rows[which] * a.heads[which] * units;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const long long item = i / units, row = item / a.heads[which];
    const int unit = (int)(i - item * units), head = (int)(item - row * a.heads[which]);
    const T *src = reinterpret_cast<const T *>(a.src[which]) + row * a.row[which] + head * a.head[which] + 8 * unit;
    __align__(16) T v[8];
#pragma unroll
    for (int x = 0; x < 8; x++) v[x] = 8 * unit + x < a.d ? src[x] : from_f32<T>(0.f);
    reinterpret_cast<uint4 *>(a.dst[which])[i] = *reinterpret_cast<const uint4 *>(v);
  }
}

// What a CTA works on next: two query tiles, or a part of their keys.
struct PromptItem {
  int valid, head, part, tile0;  // part of the keys, its first key tile
  int q_row, n, k_row, m, row0;  // first query row of the tensor, queries, first key row, keys of the sequence
  int steps[2];                               // key tiles that each query tile walks
};

template <typename T, bool BIAS, bool SPLIT>
__global__ void __launch_bounds__(kPromptThreads, 1) k_prompt_tiles(const PromptArgs a, const __grid_constant__ PromptMaps maps) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);  // the swizzle repeats every 1024 bytes
  __shared__ PromptBars s_bar;
  __shared__ PromptItem s_item[kItems];
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_fail[2];
  __shared__ volatile int s_stop[2];
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int d = a.s.head_dim, chunks = 2 * ((d + 15) / 16), blocks = (d + 63) / 64, tile_bytes = blocks * kBlockBytes;
  const int group = a.s.heads / a.s.kv_heads;
  uint8_t *q_tile = smem, *ring = smem + 2 * tile_bytes, *stage_out = ring + kStages * tile_bytes;

  auto bar = [&](uint64_t &b) { return smem_u32(&b); };
  auto wait_or_fail = [&](uint32_t at, uint32_t parity, volatile int *fail) { return wait_until(at, parity, fail, a.wait_ns); };
  if (tid == 0) {
    for (int i = 0; i < 2; i++) {
      mbar_init(bar(s_bar.s_full[i]), 1);
      mbar_init(bar(s_bar.p_full[i][0]), kTileRows);
      mbar_init(bar(s_bar.p_full[i][1]), kTileRows);
      mbar_init(bar(s_bar.pv_done[i]), 1);
    }
    for (int i = 0; i < kStages; i++) {
      mbar_init(bar(s_bar.kv_full[i]), 1);
      mbar_init(bar(s_bar.kv_empty[i]), 1);
    }
    for (int i = 0; i < kItems; i++) {
      mbar_init(bar(s_bar.item_full[i]), 1);
      mbar_init(bar(s_bar.item_empty[i]), kItemReaders);
    }
    mbar_init(bar(s_bar.q_full), 1);
    mbar_init(bar(s_bar.q_empty), 1);
    mbar_init(bar(s_bar.drain), 1);
    s_fail[0] = s_fail[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) tmem_alloc(smem_u32(&s_tmem), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  // Item number `x` of this CTA, by every thread that uses it; false when a wait ran out.  Given back by
  // done_item, once per warp that reads items (the copying warps: once).
  auto get_item = [&](int x, PromptItem &item) {
    const bool ok = wait_or_fail(bar(s_bar.item_full[x % kItems]), (x / kItems) & 1, s_fail);
    item = s_item[x % kItems];
    return ok;
  };
  auto done_item = [&](int x) { mbar_arrive(bar(s_bar.item_empty[x % kItems])); };

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp >= 12) {
      // ---- copies: Q, then K 0, V 0, K 1, V 1, ... of one item after another
      const int t = tid - 384;
      bool ok = true;
      unsigned long long copied = 0, first = 0;  // buffers filled so far, at the beginning of the item
      int q_item = -1;                           // last item whose queries came
      for (int x = 0;; x++) {
        PromptItem item;
        // one decision for all, thread 0's: how often the threads meet below depends on the item, which must not have
        // come to some of them only
        if (t == 0) {
          ok = get_item(x, item) && ok;
          s_stop[0] = !ok || !item.valid;
        }
        named_sync(1, kTileRows);
        const bool stop = s_stop[0];
        item = s_item[x % kItems];
        named_sync(1, kTileRows);
        if (stop) break;
        const int n_steps = max(item.steps[0], item.steps[1]), kv = item.head / group;
        const int n_tma = 2 * max(0, min(n_steps, item.m / kTileRows - (SPLIT ? item.tile0 : 0)));  // whole key tiles come by bulk copies
        if (n_steps > 0) {
          if (t == 0 && x > 0) ok = wait_or_fail(bar(s_bar.q_empty), (x - 1) & 1, s_fail);
          if (t == 0 && ok) {
            const uint32_t q_full = bar(s_bar.q_full);
            mbar_arrive_tx(q_full, (uint32_t)((item.steps[0] > 0) + (item.steps[1] > 0)) * tile_bytes);
            for (int i = 0; i < 2; i++)
              for (int b = 0; item.steps[i] > 0 && b < blocks; b++)
                tma_load3(smem_u32(q_tile) + i * tile_bytes + b * kBlockBytes, &maps.q, 64 * b, item.head + i * a.head_step,
                          item.q_row + item.row0 + i * a.row_step, q_full);
            q_item = x;
          }
        } else if (t == 0) {
          if (x > 0) ok = wait_or_fail(bar(s_bar.q_empty), (x - 1) & 1, s_fail);
          if (ok) {
            mbar_arrive(bar(s_bar.q_full));  // nothing to copy: the phases go on
            q_item = x;
          }
        }
        if (t == 0) {
          for (int c = 0; ok && c < n_tma; c++) {
            const unsigned long long at = first + c;
            const int stage = at % kStages;
            if (at >= kStages) ok = wait_or_fail(bar(s_bar.kv_empty[stage]), (at / kStages - 1) & 1, s_fail);
            if (!ok) break;
            const uint32_t full = bar(s_bar.kv_full[stage]);
            mbar_arrive_tx(full, tile_bytes);
            for (int b = 0; b < blocks; b++)
              tma_load3(smem_u32(ring) + stage * tile_bytes + b * kBlockBytes, (c & 1) ? &maps.v : &maps.k, 64 * b, kv,
                        item.k_row + ((SPLIT ? item.tile0 : 0) + (c >> 1)) * kTileRows, full);
            copied = at + 1;
          }
        }
        __syncwarp();
        bool gave_up = false;
        for (int c = n_tma; c < 2 * n_steps; c++) {
          const unsigned long long at = first + c;
          const int stage = at % kStages;
          if (t == 0) {
            if (ok && at >= kStages) ok = wait_or_fail(bar(s_bar.kv_empty[stage]), (at / kStages - 1) & 1, s_fail);
            s_stop[c & 1] = !ok;
          }
          named_sync(1, kTileRows);
          gave_up = s_stop[c & 1];  // one decision for all: the other entry is written next
          if (gave_up) break;
          const int key0 = ((SPLIT ? item.tile0 : 0) + (c >> 1)) * kTileRows;
          const bool is_v = c & 1;
          const long long pitch = is_v ? a.s.v_row : a.s.k_row;
          const T *src = reinterpret_cast<const T *>(is_v ? a.v : a.k) + (item.k_row + (long long)key0) * pitch +
                         kv * (is_v ? a.s.v_head : a.s.k_head);
          load_tile<T, kTileRows>(ring + stage * tile_bytes, src, pitch, min(kTileRows, item.m - key0), d, chunks, t);
          cp_async_commit();
          cp_async_wait<0>();
          fence_async_proxy();
          named_sync(1, kTileRows);
          if (t == 0) {
            mbar_arrive(bar(s_bar.kv_full[stage]));
            copied = at + 1;
          }
        }
        named_sync(1, kTileRows);  // s_stop is written again; the item has been read by all
        if (gave_up) break;
        first += 2 * n_steps;
        if (t == 0) done_item(x);
      }
      // Copies in flight land before the block ends, whoever gave up and whenever; of every buffer its last filling.
      if (t == 0) {
        if (q_item >= 0) mbar_wait(bar(s_bar.q_full), q_item & 1);
        for (unsigned long long c = copied > kStages ? copied - kStages : 0; c < copied; c++)
          mbar_wait(bar(s_bar.kv_full[c % kStages]), (c / kStages) & 1);
      }
    } else if (warp == 9) {
      // ---- what to work on.  Of 32 sequences at a time, the tiles with the most key tiles first, every tile for all
      // heads (and parts); dealt out to the CTAs forwards and backwards in turn.  Lane l holds sequence s0 + l and its
      // next tile, counted from the sequence's end.
      // (Sequence after sequence and only forwards, 16 uneven prompts of 8192 tokens took 125 us instead of 109, one of
      // 8192 tokens 551 instead of 506; in this order but only forwards 120 and 552.  Taking over CTAs that had not been
      // started, item by item, was no better than forwards.)
      const int item_rows = kTileRows + a.row_step, item_heads = 1 + a.head_step;
      const int of_heads = a.s.heads / item_heads, per_tile = SPLIT ? of_heads * a.n_parts : of_heads;
      int s0 = 0, next = -1, level = -1;
      int2 rq = make_int2(0, 0), rk = rq;
      long long before = 0;
      bool loaded = false;
      auto key_tiles = [&](int i) {  // of the last row of tile i
        const int last = min((i + 1) * item_rows, rq.y - rq.x) - 1 + (rk.y - rk.x) - (rq.y - rq.x);
        return i < 0 ? -1 : (last < 0 ? 0 : last / kTileRows + 1);
      };
      for (int x = 0;; x++) {
        const long long number = (long long)x * gridDim.x + ((x & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
        PromptItem item{};
        while (s0 < a.s.n_seqs) {
          if (!loaded) {
            const bool in = s0 + lane < a.s.n_seqs;
            rq = in ? packed_rows(a.cu_q, s0 + lane, a.s.total_q) : make_int2(0, 0);
            rk = in ? packed_rows(a.cu_k, s0 + lane, a.s.total_k) : make_int2(0, 0);
            next = (rq.y - rq.x + item_rows - 1) / item_rows - 1;
            level = key_tiles(next);
            loaded = true;
          }
          const int top = __reduce_max_sync(0xffffffffu, level);
          if (top < 0) {
            s0 += 32;
            loaded = false;
            continue;
          }
          const unsigned who = __ballot_sync(0xffffffffu, level == top);
          const long long count = (long long)__popc(who) * per_tile;
          if (number < before + count) {
            const long long in_level = number - before;
            const int in_tile = (int)(in_level % per_tile), l = __fns(who, 0, (int)(in_level / per_tile) + 1);
            item.valid = 1;
            item.part = SPLIT ? in_tile / of_heads : 0;
            item.head = (in_tile - item.part * of_heads) * item_heads;
            item.q_row = __shfl_sync(0xffffffffu, rq.x, l);
            item.n = __shfl_sync(0xffffffffu, rq.y, l) - item.q_row;
            item.k_row = __shfl_sync(0xffffffffu, rk.x, l);
            item.m = __shfl_sync(0xffffffffu, rk.y, l) - item.k_row;
            item.row0 = __shfl_sync(0xffffffffu, next, l) * item_rows;
#pragma unroll
            for (int i = 0; i < 2; i++) {
              const int r = item.row0 + i * a.row_step, rows = min(kTileRows, item.n - r);
              const int last = r + rows - 1 + item.m - item.n;
              item.steps[i] = rows <= 0 || last < 0 ? 0 : last / kTileRows + 1;
            }
            if (SPLIT) {
              const int len = (max(item.steps[0], item.steps[1]) + a.n_parts - 1) / a.n_parts;
              item.tile0 = item.part * len;
#pragma unroll
              for (int i = 0; i < 2; i++) item.steps[i] = max(0, min(len, item.steps[i] - item.tile0));
            }
            break;
          }
          before += count;
          if (level == top) level = key_tiles(--next);
        }
        bool ok = x < kItems || wait_or_fail(bar(s_bar.item_empty[x % kItems]), (x / kItems - 1) & 1, s_fail);
        if (!__all_sync(0xffffffffu, ok)) break;
        if (lane == 0) {
          s_item[x % kItems] = item;
          mbar_arrive(bar(s_bar.item_full[x % kItems]));
        }
        __syncwarp();
        if (!item.valid) break;
      }
    } else if (warp == 8) {
      // ---- matrix instructions: the whole warp walks along, one elected lane issues
      const bool bf16 = a.s.dtype == QMOE_BF16;
      const uint32_t idesc_s = make_instr_desc(kTileRows, kTileRows, bf16);
      const uint32_t idesc_o = make_instr_desc(kTileRows, 8 * chunks, bf16, true);
      uint32_t first = 0, done[2] = {0, 0};  // buffers used and products of each tile before this item; may wrap round
      auto tile_addr = [&](int c) { return smem_u32(ring) + ((first + c) % kStages) * tile_bytes; };
      auto wait_tile = [&](int c) {
        return __all_sync(0xffffffffu, wait_or_fail(bar(s_bar.kv_full[(first + c) % kStages]), ((first + c) / kStages) & 1, s_fail));
      };
      auto scores = [&](int i, int j) {
        const uint64_t qa = make_swizzled_desc(smem_u32(q_tile) + i * tile_bytes, 16, 1024);
        const uint64_t ka = make_swizzled_desc(tile_addr(2 * j), 16, 1024);
        for (int c = 0; c < chunks / 2; c++) {  // 16 columns each
          const uint32_t at = ((c >> 2) * kBlockBytes + (c & 3) * 32) >> 4;
          mma_f16_warp(tmem + i * kTileRows, qa + at, ka + at, idesc_s, c > 0);
        }
        mma_commit_warp(bar(s_bar.s_full[i]));
      };
      bool ok = true;
      for (int x = 0;; x++) {
        PromptItem item;
        ok = __all_sync(0xffffffffu, get_item(x, item));
        if (!ok || !item.valid) break;
        const int n_steps = max(item.steps[0], item.steps[1]);
        ok = __all_sync(0xffffffffu, wait_or_fail(bar(s_bar.q_full), x & 1, s_fail));
        if (n_steps > 0) {
          ok = ok && wait_tile(0);
          if (!ok) break;
          tc_fence_after();
          for (int i = 0; i < 2; i++)
            if (item.steps[i] > 0) scores(i, 0);
          mma_commit_warp(bar(s_bar.kv_empty[first % kStages]));
        }
        if (!ok) break;
        if (n_steps <= 1) mma_commit_warp(bar(s_bar.q_empty));
        for (int j = 0; ok && j < n_steps; j++) {
          const bool more = j + 1 < n_steps;
          ok = wait_tile(2 * j + 1) && (!more || wait_tile(2 * j + 2));
#pragma unroll
          for (int i = 0; i < 2; i++) {
            if (!ok || j >= item.steps[i]) continue;
            uint64_t va = make_swizzled_desc(tile_addr(2 * j + 1), kBlockBytes, 1024);
#pragma unroll
            for (int half = 0; half < 2; half++) {
              ok = ok && __all_sync(0xffffffffu, wait_or_fail(bar(s_bar.p_full[i][half]), (done[i] + j) & 1, s_fail));
              if (!ok) continue;
              tc_fence_after();
#pragma unroll
              for (int kk = 4 * half; kk < 4 * half + 4; kk++, va += 2048 >> 4)  // 16 keys each
                mma_f16_ta_warp(tmem + 256 + i * kTileRows, tmem + i * kTileRows + 8 * kk, va, idesc_o, j > 0 || kk > 0);
            }
            if (!ok) continue;
            mma_commit_warp(bar(s_bar.pv_done[i]));
            if (j + 1 < item.steps[i]) scores(i, j + 1);
          }
          if (ok) {
            mma_commit_warp(bar(s_bar.kv_empty[(first + 2 * j + 1) % kStages]));
            if (more) mma_commit_warp(bar(s_bar.kv_empty[(first + 2 * j + 2) % kStages]));
            if (j + 2 == n_steps) mma_commit_warp(bar(s_bar.q_empty));  // the last scores have been issued
          }
        }
        if (!ok) break;
        first += 2 * n_steps;
        done[0] += item.steps[0];
        done[1] += item.steps[1];
        if (lane == 0) done_item(x);
      }
      // Whatever is still in flight ends before tensor memory is freed, also when only the softmax warps gave up.
      mma_commit_warp(bar(s_bar.drain));
      mbar_wait(bar(s_bar.drain), 0);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    // ---- softmax and output: thread t of the warpgroup owns query row t of its tile
    const int i = warp >> 2, t = tid & (kTileRows - 1);
    const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t t_s = lane_base + i * kTileRows, t_o = lane_base + 256 + i * kTileRows;
    const int o_cols = 8 * chunks;
    const float sl2 = a.s.scale * kLog2e;
    uint32_t done = 0;  // key tiles before this item; may wrap round
    bool ok = true;
    for (int x = 0;; x++) {
      PromptItem item;
      ok = __all_sync(0xffffffffu, get_item(x, item));
      if (!ok || !item.valid) break;
      __syncwarp();
      if (lane == 0) done_item(x);
      const int steps = item.steps[i], n = item.n, shift = item.m - item.n, head = item.head + i * a.head_step, tile0 = item.row0 + i * a.row_step;
      const int row = tile0 + t;
      const bool live = row < n;
      const int last = live ? row + shift : -1;  // last key that the query sees
      const float *bias = BIAS ? a.bias + (size_t)head * a.s.n_dist : nullptr;
      float top = -INFINITY, sum = 0.f;  // maximum that O and the sum are relative to, in units of log 2
      bool lost = false;                 // a score was NaN or +inf
      bool rough = false;                // `top` is not near the largest score any more
      float *near_bias = reinterpret_cast<float *>(stage_out + warp * 4096);
      const float far_bias = BIAS ? in_log2(bias[a.s.n_dist - 1]) : 0.f;
      for (int j = 0; j < steps; j++) {
        bool far = true;
        uint32_t gone[5];  // of the 160 distances from the largest on: the bias is -inf
        if (BIAS) {
          // Distances of the tile's keys from the warp's queries: where all are behind the last column, one value for
          // all; else the 32 + 127 values that they can have, looked up while the scores are computed.  Query t
          // and key c find theirs at t + 127 - c.  (Looked up by every query for every key instead, 2049 queries
          // with 2826 keys and 12 heads of 64 took 45 us instead of 37.)
          const int nearest = tile0 + (t & ~31) + shift - ((SPLIT ? item.tile0 : 0) + j) * kTileRows - (kTileRows - 1);
          far = nearest >= a.s.n_dist - 1;
          if (!far) {
            __syncwarp();  // the last ones have been read
#pragma unroll
            for (int x = 0; x < 5; x++) {
              const float b = in_log2(__ldg(bias + max(0, min(nearest + lane + 32 * x, a.s.n_dist - 1))));
              near_bias[lane + 32 * x] = b;
              gone[4 - x] = __brev(__ballot_sync(0xffffffffu, b == -INFINITY));
            }
            __syncwarp();
          } else {
#pragma unroll
            for (int x = 0; x < 5; x++) gone[x] = far_bias == -INFINITY ? 0xffffffffu : 0u;
          }
        }
        ok = wait_or_fail(bar(s_bar.s_full[i]), (done + j) & 1, s_fail);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        tc_fence_after();
        float s[kTileRows];
#pragma unroll
        for (int c = 0; c < 4; c++) tmem_ld32(t_s + 32 * c, reinterpret_cast<uint32_t *>(s) + 32 * c);
#pragma unroll
        for (int c = 0; c < 4; c++) tmem_wait_ld32(reinterpret_cast<uint32_t *>(s) + 32 * c);
        const int key0 = ((SPLIT ? item.tile0 : 0) + j) * kTileRows;
        if (BIAS) {
          if (far) {
#pragma unroll
            for (int c = 0; c < kTileRows; c++) s[c] = fmaf(s[c], sl2, far_bias);
          } else {
#pragma unroll
            for (int c = 0; c < kTileRows; c++) s[c] = fmaf(s[c], sl2, near_bias[lane + kTileRows - 1 - c]);
          }
          // A key that the bias masks may hold anything: its score is replaced, not added to.
          if ((gone[0] | gone[1] | gone[2] | gone[3] | gone[4]) != 0u) {
#pragma unroll
            for (int w = 0; w < 4; w++) {
              const uint32_t mine = __funnelshift_l(gone[w], gone[w + 1], lane);  // bit c: key 32 w + c
#pragma unroll
              for (int c = 0; c < 32; c++) s[32 * w + c] = (mine >> c) & 1u ? -INFINITY : s[32 * w + c];
            }
          }
        }
        const int edge = last - key0;  // columns behind it are masked
        const bool masked = __any_sync(0xffffffffu, edge < kTileRows - 1);
        if (masked) {
#pragma unroll
          for (int c = 0; c < kTileRows; c++) s[c] = c <= edge ? s[c] : -INFINITY;
        }
        float m0 = s[0], m1 = s[1], m2 = s[2], m3 = s[3];
#pragma unroll
        for (int c = 4; c < kTileRows - 4; c += 8) {
          m0 = max3(m0, s[c], s[c + 4]);
          m1 = max3(m1, s[c + 1], s[c + 5]);
          m2 = max3(m2, s[c + 2], s[c + 6]);
          m3 = max3(m3, s[c + 3], s[c + 7]);
        }
        m0 = max3(m0, s[kTileRows - 4], s[kTileRows - 3]);
        m1 = max3(m1, s[kTileRows - 2], s[kTileRows - 1]);
        float tile_top = max2(max3(m0, m1, m2), m3);
        lost = lost || !(tile_top < INFINITY);
        const float raw_top = tile_top;
        if (!BIAS) tile_top *= sl2;
        const bool grow = tile_top > top + 8.f || (top == -INFINITY && tile_top > top);
        if (__any_sync(0xffffffffu, grow)) {
          const float next = grow ? tile_top : top;
          const float keep = grow ? exp2_approx(top - next) : 1.f;
          if (!BIAS) rough = rough || (grow && fabsf(fmaf(raw_top, sl2, -next)) > 4.f);
          top = next;
          sum *= keep;
          if (j > 0) {
            ok = wait_or_fail(bar(s_bar.pv_done[i]), (done + j - 1) & 1, s_fail);
            if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            tc_fence_after();
            for (int c = 0; c < o_cols; c += 16) {
              uint32_t o[16];
              tmem_ld16(t_o + c, o);
#pragma unroll
              for (int x = 0; x < 16; x++) o[x] = __float_as_uint(__uint_as_float(o[x]) * keep);
              tmem_st16(t_o + c, o);
            }
          }
        }
        const float base = top == -INFINITY ? 0.f : top;
        const pair_t minus = pair_of(-base, -base), by = pair_of(sl2, sl2);
        pair_t sums = pair_of(0.f, 0.f);
        // `poly` of 8 pairs go through pair_exp2 (tiles without masked keys: it has no weight of exactly 0)
        auto weights = [&](auto poly) {
#pragma unroll
          for (int half = 0; half < 2; half++) {
#pragma unroll
            for (int c0 = half * 64; c0 < half * 64 + 64; c0 += 32) {
              uint32_t p[16];
#pragma unroll
              for (int c = 0; c < 16; c++) {
                const pair_t v = pair_of(s[c0 + 2 * c], s[c0 + 2 * c + 1]);
                const pair_t x = BIAS ? pair_add(v, minus) : pair_fma(v, by, minus);
                float lo, hi;
                pair_t e;
                if ((c * decltype(poly)::value) % 8 + decltype(poly)::value > 7 && decltype(poly)::value > 0) {
                  e = pair_exp2(x);
                  pair_split(e, lo, hi);
                } else {
                  pair_split(x, lo, hi);
                  lo = exp2_approx(lo);
                  hi = exp2_approx(hi);
                  e = pair_of(lo, hi);
                }
                sums = pair_add(sums, e);
                p[c] = pack2<T>(lo, hi);
              }
              tmem_st16(t_s + c0 / 2, p);
            }
            // the product over these 64 keys starts while the next are worked on
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(bar(s_bar.p_full[i][half]));
          }
        };
        if (BIAS || masked) weights(std::integral_constant<int, 0>());
        else weights(std::integral_constant<int, kPolyPairs>());
        float sum0, sum1;
        pair_split(sums, sum0, sum1);
        sum += sum0 + sum1;
      }
      if (!ok) break;
      if (steps > 0) {
        ok = wait_or_fail(bar(s_bar.pv_done[i]), (done + steps - 1) & 1, s_fail);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
      }
      if (!ok) break;
      done += steps;
      if (SPLIT) {
        const long long at = ((item.q_row + (long long)row) * a.s.heads + head) * a.n_parts + item.part;
        if (live) a.part_stat[at] = make_float2(lost ? __int_as_float(0x7fffffff) : top, rough ? __int_as_float(0x7fffffff) : sum);
        // rows through shared memory, 32 columns at a time (stores by the thread that owns the row took 20 us more
        // for 1024 queries of 32 heads in two parts)
        uint8_t *stage = stage_out + warp * 4096;
        const int t0 = t & ~31, rows = min(32, n - (tile0 + t0));  // of this warp
        const long long pitch = (long long)a.s.heads * a.n_parts * o_cols;
        float *to = a.part_out + (((item.q_row + (long long)(tile0 + t0)) * a.s.heads + head) * a.n_parts + item.part) * o_cols;
        for (int c0 = 0; steps > 0 && c0 < o_cols; c0 += 32) {
          for (int c = c0; c < min(o_cols, c0 + 32); c += 16) {
            uint32_t o[16];
            tmem_ld16(t_o + c, o);
#pragma unroll
            for (int y = 0; y < 4; y++) {
              const int unit = ((c & 31) >> 2) + y;
              *reinterpret_cast<uint4 *>(stage + lane * 128 + ((unit ^ (lane & 7)) << 4)) = make_uint4(o[4 * y], o[4 * y + 1], o[4 * y + 2], o[4 * y + 3]);
            }
          }
          __syncwarp();
          const int u = lane & 7;
          for (int r = lane >> 3; r < rows && c0 + 4 * u < o_cols; r += 4)
            *reinterpret_cast<uint4 *>(to + r * pitch + c0 + 4 * u) = *reinterpret_cast<const uint4 *>(stage + r * 128 + ((u ^ (r & 7)) << 4));
          __syncwarp();
        }
        tc_fence_before();
        continue;
      }
      // Rows go through shared memory, 64 columns at a time, so that a warp writes them one after another instead
      // of one piece of 32 rows at a time.
      const float inv = lost ? __int_as_float(0x7fffffff) : (sum == 0.f ? 0.f : 1.f / sum);
      uint8_t *stage = stage_out + warp * 4096;
      const int t0 = t & ~31, rows = min(32, n - (tile0 + t0));  // of this warp
      T *out = reinterpret_cast<T *>(a.out) + (item.q_row + (long long)(tile0 + t0)) * a.s.out_row + head * a.s.out_head;
      const bool vec = ((reinterpret_cast<uintptr_t>(out) | (uintptr_t)(a.s.out_row * 2) | (uintptr_t)(d * 2)) & 15u) == 0;
      bool finite = true;
      for (int c0 = 0; c0 < o_cols; c0 += 64) {
        for (int c = c0; c < min(o_cols, c0 + 64); c += 16) {
          uint32_t o[16], w[8];
          if (steps > 0) {
            tmem_ld16(t_o + c, o);
          } else {
#pragma unroll
            for (int y = 0; y < 16; y++) o[y] = 0u;
          }
#pragma unroll
          for (int y = 0; y < 8; y++) {
            const float lo = __uint_as_float(o[2 * y]) * inv, hi = __uint_as_float(o[2 * y + 1]) * inv;
            finite = finite && fabsf(lo) <= FLT_MAX && fabsf(hi) <= FLT_MAX;
            w[y] = pack2<T>(lo, hi);
          }
          const int unit = (c & 63) >> 3;
          *reinterpret_cast<uint4 *>(stage + lane * 128 + ((unit ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
          *reinterpret_cast<uint4 *>(stage + lane * 128 + (((unit + 1) ^ (lane & 7)) << 4)) = make_uint4(w[4], w[5], w[6], w[7]);
        }
        __syncwarp();
        const int cols = min(64, d - c0);
        if (vec) {
          const int u = lane & 7;
          for (int r = lane >> 3; r < rows && u < cols / 8; r += 4)
            *reinterpret_cast<uint4 *>(out + r * a.s.out_row + c0 + 8 * u) = *reinterpret_cast<const uint4 *>(stage + r * 128 + ((u ^ (r & 7)) << 4));
        } else {
          for (int r0 = 0; r0 < rows; r0 += 8) {
            for (int c = lane; c < cols; c += 32) {
              T v[8];
#pragma unroll
              for (int r = 0; r < 8; r++)
                v[r] = *reinterpret_cast<const T *>(stage + (r0 + r) * 128 + (((c >> 3) ^ (r & 7)) << 4) + 2 * (c & 7));
#pragma unroll
              for (int r = 0; r < 8; r++)
                if (r0 + r < rows) out[(r0 + r) * a.s.out_row + c0 + c] = v[r];
            }
          }
        }
        __syncwarp();
      }
      tc_fence_before();
      unsigned again = __ballot_sync(0xffffffffu, live && (!finite || rough) && !lost);
      while (again != 0) {
        const int l = __ffs(again) - 1;
        again &= again - 1;
        attend_row<T, 4>(a, head, item.q_row + tile0 + t0 + l, make_int2(item.q_row, item.q_row + n), make_int2(item.k_row, item.k_row + item.m),
                         const_cast<int *>(&s_fail[1]));
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && s_fail[0]) atomicAdd(&d_prompt_timeouts, 1);
  if (warp == 0) tmem_dealloc(tmem, 512);
}

// Joins the parts of split keys, a warp per row and head: out = sum_p 2^(top_p - top) O_p / sum_p 2^(top_p - top) sum_p.
constexpr int kPartsThreads = 256;
template <typename T>
__global__ void __launch_bounds__(kPartsThreads) k_prompt_join(const PromptArgs a) {
  const int lane = threadIdx.x & 31, d = a.s.head_dim, cols = 16 * ((d + 15) / 16);
  const long long item = (long long)blockIdx.x * (kPartsThreads / 32) + (threadIdx.x >> 5);
  const int row = (int)(item / a.s.heads), head = (int)(item - (long long)row * a.s.heads);
  if (row >= a.s.total_q) return;
  const int seq = packed_seq(a.cu_q, a.s.n_seqs, row);
  if (seq < 0) return;
  const int2 rq = packed_rows(a.cu_q, seq, a.s.total_q), rk = packed_rows(a.cu_k, seq, a.s.total_k);
  asm volatile("griddepcontrol.wait;" ::: "memory");  // launched as the last CTAs of the first kernel end
  const float2 stat = lane < a.n_parts ? a.part_stat[item * a.n_parts + lane] : make_float2(-INFINITY, 0.f);
  float top = stat.x;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float weight = stat.y == 0.f ? 0.f : exp2_approx(stat.x - (top == -INFINITY ? 0.f : top));
  float sum = stat.y == 0.f ? 0.f : weight * stat.y;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  const float4 *from = reinterpret_cast<const float4 *>(a.part_out + item * a.n_parts * cols) + lane;
#pragma unroll 4
  for (int p = 0; p < a.n_parts; p++) {
    const float w = __shfl_sync(0xffffffffu, weight, p);
    if (4 * lane >= cols || w == 0.f) continue;  // a part without keys has not been written
    const float4 v = from[(long long)p * (cols / 4)];
    acc[0] += w * v.x;
    acc[1] += w * v.y;
    acc[2] += w * v.z;
    acc[3] += w * v.w;
  }
  bool finite = true;
  T *out = reinterpret_cast<T *>(a.out) + row * a.s.out_row + head * a.s.out_head + 4 * lane;
  const bool lost = __any_sync(0xffffffffu, isnan(stat.x));  // a score was NaN or +inf
  const float inv = lost ? __int_as_float(0x7fffffff) : (sum == 0.f ? 0.f : 1.f / sum);
  __align__(8) T v[4];
#pragma unroll
  for (int x = 0; x < 4; x++) {
    const float o = acc[x] * inv;
    finite = finite && (4 * lane + x >= d || fabsf(o) <= FLT_MAX);
    v[x] = from_f32<T>(o);
  }
  if (!lost && !__all_sync(0xffffffffu, finite)) {
    attend_row<T, 4>(a, head, row, rq, rk);
  } else if (4 * lane + 4 <= d && (reinterpret_cast<uintptr_t>(out) & 7u) == 0) {
    *reinterpret_cast<uint2 *>(out) = *reinterpret_cast<const uint2 *>(v);
  } else {
#pragma unroll
    for (int x = 0; x < 4; x++)
      if (4 * lane + x < d) out[x] = v[x];
  }
}

int set_prompt_wait_limit(int64_t ns) {
  QMOE_REQUIRE(ns >= 0, "a wait cannot be negative");
  g_prompt_wait_ns.store(ns, std::memory_order_relaxed);
  return QMOE_OK;
}

int prompt_timeouts(int reset, int *count) {
  QMOE_CUDA(cudaMemcpyFromSymbol(count, d_prompt_timeouts, sizeof(int)));
  const int zero = 0;
  if (reset) QMOE_CUDA(cudaMemcpyToSymbol(d_prompt_timeouts, &zero, sizeof(int)));
  return QMOE_OK;
}

// Tensor map of [rows][heads][head_dim] with boxes of 64 values, one head and 128 rows; false where the
// driver has no such map.
static bool make_map(CUtensorMap *map, const void *base, int dtype, int d, int heads, int64_t rows, int64_t head_stride,
                     int64_t row_stride) {
  using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                              const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static Encode encode = [] {
    void *f = nullptr;
    cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      return Encode(nullptr);
    }
    return reinterpret_cast<Encode>(f);
  }();
  if (encode == nullptr || rows < 1) return false;
  if (heads == 1) head_stride = 8;  // strides of axes of one entry are not used, but checked
  if (rows == 1) row_stride = 8;
  const cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)heads, (cuuint64_t)rows};
  const cuuint64_t strides[2] = {(cuuint64_t)head_stride * 2, (cuuint64_t)row_stride * 2};
  const cuuint32_t box[3] = {64, 1, (cuuint32_t)kTileRows}, steps[3] = {1, 1, 1};
  return encode(map, dtype == QMOE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                const_cast<void *>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Whether a tensor has to be packed before the tiles can be copied: rows off 16-byte boundaries, or a stride that
// a tensor map does not take (0: one head broadcast to all).
static bool needs_packing(const void *base, int64_t rows, int heads, int64_t row, int64_t head) {
  if (rows <= 0) return false;
  const bool row_ok = rows == 1 || (row > 0 && row % 8 == 0 && row < (1LL << 38)), head_ok = heads == 1 || (head > 0 && head % 8 == 0 && head < (1LL << 38));
  return (reinterpret_cast<uintptr_t>(base) & 15u) != 0 || !row_ok || !head_ok;
}
// An item's two query tiles are the same 128 queries of two neighbouring heads where those share a key head, else 256
// queries of one head.  Two heads walk the same keys, so neither tile waits for the other's last step, and short
// sequences fill both tiles: 64 sequences of 64 tokens 49 instead of 75 us, 8 of 128 queries with 4096 keys 71 instead
// of 125, 16 of 512 tokens 68 instead of 79; one of 8192 tokens 474 instead of 479 (32 query and 8 key heads of 128).
static bool two_heads(const qmoe_prompt_args &s) { return s.heads / s.kv_heads % 2 == 0; }
static int64_t most_items(const qmoe_prompt_args &s, int64_t more) {
  return two_heads(s) ? s.heads / 2 * ((s.total_q + kTileRows - 1) / kTileRows + more)
                      : s.heads * ((s.total_q + 2 * kTileRows - 1) / (2 * kTileRows) + more);
}
// Parts that the keys of every item are split into: as many as leave all items in one wave of CTAs, of two key tiles
// at least in a sequence of mean length.  256 queries with 8192 keys and 8 heads of 128: 22 instead of 118 us, 1024
// tokens 17 instead of 22.  With items for more than half of the SMs the parts' way through memory and the second
// kernel cost as much as the balance gives: 1024 tokens of 32 heads, 128 items, 35 instead of 23 us in two parts.
static int key_parts(const qmoe_prompt_args &s) {
  if (s.head_dim > kTileRows || s.n_seqs < 1 || s.total_q < 1) return 1;
  const int64_t items = std::max(most_items(s, 0), most_items(s, s.n_seqs) - most_items(s, 0));
  const int64_t tiles = (s.total_k / s.n_seqs + kTileRows - 1) / kTileRows;
  return items < 1 ? 1 : (int)std::max<int64_t>(1, std::min<int64_t>({kWave / items, tiles / 2, kMaxParts}));
}
static int64_t part_bytes(const qmoe_prompt_args &s, int parts) {
  return parts <= 1 ? 0 : (s.total_q * s.heads * parts * (16 * ((s.head_dim + 15) / 16) + 2) * 4 + 255) / 256 * 256;
}
static int64_t packed_bytes(int64_t rows, int heads, int d) { return (rows * heads * ((d + 7) / 8 * 16) + 255) / 256 * 256; }

template <typename T>
static int run_prompt(PromptArgs a, void *work, int device, cudaStream_t stream) {
  if (a.s.head_dim > kTileRows) {
    const dim3 grid((unsigned)a.s.heads, (unsigned)((a.s.total_q + 3) / 4));
    QMOE_LAUNCH((k_prompt_rows<T>), grid, 128, 0, stream, a);
    QMOE_CUDA(cudaGetLastError());
    return QMOE_OK;
  }
  // tensors that need it are packed first
  PackArgs pack{};
  pack.d = a.s.head_dim;
  pack.pitch = (a.s.head_dim + 7) / 8 * 8;
  uint8_t *at = reinterpret_cast<uint8_t *>(work);
  long long largest = 0;
  auto prepare = [&](int i, const void *&base, int64_t rows, int heads, int64_t &row, int64_t &head) {
    if (!needs_packing(base, rows, heads, row, head)) return;
    pack.src[i] = base;
    pack.dst[i] = at;
    pack.row[i] = row;
    pack.head[i] = head;
    pack.rows[i] = rows;
    pack.heads[i] = heads;
    base = at;
    head = pack.pitch;
    row = (int64_t)heads * pack.pitch;
    at += packed_bytes(rows, heads, a.s.head_dim);
    largest = largest > rows * heads * (pack.pitch / 8) ? largest : rows * heads * (pack.pitch / 8);
  };
  prepare(0, a.q, a.s.total_q, a.s.heads, a.s.q_row, a.s.q_head);
  prepare(1, a.k, a.s.total_k, a.s.kv_heads, a.s.k_row, a.s.k_head);
  prepare(2, a.v, a.s.total_k, a.s.kv_heads, a.s.v_row, a.s.v_head);
  if (largest > 0) {
    const long long blocks = (largest + 255) / 256;
    QMOE_LAUNCH((k_prompt_pack<T>), dim3((unsigned)(blocks < 16384 ? blocks : 16384), 3), 256, 0, stream, pack);
    QMOE_CUDA(cudaGetLastError());
  }
  a.n_parts = key_parts(a.s);
  a.row_step = two_heads(a.s) ? 0 : kTileRows;
  a.head_step = two_heads(a.s) ? 1 : 0;
  const bool split = a.n_parts > 1;
  const long long wait_ns = g_prompt_wait_ns.load(std::memory_order_relaxed);
  a.wait_ns = wait_ns > 0 ? (unsigned long long)wait_ns : kPromptWait;
  a.part_out = reinterpret_cast<float *>(at);
  a.part_stat = reinterpret_cast<float2 *>(a.part_out + a.s.total_q * a.s.heads * a.n_parts * (16 * ((a.s.head_dim + 15) / 16)));
  PromptMaps maps{};
  // without keys no tile is copied
  if (a.s.total_k > 0 &&
      !(make_map(&maps.q, a.q, a.s.dtype, a.s.head_dim, a.s.heads, a.s.total_q, a.s.q_head, a.s.q_row) &&
                   make_map(&maps.k, a.k, a.s.dtype, a.s.head_dim, a.s.kv_heads, a.s.total_k, a.s.k_head, a.s.k_row) &&
                   make_map(&maps.v, a.v, a.s.dtype, a.s.head_dim, a.s.kv_heads, a.s.total_k, a.s.v_head, a.s.v_row))) {
    set_error("qmoe_prompt_attention: the driver took no tensor map of q, k or v");
    return QMOE_ERR_UNSUPPORTED;
  }
  const int smem = (2 + kStages) * ((a.s.head_dim + 63) / 64) * kBlockBytes + 8 * 4096 + 1024;
  auto kernel = a.bias != nullptr ? (split ? k_prompt_tiles<T, true, true> : k_prompt_tiles<T, true, false>)
                                  : (split ? k_prompt_tiles<T, false, true> : k_prompt_tiles<T, false, false>);
  // the warpgroups' register shares have to fit what the block is launched with
  const int allowed = allow_shared(reinterpret_cast<const void *>(kernel), smem, device, kPromptRegs);
  if (allowed != QMOE_OK) return allowed;
  const long long n_items = most_items(a.s, a.s.n_seqs) * a.n_parts;
  QMOE_REQUIRE(n_items <= 0x7fffffff, "too many heads");
  const long long ctas = n_items < sm_count(device) ? n_items : sm_count(device);
  QMOE_LAUNCH(kernel, (unsigned)ctas, kPromptThreads, smem, stream, a, maps);
  QMOE_CUDA(cudaGetLastError());
  if (split) {
    cudaLaunchAttribute overlap{};
    overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    overlap.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3((unsigned)((a.s.total_q * a.s.heads + kPartsThreads / 32 - 1) / (kPartsThreads / 32)));
    config.blockDim = dim3(kPartsThreads);
    config.stream = stream;
    config.attrs = &overlap;
    config.numAttrs = 1;
    QMOE_CUDA(cudaLaunchKernelEx(&config, k_prompt_join<T>, a));
    count_launch();
  }
  return QMOE_OK;
}

}  // namespace qmoe

using namespace qmoe;

extern "C" int64_t qmoe_prompt_work_bytes(const qmoe_prompt_args *args) {
  if (args == nullptr || args->head_dim > kTileRows || args->head_dim < 1 || args->heads < 1 || args->kv_heads < 1) return 0;
  const qmoe_prompt_args &s = *args;
  int64_t bytes = part_bytes(s, key_parts(s));
  if (needs_packing(s.q_dev, s.total_q, s.heads, s.q_row, s.q_head)) bytes += packed_bytes(s.total_q, s.heads, s.head_dim);
  if (needs_packing(s.k_dev, s.total_k, s.kv_heads, s.k_row, s.k_head)) bytes += packed_bytes(s.total_k, s.kv_heads, s.head_dim);
  if (needs_packing(s.v_dev, s.total_k, s.kv_heads, s.v_row, s.v_head)) bytes += packed_bytes(s.total_k, s.kv_heads, s.head_dim);
  return bytes;
}

extern "C" int qmoe_prompt_attention(const qmoe_prompt_args *args, int device, void *stream) {
  QMOE_REQUIRE(args != nullptr && args->cu_q_dev && args->cu_k_dev, "null pointer");
  PromptArgs a{args->q_dev, args->k_dev, args->v_dev, args->out_dev, args->cu_q_dev, args->cu_k_dev, args->rel_bias_dev, *args};
  QMOE_REQUIRE(a.s.n_seqs >= 0 && a.s.total_q >= 0 && a.s.total_k >= 0, "negative size");
  QMOE_REQUIRE(a.s.heads >= 1 && a.s.kv_heads >= 1 && a.s.heads % a.s.kv_heads == 0 && a.s.head_dim >= 1,
               "heads must be a positive multiple of kv_heads");
  QMOE_REQUIRE(a.s.dtype == QMOE_BF16 || a.s.dtype == QMOE_FP16, "q, k and v are bf16 or fp16");
  QMOE_REQUIRE((a.bias == nullptr) == (a.s.n_dist == 0) && a.s.n_dist >= 0, "bias and n_dist do not agree");
  QMOE_REQUIRE(isfinite(a.s.scale), "scale is not finite");
  if (a.s.n_seqs == 0 || a.s.total_q == 0) return QMOE_OK;
  QMOE_REQUIRE(a.q && a.out && (a.s.total_k == 0 || (a.k && a.v)), "null device pointer");
  // Keys: an item's 2^18 tiles take about half a second, far less than a wait's bound.  Queries of wide heads: the rows
  // kernel's grid.
  if (a.s.head_dim > 256 || a.s.total_q > (a.s.head_dim > kTileRows ? (1 << 18) - 4 : 1 << 25) || a.s.total_k > (1 << 25) || a.s.n_seqs > 32768) {
    set_error("%s: head_dim <= 256, 2^25 query rows (262140 of more than 128 values), 2^25 key rows and 32768 sequences are supported", __func__);
    return QMOE_ERR_UNSUPPORTED;
  }
  QMOE_REQUIRE(qmoe_prompt_work_bytes(args) == 0 || (args->work_dev != nullptr && (reinterpret_cast<uintptr_t>(args->work_dev) & 255u) == 0),
               "workspace is missing or not 256-byte aligned");
  if (a.s.scale <= 0.f) a.s.scale = 1.f / sqrtf((float)a.s.head_dim);
  DeviceGuard guard(device);
  if (!guard.ok) return cuda_fail(cudaGetLastError(), "cudaSetDevice");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return a.s.dtype == QMOE_BF16 ? run_prompt<__nv_bfloat16>(a, args->work_dev, device, st)
                                  : run_prompt<__half>(a, args->work_dev, device, st);
}
