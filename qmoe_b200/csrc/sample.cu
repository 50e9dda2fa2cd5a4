// Sampling of one token per row of logits (qmoe_sample).
#include <cooperative_groups.h>
#include <math.h>

#include "serving.cuh"

namespace qmoe {

constexpr int kMaxVocab = 262144;
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

// Masses: exp((l - max) / temperature) as multiples of 2^-45.  At most 2^18 of them, each at most 2^45, fit 64 bits,
// and integer sums are the same in every order.
// The kept mass that the token's has to exceed: u of `total`, u clamped to [0, 1).
__device__ __forceinline__ unsigned long long target_of(float u, unsigned long long total) {
  const double at = (u > 0.f ? (double)u : 0.0) * (double)total;
  const unsigned long long target = at >= (double)total ? total - 1 : (unsigned long long)at;
  return target >= total ? total - 1 : target;
}

// The mass without the library's exponential: 2^y, y = (l - top) / temperature * log2 e, from a table of 2^(j/256)
// and a polynomial for the rest of the exponent (Tang's table-driven method), all in 64 bits: a relative error
// of 2^-44 with eleven operations, where exp and a conversion take four times as many.  The exponent is added to
// the table's entry; 2^52 is added so that the integer stands in the sum's low bits.
struct MassTable {
  double power[256];
  double top, scale;  // scale = log2 e / temperature
};
__device__ __forceinline__ unsigned long long mass_at(const MassTable &m, float l) {
  const double y = ((double)l - m.top) * m.scale;
  const double n = fma(y, 256.0, 6755399441055744.0);  // nearest integer to 256 y in the low bits
  const int j = __double2loint(n);
  const double r = fma(n - 6755399441055744.0, -0.00390625, y);
  double v = 0.055504112479583289971;
  v = fma(v, r, 0.24022653447679007866);
  v = fma(v, r, 0.69314718055994530942);
  v = fma(v, r, 1.0);
  const double t = m.power[j & 255];
  const double unit = __hiloint2double(__double2hiint(t) + (((j >> 8) + 45) << 20), __double2loint(t));
  const double sum = fma(v, unit, 4503599627370496.0);
  return y > -46.5 ? (unsigned long long)__double_as_longlong(sum) & 0xfffffffffffffull : 0ull;
}

// Log of a token's share of the kept mass, from its own logit (its mass may have few bits).
__device__ __forceinline__ float logprob_of(float l, const MassTable &m, unsigned long long total) {
  return (float)(((double)l - m.top) * m.scale * 0.69314718055994530942 - log((double)total / kMassUnit));
}

template <typename V>
__device__ __forceinline__ V block_total(V v, V *scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  V t = 0;
  for (int w = 0; w < (int)(blockDim.x >> 5); w++) t += scratch[w];
  return t;
}

// ---- one row, by a cluster of CTAs ------------------------------------------------------------------
// The row is read once: every CTA of the cluster keeps a slice of it in shared memory, and what the CTAs find
// out is exchanged through distributed shared memory.
//   1. largest logit (and whether the row has a distribution at all)
//   2. where something is cut off, the logits are put into kBins bins of equal width below the largest, and the
//      bins select a short list of tokens that the cut must be among ("candidates", in index order), so that
//      what is expensive is done for those only:
//      top_k  the k-th largest of the threads' own maxima bounds the k-th largest logit from below; little more
//             than k logits lie above that bound.  Where they are few they are gathered in the first CTA, which
//             does the rest on them
//      top_p  the exact mass of all that is kept; counts per bin bound the bins in which the mass reaches the
//             goal; exact masses of those; the tokens of the one bin gathered, their order by counting.  What is
//             kept is then everything above the borderline token (by logit, then by index)
//   3. kept mass, and the token that the uniform number falls into
// The bins only select, so their rounding does not matter; everything that decides is done on the logits'
// order and on integer masses.  A bin that holds more than kList tokens (a row of almost equal logits) sends
// the row to sample_by_radix, which reads it again from global memory.
// What bounds it: the passes over a slice and the exchanges between them (a barrier of the cluster and a trip through
// distributed shared memory, a microsecond and more each), during which a CTA requests nothing: a cluster has one
// row, and only the SM's second CTA works meanwhile.  With a top_p, of a row's 43 us loading takes 6.5, the masses and
// counts 8.4, selecting and gathering 9.  The 64-bit exponentials (eleven operations a logit at 64 a clock and SM)
// are 20 us of the times below.
// 256 rows of 131072 fp32 logits (134 MB): 84 us for the largest alone, 155 with the masses of the whole row, 164 with a
// top_k of 50, 354 with a top_p of 0.9 (bf16: 77, 149, 162, 363).  Four rows of 32128: 8 us.
constexpr int kRowThreads = 512;
constexpr int kRowWarps = kRowThreads / 32;
constexpr int kBins = 1024;
constexpr int kList = 1024;
constexpr int kCandidates = 8192;  // of a slice
constexpr int kMaxCluster = 8;

struct RowShared {
  MassTable table;
  unsigned long long sum[kRowWarps];
  union {  // the masses are merged before the next list is begun
    struct {
      unsigned long long list[kList], mass[kList];
    };
    uint32_t limb[3][kBins];  // exact masses of the bins in question, in three limbs
  };
  alignas(16) uint32_t hist[kBins];
  uint16_t candidate[kCandidates];
  unsigned long long total, below, pick, above_mass;  // kept mass, mass of sure bins, borderline token
  uint32_t top_key, low_key, inside;
  float red[kRowWarps];
  int bad, first, bin, b_lo, b_hi, above, scan[kRowWarps];
};
constexpr int kRowSharedBytes = (int)((sizeof(RowShared) + 15) / 16 * 16);

// Inclusive prefix sums of the block's threads.
template <typename V>
__device__ __forceinline__ V block_scan(V v, V *scratch, V &all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  __syncthreads();
  if (lane == 31) scratch[warp] = v;
  __syncthreads();
  V before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < kRowWarps; w++) {
    const V x = scratch[w];
    if (w < warp) before += x;
    all += x;
  }
  return v + before;
}

// The same for a row in which too many tokens lie in one bin: one CTA, which reads the row again for every step.
// Keys of the k-th largest and of the cut by mass by radix selection on counts and on masses.
template <typename T>
__device__ void sample_by_radix(const SampleArgs &a, int row, uint32_t top_key, uint32_t least_key, const MassTable &table,
                                unsigned long long *s_sum, unsigned long long *s_hist) {
  __shared__ int s_cnt[32];
  __shared__ uint32_t s_prefix;
  __shared__ unsigned long long s_left;
  __shared__ int s_found;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = a.vocab;
  const T *logits = reinterpret_cast<const T *>(a.logits) + row * a.row_stride;

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
      for (int i = tid; i < n; i += kRowThreads) {
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
    for (int i = tid; i < n; i += kRowThreads) {
      const float l = to_f32(logits[i]);
      const uint32_t key = order_key(l);
      if (key > edge || (!cut_k && key == edge)) z += mass_at(table, l);
    }
    z = block_total(z, s_sum);
    const unsigned long long edge_mass = cut_k ? mass_at(table, key_value(edge)) : 0ull;
    z += edge_mass * (unsigned long long)(cut_k ? edge_count : 0);
    // tokens before which less than `goal` lies: integers below p * z
    const unsigned long long goal = p > 0.f ? (unsigned long long)ceil((double)p * (double)z) : 0ull;
    uint32_t prefix = 0;
    unsigned long long above = 0;  // mass of the keys above the prefix's range
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) s_hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += kRowThreads) {
        const float l = to_f32(logits[i]);
        const uint32_t key = order_key(l);
        if ((key > edge || (!cut_k && key == edge)) && (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))))
          atomicAdd(&s_hist[(key >> shift) & 255], mass_at(table, l));
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
    const unsigned long long w = mass_at(table, key_value(prefix));
    const unsigned long long need = max(goal, 1ull) - above;  // > 0
    const unsigned long long count = w > 0 ? (need + w - 1) / w : (unsigned long long)n;
    const int limit = prefix == edge && cut_k ? edge_count : n;
    edge = prefix;
    edge_count = (int)min(count, (unsigned long long)limit);
  }
  // segments of 32-element strides, one per warp: tokens equal to the edge, then kept mass
  const int per_warp = (n + 32 * kRowWarps - 1) / (32 * kRowWarps) * 32;
  const int begin = min(n, warp * per_warp), end = min(n, begin + per_warp);
  int ties = 0;
  for (int i = begin + lane; i < end; i += 32) ties += order_key(to_f32(logits[i])) == edge;
  ties = __reduce_add_sync(0xffffffffu, ties);
  if (lane == 0) s_cnt[warp] = ties;
  __syncthreads();
  int ties_before = 0;
  for (int w = 0; w < warp; w++) ties_before += s_cnt[w];
  auto kept_mass = [&](int i, int &seen) {
    const float l = i < end ? to_f32(logits[i]) : -INFINITY;
    const uint32_t key = i < end ? order_key(l) : 0u;
    const unsigned tied = __ballot_sync(0xffffffffu, i < end && key == edge);
    const int rank = seen + __popc(tied & ((1u << lane) - 1u));
    seen += __popc(tied);
    const bool kept = i < end && (key > edge || (key == edge && rank < edge_count)) && key >= least_key;
    return kept ? mass_at(table, l) : 0ull;
  };
  unsigned long long mine = 0;
  int seen = ties_before;
  for (int i = begin; i < end; i += 32) mine += kept_mass(i + lane, seen);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  __syncthreads();
  if (lane == 0) s_sum[warp] = mine;
  __syncthreads();
  unsigned long long total = 0, before = 0;
  for (int v = 0; v < kRowWarps; v++) {
    if (v == warp) before = total;
    total += s_sum[v];
  }
  const float u = a.uniform[row];
  const unsigned long long target = target_of(u, total);
  if (target < before || target >= before + mine) return;
  seen = ties_before;
  for (int i = begin; i < end; i += 32) {
    const unsigned long long m = kept_mass(i + lane, seen);
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
        if (a.logprob != nullptr) a.logprob[row] = logprob_of(to_f32(logits[i + lane]), table, total);
      }
      return;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
}


template <typename T>
__global__ void __launch_bounds__(kRowThreads) k_sample(const SampleArgs a, const int slice) {
  namespace cg = cooperative_groups;
  extern __shared__ __align__(16) uint8_t row_smem[];
  RowShared &sh = *reinterpret_cast<RowShared *>(row_smem);
  float *s_logit = reinterpret_cast<float *>(row_smem + kRowSharedBytes);  // slice
  const cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), row = blockIdx.x / ranks;
  const int first_index = rank * slice, n = max(0, min(slice, a.vocab - first_index));
  const T *logits = reinterpret_cast<const T *>(a.logits) + row * a.row_stride + first_index;
  const float t = a.temperature != nullptr ? a.temperature[row] : 1.f;
  const int k = a.top_k != nullptr ? a.top_k[row] : 0;
  const float p = a.top_p != nullptr ? a.top_p[row] : 1.f, u = a.uniform[row];
  const float least = a.min_p != nullptr ? a.min_p[row] : 0.f;
  const bool cut_k = k > 0 && k < a.vocab, cut_p = p < 1.f;
  auto peer = [&](int r) { return cluster.map_shared_rank(&sh, r); };
  auto leave = [&](long long token, float logprob) {  // by one thread
    a.tokens[row] = token;
    if (a.logprob != nullptr) a.logprob[row] = logprob;
  };

  // ---- 1. the slice, its largest logit and the smallest that is not a mask
  bool bad = false;
  uint32_t top_key = 0, low_key = 0xffffffffu;
  auto take = [&](int i, float l) {
    s_logit[i] = l;
    bad = bad || !(l <= FLT_MAX);
    const uint32_t key = order_key(l);
    top_key = max(top_key, key);
    if (l > -1e30f) low_key = min(low_key, key);
  };
  constexpr int kVec = 16 / sizeof(T);
  if ((reinterpret_cast<uintptr_t>(logits) & 15u) == 0) {
    constexpr int kAhead = 8;  // loads under way
    for (int i0 = kVec * tid; i0 + kVec <= n; i0 += kAhead * kVec * kRowThreads) {
      uint4 v[kAhead];
#pragma unroll
      for (int y = 0; y < kAhead; y++) {
        const int i = i0 + y * kVec * kRowThreads;
        if (i + kVec <= n) v[y] = __ldg(reinterpret_cast<const uint4 *>(logits + i));
      }
#pragma unroll
      for (int y = 0; y < kAhead; y++) {
        const int i = i0 + y * kVec * kRowThreads;
        if (i + kVec > n) break;
        const T *e = reinterpret_cast<const T *>(&v[y]);
#pragma unroll
        for (int x = 0; x < kVec; x++) take(i + x, to_f32(e[x]));
      }
    }
    for (int i = n / kVec * kVec + tid; i < n; i += kRowThreads) take(i, to_f32(logits[i]));
  } else {
#pragma unroll 4
    for (int i = tid; i < n; i += kRowThreads) take(i, to_f32(logits[i]));
  }
  if (tid == 0) {
    sh.top_key = 0;
    sh.low_key = 0xffffffffu;
    sh.bad = 0;
    sh.first = 0x7fffffff;
  }
  for (int i = tid; i < kBins; i += kRowThreads) sh.hist[i] = 0;
  if (tid < 256) sh.table.power[tid] = exp2((double)tid / 256.0);
  __syncthreads();
  const uint32_t thread_top = top_key;
  top_key = __reduce_max_sync(0xffffffffu, top_key);
  low_key = __reduce_min_sync(0xffffffffu, low_key);
  bad = __any_sync(0xffffffffu, bad);
  if (lane == 0) {
    atomicMax(&sh.top_key, top_key);
    atomicMin(&sh.low_key, low_key);
    if (bad) sh.bad = 1;
  }
  cluster.sync();
  {
    const RowShared *of = peer(lane < ranks ? lane : rank);
    top_key = __reduce_max_sync(0xffffffffu, of->top_key);
    low_key = __reduce_min_sync(0xffffffffu, of->low_key);
    bad = __any_sync(0xffffffffu, of->bad != 0);
  }
  const float top = key_value(top_key);
  if (bad || top == -INFINITY || !(t >= 0.f) || t > FLT_MAX) {
    if (rank == 0 && tid == 0) leave(-1, __int_as_float(0x7fffffff));
    cluster.sync();
    return;
  }
  if (t == 0.f) {
    for (int i = tid; i < n; i += kRowThreads)
      if (order_key(s_logit[i]) == top_key) {
        atomicMin(&sh.first, first_index + i);
        break;
      }
    cluster.sync();
    if (rank == 0 && tid == 0) {
      int first = 0x7fffffff;
      for (int r = 0; r < ranks; r++) first = min(first, peer(r)->first);
      leave(first, 0.f);
    }
    cluster.sync();
    return;
  }
  if (tid == 0) {
    sh.table.top = (double)top;
    sh.table.scale = 1.4426950408889634074 / (double)t;
  }
  __syncthreads();
  const MassTable &table = sh.table;
  auto entry = [](float l, int index) { return (unsigned long long)order_key(l) << 32 | (uint32_t)~index; };  // order: logit, then lower index
  auto entry_mass = [&](unsigned long long e) { return mass_at(table, key_value((uint32_t)(e >> 32))); };
  // Smallest key with at least min_p of the largest weight: a search among all keys, 32 at a time.
  uint32_t least_key = 0;
  if (least > 0.f) {
    const double min_w = fmin((double)least, 1.0);
    uint32_t low = order_key(-FLT_MAX), high = top_key;  // the largest has enough
    while (low < high) {
      const uint32_t step = (high - low) / 32 + 1;
      const unsigned long long at = (unsigned long long)low + (unsigned long long)lane * step;
      const uint32_t key = (uint32_t)min(at, (unsigned long long)high);
      const bool enough = exp(((double)key_value(key) - (double)top) / (double)t) >= min_w;
      const unsigned who = __ballot_sync(0xffffffffu, enough);
      const int f = who == 0 ? 32 : __ffs(who) - 1;
      const unsigned long long new_low = f == 0 ? low : (unsigned long long)low + (unsigned long long)(f - 1) * step + 1;
      if (f < 32) high = (uint32_t)min((unsigned long long)high, (unsigned long long)low + (unsigned long long)f * step);
      low = (uint32_t)min(new_low, (unsigned long long)high);
    }
    least_key = high;
  }
  unsigned long long edge = 0;  // kept: entries not below it
  // A value of every CTA, read by the lanes at once: their sum, and that of the CTAs before this one.
  auto exchange = [&](auto of, auto &before_this) {
    auto v = of(lane < ranks ? peer(lane) : &sh);
    if (lane >= ranks) v = 0;
    auto upto = v;
#pragma unroll
    for (int o = 1; o < kMaxCluster; o <<= 1) {
      const auto x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    before_this = __shfl_sync(0xffffffffu, upto, rank) - __shfl_sync(0xffffffffu, v, rank);
    return __shfl_sync(0xffffffffu, upto, kMaxCluster - 1);
  };
  // Tokens that are still in question: the slice's, or the candidates among them, in index order.
  int n_left = n;
  bool selected = false;
  auto place = [&](int j) { return selected ? (int)sh.candidate[j] : j; };

  if (cut_k || cut_p) {
    // ---- 2. bins
    const float span = fminf(40.f * t, top - (low_key == 0xffffffffu ? top : key_value(low_key)));
    const float per_bin = span > 0.f ? (kBins - 1) / span : 0.f;
    auto bin_of = [&](float l) {  // 2^23 is added so that the nearest integer stands in the low bits; a mask's bin is the last
      return l > -1e30f ? __float_as_int(fminf((top - l) * per_bin, kBins - 1) + 8388608.f) - 0x4b000000 : kBins - 1;
    };
    constexpr int kPer = kBins / kRowThreads;
    uint32_t count[kPer];
    // The cluster's counts of this thread's bins.
    auto merge = [&]() {
      cluster.sync();
      uint2 h[kMaxCluster];
#pragma unroll
      for (int r = 0; r < kMaxCluster; r++) h[r] = *reinterpret_cast<const uint2 *>(&peer(r < ranks ? r : rank)->hist[tid * kPer]);
      count[0] = count[1] = 0;
#pragma unroll
      for (int r = 0; r < kMaxCluster; r++) {
        count[0] += r < ranks ? h[r].x : 0u;
        count[1] += r < ranks ? h[r].y : 0u;
      }
    };
    static_assert(kPer == 2, "two bins a thread");
    // First bin up to which `goal` tokens lie (kBins: none), and the tokens before it.
    auto bin_of_rank = [&](uint32_t goal) {
      uint32_t all;
      uint32_t before = block_scan(count[0] + count[1], reinterpret_cast<uint32_t *>(sh.scan), all) - count[0] - count[1];
      if (tid == 0) sh.bin = kBins;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kPer; i++) {
        if (before < goal && before + count[i] >= goal) {
          sh.bin = tid * kPer + i;
          sh.above = (int)before;
        }
        before += count[i];
      }
      __syncthreads();
      return sh.bin;
    };
    auto clear_counts = [&]() {
      cluster.sync();  // they have been read
      for (int i = tid; i < kBins; i += kRowThreads) sh.hist[i] = 0;
      __syncthreads();
    };
    // Leaves the tokens in bins [0, to] in question, unless there are too many.  Every warp looks at a segment of
    // what is in question, so that the order stays.
    auto select = [&](int to) {
      const int part = (n_left + 32 * kRowWarps - 1) / (32 * kRowWarps) * 32;
      const int begin = min(n_left, warp * part), end = min(n_left, begin + part);
      uint32_t mine = 0, all;
#pragma unroll 4
      for (int j = begin + lane; j < end; j += 32) mine += bin_of(s_logit[place(j)]) <= to;
      mine = __reduce_add_sync(0xffffffffu, mine);
      uint32_t at = block_scan<uint32_t>(lane == 0 ? mine : 0u, reinterpret_cast<uint32_t *>(sh.scan), all);
      if (all > kCandidates || selected) return;  // narrowed down once only: the list is not written over itself
      at = __shfl_sync(0xffffffffu, at, 0) - mine;
      for (int j0 = begin; j0 < end; j0 += 32) {
        const bool in = j0 + lane < end && bin_of(s_logit[j0 + lane]) <= to;
        const unsigned who = __ballot_sync(0xffffffffu, in);
        if (in) sh.candidate[at + __popc(who & ((1u << lane) - 1u))] = (uint16_t)(j0 + lane);
        at += __popc(who);
      }
      __syncthreads();
      n_left = (int)all;
      selected = true;
    };
    // The entries of the tokens in question that lie in bins [from, to], in index order, to the first CTA's list,
    // the slices one after another.  Returns their number; more than kList of them are not written.
    auto gather = [&](int from, int to) {
      const int part = (n_left + 32 * kRowWarps - 1) / (32 * kRowWarps) * 32;
      const int begin = min(n_left, warp * part), end = min(n_left, begin + part);
      auto inside = [&](int j) {
        if (j >= end) return false;
        const int b = bin_of(s_logit[place(j)]);
        return b >= from && b <= to;
      };
      uint32_t mine = 0, all, at_slice;
#pragma unroll 4
      for (int j = begin + lane; j < end; j += 32) mine += inside(j);
      mine = __reduce_add_sync(0xffffffffu, mine);
      uint32_t at = block_scan<uint32_t>(lane == 0 ? mine : 0u, reinterpret_cast<uint32_t *>(sh.scan), all);
      at = __shfl_sync(0xffffffffu, at, 0) - mine;
      if (tid == 0) sh.inside = all;
      cluster.sync();
      const uint32_t total = exchange([](const RowShared *r) { return r->inside; }, at_slice);
      at += at_slice;
      if (total <= kList && mine > 0) {
        unsigned long long *list = peer(0)->list;
        for (int j0 = begin; j0 < end; j0 += 32) {
          const bool in = inside(j0 + lane);
          const unsigned who = __ballot_sync(0xffffffffu, in);
          if (in) {
            const int i = place(j0 + lane);
            list[at + __popc(who & ((1u << lane) - 1u))] = entry(s_logit[i], first_index + i);
          }
          at += __popc(who);
        }
      }
      cluster.sync();
      return (int)total;
    };
    // Of the gathered entries of one bin (first CTA): the last in falling order that is kept, which is the edge.
    auto borderline = [&](int count_in, bool by_mass, unsigned long long ahead_mass, unsigned long long goal, int need) {
      if (rank == 0) {
        if (by_mass) {
          for (int j = tid; j < count_in; j += kRowThreads) sh.mass[j] = sh.list[j] >= edge ? entry_mass(sh.list[j]) : 0ull;
        }
        if (tid == 0) sh.pick = ~0ull;
        __syncthreads();
        for (int j = tid; j < count_in; j += kRowThreads) {
          const unsigned long long e = sh.list[j];
          int o = 0;
          unsigned long long sum = ahead_mass;
#pragma unroll 4
          for (int i = 0; i < count_in; i++) {
            const bool larger = sh.list[i] > e;
            o += larger;
            if (by_mass) sum += larger ? sh.mass[i] : 0ull;
          }
          if (by_mass ? (sum < goal && e >= edge) : o < need) atomicMin(&sh.pick, e);
        }
      }
      cluster.sync();
      edge = max(edge, peer(0)->pick);
      cluster.sync();  // the list and the pick are used again
    };

    bool lost = false;  // a bin with too many tokens
    if (cut_k) {
      int gathered = kList + 1, b_k = kBins;
      if (k <= ranks * kRowThreads / 4) {
        if (thread_top != 0) atomicAdd(&sh.hist[bin_of(key_value(thread_top))], 1u);
        merge();
        b_k = bin_of_rank((uint32_t)k);
        if (b_k < kBins) {
          select(b_k);
          gathered = gather(0, b_k);
        }
        if (gathered > kList) clear_counts();
      }
      if (gathered > kList) {  // counts of all logits
        for (int j = tid; j < n_left; j += kRowThreads) atomicAdd(&sh.hist[bin_of(s_logit[place(j)])], 1u);
        merge();
        b_k = bin_of_rank((uint32_t)k);
        const int above = sh.above;
        select(b_k);
        gathered = gather(0, b_k);
        if (gathered > kList) {
          const int in_bin = gather(b_k, b_k);
          lost = in_bin > kList;
          if (!lost) borderline(in_bin, false, 0, 0, k - above);
          clear_counts();
        }
      }
      if (gathered <= kList) {
        // All that can be kept is in the first CTA; nobody looks into the others any more.
        if (rank == 0) {
          const int m = gathered;
          for (int j = tid; j < m; j += kRowThreads) sh.mass[j] = entry_mass(sh.list[j]);
          __syncthreads();
          unsigned long long z = 0, ahead[kList / kRowThreads];
          int order[kList / kRowThreads];
#pragma unroll
          for (int x = 0; x < kList / kRowThreads; x++) {
            const int j = tid + x * kRowThreads;
            ahead[x] = 0;
            order[x] = kList;
            if (j >= m) continue;
            const unsigned long long e = sh.list[j];
            int o = 0;
            unsigned long long sum = 0;
#pragma unroll 4
            for (int i = 0; i < m; i++) {
              const bool larger = sh.list[i] > e;
              o += larger;
              sum += larger ? sh.mass[i] : 0ull;
            }
            order[x] = o;
            ahead[x] = sum;
            if (o < k) z += sh.mass[j];
          }
          z = block_total(z, sh.sum);
          const unsigned long long goal = p > 0.f ? (unsigned long long)ceil((double)p * (double)z) : 0ull;
          __syncthreads();
#pragma unroll
          for (int x = 0; x < kList / kRowThreads; x++) {
            const int j = tid + x * kRowThreads;
            if (j >= m) continue;
            const bool kept = order[x] < k && (!cut_p || ahead[x] < goal || order[x] == 0) && (uint32_t)(sh.list[j] >> 32) >= least_key;
            if (!kept) sh.mass[j] = 0;
          }
          __syncthreads();
          // list order is index order: neighbouring entries per thread
          constexpr int kEach = kList / kRowThreads;
          unsigned long long own = 0, total;
#pragma unroll
          for (int x = 0; x < kEach; x++) own += kEach * tid + x < m ? sh.mass[kEach * tid + x] : 0ull;
          unsigned long long upto = block_scan(own, sh.sum, total);
          const unsigned long long target = target_of(u, total);
          upto -= own;
          for (int x = 0; x < kEach; x++) {
            const int j = kEach * tid + x;
            const unsigned long long here = j < m ? sh.mass[j] : 0ull;
            if (here > 0 && target >= upto && target < upto + here)
              leave((long long)(uint32_t)~(uint32_t)sh.list[j], logprob_of(key_value((uint32_t)(sh.list[j] >> 32)), table, total));
            upto += here;
          }
        }
        return;
      }
    }
    if (cut_p && !lost) {
      // the mass of all that is kept, and counts per bin
      unsigned long long total = 0, below = 0, unused;
#pragma unroll 2
      for (int j = tid; j < n_left; j += kRowThreads) {
        const int i = place(j);
        const float l = s_logit[i];
        if (entry(l, first_index + i) < edge) continue;
        total += mass_at(table, l);
        atomicAdd(&sh.hist[bin_of(l)], 1u);
      }
      total = block_total(total, sh.sum);
      if (tid == 0) sh.total = total;
      merge();
      total = exchange([](const RowShared *r) { return r->total; }, unused);
      const unsigned long long goal = max(1ull, p > 0.f ? (unsigned long long)ceil((double)p * (double)total) : 0ull);
      // Bounds: a token of bin b weighs between 2^(-(b + 1/2) step) and 2^(-(b - 1/2) step); what lies behind the
      // last bin as little as nothing.  The bins in which the mass may reach the goal:
      const float step = per_bin > 0.f ? 1.4426950408889634f / (per_bin * t) : 0.f, goal_f = (float)goal * (float)(1.0 / kMassUnit);
      float low[kPer], high[kPer], unused_f;
#pragma unroll
      for (int i = 0; i < kPer; i++) {
        const int b = tid * kPer + i;
        low[i] = b == kBins - 1 ? 0.f : (float)count[i] * exp2f(-((float)b + 0.5f) * step);
        high[i] = (float)count[i] * exp2f(-((float)b - 0.5f) * step);
      }
      float low_upto = block_scan(low[0] + low[1], sh.red, unused_f) - low[1];
      float high_upto = block_scan(high[0] + high[1], sh.red, unused_f) - high[1];
      if (tid == 0) sh.b_lo = sh.b_hi = kBins - 1;
      for (int i = tid; i < kBins; i += kRowThreads) sh.limb[0][i] = sh.limb[1][i] = sh.limb[2][i] = 0;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kPer; i++) {
        if (high_upto * 1.001f >= goal_f) atomicMin(&sh.b_lo, tid * kPer + i);
        if (low_upto * 0.999f >= goal_f) atomicMin(&sh.b_hi, tid * kPer + i);
        low_upto += low[1];
        high_upto += high[1];
      }
      __syncthreads();
      const int b_lo = sh.b_lo, b_hi = sh.b_hi;
      select(b_hi);
      // exact masses: of the bins before b_lo together, of every bin from there to b_hi
      for (int j = tid; j < n_left; j += kRowThreads) {
        const int i = place(j);
        const float l = s_logit[i];
        const int b = bin_of(l);
        if (b > b_hi || entry(l, first_index + i) < edge) continue;
        const unsigned long long m = mass_at(table, l);
        if (b < b_lo) {
          below += m;
        } else {
          atomicAdd(&sh.limb[0][b], (uint32_t)(m & 0xffffu));
          atomicAdd(&sh.limb[1][b], (uint32_t)((m >> 16) & 0xffffu));
          atomicAdd(&sh.limb[2][b], (uint32_t)(m >> 32));
        }
      }
      below = block_total(below, sh.sum);
      if (tid == 0) {
        sh.below = below;
        sh.bin = -1;
      }
      cluster.sync();
      below = exchange([](const RowShared *r) { return r->below; }, unused);
      // the bin in which the goal is reached
      unsigned long long m[kPer], all_mass;
#pragma unroll
      for (int i = 0; i < kPer; i++) {
        const int b = tid * kPer + i;
        m[i] = 0;
        if (b < b_lo || b > b_hi) continue;
#pragma unroll
        for (int r = 0; r < kMaxCluster; r++) {
          const RowShared *from = peer(r < ranks ? r : rank);
          const unsigned long long of =
              from->limb[0][b] + ((unsigned long long)from->limb[1][b] << 16) + ((unsigned long long)from->limb[2][b] << 32);
          m[i] += r < ranks ? of : 0ull;
        }
      }
      unsigned long long ahead = below + block_scan(m[0] + m[1], sh.sum, all_mass) - m[0] - m[1];
#pragma unroll
      for (int i = 0; i < kPer; i++) {
        if (ahead < goal && ahead + m[i] >= goal && m[i] > 0) {
          sh.bin = tid * kPer + i;
          sh.above_mass = ahead;
        }
        ahead += m[i];
      }
      __syncthreads();
      const int bin = sh.bin;
      const unsigned long long above = sh.above_mass;
      const int in_bin = bin < 0 ? kList + 1 : gather(bin, bin);  // the same in every CTA
      lost = in_bin > kList;
      if (!lost) borderline(in_bin, true, above, goal, 0);
    }
    if (lost) {
      cluster.sync();  // the exchanged values have been read
      if (rank == 0) sample_by_radix<T>(a, row, top_key, least_key, table, sh.sum, sh.list);
      return;
    }
  }

  // ---- 3. kept mass of every warp's segment of what is in question, then the token
  edge = max(edge, (unsigned long long)least_key << 32);
  const int part = (n_left + 32 * kRowWarps - 1) / (32 * kRowWarps) * 32;
  const int begin = min(n_left, warp * part), end = min(n_left, begin + part);
  auto kept_mass = [&](int j) {
    const int i = place(j);
    const float l = s_logit[i];
    return entry(l, first_index + i) >= edge ? mass_at(table, l) : 0ull;
  };
  unsigned long long mine = 0;
#pragma unroll 4
  for (int j = begin + lane; j < end; j += 32) mine += kept_mass(j);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  __syncthreads();
  if (lane == 0) sh.sum[warp] = mine;
  __syncthreads();
  if (tid == 0) {
    unsigned long long all = 0;
#pragma unroll
    for (int w = 0; w < kRowWarps; w++) all += sh.sum[w];
    sh.total = all;
  }
  cluster.sync();
  unsigned long long before;
  const unsigned long long total = exchange([](const RowShared *r) { return r->total; }, before);
  const unsigned long long target = target_of(u, total);
  int seg = -1;  // the segment it falls into
  unsigned long long seg_before = before;
#pragma unroll
  for (int w = 0; w < kRowWarps; w++) {
    const unsigned long long of = sh.sum[w];
    if (target >= before && target < before + of) {
      seg = w;
      seg_before = before;
    }
    before += of;
  }
  if (seg >= 0) {  // the whole CTA looks at its tokens, neighbouring tokens per thread
    const int seg_begin = min(n_left, seg * part), seg_end = min(n_left, seg_begin + part);
    for (int j0 = seg_begin; j0 < seg_end; j0 += 2 * kRowThreads) {
      const int j = j0 + 2 * tid;
      const unsigned long long m0 = j < seg_end ? kept_mass(j) : 0ull, m1 = j + 1 < seg_end ? kept_mass(j + 1) : 0ull;
      unsigned long long all;
      const unsigned long long upto = seg_before + block_scan(m0 + m1, sh.sum, all);
      if (target < upto && target >= upto - m0 - m1) {
        const int at = place(target < upto - m1 ? j : j + 1);
        leave(first_index + at, logprob_of(s_logit[at], table, total));
      }
      seg_before += all;
    }
  }
  cluster.sync();  // the totals have been read
}

}  // namespace qmoe

using namespace qmoe;

extern "C" int qmoe_sample(const qmoe_sample_args *args, int device, void *stream) {
  QMOE_REQUIRE(args != nullptr, "null pointer");
  const int rows = args->rows, vocab = args->vocab, dtype = args->dtype;
  QMOE_REQUIRE(rows >= 0 && vocab >= 1 && args->row_stride >= 0, "bad shape");
  QMOE_REQUIRE(dtype == QMOE_FP32 || dtype == QMOE_BF16 || dtype == QMOE_FP16, "logits are fp32, bf16 or fp16");
  if (rows == 0) return QMOE_OK;
  QMOE_REQUIRE(rows <= 0x7fffffff / kMaxCluster, "too many rows");
  QMOE_REQUIRE(args->logits_dev && args->uniform_dev && args->tokens_dev, "null device pointer");
  if (vocab > kMaxVocab) {
    set_error("%s: at most %d logits a row are supported", __func__, kMaxVocab);
    return QMOE_ERR_UNSUPPORTED;
  }
  const SampleArgs a{args->logits_dev, args->row_stride, vocab, args->temperature_dev, args->top_p_dev, args->min_p_dev,
                     args->uniform_dev, args->top_k_dev, reinterpret_cast<long long *>(args->tokens_dev), args->logprob_dev};
  DeviceGuard guard(device);
  if (!guard.ok) return cuda_fail(cudaGetLastError(), "cudaSetDevice");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  // CTAs of a row's cluster: slices of at most 16384 logits where 8 CTAs are enough for that, more CTAs for few
  // rows so that they do not leave most of the GPU idle (slices of 1024 at least)
  int ranks = 1;
  while (ranks < kMaxCluster && (vocab + ranks - 1) / ranks > 16384) ranks *= 2;
  while (ranks < kMaxCluster && 2 * ranks * (int64_t)rows <= sm_count(device) && vocab / (2 * ranks) >= 1024) ranks *= 2;
  const int slice = ((vocab + ranks - 1) / ranks + 7) / 8 * 8;
  auto kernel = dtype == QMOE_FP32 ? k_sample<float> : (dtype == QMOE_BF16 ? k_sample<__nv_bfloat16> : k_sample<__half>);
  const size_t smem = kRowSharedBytes + (size_t)slice * sizeof(float);
  const int allowed = allow_shared(reinterpret_cast<const void *>(kernel), (int)smem, device);
  if (allowed != QMOE_OK) return allowed;
  cudaLaunchAttribute cluster{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = (unsigned)ranks;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3((unsigned)(rows * ranks));
  config.blockDim = dim3(kRowThreads);
  config.dynamicSmemBytes = smem;
  config.stream = st;
  config.attrs = &cluster;
  config.numAttrs = 1;
  QMOE_CUDA(cudaLaunchKernelEx(&config, kernel, a, slice));
  count_launch();
  return QMOE_OK;
}
