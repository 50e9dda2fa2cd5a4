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

// exp((l - max) / temperature) in 64 bits, and as a multiple of 2^-45: at most 2^18 of them, each at
// most 1, fit 64 bits, and integer sums are the same in every order.
__device__ __forceinline__ double weight_of(float l, double top, double inv_t) { return exp(((double)l - top) * inv_t); }
__device__ __forceinline__ unsigned long long mass_of(double w) { return __double2ull_rn(w * kMassUnit); }

// The kept mass that the token's has to exceed: u of `total`, u clamped to [0, 1).
__device__ __forceinline__ unsigned long long target_of(float u, unsigned long long total) {
  const double at = (u > 0.f ? (double)u : 0.0) * (double)total;
  const unsigned long long target = at >= (double)total ? total - 1 : (unsigned long long)at;
  return target >= total ? total - 1 : target;
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
//   2. where something is cut off: counts of the logits in kBins bins of equal width below the largest, which
//      give the bin of the k-th largest exactly and bounds on the bin in which the mass reaches top_p
//   3. a) the tokens up to the k-th largest's bin are few: they are gathered in index order, and the first CTA
//         does the rest on them;
//      b) else the borderline token of each cut is found: the exact mass up to every bin in question, the
//         tokens of the one bin gathered, their order by counting; what is kept is then everything above the
//         borderline token (by logit, then by index)
//   4. kept mass per warp's segment, the segment and the token that the uniform number falls into
// The bins only select, so their rounding does not matter; everything that decides is done on the logits'
// order and on integer masses.  A bin that holds more than kList tokens (a row of almost equal logits) sends
// the row to sample_by_radix, which reads it again from global memory.
constexpr int kRowThreads = 512;
constexpr int kRowWarps = kRowThreads / 32;
constexpr int kBins = 2048;
constexpr int kList = 1024;
constexpr int kMaxCluster = 8;

struct RowShared {
  unsigned long long sum[kRowWarps], list[kList], mass[kList];
  unsigned long long total, below, pick[2];      // exchanged: kept mass, mass of sure bins, borderline token
  uint32_t hist[kBins], limb[3][kBins];          // counts; exact masses of the bins in question in 3 limbs
  uint32_t top_key, low_key;
  float red[kRowWarps];
  int bad, first, flag, scan[kRowWarps];
  int b_k, above_k, upto_k, b_lo, b_hi, above_p, in_p;
  unsigned long long above_mass;
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
  for (int w = 0; w < kRowWarps; w++) {
    if (w < warp) before += scratch[w];
    all += scratch[w];
  }
  return v + before;
}

// The same for a row in which too many tokens lie in one bin: one CTA, which reads the row again for every step.
// Keys of the k-th largest and of the cut by mass by radix selection on counts and on masses.
template <typename T>
__device__ void sample_by_radix(const SampleArgs &a, int row, uint32_t top_key, unsigned long long *s_sum, unsigned long long *s_hist) {
  __shared__ int s_cnt[32];
  __shared__ uint32_t s_prefix;
  __shared__ unsigned long long s_left;
  __shared__ int s_found;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = a.vocab;
  const T *logits = reinterpret_cast<const T *>(a.logits) + row * a.row_stride;
  const float t = a.temperature != nullptr ? a.temperature[row] : 1.f;

  const float top = key_value(top_key);
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
      for (int i = tid; i < n; i += kRowThreads) {
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
  const int per_warp = (n + 32 * kRowWarps - 1) / (32 * kRowWarps) * 32;
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
  for (int v = 0; v < kRowWarps; v++) {
    if (v == warp) before = total;
    total += s_sum[v];
  }
  const float u = a.uniform[row];
  const unsigned long long target = target_of(u, total);
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
  const double min_w = least > 0.f ? fmin((double)least, 1.0) : 0.0;
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
    for (int i = kVec * tid; i + kVec <= n; i += kVec * kRowThreads) {
      const uint4 v = __ldg(reinterpret_cast<const uint4 *>(logits + i));
      const T *e = reinterpret_cast<const T *>(&v);
#pragma unroll
      for (int x = 0; x < kVec; x++) take(i + x, to_f32(e[x]));
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
    sh.total = sh.below = 0;
  }
  for (int i = tid; i < kBins; i += kRowThreads) sh.hist[i] = sh.limb[0][i] = sh.limb[1][i] = sh.limb[2][i] = 0;
  __syncthreads();
  top_key = __reduce_max_sync(0xffffffffu, top_key);
  low_key = __reduce_min_sync(0xffffffffu, low_key);
  bad = __any_sync(0xffffffffu, bad);
  if (lane == 0) {
    atomicMax(&sh.top_key, top_key);
    atomicMin(&sh.low_key, low_key);
    if (bad) sh.bad = 1;
  }
  cluster.sync();
  bad = false;
  for (int r = 0; r < ranks; r++) {
    top_key = max(top_key, peer(r)->top_key);
    low_key = min(low_key, peer(r)->low_key);
    bad = bad || peer(r)->bad != 0;
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
  const double dtop = (double)top, inv_t = 1.0 / (double)t;
  auto entry = [](float l, int index) { return (unsigned long long)order_key(l) << 32 | (uint32_t)~index; };  // order: logit, then lower index
  auto entry_weight = [&](unsigned long long e) { return weight_of(key_value((uint32_t)(e >> 32)), dtop, inv_t); };
  unsigned long long edge = 0;  // kept: entries not below it

  if (cut_k || cut_p) {
    // ---- 2. bins
    const float span = fminf(40.f * t, top - (low_key == 0xffffffffu ? top : key_value(low_key)));
    const float per_bin = span > 0.f ? (kBins - 1) / span : 0.f;
    auto bin_of = [&](float l) { return l > -1e30f ? min(kBins - 1, (int)((top - l) * per_bin)) : kBins - 1; };
    for (int i = tid; i < n; i += kRowThreads) atomicAdd(&sh.hist[bin_of(s_logit[i])], 1u);
    cluster.sync();
    constexpr int kPer = kBins / kRowThreads;
    uint32_t count[kPer], mine = 0, all;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      count[i] = 0;
      for (int r = 0; r < ranks; r++) count[i] += peer(r)->hist[tid * kPer + i];
      mine += count[i];
    }
    uint32_t before = block_scan(mine, reinterpret_cast<uint32_t *>(sh.scan), all) - mine;
    const uint32_t before0 = before;
    if (tid == 0) {
      sh.b_k = kBins;
      sh.above_k = sh.upto_k = a.vocab;
    }
    __syncthreads();
    if (cut_k) {
#pragma unroll
      for (int i = 0; i < kPer; i++) {
        if (before < (uint32_t)k && before + count[i] >= (uint32_t)k) {
          sh.b_k = tid * kPer + i;
          sh.above_k = (int)before;
          sh.upto_k = (int)(before + count[i]);
        }
        before += count[i];
      }
    }
    __syncthreads();
    const int b_k = sh.b_k, above_k = sh.above_k, upto_k = sh.upto_k;

    // The entries of the slice's tokens in bins [from, to], in index order, to the first CTA's list, the slices
    // one after another.  Whole cluster; the counts are known to fit.
    auto gather = [&](int from, int to) {
      uint32_t at = 0;  // entries of the CTAs before this one, from their histograms
      for (int r = 0; r < rank; r++)
        for (int b = from + tid; b <= to; b += kRowThreads) at += peer(r)->hist[b];
      at = block_total(at, reinterpret_cast<uint32_t *>(sh.scan));
      unsigned long long *list = peer(0)->list;
      for (int i0 = 0; i0 < n; i0 += kRowThreads) {
        const int i = i0 + tid;
        const int b = i < n ? bin_of(s_logit[i]) : kBins;
        const bool in = b >= from && b <= to;
        if (__syncthreads_or(in) == 0) continue;
        uint32_t here;
        const uint32_t upto = block_scan<uint32_t>(in, reinterpret_cast<uint32_t *>(sh.scan), here);
        if (in) list[at + upto - 1] = entry(s_logit[i], first_index + i);
        at += here;
        __syncthreads();
      }
      cluster.sync();
    };

    if (cut_k && upto_k <= kList) {
      // ---- 3a. all that can be kept in the first CTA
      gather(0, b_k);
      if (rank == 0) {
        const int m = upto_k;
        for (int j = tid; j < m; j += kRowThreads) sh.mass[j] = mass_of(entry_weight(sh.list[j]));
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
          const bool kept = order[x] < k && (!cut_p || ahead[x] < goal || order[x] == 0) && entry_weight(sh.list[j]) >= min_w;
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
            leave((long long)(uint32_t)~(uint32_t)sh.list[j], (float)log(entry_weight(sh.list[j]) * kMassUnit / (double)total));
          upto += here;
        }
      }
      cluster.sync();
      return;
    }

    // ---- 3b. borderline tokens
    // Of the gathered entries of one bin (first CTA): the last in falling order for which `keep(order, mass ahead)`.
    bool lost = false;  // a bin with too many tokens
    auto borderline = [&](int count_in, bool by_mass, unsigned long long ahead_mass, unsigned long long goal, int need) {
      if (rank == 0) {
        if (by_mass) {
          for (int j = tid; j < count_in; j += kRowThreads) sh.mass[j] = sh.list[j] >= edge ? mass_of(entry_weight(sh.list[j])) : 0ull;
        }
        if (tid == 0) sh.pick[0] = ~0ull;
        __syncthreads();
        for (int j = tid; j < count_in; j += kRowThreads) {
          const unsigned long long e = sh.list[j];
          int o = 0;
          unsigned long long sum = ahead_mass;
          for (int i = 0; i < count_in; i++) {
            const bool larger = sh.list[i] > e;
            o += larger;
            if (by_mass) sum += larger ? sh.mass[i] : 0ull;
          }
          if (by_mass ? (sum < goal && e >= edge) : o < need) atomicMin(&sh.pick[0], e);
        }
      }
      cluster.sync();
      edge = max(edge, peer(0)->pick[0]);
      cluster.sync();  // the list and the pick are used again
    };
    if (cut_k) {
      lost = upto_k - above_k > kList;
      if (!lost) {
        gather(b_k, b_k);
        borderline(upto_k - above_k, false, 0, 0, k - above_k);
      }
    }
    if (cut_p && !lost) {
      // bounds: a token of bin b weighs between exp2(-(b + 1) / per_bin / t * log2 e) and the same of b
      const float step = per_bin > 0.f ? 1.4426950408889634f / (per_bin * t) : 0.f;
      float low_mass = 0.f, high_mass = 0.f, low_all, high_all;
      uint32_t seen = before0;
#pragma unroll
      for (int i = 0; i < kPer; i++) {
        const int b = tid * kPer + i;
        // of the k-th largest's bin some are kept; the last bin reaches down to nothing
        const float kept_low = b < b_k ? (float)count[i] : 0.f, kept_high = b <= b_k ? (float)count[i] : 0.f;
        low_mass += kept_low * (b == kBins - 1 ? 0.f : exp2f(-(float)(b + 1) * step));
        high_mass += kept_high * exp2f(-(float)b * step);
        seen += count[i];
      }
      const float low_upto = block_scan(low_mass, sh.red, low_all), high_upto = block_scan(high_mass, sh.red, high_all);
      // first bin that may hold the cut: the upper bound of the mass up to it reaches the lower bound of the goal
      const float goal_low = p * low_all * 0.999f, goal_high = p * high_all * 1.001f;
      if (tid == 0) {
        sh.b_lo = kBins - 1;
        sh.b_hi = kBins - 1;
      }
      __syncthreads();
      float lo = low_upto - low_mass, hi = high_upto - high_mass;
#pragma unroll
      for (int i = 0; i < kPer; i++) {
        const int b = tid * kPer + i;
        lo += (b < b_k ? (float)count[i] : 0.f) * (b == kBins - 1 ? 0.f : exp2f(-(float)(b + 1) * step));
        hi += (b <= b_k ? (float)count[i] : 0.f) * exp2f(-(float)b * step);
        if (hi * 1.001f >= goal_low) atomicMin(&sh.b_lo, b);
        if (lo * 0.999f >= goal_high) atomicMin(&sh.b_hi, b);
      }
      __syncthreads();
      const int b_lo = sh.b_lo, b_hi = min(sh.b_hi, b_k);
      // exact masses: of everything kept, of the bins before b_lo, and of every bin from there to b_hi
      unsigned long long total = 0, below = 0;
      for (int i = tid; i < n; i += kRowThreads) {
        const float l = s_logit[i];
        if (entry(l, first_index + i) < edge) continue;
        const unsigned long long m = mass_of(weight_of(l, dtop, inv_t));
        const int b = bin_of(l);
        total += m;
        if (b < b_lo) below += m;
        else if (b <= b_hi) {
          atomicAdd(&sh.limb[0][b], (uint32_t)(m & 0xffffu));
          atomicAdd(&sh.limb[1][b], (uint32_t)((m >> 16) & 0xffffu));
          atomicAdd(&sh.limb[2][b], (uint32_t)(m >> 32));
        }
      }
      total = block_total(total, sh.sum);
      below = block_total(below, sh.sum);
      if (tid == 0) {
        sh.total = total;
        sh.below = below;
        sh.b_lo = -1;
      }
      cluster.sync();
      total = below = 0;
      for (int r = 0; r < ranks; r++) {
        total += peer(r)->total;
        below += peer(r)->below;
      }
      const unsigned long long goal = max(1ull, p > 0.f ? (unsigned long long)ceil((double)p * (double)total) : 0ull);
      // the bin in which the goal is reached
      unsigned long long m[kPer], own = 0, all_mass;
#pragma unroll
      for (int i = 0; i < kPer; i++) {
        m[i] = 0;
        const int b = tid * kPer + i;
        if (b >= b_lo && b <= b_hi)
          for (int r = 0; r < ranks; r++)
            m[i] += peer(r)->limb[0][b] + ((unsigned long long)peer(r)->limb[1][b] << 16) + ((unsigned long long)peer(r)->limb[2][b] << 32);
        own += m[i];
      }
      unsigned long long ahead = below + block_scan(own, sh.sum, all_mass) - own;
#pragma unroll
      for (int i = 0; i < kPer; i++) {
        if (ahead < goal && ahead + m[i] >= goal && m[i] > 0) {
          sh.b_lo = tid * kPer + i;
          sh.above_mass = ahead;
          sh.in_p = (int)count[i];
        }
        ahead += m[i];
      }
      __syncthreads();
      const int bin = sh.b_lo;
      lost = bin < 0 || sh.in_p > kList;  // the same in every CTA
      if (!lost) {
        const unsigned long long above = sh.above_mass;
        const int in_p = sh.in_p;
        gather(bin, bin);
        borderline(in_p, true, above, goal, 0);
      }
    }
    if (lost) {
      if (rank == 0) sample_by_radix<T>(a, row, top_key, sh.sum, sh.list);
      cluster.sync();
      return;
    }
  }

  // ---- 4. kept mass of every warp's segment, then the token
  const int per_warp = (slice + 32 * kRowWarps - 1) / (32 * kRowWarps) * 32;
  const int begin = min(n, warp * per_warp), end = min(n, begin + per_warp);
  auto kept_weight = [&](int i) {
    const float l = s_logit[i];
    if (entry(l, first_index + i) < edge) return 0.0;
    const double w = weight_of(l, dtop, inv_t);
    return w >= min_w ? w : 0.0;
  };
  unsigned long long mine = 0;
  for (int i = begin + lane; i < end; i += 32) mine += mass_of(kept_weight(i));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  __syncthreads();
  if (lane == 0) sh.sum[warp] = mine;
  __syncthreads();
  if (tid == 0) {
    unsigned long long all = 0;
    for (int w = 0; w < kRowWarps; w++) all += sh.sum[w];
    sh.total = all;
  }
  cluster.sync();
  unsigned long long total = 0, before = 0;
  for (int r = 0; r < ranks; r++) {
    const unsigned long long of = peer(r)->total;
    if (r < rank) before += of;
    total += of;
  }
  for (int w = 0; w < warp; w++) before += sh.sum[w];
  const unsigned long long target = target_of(u, total);
  if (target >= before && target < before + mine) {
    for (int i0 = begin; i0 < end; i0 += 32) {
      const double w = i0 + lane < end ? kept_weight(i0 + lane) : 0.0;
      unsigned long long upto = mass_of(w);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + upto > target);
      if (hit != 0) {
        if (lane == __ffs(hit) - 1) leave(first_index + i0 + lane, (float)log(w * kMassUnit / (double)total));
        break;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  cluster.sync();  // the totals have been read
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
  QMOE_REQUIRE(rows <= 0x7fffffff / kMaxCluster, "too many rows");
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
  // CTAs of a row's cluster: slices of at most 16384 logits where 8 CTAs are enough for that, more CTAs for few
  // rows so that they do not leave most of the GPU idle (slices of 1024 at least)
  int ranks = 1;
  while (ranks < kMaxCluster && (vocab + ranks - 1) / ranks > 16384) ranks *= 2;
  while (ranks < kMaxCluster && 2 * ranks * (int64_t)rows <= sm_count(device) && vocab / (2 * ranks) >= 1024) ranks *= 2;
  const int slice = ((vocab + ranks - 1) / ranks + 7) / 8 * 8;
  auto kernel = dtype == QMOE_FP32 ? k_sample<float> : (dtype == QMOE_BF16 ? k_sample<__nv_bfloat16> : k_sample<__half>);
  const size_t smem = kRowSharedBytes + (size_t)slice * sizeof(float);
  QMOE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
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
