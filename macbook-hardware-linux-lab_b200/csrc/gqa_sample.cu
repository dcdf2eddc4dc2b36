// One token per row of logits by temperature, top-k, top-p and min-p from a
// given uniform number.
//
// The reference's host loop takes the largest logit (qwen_server.c:998-1005);
// its greedy rule (first of the largest) is kept here for temperature 0.
//
// With the row sorted by descending logit, equal logits by ascending index, and
// w = exp((x - max) / temperature), every filter keeps a prefix of that order:
// top-k the first k, top-p the shortest prefix whose weight reaches p times what
// top-k kept, min-p the weights of at least min_p.  So no sort is needed, only
// the last element that is kept, as the pair (logit, index): `ord` below.  The
// token is then the first, in index order, whose cumulative kept weight exceeds
// u times the total.
//
// Weights are formed in 64 bits and summed as integers (units of 2^-wshift of the
// largest weight): a sum is exact in any order, so neither the order of atomics nor
// the split of a row over threads can change a token.  Logits whose weight rounds to
// zero in these units take part in nothing.
//
// A row belongs to a cluster of CTAs, each with a contiguous slice of it in shared
// memory (logits past what fits are read again from memory), so a row is read from
// memory once.  The last kept element is found in two steps: a histogram over 4096
// equal steps of the exponent (they hold few elements each, wherever the logits lie,
// and equal logits fall together), merged over the cluster by reads of the other CTAs'
// shared memory, gives the step; its few elements are listed and ranked by comparing all
// pairs.  Should a step hold more than the list takes (a high temperature, many ties),
// the step is cut again by the pair's 64 bits.  For top-p the histogram holds weights
// rounded to 14 bits; they only propose the step, which the exact sums confirm or move.
//
// Measured: one row of 151936 in fp32 with top-k, top-p and min-p 11.9 us (latency: the load, three
// exchanges over the cluster and the barrier at its end, the ranks); 64 rows with a setting each of
// their own 60 us for two to four passes over the row (the 39 MB take 6).  What bounds the passes is
// not settled: issue slots are 30 % busy, and weights in fp32 took 2 % off.
#include <algorithm>

#include <math_constants.h>

#include "gqa_paged.cuh"
#include "gqa_sample.cuh"

namespace gqa {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 4096;       // eight per thread
constexpr int kList = 512;
// A top_k up to which the row's first k are looked for by way of the threads' largest logits.
constexpr int kSmallK = 256;
constexpr int kMaxCluster = 8;
constexpr int kBlock = kThreads * 4;  // elements of one turn of the CTA's threads

using u64 = unsigned long long;

constexpr int kGroups = 64;                 // of the steps, for the first look over the cluster
constexpr int kInGroup = kBins / kGroups;   // 64: two per lane of a warp
constexpr int kSums = (1 << 20) / kMaxCluster / 128 + kWarps;  // of the largest slice

struct alignas(16) Shared {  // (the slice of the row follows it)
  union {
    uint32_t hist[kBins];
    u64 sums[kSums];  // for the pick: weights of 128 elements each
    struct {          // for the finish, by rank
      u64 ord[kList], w[kList], i[kList], kept[kList];
    } by_rank;
  };
  alignas(16) u64 group[kGroups];      // sums of the histogram's groups
  u64 list_ord[kList];                 // this CTA's elements of the step
  u64 over_ord[kList];                 // and those before it, while they fit
  u64 all_ord[kList], all_w[kList];    // the cluster's
  u64 x[2][4];                         // values exchanged over the cluster
  u64 got[kMaxCluster][4];
  u64 red[kWarps][4];
  double pow2[64];                     // 2^(j / 64 + wshift)
  u64 found_before, found_all, cut;
  int found, row;
  uint32_t n_list, n_over;
  alignas(16) u64 counts[kWarps];  // rows of each class by warp, ten bits a class
};

// Keys in the order of the logits: larger logit, larger key.
__device__ __forceinline__ uint32_t logit_key(float x) {
  const uint32_t u = __float_as_uint(x);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_logit(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}
// -0 as 0, NaN as -inf.
__device__ __forceinline__ float clean(float x) { return fmaxf(x, -CUDART_INF_F) + 0.0f; }

__device__ __forceinline__ u64 ld_cluster_u64(uint32_t addr) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void ld_cluster_v2(uint32_t addr, u64 (&v)[2]) {
  asm volatile("ld.shared::cluster.v2.u64 {%0, %1}, [%2];" : "=l"(v[0]), "=l"(v[1]) : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ld_cluster_v2(uint32_t addr, uint32_t (&v)[2]) {
  asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ u64 warp_sum(u64 x) {
#pragma unroll
  for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
  return x;
}
__device__ __forceinline__ u64 warp_scan(u64 x, int lane) {  // inclusive
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const u64 y = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += y;
  }
  return x;
}

template <typename T>
struct Row {
  const SampleParams& p;
  Shared& sm;
  const T* logits;  // of the slice
  const float* held;
  int lo, n, n_held;  // the slice's first index, its elements, those in shared memory
  int rank, ranks, tid, lane, warp, turn = 0;
  float top;          // largest logit
  bool infinite = false;      // it was infinite: it counts as 0, and all others as -inf
  u64 top_ord;
  int range;          // the steps cover weights down to 2^-range; others round to zero
  float logits_per_step;
  float half_top, rate;  // step of a logit: (half_top - x / 2) * rate
  float floor_x;      // no logit up to this one has a weight
  double t_scale, t_shift;  // a logit's exponent in 64ths: x * t_scale + t_shift
  double most;              // weight of the largest (2^wshift, to the rounding of t_shift)
  float min_p;

  __device__ void settle(u64 best, float temp) {
    top_ord = best;
    top = key_logit((uint32_t)(top_ord >> 32));
    range = p.wshift + 2;
    const double ct = 1.4426950408889634074 / (double)temp;  // of the exponent, per logit
    t_scale = 64.0 * ct;
    t_shift = -(double)top * t_scale;
    half_top = 0.5f * top;
    rate = (float)(2.0 * ct * kBins / range);
    logits_per_step = (float)(range / ct / kBins);
    // Where float logits lie so far apart that the next one below the largest weighs nothing,
    // only the largest (and its equals) count.
    floor_x = -CUDART_INF_F;
    const float next = prev_logit(top);
    if (((double)top - (double)next) * ct > range) {
      floor_x = next;
      t_scale = t_shift = 0.0;
    } else {
      floor_x = below(kBins);
    }
    weight(top, true, most);
  }

  static __device__ __forceinline__ float prev_logit(float x) {
    const uint32_t k = logit_key(x) - 1;
    return key_logit(k == 0x7fffffffu ? k - 1 : k);  // (-0 is not below 0)
  }

  // A logit below all those of step `steps` and less that have a weight.
  __device__ __forceinline__ float below(int steps) const {
    if (steps >= kBins - 1) steps = kBins;  // (the last step takes in what rounds past it)
    return fmaxf(floor_x, top - (steps + 1.5f) * logits_per_step - 1e-6f * fabsf(top));
  }

  __device__ __forceinline__ u64 ord(float x, int i) const {
    return (u64)logit_key(x) << 32 | (0xffffffffu - (uint32_t)(lo + i));
  }

  __device__ __forceinline__ void get4(int i, float (&v)[4]) const {
    if (i < n_held) {  // (n_held is a multiple of 4, padded with -inf)
      const float4 x = *reinterpret_cast<const float4*>(held + i);
      v[0] = x.x;
      v[1] = x.y;
      v[2] = x.z;
      v[3] = x.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        v[e] = i + e < n ? finite(clean(Elem<T>::get(logits[i + e]))) : -CUDART_INF_F;
    }
  }
  __device__ __forceinline__ float finite(float x) const {
    return !infinite ? x : x == CUDART_INF_F ? 0.f : -CUDART_INF_F;
  }

  // f(v, i) for the slice's elements i .. i + 3, four at a time per thread, where one of them
  // is above `least`.
  template <typename F>
  __device__ __forceinline__ void each4(float least, F&& f) const {
#pragma unroll 2
    for (int b = 0; b < n; b += kBlock) {
      const int i = b + 4 * tid;
      float v[4];
      get4(i, v);
      if (fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])) > least) f(v, i);
    }
  }
  // f(x, i) for the elements above `least`.
  template <typename F>
  __device__ __forceinline__ void each(float least, F&& f) const {
    each4(least, [&](const float (&v)[4], int i) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (v[e] > least) f(v[e], i + e);
    });
  }

  // The step of a logit above floor_x: how far below the largest it lies, in equal parts of
  // the exponent.  Non-decreasing in falling x, so steps cut the sorted order; halves keep the
  // difference of two far logits finite.
  __device__ __forceinline__ int step_of(float x) const {
    const int s = (int)(fmaf(-0.5f, x, half_top) * rate);
    return min(s, kBins - 1);
  }

  // The weight in units of 2^-wshift, from 64 bits: 2^(t/64) as 2^(k/64) times the series of
  // the rest (|rest| <= 1/2; Tang's table method, the series to the fourth power is off by
  // 4e-14).  `on`: the logit is above floor_x (others weigh nothing).  No branches, so that the
  // four elements a thread has at a time go through the 64-bit pipe side by side.
  __device__ __forceinline__ u64 weight(float x, bool on, double& w) const {
    const double t = fma((double)x, t_scale, t_shift);
    return weight_at(__hiloint2double(on ? __double2hiint(t) : (int)0xc0ef4000, __double2loint(t)),
                     w);
  }
  __device__ __forceinline__ u64 weight_at(double t, double& w) const {
    constexpr double c = 0.693147180559945309 / 64.0;
    const double magic = 6755399441055744.0;  // 1.5 * 2^52: rounds to an integer
    const double km = t + magic;
    const int k = __double2loint(km);
    const double y = t - (km - magic);
    double q = fma(y, c * c * c * c / 24.0, c * c * c / 6.0);
    q = fma(q, y, c * c / 2.0);
    q = fma(q, y, c);
    q *= y;
    const double b = sm.pow2[k & 63];
    const double m = fma(b, q, b);
    w = __hiloint2double(__double2hiint(m) + ((k & ~63) << 14), __double2loint(m));
    // (a product of at most 2^50 plus 2^52 holds the rounded integer in its low bits)
    return __double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffull;
  }

  // Sums or maxima of N values over the block.
  template <bool kMax, int N>
  __device__ void block_reduce(u64 (&v)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
      for (int d = 16; d; d >>= 1) {
        const u64 y = __shfl_xor_sync(0xffffffffu, v[j], d);
        v[j] = kMax ? (y > v[j] ? y : v[j]) : v[j] + y;
      }
    __syncthreads();
    if (lane == 0)
#pragma unroll
      for (int j = 0; j < N; ++j) sm.red[warp][j] = v[j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < N; ++j) {
      u64 x = sm.red[lane % kWarps][j];
#pragma unroll
      for (int d = kWarps / 2; d; d >>= 1) {
        const u64 y = __shfl_xor_sync(0xffffffffu, x, d);
        x = kMax ? (y > x ? y : x) : x + y;
      }
      v[j] = x;
    }
  }

  // Every CTA's values into sm.got[rank] (a cluster barrier; what a CTA wrote to its
  // shared memory before it, the others may read after it).  The two places alternate: a CTA
  // is past the next barrier only when all have read this one's.
  __device__ void exchange(u64 a, u64 b = 0, u64 c = 0, u64 d = 0) {
    u64* mine = sm.x[turn & 1];
    if (tid < 4) mine[tid] = tid == 0 ? a : tid == 1 ? b : tid == 2 ? c : d;
    __syncwarp();
    cluster_sync();
    if (tid < ranks * 4)
      sm.got[tid >> 2][tid & 3] = ld_cluster_u64(cluster_map(mine + (tid & 3), tid >> 2));
    __syncthreads();
    ++turn;
  }
  __device__ __forceinline__ u64 total(int j) const {
    u64 x = 0;
    for (int r = 0; r < ranks; ++r) x += sm.got[r][j];
    return x;
  }

  __device__ void clear_hist() {
    static_assert(kBins == 8 * kThreads, "eight steps a thread");
#pragma unroll
    for (int j = 0; j < 8; j += 4)
      *reinterpret_cast<uint4*>(&sm.hist[8 * tid + j]) = make_uint4(0, 0, 0, 0);
    if (tid == 0) sm.n_list = sm.n_over = 0;
    __syncthreads();
  }

  // A weight in a histogram of steps: its leading 14 bits or so, shifted by the step's exponent
  // (the same for all of a step, so sums keep their meaning).
  __device__ __forceinline__ int shift_of(int step) const {
    return max(p.wshift - 14 - (step * range / kBins), 0);
  }

  // Puts the sums of the histogram's groups beside it (before an exchange).
  __device__ void sum_groups(bool by_weight) {
    __syncthreads();
    const int s = 8 * tid;
    u64 x = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) x += (u64)sm.hist[s + j] << (by_weight ? shift_of(s + j) : 0);
#pragma unroll
    for (int d = kInGroup / 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    if (tid % (kInGroup / 8) == 0) sm.group[tid / (kInGroup / 8)] = x;
  }

  // After the exchange: the step of the cluster's histogram at which the running sum reaches
  // want (by_weight: that share of the total), into sm.found, the sum before it and the total.
  // The last non-empty one if none does.  By one warp: the groups first, then the group's steps.
  __device__ void find_step(double want, bool share, bool by_weight) {
    if (warp == 0) {
      u64 part[kMaxCluster][2], g[2] = {0, 0};
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r)
        ld_cluster_v2(cluster_map(&sm.group[2 * lane], min(r, ranks - 1)), part[r]);
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r)
        if (r < ranks) {
          g[0] += part[r][0];
          g[1] += part[r][1];
        }
      const u64 incl = warp_scan(g[0] + g[1], lane);
      const u64 all = __shfl_sync(0xffffffffu, incl, 31);
      if (share) want *= (double)all;
      // the last non-empty group before which the sum is below `want`
      const u64 b0 = incl - g[0] - g[1], b1 = incl - g[1];
      int at = -1;
      if (g[0] && (double)b0 < want) at = 2 * lane;
      if (g[1] && (double)b1 < want) at = 2 * lane + 1;
      const int gr = max(__reduce_max_sync(0xffffffffu, at), 0);
      u64 before = __shfl_sync(0xffffffffu, gr & 1 ? b1 : b0, gr >> 1);
      const int s = gr * kInGroup + 2 * lane;
      uint32_t ph[kMaxCluster][2];
      u64 h[2] = {0, 0};
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r)
        ld_cluster_v2(cluster_map(&sm.hist[s], min(r, ranks - 1)), ph[r]);
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r)
        if (r < ranks) {
          h[0] += ph[r][0];
          h[1] += ph[r][1];
        }
      if (by_weight) {
        h[0] <<= shift_of(s);
        h[1] <<= shift_of(s + 1);
      }
      const u64 c0 = before + warp_scan(h[0] + h[1], lane) - h[0] - h[1], c1 = c0 + h[0];
      at = -1;
      if (h[0] && (double)c0 < want) at = 2 * lane;
      if (h[1] && (double)c1 < want) at = 2 * lane + 1;
      const int in = max(__reduce_max_sync(0xffffffffu, at), 0);
      before = __shfl_sync(0xffffffffu, in & 1 ? c1 : c0, in >> 1);
      if (lane == 0) {
        sm.found = gr * kInGroup + in;
        sm.found_before = before;
        sm.found_all = all;
      }
    }
    __syncthreads();
  }

  // The nearest non-empty step after (or before) `step`, or -1 (rarely needed).
  __device__ int neighbour(int step, bool after) {
    int best = -1;
    for (int s = tid; s < kBins; s += kThreads) {
      if (after ? s <= step : s >= step) continue;
      uint32_t h = 0;
      for (int r = 0; r < ranks; ++r) h |= ld_cluster_u32(cluster_map(&sm.hist[s], r));
      if (h) best = max(best, after ? kBins - s : s);
    }
    u64 v[1] = {(u64)(best + 1)};
    block_reduce<true, 1>(v);
    best = (int)v[0] - 1;
    return best < 0 ? -1 : after ? kBins - best : best;
  }

  // Appends an element to a list of the CTA.
  __device__ __forceinline__ static void put(uint32_t& count, u64* list, u64 o) {
    const uint32_t at = atomicAdd(&count, 1u);
    if (at < kList) list[at] = o;
  }

  // The cluster's lists of the step into sm.all_* (counts in the exchange's last value: the
  // step's elements low, those before it high).
  __device__ void collect(bool weights, bool over) {
    int at = 0;
    for (int r = 0; r < ranks; ++r) {
      const int c = (int)(uint32_t)sm.got[r][3], o = over ? (int)(sm.got[r][3] >> 32) : 0;
      for (int i = tid; i < c + o; i += kThreads) {
        const u64* from = i < c ? &sm.list_ord[i] : &sm.over_ord[i - c];
        const u64 e = ld_cluster_u64(cluster_map(from, r));
        sm.all_ord[at + i] = e;
        if (weights) {
          const float x = key_logit((uint32_t)(e >> 32));
          double w64;
          sm.all_w[at + i] = weight(x, x > floor_x, w64);
        }
      }
      at += c + o;
    }
    __syncthreads();
  }

  // Whether the first k of the row are all among n collected elements, found by way of the
  // threads' own largest logits: at least k elements are at or above the k-th largest of
  // those, and few more where the logits are in no particular order.  One count per thread
  // in place of one per logit.
  __device__ bool gather_first(int k, float best, int& n_all) {
    clear_hist();
    if (best > floor_x) atomicAdd(&sm.hist[step_of(best)], 1u);
    sum_groups(false);
    exchange(0);
    find_step(k, false, false);
    // (fewer threads than k have a weight: all that have one)
    const int upto = sm.found_all < (u64)k ? kBins - 1 : sm.found;
    each(below(upto), [&](float x, int i) {
      if (step_of(x) <= upto) put(sm.n_list, sm.list_ord, ord(x, i));
    });
    __syncthreads();
    exchange(0, 0, 0, sm.n_list);
    const u64 count = total(3);
    n_all = (int)min(count, (u64)(1 << 30));
    if (count <= kList) return true;
    __syncthreads();
    cluster_sync();  // (the lists are reused)
    return false;
  }

  // The token from n collected elements that hold all of the row's first k (and, where a
  // target is given, all that it takes to reach it).  By one CTA: ranks by comparing all
  // pairs, prefixes by a scan, and the index order again by pairs.
  __device__ void finish(int n_all, int k, double target, double share, float u, int* token) {
    const int m = min(n_all, k);
    if (tid < n_all) {
      const u64 o = sm.all_ord[tid];
      int at = 0;
#pragma unroll 8
      for (int j = 0; j < n_all; ++j) at += sm.all_ord[j] > o;
      const float x = key_logit((uint32_t)(o >> 32));
      double w64;
      const u64 w = weight(x, x > floor_x, w64);
      sm.by_rank.ord[at] = o;
      // the weight, and whether min_p leaves it out in the top bit (weights stay below 2^51)
      sm.by_rank.w[at] = w | (u64)(w64 < (double)min_p * most && at > 0) << 63;
    }
    __syncthreads();
    // cumulative weight in rank order, one rank a thread
    static_assert(kList <= kThreads, "a thread per element");
    const u64 marked = tid < m ? sm.by_rank.w[tid] : 0;
    const u64 w = marked & (~0ull >> 1);
    u64 incl = warp_scan(w, lane);
    if (lane == 31) sm.red[warp][0] = incl;
    __syncthreads();
    u64 all = 0;
    for (int j = 0; j < kWarps; ++j) {
      if (j < warp) incl += sm.red[j][0];
      all += sm.red[j][0];
    }
    if (target < 0.0) target = share * (double)all;
    // rank i stays while the weight before it is below the target
    const bool stays = tid < m && !(marked >> 63) &&
                       (tid == 0 || !(share < 1.0) || (double)(incl - w) < target);
    u64 mass[1] = {stays ? w : 0};
    if (tid < m) {
      sm.by_rank.i[tid] = stays ? 0xffffffffu - (uint32_t)sm.by_rank.ord[tid] : 0xffffffffu;
      sm.by_rank.kept[tid] = mass[0];
    }
    block_reduce<false, 1>(mass);
    u = u > 0.f ? u : 0.f;
    const double ut = (double)u * (double)mass[0];
    const u64 pick = ut < (double)mass[0] ? (u64)ut : mass[0] - 1;
    if (stays && w) {
      const u64 me = sm.by_rank.i[tid];
      u64 run = 0;
#pragma unroll 8
      for (int j = 0; j < m; ++j) run += sm.by_rank.i[j] <= me ? sm.by_rank.kept[j] : 0;
      if (run > pick && run - w <= pick) *token = (int)me;
    }
  }

  // [first, last] from the largest ord and the largest complement that were exchanged.
  __device__ void narrow(u64& first, u64& last) {
    u64 hi = 0, lo_c = 0;
    for (int r = 0; r < ranks; ++r) {
      hi = max(hi, sm.got[r][0]);
      lo_c = max(lo_c, sm.got[r][1]);
    }
    last = hi;
    first = ~lo_c;
    __syncthreads();
  }

  // Element k (from 1) of the sorted row, as an ord; 0 if fewer have a weight.
  __device__ u64 find_kth(int k) {
    clear_hist();
    each(floor_x, [&](float x, int) { atomicAdd(&sm.hist[step_of(x)], 1u); });
    sum_groups(false);
    exchange(0);
    find_step(k, false, false);
    if (sm.found_all <= (u64)k) {
      __syncthreads();
      cluster_sync();  // (the next step reuses the histograms that the other CTAs may be reading)
      return 0;
    }
    const int step = sm.found;
    u64 want = k - sm.found_before;  // rank within the interval
    u64 first = 0, last = ~0ull;     // ords of the interval
    bool by_step = true;
    // (each turn narrows the interval to one of 4096 parts: 64 bits take six)
    for (int guard = 0; guard < 16; ++guard) {
      u64 mm[2] = {0, 0};  // largest ord, largest ~ord
      each(by_step ? below(step) : below(kBins), [&](float x, int i) {
        const u64 o = ord(x, i);
        if (by_step ? step_of(x) == step : o >= first && o <= last) {
          put(sm.n_list, sm.list_ord, o);
          mm[0] = max(mm[0], o);
          mm[1] = max(mm[1], ~o);
        }
      });
      block_reduce<true, 2>(mm);
      exchange(mm[0], mm[1], 0, sm.n_list);
      const u64 count = total(3);
      if (count <= kList) {
        collect(false, false);
        for (int i = tid; i < (int)count; i += kThreads) {
          const u64 o = sm.all_ord[i];
          int at = 0;
#pragma unroll 8
          for (int j = 0; j < (int)count; ++j) at += sm.all_ord[j] > o;
          if (at == (int)want - 1) sm.cut = o;
        }
        __syncthreads();
        return sm.cut;
      }
      narrow(first, last);
      by_step = false;
      const int shift = max(0, 52 - __clzll(last - first));  // (last - first) >> shift < kBins
      clear_hist();
      each(below(kBins), [&](float x, int i) {
        const u64 o = ord(x, i);
        if (o >= first && o <= last) atomicAdd(&sm.hist[(last - o) >> shift], 1u);
      });
      sum_groups(false);
      exchange(0);
      find_step((double)want, false, false);
      want -= sm.found_before;
      last -= (u64)sm.found << shift;
      if (last - first >> shift) first = last - ((1ull << shift) - 1);
      __syncthreads();
    }
    return 0;
  }

  // The last element of the shortest prefix, among the ords from `cut` up, whose weight
  // reaches share times theirs.  n_all > 0: instead, so many elements that hold all of that
  // prefix are listed, and `target` is the weight to reach.
  __device__ u64 find_share(u64 cut, double share, int& n_all, double& target) {
    n_all = 0;
    if (!(share > 0.0)) return top_ord;
    clear_hist();
    const float least = cut ? fmaxf(floor_x, before_cut(cut)) : floor_x;
    u64 v[1] = {0};
    each4(least, [&](const float (&x)[4], int i) {
      bool on[4];
      u64 w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        double w64;
        on[e] = x[e] > floor_x && ord(x[e], i + e) >= cut;
        w[e] = weight(x[e], on[e], w64);
        v[0] += w[e];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (on[e]) {
          const int s = step_of(x[e]);
          atomicAdd(&sm.hist[s], (uint32_t)(w[e] >> shift_of(s)));
        }
    });
    block_reduce<false, 1>(v);
    sum_groups(true);
    exchange(v[0]);
    target = share * (double)total(0);
    find_step(share, true, true);
    int step = sm.found;
    u64 first = cut, last = ~0ull;  // the interval, cut into steps
    int shift = -1;                 // -1: by exponent
    u64 above = 0;                  // exact weight of the kept elements before the interval
    for (int guard = 0; guard < 4 * kBins; ++guard) {
      if (tid == 0) sm.n_list = sm.n_over = 0;
      __syncthreads();
      u64 s[2] = {0, 0};  // weight before the step, of the step
      each(shift < 0 ? fmaxf(floor_x, below(step)) : least, [&](float x, int i) {
        const u64 o = ord(x, i);
        if (o < first || o > last) return;
        const int b = shift < 0 ? step_of(x) : (int)((last - o) >> shift);
        if (b > step) return;
        double w64;
        const u64 w = weight(x, x > floor_x, w64);
        if (b < step) {
          s[0] += w;
          if (shift < 0 && *(volatile uint32_t*)&sm.n_over < kList) put(sm.n_over, sm.over_ord, o);
        } else {
          s[1] += w;
          put(sm.n_list, sm.list_ord, o);
        }
      });
      block_reduce<false, 2>(s);
      exchange(s[0], s[1], 0, sm.n_list | (u64)sm.n_over << 32);
      const u64 before = above + total(0), in = total(1);
      u64 n_in = 0, n_over = 0;
      for (int r = 0; r < ranks; ++r) {
        n_in += (uint32_t)sm.got[r][3];
        n_over += sm.got[r][3] >> 32;
      }
      const bool early = (double)before >= target, late = (double)(before + in) < target;
      if (early || late) {  // the short weights were too coarse: on to the next step that way
        const int next = neighbour(step, late);
        if (next < 0) {
          __syncthreads();
          cluster_sync();
          return late ? 0 : top_ord;
        }
        step = next;
        continue;
      }
      if (shift < 0 && n_in + n_over <= kList) {
        n_all = (int)(n_in + n_over);
        return 0;
      }
      if (n_in <= kList) {
        collect(true, false);
        for (int i = tid; i < (int)n_in; i += kThreads) {
          const u64 o = sm.all_ord[i];
          u64 incl = before;
#pragma unroll 8
          for (int j = 0; j < (int)n_in; ++j) incl += sm.all_ord[j] >= o ? sm.all_w[j] : 0;
          if ((double)incl >= target && (double)(incl - sm.all_w[i]) < target) sm.cut = o;
        }
        __syncthreads();
        return sm.cut;
      }
      // Too many for the list: cut the step by the ords it spans.
      u64 mm[2] = {0, 0};
      each(least, [&](float x, int i) {
        const u64 o = ord(x, i);
        if (x <= floor_x || o < first || o > last) return;
        if ((shift < 0 ? step_of(x) : (int)((last - o) >> shift)) != step) return;
        mm[0] = max(mm[0], o);
        mm[1] = max(mm[1], ~o);
      });
      block_reduce<true, 2>(mm);
      exchange(mm[0], mm[1]);
      narrow(first, last);
      above = before;
      shift = max(0, 52 - __clzll(last - first));
      clear_hist();
      double largest;
      weight(key_logit((uint32_t)(last >> 32)), true, largest);
      const float unit = (float)(16384.0 / largest);
      each(least, [&](float x, int i) {
        const u64 o = ord(x, i);
        if (o < first || o > last) return;
        double w;
        weight(x, x > floor_x, w);
        atomicAdd(&sm.hist[(last - o) >> shift], (uint32_t)((float)w * unit + 0.5f));
      });
      sum_groups(false);
      exchange(0);
      find_step(fmax((target - (double)above) * unit, 0.5), false, false);
      step = sm.found;
    }
    return cut;
  }

  // The largest logit below the cut's.
  __device__ __forceinline__ float before_cut(u64 cut) const {
    return prev_logit(key_logit((uint32_t)(cut >> 32)));
  }

  // The first index whose cumulative kept weight exceeds u times the total; the CTA that
  // holds it writes it.
  __device__ void pick(u64 cut, float u, int* token) {
    // min_p's logits lie above a bound; the comparison itself is in 64 bits.
    float least = floor_x;
    if (cut) least = fmaxf(least, before_cut(cut));
    if (min_p > 0.f)
      least = fmaxf(least, below((int)fminf(-log2f(min_p) * (1.f * kBins / range) + 2.f, kBins)));
    const float cut_x = cut ? key_logit((uint32_t)(cut >> 32)) : -CUDART_INF_F;
    const int cut_i = (int)(0xffffffffu - (uint32_t)cut) - lo;  // the last of its ties
    const double min_w = (double)min_p * most;
    const auto weights4 = [&](const float (&x)[4], int i, u64 (&w)[4]) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        double w64;
        const bool on = x[e] > least && (x[e] != cut_x || i + e <= cut_i);
        w[e] = weight(x[e], on, w64);
        if (w64 < min_w) w[e] = 0;
      }
    };
    u64 v[1] = {0};
    for (int b = 0; b < n; b += kBlock) {
      const int i = b + 4 * tid;
      float x[4];
      get4(i, x);
      const bool any = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) > least;
      u64 sum = 0;
      if (__any_sync(0xffffffffu, any)) {
        u64 w[4];
        weights4(x, i, w);
        sum = warp_sum(w[0] + w[1] + w[2] + w[3]);
      }
      if (lane == 0) {
        sm.sums[b / kBlock * kWarps + warp] = sum;
        v[0] += sum;
      }
    }
    block_reduce<false, 1>(v);
    exchange(v[0]);
    u64 before = 0, all = 0;
    for (int r = 0; r < ranks; ++r) {
      if (r < rank) before += sm.got[r][0];
      all += sm.got[r][0];
    }
    u = u > 0.f ? u : 0.f;
    const double ut = (double)u * (double)all;
    const u64 target = ut < (double)all ? (u64)ut : all - 1;
    if (warp != 0 || target < before || target >= before + sm.got[rank][0]) return;
    // The entry of sums, then the element of its 128.
    const int entries = (n + kBlock - 1) / kBlock * kWarps;
    int entry = 0;
    for (int e0 = 0; e0 < entries; e0 += 32) {
      const u64 w = e0 + lane < entries ? sm.sums[e0 + lane] : 0;
      const u64 incl = warp_scan(w, lane);
      const unsigned over = __ballot_sync(0xffffffffu, before + incl > target);
      if (over) {
        const int l = __ffs(over) - 1;
        entry = e0 + l;
        before += __shfl_sync(0xffffffffu, incl - w, l);
        break;
      }
      before += __shfl_sync(0xffffffffu, incl, 31);
    }
    const int i = entry / kWarps * kBlock + entry % kWarps * 128 + 4 * lane;
    float x[4];
    u64 w[4];
    get4(i, x);
    weights4(x, i, w);
    const u64 mine = w[0] + w[1] + w[2] + w[3];
    u64 run = before + warp_scan(mine, lane) - mine;
    if (run <= target && run + mine > target) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (run <= target && run + w[e] > target) *token = lo + i + e;
        run += w[e];
      }
    }
  }
};

// The slice into shared memory in 16-byte loads, several in flight per thread, and the
// thread's largest logit (the first of them).  Element `skip` of base is the slice's first;
// base is 16-byte aligned, and what stands before the slice is held as -inf.
template <typename T>
__device__ void load_slice(const T* base, int skip, int n, int n_held, float* held, float& best,
                           int& at) {
  constexpr int V = 16 / (int)sizeof(T), kAhead = 4;
  best = -CUDART_INF_F;
  at = 0;
  const int tid = threadIdx.x;
  const int g0 = skip ? 1 : 0, g1 = max(g0, min(n, n_held) / V);  // whole vectors
  for (int g = g0 + tid; g < g1; g += kAhead * kThreads) {
    uint4 r[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (g + u * kThreads < g1)
        r[u] = __ldg(reinterpret_cast<const uint4*>(base) + g + u * kThreads);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = (g + u * kThreads) * V;
      if (g + u * kThreads < g1) {
        const T* e = reinterpret_cast<const T*>(&r[u]);
        float v[V];
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = clean(Elem<T>::get(e[j]));
        float most = v[0];
#pragma unroll
        for (int j = 1; j < V; ++j) most = fmaxf(most, v[j]);
        if (most > best) {
          best = most;
          at = i;  // (of the vector; the element is looked up below)
        }
#pragma unroll
        for (int j = 0; j < V; j += 4)
          *reinterpret_cast<float4*>(held + i + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
      }
    }
  }
  if (best > -CUDART_INF_F) {
    const int i = at;
#pragma unroll
    for (int j = V - 1; j >= 0; --j)
      if (held[i + j] == best) at = i + j;
  }
  const auto one = [&](int i) {
    const float v = i >= skip && i < n ? clean(Elem<T>::get(base[i])) : -CUDART_INF_F;
    if (i < n_held) held[i] = v;
    if (v > best || (v == best && i < at)) {
      best = v;
      at = i;
    }
  };
  for (int i = tid; i < g0 * V; i += kThreads) one(i);
  for (int i = g1 * V + tid; i < max(n, n_held); i += kThreads) one(i);
}

// The row of cluster q when there are more clusters than run at once: within each 512 rows those
// of the costliest settings come first, so that no long row starts when the others are done.
__device__ int ordered_row(const SampleParams& p, Shared& sm, int q) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int base = q / kThreads * kThreads, row = base + tid;
  int cls = -1;
  if (row < p.n_rows) {
    const float temp = p.temperature ? p.temperature[row] : 1.f;
    const int k = p.top_k ? p.top_k[row] : 0;
    const float top_p = p.top_p ? p.top_p[row] : 1.f;
    const bool by_count = k > 0 && k < p.vocab;
    cls = !(temp > 0.f) ? 0
          : by_count && k <= kSmallK ? 1
                                     : 2 + (top_p < 1.f ? 1 : 0) + (by_count ? 2 : 0);
  }
  static_assert(kThreads < 1024, "ten bits hold a class's rows");
  u64 packed = 0;
  int mine = 0;  // rows that come before the thread's
#pragma unroll
  for (int c = 0; c < 6; ++c) {
    const unsigned in = __ballot_sync(0xffffffffu, cls == c);
    packed |= (u64)__popc(in) << (10 * c);
    if (cls == c) mine = __popc(in & ((1u << lane) - 1));
  }
  if (lane == 0) sm.counts[warp] = packed;
  __syncthreads();
  u64 all = 0, before = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const u64 x = sm.counts[w];
    all += x;
    before += w < warp ? x : 0;
  }
  if (cls >= 0) mine += (int)(before >> (10 * cls)) & 1023;
#pragma unroll
  for (int c = 1; c < 6; ++c) mine += c > cls ? (int)(all >> (10 * c)) & 1023 : 0;
  if (cls >= 0 && mine == q - base) sm.row = row;
  __syncthreads();
  return sm.row;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2)
    sample_kernel(const SampleParams p, const int ranks, const int per, const int room,
                  const bool order) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  Shared& sm = *reinterpret_cast<Shared*>(smem_raw);
  float* held = reinterpret_cast<float*>(smem_raw + sizeof(Shared));
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = blockIdx.x % ranks;
  if (tid < 64) sm.pow2[tid] = exp2(tid / 64.0 + p.wshift);
  pdl_wait();
  const int row = order ? ordered_row(p, sm, blockIdx.x / ranks) : blockIdx.x / ranks;
  const int lo = min(rank * per, p.vocab);
  const T* x = static_cast<const T*>(p.logits) + (long long)row * p.logits_stride + lo;
  const int skip = (int)(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));
  const int n = lo < p.vocab ? min(per, p.vocab - lo) + skip : 0;
  static_assert(sizeof(Shared) % 16 == 0, "the slice is read 16 bytes at a time");
  const int n_held = min((n + 7) & ~7, room);

  float best;
  int at;
  load_slice(x - skip, skip, n, n_held, held, best, at);
  const float temp = p.temperature ? p.temperature[row] : 1.f;
  const int k = p.top_k ? p.top_k[row] : 0;
  const float top_p = p.top_p ? p.top_p[row] : 1.f;
  const float u = p.uniform[row];
  Row<T> r{p, sm, x - skip, held, lo - skip, n, n_held, rank, ranks, tid, lane, warp};
  u64 v[1] = {best == -CUDART_INF_F ? 0 : r.ord(best, at)};
  r.template block_reduce<true, 1>(v);
  r.exchange(v[0]);
  u64 top_ord = 0;
  for (int i = 0; i < ranks; ++i) top_ord = max(top_ord, sm.got[i][0]);
  int* token = p.tokens + row;
  if (top_ord == 0 || !(temp > 0.f)) {  // nothing above -inf, or greedy
    if (rank == 0 && tid == 0) *token = top_ord == 0 ? 0 : (int)(0xffffffffu - (uint32_t)top_ord);
  } else {
    if (top_ord >> 32 == logit_key(CUDART_INF_F)) {
      // an infinite logit: only its equals count, all alike
      r.infinite = true;
      for (int i = tid; i < n_held; i += kThreads) held[i] = r.finite(held[i]);
      best = r.finite(best);
      top_ord = (top_ord & 0xffffffffull) | (u64)logit_key(0.f) << 32;
      __syncthreads();
    }
    r.settle(top_ord, temp);
    r.min_p = p.min_p ? p.min_p[row] : 0.f;
    if (!(r.min_p <= 1.f)) r.min_p = 2.f;  // (a NaN too) only the first token
    const bool by_count = k > 0 && k < p.vocab;
    const bool small = by_count && k <= kSmallK;
    int listed = 0;        // elements listed that hold all that is kept
    u64 cut = 0;           // otherwise: the last kept element
    double target = -1.0;  // the weight that top-p keeps, where it is known
    if (!small || !r.gather_first(k, best, listed)) {
      listed = 0;
      if (by_count) cut = r.find_kth(k);
      if (top_p < 1.f) {
        const u64 c = r.find_share(cut, (double)top_p, listed, target);
        cut = max(cut, c);
      }
      if (r.min_p > 1.f && listed == 0) {
        cut = top_ord;
        r.min_p = 0.f;
      }
    }
    if (listed == 0) {
      r.pick(cut, u, token);
    } else if (rank == 0) {
      r.collect(false, target >= 0.0);
      r.finish(listed, target >= 0.0 ? kList : k, target, (double)top_p, u, token);
    }
  }
  __syncthreads();
  cluster_sync();  // no CTA leaves while another may read its shared memory
}

template <typename T>
cudaError_t launch_one(const SampleParams& p, int ranks, int per, int room, size_t smem,
                       bool order, cudaStream_t st, bool pdl) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.n_rows * ranks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ranks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, sample_kernel<T>, p, ranks, per, room, order);
}

constexpr int kMaxSmem = 227 * 1024;

}  // namespace

cudaError_t prepare_sample() {
  cudaError_t e = cudaFuncSetAttribute((const void*)sample_kernel<float>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute((const void*)sample_kernel<__nv_bfloat16>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute((const void*)sample_kernel<__half>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
  return e;
}

cudaError_t launch_sample(const SampleParams& p, int dtype, int n_sm, cudaStream_t st, bool pdl) {
  // CTAs per row: as many as let two CTAs share an SM with the whole row in shared memory, and
  // more while the rows alone do not fill the SMs and a slice keeps the threads busy.
  const int two = (kMaxSmem / 2 - 1024 - (int)sizeof(Shared)) / 4;  // logits that fit beside another CTA
  int ranks = 1;
  while (ranks < kMaxCluster &&
         (p.vocab > two * ranks ||
          ((long long)p.n_rows * ranks < 2 * n_sm && p.vocab > 2 * kBlock * ranks)))
    ranks *= 2;
  const int per = ((p.vocab + ranks - 1) / ranks + 7) & ~7;
  // (a slice that starts off a 16-byte boundary is held from that boundary on)
  const int room = std::min(per + 8, (kMaxSmem - (int)sizeof(Shared)) / 4 & ~7);
  size_t smem = sizeof(Shared) + (size_t)room * 4;
  // Few clusters would share SMs while others are idle: each CTA asks for more than half of one.
  // (Not as soon as the CTAs outnumber half the SMs: a cluster lies within one of the device's
  // parts, which then holds fewer of them.  16 rows took 25 us in place of 19.)
  constexpr int kHalf = kMaxSmem / 2 - 1024;
  const long long ctas = (long long)p.n_rows * ranks;
  if (ctas <= n_sm / 2) smem = std::max<size_t>(smem, kMaxSmem / 2 + 1024);
  const bool order = ctas > (long long)n_sm * (smem <= kHalf ? 2 : 1);
  if (dtype == kDtypeF32) return launch_one<float>(p, ranks, per, room, smem, order, st, pdl);
  if (dtype == kDtypeBf16) return launch_one<__nv_bfloat16>(p, ranks, per, room, smem, order, st, pdl);
  return launch_one<__half>(p, ranks, per, room, smem, order, st, pdl);
}

}  // namespace gqa
