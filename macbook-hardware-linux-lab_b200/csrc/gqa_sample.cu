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
// memory once.  The last kept element is found in two steps: a histogram over 2048
// equal steps of the exponent (they hold few elements each, wherever the logits lie,
// and equal logits fall together), merged over the cluster by reads of the other CTAs'
// shared memory, gives the step; its few elements are listed and ranked by comparing all
// pairs.  Should a step hold more than the list takes (a high temperature, many ties),
// the step is cut again by the pair's 64 bits.  For top-p the histogram holds weights
// rounded to 14 bits; they only propose the step, which the exact sums confirm or move.
#include <algorithm>

#include <math_constants.h>

#include "gqa_paged.cuh"
#include "gqa_sample.cuh"

namespace gqa {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;       // four per thread
constexpr int kList = 512;
// A top_k up to which the row's first k are looked for by way of the threads' largest logits.
constexpr int kSmallK = 256;
constexpr int kMaxCluster = 8;
constexpr int kBlock = kThreads * 4;  // elements of one turn of the CTA's threads

using u64 = unsigned long long;

struct alignas(16) Shared {  // (the slice of the row follows it)
  union {
    uint32_t hist[kBins];
    u64 sums[kBins / 2 + kWarps];  // for the pick: weights of 128 elements each
  };
  u64 list_ord[kList], list_w[kList];  // this CTA's elements of the step
  u64 over_ord[kList], over_w[kList];  // and those before it, while they fit
  u64 all_ord[kList], all_w[kList];    // the cluster's
  u64 x[2][4];                         // values exchanged over the cluster
  u64 got[kMaxCluster][4];
  u64 red[kWarps][4];
  double pow2[64];                     // 2^(j / 64)
  u64 found_before, cut;
  int found;
  uint32_t n_list, n_over;
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
__device__ __forceinline__ float clean(float x) { return x != x ? -CUDART_INF_F : x + 0.0f; }

__device__ __forceinline__ uint4 ld_cluster_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ u64 ld_cluster_u64(uint32_t addr) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ u64 warp_sum(u64 x) {
#pragma unroll
  for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
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
  bool infinite;      // it is infinite: only its equals have a weight, and the same one
  u64 top_ord;
  float c2;           // twice log2(e) / temperature, for the steps
  double ct;          // log2(e) / temperature
  float range;        // steps cover weights down to 2^-range
  float per_step;     // kBins / range
  double scale;       // 2^wshift
  float min_p;

  __device__ __forceinline__ u64 ord(float x, int i) const {
    return (u64)logit_key(x) << 32 | (0xffffffffu - (uint32_t)(lo + i));
  }

  // f(x, i) for the elements of the slice, four at a time per thread.
  template <typename F>
  __device__ __forceinline__ void each(F&& f) const {
#pragma unroll 2
    for (int b = 0; b < n; b += kBlock) {
      const int i = b + 4 * tid;
      float v[4];
      get4(i, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) f(v[e], i + e);
    }
  }
  // f(x, i, step, d, on) with the weights of the elements that f wants (`want` says which, by
  // ord and step), computed for four elements side by side where a warp has any.
  template <typename W, typename F>
  __device__ __forceinline__ void each_weight(W&& want, F&& f) const {
    for (int b = 0; b < n; b += kBlock) {
      const int i = b + 4 * tid;
      float v[4], d[4];
      int s[4];
      bool on[4], any = false;
      get4(i, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[e] = step_of(v[e], d[e]);
        on[e] = s[e] < kBins && want(ord(v[e], i + e), s[e]);
        any |= on[e];
      }
      if (!__any_sync(0xffffffffu, any)) continue;
      u64 w[4];
      double w64[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = weight(v[e], on[e], w64[e]);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (on[e]) f(i + e, ord(v[e], i + e), s[e], d[e], w[e], w64[e]);
    }
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
        v[e] = i + e < n ? clean(Elem<T>::get(logits[i + e])) : -CUDART_INF_F;
    }
  }

  // log2 of top's weight over x's, and the step it falls in (kBins: beyond every weight).
  // Non-decreasing in falling x, so steps cut the sorted order; halves keep the difference
  // of two far logits finite.
  __device__ __forceinline__ int step_of(float x, float& d) const {
    d = x == top ? 0.f : (0.5f * top - 0.5f * x) * c2;
    return d < range ? min((int)(d * per_step), kBins - 1) : kBins;
  }

  // The weight in 64 bits: 2^t as 2^(k/64) times the series of the rest (|rest| <= 2^-7 ln 2;
  // Tang's table method), and in units of 2^-wshift.  `on`: the logit is within the steps
  // (others weigh nothing).  No branches, so that the four elements a thread has at a time
  // go through the 64-bit pipe side by side.
  __device__ __forceinline__ u64 weight(float x, bool on, double& w) const {
    double t = ((double)(on ? x : top) - (double)top) * ct;
    if (infinite) t = 0.0;
    const double magic = 6755399441055744.0;  // 1.5 * 2^52: rounds to an integer
    const double km = fma(t, 64.0, magic);
    const int k = __double2loint(km);
    const double y = fma(km - magic, -1.0 / 64.0, t) * 0.693147180559945309;
    double q = fma(y, 1.0 / 120.0, 1.0 / 24.0);
    q = fma(q, y, 1.0 / 6.0);
    q = fma(q, y, 0.5);
    q = fma(q, y, 1.0);
    q *= y;
    const double b = sm.pow2[k & 63];
    const double m = fma(b, q, b);
    w = __hiloint2double(__double2hiint(m) + ((k >> 6) << 20), __double2loint(m));
    // (a product of at most 2^50 plus 2^52 holds the rounded integer in its low bits)
    const u64 bits = __double_as_longlong(fma(w, scale, 4503599627370496.0)) & 0xfffffffffffffull;
    if (!on) w = 0.0;
    return on ? bits : 0ull;
  }

  // Sums (or, for `largest`, maxima) of four values over the block.
  template <bool kMax>
  __device__ void block_reduce(u64 (&v)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int d = 16; d; d >>= 1) {
        const u64 y = __shfl_xor_sync(0xffffffffu, v[j], d);
        v[j] = kMax ? (y > v[j] ? y : v[j]) : v[j] + y;
      }
    __syncthreads();
    if (lane < 4) sm.red[warp][lane] = lane == 0 ? v[0] : lane == 1 ? v[1] : lane == 2 ? v[2] : v[3];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      u64 x = 0;
      for (int w = 0; w < kWarps; ++w) {
        const u64 y = sm.red[w][j];
        x = kMax ? (y > x ? y : x) : x + y;
      }
      v[j] = x;
    }
  }

  // Every CTA's four values into sm.got[rank] (a cluster barrier; what a CTA wrote to its
  // shared memory before it, the others may read after it).  The two places alternate: a CTA
  // is past the next barrier only when all have read this one's.
  __device__ void exchange(const u64 (&v)[4]) {
    u64* mine = sm.x[turn & 1];
    if (tid < 4) mine[tid] = tid == 0 ? v[0] : tid == 1 ? v[1] : tid == 2 ? v[2] : v[3];
    __syncwarp();
    cluster_sync();
    if (tid < ranks * 4) sm.got[tid >> 2][tid & 3] = ld_cluster_u64(cluster_map(mine + (tid & 3), tid >> 2));
    __syncthreads();
    ++turn;
  }
  __device__ __forceinline__ u64 total(int j) const {
    u64 x = 0;
    for (int r = 0; r < ranks; ++r) x += sm.got[r][j];
    return x;
  }

  __device__ void clear_hist() {
    *reinterpret_cast<uint4*>(&sm.hist[4 * tid]) = make_uint4(0, 0, 0, 0);
    if (tid == 0) sm.n_list = sm.n_over = 0;
    __syncthreads();
  }

  // This thread's four steps of the cluster's histogram (after a barrier).
  __device__ void merged(u64 (&h)[4]) {
    uint4 v[kMaxCluster];
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r)
      v[r] = r < ranks ? ld_cluster_v4(cluster_map(&sm.hist[4 * tid], r)) : make_uint4(0, 0, 0, 0);
    h[0] = h[1] = h[2] = h[3] = 0;
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) {
      h[0] += v[r].x;
      h[1] += v[r].y;
      h[2] += v[r].z;
      h[3] += v[r].w;
    }
  }

  // The step at which the running sum of h reaches `want` (below zero: that share of the
  // total), the sum before it and the total.
  __device__ int find_step(const double (&h)[4], double want, double& before, double& all) {
    __syncthreads();
    double mine = h[0] + h[1] + h[2] + h[3], incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += y;
    }
    double* red = reinterpret_cast<double*>(sm.red);
    if (lane == 31) red[warp] = incl;
    if (tid == 0) sm.found = -1;
    __syncthreads();
    double base = 0.0;
    all = 0.0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) base += red[w];
      all += red[w];
    }
    if (want < 0.0) want = -want * all;
    double run = base + incl - mine;
    // The last non-empty step before which the sum is below `want`: unlike a test of both
    // ends, this always names one, however the sums are rounded.
    int at = -1;
    double at_before = 0.0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (h[j] > 0.0 && run < want) {
        at = 4 * tid + j;
        at_before = run;
      }
      run += h[j];
    }
    if (at >= 0) atomicMax(&sm.found, at);
    __syncthreads();
    if (at >= 0 && sm.found == at) *reinterpret_cast<double*>(&sm.found_before) = at_before;
    __syncthreads();
    before = *reinterpret_cast<double*>(&sm.found_before);
    return sm.found;
  }

  // Appends this thread's element to a list of the CTA.
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
        sm.all_ord[at + i] = ld_cluster_u64(cluster_map(from, r));
        if (weights) {
          from = i < c ? &sm.list_w[i] : &sm.over_w[i - c];
          sm.all_w[at + i] = ld_cluster_u64(cluster_map(from, r));
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
  __device__ bool gather_first(int k, float best, int& n) {
    clear_hist();
    float d;
    const int mine = step_of(best, d);
    if (mine < kBins) atomicAdd(&sm.hist[mine], 1u);
    u64 v[4] = {0, 0, 0, 0};
    __syncthreads();
    exchange(v);
    u64 h[4];
    merged(h);
    const double hd[4] = {(double)h[0], (double)h[1], (double)h[2], (double)h[3]};
    double before, all;
    const int step = find_step(hd, k, before, all);
    const int upto = all < k ? kBins - 1 : step;  // (fewer: all that have a weight)
    each([&](float x, int i) {
      if (step_of(x, d) <= upto) put(sm.n_list, sm.list_ord, ord(x, i));
    });
    __syncthreads();
    v[3] = min(sm.n_list, 1u << 30);
    exchange(v);
    const u64 count = total(3);
    n = (int)count;
    if (count > kList) {
      __syncthreads();
      cluster_sync();  // (the lists are reused)
      return false;
    }
    return true;
  }

  // The token from n collected elements that hold all of the row's first k (and, with
  // weights, all that top-p keeps, whose weight the target is).  By one CTA: ranks by
  // comparing all pairs, prefixes by a scan, and the index order again by pairs.
  __device__ void finish(int n, int k, bool weighed, double target, double share, float u,
                         int* token) {
    const int m = min(n, k);
    for (int i = tid; i < n; i += kThreads) {  // (n <= kList: one element a thread)
      const u64 o = sm.all_ord[i];
      int at = 0;
      for (int j = 0; j < n; ++j) at += sm.all_ord[j] > o;
      u64 w;
      double w64;
      const float x = key_logit((uint32_t)(o >> 32));
      float d;
      w = weight(x, step_of(x, d) < kBins, w64);
      sm.over_ord[at] = o;
      // the weight with min_p's answer in the sign bit (weights stay below 2^50)
      sm.over_w[at] = w | (u64)(!(w64 >= (double)min_p) && at > 0) << 63;
    }
    __syncthreads();
    constexpr u64 kMask = ~0ull >> 1;
    // cumulative weight in rank order, one rank a thread
    static_assert(kList <= kThreads, "a thread per element");
    const u64 w = tid < m ? sm.over_w[tid] & kMask : 0;
    u64 incl = w;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const u64 y = __shfl_up_sync(0xffffffffu, incl, s);
      if (lane >= s) incl += y;
    }
    __syncthreads();
    if (lane == 31) sm.red[warp][0] = incl;
    __syncthreads();
    u64 all = 0;
    for (int j = 0; j < kWarps; ++j) {
      if (j < warp) incl += sm.red[j][0];
      all += sm.red[j][0];
    }
    if (!weighed) target = share * (double)all;
    // rank i stays while the weight before it is below the target
    const bool stays = tid < m && !(sm.over_w[tid] >> 63) &&
                       (tid == 0 || !(share < 1.0) || (double)(incl - w) < target);
    u64 mass[4] = {stays ? w : 0, 0, 0, 0};
    // kept elements, for the index order
    if (tid < n) {
      sm.list_ord[tid] = stays ? 0xffffffffu - (uint32_t)sm.over_ord[tid] : 0xffffffffu;
      sm.list_w[tid] = mass[0];
    }
    block_reduce<false>(mass);
    u = u > 0.f ? u : 0.f;
    const double ut = (double)u * (double)mass[0];
    const u64 pick = ut < (double)mass[0] ? (u64)ut : mass[0] - 1;
    if (stays && w) {
      const u64 me = sm.list_ord[tid];
      u64 run = 0;
      for (int j = 0; j < m; ++j) run += sm.list_ord[j] <= me ? sm.list_w[j] : 0;
      if (run > pick && run - w <= pick) *token = (int)me;
    }
  }

  // Element k (from 1) of the sorted row, as an ord; 0 if fewer have a weight.
  __device__ u64 find_kth(int k) {
    clear_hist();
    each([&](float x, int) {
      float d;
      const int s = step_of(x, d);
      if (s < kBins) atomicAdd(&sm.hist[s], 1u);
    });
    u64 v[4] = {0, 0, 0, 0};
    __syncthreads();
    exchange(v);
    u64 h[4];
    merged(h);
    double hd[4] = {(double)h[0], (double)h[1], (double)h[2], (double)h[3]};
    double before, all;
    int step = find_step(hd, k, before, all);
    if (all <= k) {
      __syncthreads();
      cluster_sync();  // (the next step reuses the histograms that the other CTAs may be reading)
      return 0;
    }
    double want = k - before;     // rank within the interval
    u64 first = 0, last = ~0ull;  // ords of the interval
    bool by_step = true;
    // (each turn narrows the interval to one of 2048 parts: 64 bits take six)
    for (int guard = 0; guard < 16; ++guard) {
      u64 mm[4] = {0, 0, 0, 0};  // largest ord, largest ~ord
      each([&](float x, int i) {
        const u64 o = ord(x, i);
        float d;
        if (by_step ? step_of(x, d) == step : o >= first && o <= last) {
          put(sm.n_list, sm.list_ord, o);
          if (o > mm[0]) mm[0] = o;
          if (~o > mm[1]) mm[1] = ~o;
        }
      });
      block_reduce<true>(mm);
      mm[3] = sm.n_list;
      exchange(mm);
      const u64 n = total(3);
      if (n <= kList) {
        collect(false, false);
        for (int i = tid; i < (int)n; i += kThreads) {
          const u64 o = sm.all_ord[i];
          int at = 0;
          for (int j = 0; j < (int)n; ++j) at += sm.all_ord[j] > o;
          if (at == (int)want - 1) sm.cut = o;
        }
        __syncthreads();
        return sm.cut;
      }
      narrow(first, last);
      by_step = false;
      const int shift = max(0, 53 - __clzll(last - first));  // (last - first) >> shift < kBins
      clear_hist();
      each([&](float x, int i) {
        const u64 o = ord(x, i);
        if (o >= first && o <= last) atomicAdd(&sm.hist[(last - o) >> shift], 1u);
      });
      __syncthreads();
      exchange(v);
      merged(h);
#pragma unroll
      for (int j = 0; j < 4; ++j) hd[j] = (double)h[j];
      const int b = find_step(hd, want, before, all);
      want -= before;
      last -= (u64)b << shift;
      if (last - first >> shift) first = last - ((1ull << shift) - 1);
    }
    return 0;
  }

  // [first, last] from the largest ord and the largest complement that were exchanged.
  __device__ void narrow(u64& first, u64& last) {
    u64 hi = 0, lo_c = 0;
    for (int r = 0; r < ranks; ++r) {
      if (sm.got[r][0] > hi) hi = sm.got[r][0];
      if (sm.got[r][1] > lo_c) lo_c = sm.got[r][1];
    }
    last = hi;
    first = ~lo_c;
    __syncthreads();
  }

  // The last element of the shortest prefix, among the ords from `cut` up, whose weight
  // reaches share times theirs.  n > 0: instead, n elements that hold all of that prefix are
  // collected, and `target` is the weight to reach.
  __device__ u64 find_share(u64 cut, double share, int& n, double& target) {
    n = 0;
    if (!(share > 0.0)) return top_ord;
    clear_hist();
    const float width = range / kBins;
    u64 v[4] = {0, 0, 0, 0};
    each_weight([&](u64 o, int) { return o >= cut; },
                [&](int, u64, int b, float d, u64 w, double) {
                  v[0] += w;
                  atomicAdd(&sm.hist[b], (uint32_t)(exp2f(b * width - d) * 16384.f + 0.5f));
                });
    block_reduce<false>(v);
    exchange(v);
    target = share * (double)total(0);
    u64 h[4];
    merged(h);
    double hd[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) hd[j] = (double)h[j] * exp2f(-(4 * tid + j) * width);
    double unused, all;
    int step = find_step(hd, -share, unused, all);
    u64 first = cut, last = ~0ull;  // the interval, cut into steps
    int shift = -1;                 // -1: by exponent
    u64 above = 0;                  // exact weight of the kept elements before the interval
    for (int guard = 0; guard < 4 * kBins; ++guard) {
      if (tid == 0) sm.n_list = sm.n_over = 0;
      __syncthreads();
      u64 s[4] = {0, 0, 0, 0};  // weight before the step, of the step
      const auto part = [&](u64 o, int b) { return shift < 0 ? b : (int)((last - o) >> shift); };
      each_weight([&](u64 o, int b) { return o >= first && o <= last && part(o, b) <= step; },
                  [&](int, u64 o, int b, float, u64 w, double) {
                    if (part(o, b) < step) {
                      s[0] += w;
                      if (shift < 0 && *(volatile uint32_t*)&sm.n_over < kList) {
                        const uint32_t at = atomicAdd(&sm.n_over, 1u);
                        if (at < kList) {
                          sm.over_ord[at] = o;
                          sm.over_w[at] = w;
                        }
                      }
                    } else {
                      s[1] += w;
                      const uint32_t at = atomicAdd(&sm.n_list, 1u);
                      if (at < kList) {
                        sm.list_ord[at] = o;
                        sm.list_w[at] = w;
                      }
                    }
                  });
      block_reduce<false>(s);
      s[3] = sm.n_list | (u64)sm.n_over << 32;
      exchange(s);
      const u64 before = above + total(0), in = total(1);
      u64 n_in = 0, n_over = 0;
      for (int r = 0; r < ranks; ++r) {
        n_in += (uint32_t)sm.got[r][3];
        n_over += sm.got[r][3] >> 32;
      }
      const bool early = (double)before >= target, late = (double)(before + in) < target;
      if (early || late) {
        // the 14-bit weights were too coarse: the next non-empty step that way
        int other = -1;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int b = 4 * tid + j;
          if (h[j] == 0) continue;
          if (early && b < step) other = b;                      // the last before
          if (late && b > step && other < 0) other = kBins - b;  // the first after
        }
        if (tid == 0) sm.found = -1;
        __syncthreads();
        atomicMax(&sm.found, other);
        __syncthreads();
        const int next = sm.found;
        __syncthreads();
        if (next < 0) return late ? 0 : top_ord;
        step = late ? kBins - next : next;
        continue;
      }
      if (shift < 0 && n_in + n_over <= kList) {
        n = (int)(n_in + n_over);
        return 0;
      }
      if (n_in <= kList) {
        collect(true, false);
        for (int i = tid; i < (int)n_in; i += kThreads) {
          const u64 o = sm.all_ord[i];
          u64 incl = before;
          for (int j = 0; j < (int)n_in; ++j) incl += sm.all_ord[j] >= o ? sm.all_w[j] : 0;
          if ((double)incl >= target && (double)(incl - sm.all_w[i]) < target) sm.cut = o;
        }
        __syncthreads();
        return sm.cut;
      }
      // Too many for the list: cut the step by the ords it spans.
      u64 mm[4] = {0, 0, 0, 0};
      each([&](float x, int i) {
        const u64 o = ord(x, i);
        float d;
        const int b = step_of(x, d);
        if (b == kBins || o < first || o > last || part(o, b) != step) return;
        if (o > mm[0]) mm[0] = o;
        if (~o > mm[1]) mm[1] = ~o;
      });
      block_reduce<true>(mm);
      exchange(mm);
      narrow(first, last);
      above = before;
      shift = max(0, 53 - __clzll(last - first));
      clear_hist();
      double most;
      weight(key_logit((uint32_t)(last >> 32)), true, most);
      const float unit = (float)(16384.0 / most);
      each_weight([&](u64 o, int) { return o >= first && o <= last; },
                  [&](int, u64 o, int, float, u64, double w) {
                    atomicAdd(&sm.hist[(last - o) >> shift], (uint32_t)((float)w * unit + 0.5f));
                  });
      v[0] = 0;
      __syncthreads();
      exchange(v);
      merged(h);
#pragma unroll
      for (int j = 0; j < 4; ++j) hd[j] = (double)h[j];
      step = find_step(hd, fmax((target - (double)above) / scale * unit, 0.5), unused, all);
    }
    return cut;
  }

  // The first index whose cumulative kept weight exceeds u times the total; the CTA that
  // holds it writes it.
  __device__ void pick(u64 cut, float u, int* token) {
    // min_p's logits lie before the step of 2^-reach; the comparison itself is in 64 bits.
    const float reach = min_p > 0.f ? -log2f(min_p) * 1.0001f + 0.01f : range;
    const auto weights4 = [&](int i, const float (&x)[4], u64 (&w)[4]) {
      bool on[4], any = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float d;
        const u64 o = ord(x[e], i + e);
        on[e] = step_of(x[e], d) < kBins && o >= cut && (d <= reach || o == top_ord);
        any |= on[e];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = 0;
      if (!__any_sync(0xffffffffu, any)) return;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        double w64;
        w[e] = weight(x[e], on[e], w64);
        if (!(w64 >= (double)min_p) && ord(x[e], i + e) != top_ord) w[e] = 0;
      }
    };
    u64 v[4] = {0, 0, 0, 0};
    for (int b = 0; b < n; b += kBlock) {
      float x[4];
      u64 w[4];
      get4(b + 4 * tid, x);
      weights4(b + 4 * tid, x, w);
      const u64 sum = warp_sum(w[0] + w[1] + w[2] + w[3]);
      if (lane == 0) {
        sm.sums[b / kBlock * kWarps + warp] = sum;
        v[0] += sum;
      }
    }
    block_reduce<false>(v);
    exchange(v);
    u64 before = 0, all = 0;
    for (int r = 0; r < ranks; ++r) {
      if (r < rank) before += sm.got[r][0];
      all += sm.got[r][0];
    }
    u = u > 0.f ? u : 0.f;
    const double ut = (double)u * (double)all;
    const u64 target = ut < (double)all ? (u64)ut : all - 1;
    if (warp != 0 || target < before || target >= before + sm.got[rank][0]) return;
    // Lane by lane: the entry of sums, then the element of its 128.
    const int entries = (n + kBlock - 1) / kBlock * kWarps;
    int entry = 0;
    for (int e0 = 0; e0 < entries; e0 += 32) {
      const u64 w = e0 + lane < entries ? sm.sums[e0 + lane] : 0;
      u64 incl = w;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const u64 y = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += y;
      }
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
    get4(i, x);
    u64 w[4];
    weights4(i, x, w);
    const u64 mine = w[0] + w[1] + w[2] + w[3];
    u64 incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const u64 y = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += y;
    }
    u64 run = before + incl - mine;
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
  const auto see = [&](float v, int i) {
    if (v > best || (v == best && i < at)) {
      best = v;
      at = i;
    }
  };
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
        for (int j = 0; j < V; ++j) {
          v[j] = clean(Elem<T>::get(e[j]));
          see(v[j], i + j);
        }
#pragma unroll
        for (int j = 0; j < V; j += 4)
          *reinterpret_cast<float4*>(held + i + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
      }
    }
  }
  const auto one = [&](int i) {
    const float v = i >= skip && i < n ? clean(Elem<T>::get(base[i])) : -CUDART_INF_F;
    if (i < n_held) held[i] = v;
    see(v, i);
  };
  for (int i = tid; i < g0 * V; i += kThreads) one(i);
  for (int i = g1 * V + tid; i < max(n, n_held); i += kThreads) one(i);
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2)
    sample_kernel(const SampleParams p, const int ranks, const int per, const int room) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  Shared& sm = *reinterpret_cast<Shared*>(smem_raw);
  float* held = reinterpret_cast<float*>(smem_raw + sizeof(Shared));
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = blockIdx.x % ranks, row = blockIdx.x / ranks;
  const int lo = min(rank * per, p.vocab);
  const T* x = static_cast<const T*>(p.logits) + (long long)row * p.logits_stride + lo;
  const int skip = (int)(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));
  const int n = lo < p.vocab ? min(per, p.vocab - lo) + skip : 0;
  static_assert(sizeof(Shared) % 16 == 0, "the slice is read 16 bytes at a time");
  const int n_held = min((n + 7) & ~7, room);
  if (tid < 64) sm.pow2[tid] = exp2(tid / 64.0);
  pdl_wait();

  float best;
  int at;
  load_slice(x - skip, skip, n, n_held, held, best, at);
  const float temp = p.temperature ? p.temperature[row] : 1.f;
  const int k = p.top_k ? p.top_k[row] : 0;
  const float top_p = p.top_p ? p.top_p[row] : 1.f;
  const float u = p.uniform[row];
  Row<T> r{p, sm, x - skip, held, lo - skip, n, n_held, rank, ranks, tid, lane, warp};
  u64 v[4] = {r.ord(best, at), 0, 0, 0};
  if (best == -CUDART_INF_F) v[0] = 0;
  r.template block_reduce<true>(v);
  r.exchange(v);
  u64 top_ord = 0;
  for (int i = 0; i < ranks; ++i) top_ord = max(top_ord, sm.got[i][0]);
  int* token = p.tokens + row;
  if (top_ord == 0 || !(temp > 0.f)) {  // nothing above -inf, or greedy
    if (rank == 0 && tid == 0) *token = top_ord == 0 ? 0 : (int)(0xffffffffu - (uint32_t)top_ord);
  } else {
    r.top = key_logit((uint32_t)(top_ord >> 32));
    r.infinite = r.top == CUDART_INF_F;
    r.top_ord = top_ord;
    r.ct = 1.4426950408889634074 / (double)temp;
    r.c2 = (float)(2.0 * r.ct);
    r.range = (float)(p.wshift + 2);
    r.per_step = kBins / r.range;
    r.scale = (double)(1ull << p.wshift);
    r.min_p = p.min_p ? p.min_p[row] : 0.f;
    const bool by_count = k > 0 && k < p.vocab;
    int listed = 0;       // elements collected that hold all that is kept
    u64 cut = 0;          // otherwise: the last kept element
    double target = 0.0;  // the weight that top-p keeps, where it is known
    if (by_count && k <= kSmallK && r.gather_first(k, best, listed)) {
      // (all is in the list)
    } else {
      listed = 0;
      if (by_count) cut = r.find_kth(k);
      if (top_p < 1.f) {
        const u64 c = r.find_share(cut, (double)top_p, listed, target);
        cut = max(cut, c);
        if (listed) target = fmax(target, 0.0);
      }
    }
    if (listed == 0) {
      r.pick(cut, u, token);
    } else if (rank == 0) {
      const bool weighed = !(by_count && k <= kSmallK && target == 0.0);
      r.collect(false, weighed);
      r.finish(listed, weighed ? kList : k, weighed, target, (double)top_p, u, token);
    }
  }
  __syncthreads();
  cluster_sync();  // no CTA leaves while another may read its shared memory
}

template <typename T>
cudaError_t launch_one(const SampleParams& p, int ranks, int per, int room, size_t smem,
                       cudaStream_t st, bool pdl) {
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
  return cudaLaunchKernelEx(&cfg, sample_kernel<T>, p, ranks, per, room);
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
  const size_t smem = sizeof(Shared) + (size_t)room * 4;
  if (dtype == kDtypeF32) return launch_one<float>(p, ranks, per, room, smem, st, pdl);
  if (dtype == kDtypeBf16) return launch_one<__nv_bfloat16>(p, ranks, per, room, smem, st, pdl);
  return launch_one<__half>(p, ranks, per, room, smem, st, pdl);
}

}  // namespace gqa
