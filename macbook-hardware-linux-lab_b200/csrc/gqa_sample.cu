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
// the last key that is kept and how many of its ties are, found by radix
// selection over counts and over weights.  The token is then the first, in index
// order, whose cumulative kept weight exceeds u times the total.
//
// Weights are summed as integers (fixed point, 2^-wshift of the largest weight):
// a sum is exact in any order, so neither the order of atomics nor the split of
// a row over threads can change a token.
#include <math_constants.h>

#include "gqa_paged.cuh"
#include "gqa_sample.cuh"

namespace gqa {

constexpr int kSampleThreads = 1024;

// Keys in the order of the logits: larger logit, larger key; -0 as 0, NaN as -inf.
__device__ __forceinline__ uint32_t logit_key(float x) {
  if (x != x) x = -CUDART_INF_F;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_logit(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}

struct RowRule {
  double inv_t, scale;  // 1 / temperature, 2^wshift
  float top;            // largest logit
};

// The weight of a logit relative to the largest one.
__device__ __forceinline__ double weight_of(float x, const RowRule& r) {
  if (x == r.top) return 1.0;  // (also where the largest is infinite)
  if (!(x > -CUDART_INF_F) || r.top == CUDART_INF_F) return 0.0;
  return exp(((double)x - (double)r.top) * r.inv_t);
}
__device__ __forceinline__ unsigned long long fixed_weight(float x, const RowRule& r) {
  return (unsigned long long)(weight_of(x, r) * r.scale + 0.5);
}

// Exclusive scan over the block's threads; *total gets the sum.
__device__ unsigned long long block_scan(unsigned long long v, unsigned long long* total) {
  __shared__ unsigned long long part[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long x = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const unsigned long long y = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();
  if (lane == 31) part[warp] = x;
  __syncthreads();
  unsigned long long before = 0, sum = 0;
  for (int w = 0; w < kSampleThreads / 32; ++w) {
    if (w < warp) before += part[w];
    sum += part[w];
  }
  *total = sum;
  return before + x - v;
}

template <typename T>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const SampleParams p) {
  __shared__ unsigned long long hist[256];
  __shared__ unsigned long long s_best, s_sum;
  __shared__ uint32_t s_bin;
  __shared__ unsigned long long s_before;
  const int row = blockIdx.x, tid = threadIdx.x, n = p.vocab;
  const T* x = static_cast<const T*>(p.logits) + (long long)row * p.logits_stride;
  pdl_wait();
  const float temp = p.temperature ? p.temperature[row] : 1.f;
  const int k = p.top_k ? p.top_k[row] : 0;
  const float top_p = p.top_p ? p.top_p[row] : 1.f;
  const float min_p = p.min_p ? p.min_p[row] : 0.f;

  // the largest logit, the first of its ties
  if (tid == 0) s_best = 0;
  __syncthreads();
  unsigned long long best = 0;
  for (int i = tid; i < n; i += kSampleThreads) {
    const unsigned long long b =
        (unsigned long long)logit_key(Elem<T>::get(x[i])) << 32 | (0xffffffffu - (uint32_t)i);
    if (b > best) best = b;
  }
  atomicMax(&s_best, best);
  __syncthreads();
  best = s_best;
  const uint32_t top_key = (uint32_t)(best >> 32);
  const int first = (int)(0xffffffffu - (uint32_t)best);
  RowRule r;
  r.top = key_logit(top_key);
  if (!(temp > 0.f) || r.top == -CUDART_INF_F) {
    if (tid == 0) p.tokens[row] = r.top == -CUDART_INF_F ? 0 : first;
    return;
  }
  r.inv_t = 1.0 / (double)temp;
  r.scale = (double)(1ull << p.wshift);

  // The last kept key and how many of its ties are kept (all keys to begin with).
  uint32_t cut = 0;
  unsigned long long ties = ~0ull;
  if (k > 0 && k < n) {
    uint32_t prefix = 0;
    unsigned long long before = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int b = tid; b < 256; b += kSampleThreads) hist[b] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += kSampleThreads) {
        const uint32_t key = logit_key(Elem<T>::get(x[i]));
        if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8)))
          atomicAdd(&hist[(key >> shift) & 255], 1ull);
      }
      __syncthreads();
      if (tid == 0) {
        int b = 255;
        while (b > 0 && before + hist[b] < (unsigned long long)k) before += hist[b--];
        s_bin = b;
        s_before = before;
      }
      __syncthreads();
      prefix |= s_bin << shift;
      before = s_before;
    }
    cut = prefix;
    ties = (unsigned long long)k - before;
  }
  if (top_p < 1.f) {
    const unsigned long long cut_mass = ties == ~0ull ? 0 : ties * fixed_weight(key_logit(cut), r);
    if (tid == 0) s_sum = 0;
    __syncthreads();
    unsigned long long sum = 0;
    for (int i = tid; i < n; i += kSampleThreads) {
      const float v = Elem<T>::get(x[i]);
      const uint32_t key = logit_key(v);
      if (key > cut || ties == ~0ull) sum += fixed_weight(key_logit(key), r);
    }
    atomicAdd(&s_sum, sum);
    __syncthreads();
    const double target = (double)top_p * (double)(s_sum + cut_mass);
    uint32_t prefix = 0;
    unsigned long long before = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int b = tid; b < 256; b += kSampleThreads) hist[b] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += kSampleThreads) {
        const uint32_t key = logit_key(Elem<T>::get(x[i]));
        if ((key > cut || ties == ~0ull) &&
            (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))))
          atomicAdd(&hist[(key >> shift) & 255], fixed_weight(key_logit(key), r));
      }
      __syncthreads();
      if (tid == 0) {
        if (cut_mass && (shift == 24 || (cut >> (shift + 8)) == (prefix >> (shift + 8))))
          hist[(cut >> shift) & 255] += cut_mass;
        // down to the first bin whose weight reaches the target (or, should
        // rounding leave it unreached, the last bin with any weight)
        int b = 255, last = -1;
        unsigned long long at_last = before;
        for (; b >= 0; --b) {
          if (!hist[b]) continue;
          last = b;
          at_last = before;
          if ((double)(before + hist[b]) >= target) break;
          before += hist[b];
        }
        s_bin = last;
        s_before = at_last;
      }
      __syncthreads();
      prefix |= s_bin << shift;
      before = s_before;
    }
    // ties of the last key: the fewest, at least one, that reach the target
    const unsigned long long w = fixed_weight(key_logit(prefix), r);
    unsigned long long need = 1;
    if (w && (double)(before + w) < target) {
      need = (unsigned long long)ceil((target - (double)before) / (double)w);
      if (need > 1 && (double)(before + (need - 1) * w) >= target) --need;
      if ((double)(before + need * w) < target) ++need;
    }
    ties = prefix == cut && need > ties ? ties : need;
    cut = prefix;
  }

  // Cumulative weights in index order: a contiguous range of the row per thread.
  const int per = (n + kSampleThreads - 1) / kSampleThreads;
  const int lo = min(tid * per, n), hi = min(lo + per, n);
  unsigned long long mine = 0;
  for (int i = lo; i < hi; ++i) mine += logit_key(Elem<T>::get(x[i])) == cut;
  unsigned long long unused;
  const unsigned long long tie0 = block_scan(mine, &unused);
  const auto walk = [&](auto&& f) {
    unsigned long long tie = tie0;
    for (int i = lo; i < hi; ++i) {
      const uint32_t key = logit_key(Elem<T>::get(x[i]));
      bool keep = key > cut || (key == cut && tie < ties);
      tie += key == cut;
      if (!keep) continue;
      const float v = key_logit(key);
      if (i != first && weight_of(v, r) < (double)min_p) continue;
      const unsigned long long w = fixed_weight(v, r);
      if (w && !f(i, w)) break;
    }
  };
  unsigned long long weight = 0, total;
  walk([&](int, unsigned long long w) { weight += w; return true; });
  const unsigned long long before = block_scan(weight, &total);
  float u = p.uniform[row];
  u = u > 0.f ? u : 0.f;
  // the token is the first whose cumulative weight exceeds u * total (the last, should u be
  // 1 or more)
  const double ut = (double)u * (double)total;
  const unsigned long long target = ut < (double)total ? (unsigned long long)ut : total - 1;
  if (before <= target && before + weight > target) {
    unsigned long long c = before;
    walk([&](int i, unsigned long long w) {
      c += w;
      if (c <= target) return true;
      p.tokens[row] = i;
      return false;
    });
  }
}

cudaError_t launch_sample(const SampleParams& p, int dtype, cudaStream_t st, bool pdl) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.n_rows);
  cfg.blockDim = dim3(kSampleThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  if (dtype == kDtypeF32) return cudaLaunchKernelEx(&cfg, sample_kernel<float>, p);
  if (dtype == kDtypeBf16) return cudaLaunchKernelEx(&cfg, sample_kernel<__nv_bfloat16>, p);
  return cudaLaunchKernelEx(&cfg, sample_kernel<__half>, p);
}

}  // namespace gqa
