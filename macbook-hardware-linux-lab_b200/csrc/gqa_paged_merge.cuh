// Merge of the parts that the attention's shares leave (gqa_paged_decode.cu, gqa_paged_chunk.cu).
#pragma once

#include <math_constants.h>

#include "gqa_paged.cuh"
#include "gqa_paged_launch.cuh"

namespace gqa {

// A warp's merge of every `step`-th part of a pair from `first` on, for one query head.  (m, l) and
// outputs are loaded together (nothing waits for a weight), up to 8 parts at once.
constexpr int kMergeWarps = 8;

template <int D, int G>
__device__ __forceinline__ void merge_parts(const PagedPartials& part, const PagedJob& job, int g,
                                            int first, int step, float& m, float& l,
                                            float (&o)[D / 32]) {
  const int lane = threadIdx.x & 31;
  // the first part's slot, then slot 0 of each CTA after it
  const auto slot_of = [&](int i) { return i == 0 ? job.slot : 2 * (job.cta + i); };
  constexpr int E = D / 32, kAtOnce = kFewParts;
  m = -CUDART_INF_F;
  l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  for (int i0 = first; i0 < job.n_parts; i0 += kAtOnce * step) {
    const int own = i0 + (lane & (kAtOnce - 1)) * step;  // the part of this lane's (m, l)
    const float2 ml =
        own < job.n_parts ? part.ml[slot_of(own) * G + g] : make_float2(-CUDART_INF_F, 0.f);
    float x[kAtOnce][E];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int i = i0 + u * step;
      const float* src = part.o + ((long long)slot_of(i) * G + g) * D + lane * E;
#pragma unroll
      for (int e = 0; e < E; ++e) x[u][e] = i < job.n_parts ? src[e] : 0.f;
    }
    float mx = ml.y != 0.f ? ml.x : -CUDART_INF_F;
#pragma unroll
    for (int d = kAtOnce / 2; d; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
    mx = fmaxf(m, mx);
    if (mx == -CUDART_INF_F) continue;  // (nothing in any of them; alike in the warp's lanes)
    const float a = exp2f(m - mx), w = ml.y != 0.f ? exp2f(ml.x - mx) : 0.f;
    float add = w * ml.y;
#pragma unroll
    for (int d = kAtOnce / 2; d; d >>= 1) add += __shfl_xor_sync(0xffffffffu, add, d);
    m = mx;
    l = l * a + add;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] *= a;
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const float wu = __shfl_sync(0xffffffffu, w, u);
      if (wu != 0.f)  // (a part without a row holds nothing to be added)
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] += wu * x[u][e];
    }
  }
}

// A pair of few parts, a query head by a warp.
template <typename T, int D, int G>
__device__ __forceinline__ void merge_by_warp(const PagedAttnParams& p, const PagedPartials& part,
                                              const PagedJob& job, int g) {
  constexpr int E = D / 32;
  float m, l, o[E];
  merge_parts<D, G>(part, job, g, 0, 1, m, l, o);
  T* out = static_cast<T*>(p.out) + (long long)job.tok * p.out_stride +
           (long long)(job.head * G + g) * D + (threadIdx.x & 31) * E;
#pragma unroll
  for (int e = 0; e < E; ++e) out[e] = Elem<T>::put(l != 0.f ? o[e] / l : 0.f);
}

// A query head of many, by a block.
template <typename T, int D, int G>
__device__ void merge_by_block(const PagedAttnParams& p, const PagedPartials& part,
                               const PagedJob& job, int g) {
  __shared__ float sm[kMergeWarps], sl[kMergeWarps], so[kMergeWarps][D];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int E = D / 32;
  float m, l, o[E];
  merge_parts<D, G>(part, job, g, warp, kMergeWarps, m, l, o);
  __syncthreads();
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) so[warp][lane * E + e] = o[e];
  __syncthreads();
  T* out = static_cast<T*>(p.out) + (long long)job.tok * p.out_stride +
           (long long)(job.head * G + g) * D;
  for (int e = tid; e < D; e += kMergeWarps * 32) {
    float mm = -CUDART_INF_F;
#pragma unroll
    for (int w = 0; w < kMergeWarps; ++w) mm = fmaxf(mm, sm[w]);
    float ll = 0.f, oo = 0.f;
#pragma unroll
    for (int w = 0; w < kMergeWarps; ++w) {
      if (sl[w] == 0.f) continue;
      const float a = exp2f(sm[w] - mm);
      ll += a * sl[w];
      oo += a * so[w][e];
    }
    out[e] = Elem<T>::put(ll != 0.f ? oo / ll : 0.f);
  }
}

// Merges the parts of a unit that crossed shares: R rows at a time per warp, two parts at once,
// all loads of which go out together.
template <typename T, int D, int G, int R>
__device__ void merge_unit_rows(const PagedAttnParams& p, const PagedPartials& part,
                                const PagedChunkJob& job, int cta, int idx0, int step) {
  constexpr int kTok = kChunkRows / G, E = D / 32, kAtOnce = 2;
  const int lane = threadIdx.x & 31, rows = job.n_tok * G;
  const auto at = [&](int i, int r) {
    const int idx = min(idx0 + r * step, rows - 1), t = idx / G;
    const int row = t < kTok ? idx : kChunkRows + idx - kTok * G;
    return (long long)(i == 0 ? job.slot : 2 * (cta + i)) * kChunkSlotRows + row;
  };
  float m[R], l[R], o[R][E];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = -CUDART_INF_F;
    l[r] = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) o[r][e] = 0.f;
  }
  for (int i0 = 0; i0 < job.n_parts; i0 += kAtOnce) {
    float2 ml[R][kAtOnce];
    float x[R][kAtOnce][E];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const bool on = i0 + u < job.n_parts;
        const long long a = at(on ? i0 + u : 0, r);
        ml[r][u] = on ? part.chunk_ml[a] : make_float2(-CUDART_INF_F, 0.f);
#pragma unroll
        for (int e = 0; e < E; ++e) x[r][u][e] = on ? part.chunk_o[a * D + lane * E + e] : 0.f;
      }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float mx = m[r];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u)
        if (ml[r][u].y != 0.f) mx = fmaxf(mx, ml[r][u].x);
      if (mx == -CUDART_INF_F) continue;
      const float a = exp2f(m[r] - mx);
      m[r] = mx;
      l[r] *= a;
#pragma unroll
      for (int e = 0; e < E; ++e) o[r][e] *= a;
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        if (ml[r][u].y == 0.f) continue;
        const float w = exp2f(ml[r][u].x - mx);
        l[r] += w * ml[r][u].y;
#pragma unroll
        for (int e = 0; e < E; ++e) o[r][e] += w * x[r][u][e];
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int idx = idx0 + r * step;
    if (idx >= rows) break;
    T* out = static_cast<T*>(p.out) + (long long)(job.tok + idx / G) * p.out_stride +
             (long long)(job.head * G + idx % G) * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) out[e] = Elem<T>::put(l[r] != 0.f ? o[r][e] / l[r] : 0.f);
  }
}

// Blocks: one per decode CTA, which does what that CTA listed, then kUnitSlabs per chunk CTA.  All
// of a decode's fit on the device at once (a block per CTA and query head, most of which found
// nothing, took three waves: 58.6 us in place of 56.6 for 64 sequences), and registers are kept to
// what lets four share an SM: with 16 parts at once and three, 64 sequences took 3 us more.  The
// merge is 4 us of the 10 and 19 of one token over 4096 and 32768 rows in fp32, and is bound by
// the chain of its loads.  (One list of the jobs, made by every block for itself and dealt out
// evenly, took 104 us in place of 97 for four whole prompts.)
// A chunk's rows: one at a time per warp of 16 blocks (two per warp of 8 blocks: 58.1 us in place of
// 53.9 for 512 tokens over 8192 rows, the others within 1 us).
constexpr int kUnitSlabs = 16, kUnitRows = 1;

template <typename T, int D, int G>
__global__ void __launch_bounds__(kMergeWarps * 32, 4)
    paged_merge_kernel(const PagedAttnParams p, const PagedPartials part, const int n_decode) {
  pdl_wait();
  const int b = blockIdx.x;
  if (b < n_decode) {
    static_assert(kMergeWarps >= G, "a warp per query head");
    const PagedJob job = part.jobs[b];
    if (job.n_parts == 0) return;
    if (job.q_head >= 0)
      merge_by_block<T, D, G>(p, part, job, job.q_head);
    else if ((threadIdx.x >> 5) < G)
      merge_by_warp<T, D, G>(p, part, job, threadIdx.x >> 5);
    return;
  }
  const int cta = (b - n_decode) / kUnitSlabs, slab = (b - n_decode) % kUnitSlabs;
  const PagedChunkJob job = part.chunk_jobs[cta];
  if (job.n_parts == 0) return;
  constexpr int kStep = kUnitSlabs * kMergeWarps;
  for (int i = slab * kMergeWarps + (threadIdx.x >> 5); i < job.n_tok * G; i += kUnitRows * kStep)
    merge_unit_rows<T, D, G, kUnitRows>(p, part, job, cta, i, kStep);
}

}  // namespace gqa
