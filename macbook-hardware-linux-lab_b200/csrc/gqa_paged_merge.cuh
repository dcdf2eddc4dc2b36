// Merge of the parts that the attention's shares leave (gqa_paged_decode.cu, gqa_paged_chunk.cu).
#pragma once

#include <math_constants.h>

#include "gqa_paged.cuh"
#include "gqa_paged_launch.cuh"

namespace gqa {

// Merges the parts of a pair: one block per (CTA that holds a first part, query head).  The
// parts' weights first (a part per thread), so that the loads of the outputs depend on nothing
// and go out together.
constexpr int kMergeWarps = 8;
constexpr int kMaxParts = kMaxDecodeCtas;

template <typename T, int D, int G>
__device__ void merge_pair(const PagedAttnParams& p, const PagedPartials& part, int cta, int g) {
  __shared__ float weight[kMaxParts], red[2][kMergeWarps], so[kMergeWarps][D];
  const PagedJob job = part.jobs[cta];
  if (job.n_parts == 0) return;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // the first part's slot, then slot 0 of each CTA after it
  const auto slot_of = [&](int i) { return i == 0 ? job.slot : 2 * (cta + i); };
  constexpr int kOwn = kMaxParts / (kMergeWarps * 32);
  float2 ml[kOwn];
  float m = -CUDART_INF_F;
#pragma unroll
  for (int j = 0; j < kOwn; ++j) {
    const int i = tid + j * kMergeWarps * 32;
    ml[j] = i < job.n_parts ? part.ml[slot_of(i) * G + g] : make_float2(-CUDART_INF_F, 0.f);
    if (ml[j].y != 0.f) m = fmaxf(m, ml[j].x);
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  if (lane == 0) red[0][warp] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kMergeWarps; ++w) m = fmaxf(m, red[0][w]);
  float l = 0.f;
#pragma unroll
  for (int j = 0; j < kOwn; ++j) {
    const float a = ml[j].y != 0.f ? exp2f(ml[j].x - m) : 0.f;
    l += a * ml[j].y;
    weight[tid + j * kMergeWarps * 32] = a;
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
  if (lane == 0) red[1][warp] = l;
  __syncthreads();
  l = 0.f;
#pragma unroll
  for (int w = 0; w < kMergeWarps; ++w) l += red[1][w];
  constexpr int E = D / 32;
  float o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  for (int i0 = warp; i0 < job.n_parts; i0 += 8 * kMergeWarps) {
    float x[8][E], a[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = min(i0 + u * kMergeWarps, job.n_parts - 1);
      a[u] = i0 + u * kMergeWarps < job.n_parts ? weight[i] : 0.f;
      const float* src = part.o + ((long long)slot_of(i) * G + g) * D + lane * E;
#pragma unroll
      for (int e = 0; e < E; ++e) x[u][e] = src[e];
    }
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (a[u] != 0.f)  // (a part without a row holds nothing to be added)
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] += a[u] * x[u][e];
  }
#pragma unroll
  for (int e = 0; e < E; ++e) so[warp][lane * E + e] = o[e];
  __syncthreads();
  T* out = static_cast<T*>(p.out) + (long long)job.tok * p.out_stride +
           (long long)(job.head * G + g) * D;
  for (int e = tid; e < D; e += kMergeWarps * 32) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kMergeWarps; ++w) sum += so[w][e];
    out[e] = Elem<T>::put(l != 0.f ? sum / l : 0.f);
  }
}

// Merges the parts of a unit that crossed shares: a warp per row.
template <typename T, int D, int G>
__device__ void merge_unit_row(const PagedAttnParams& p, const PagedPartials& part,
                               const PagedChunkJob& job, int cta, int idx) {
  constexpr int kTok = kChunkRows / G, E = D / 32;
  const int lane = threadIdx.x & 31;
  const int t = idx / G, g = idx % G;
  if (t >= job.n_tok) return;
  const int row = t < kTok ? idx : kChunkRows + (t - kTok) * G + g;
  const auto at = [&](int i) {
    return (long long)(i == 0 ? job.slot : 2 * (cta + i)) * kChunkSlotRows + row;
  };
  // the parts' weights, a part per lane; then loads that depend on nothing
  float m = -CUDART_INF_F, l = 0.f, o[E];
  for (int i = lane; i < job.n_parts; i += 32) {
    const float2 ml = part.chunk_ml[at(i)];
    if (ml.y != 0.f) m = fmaxf(m, ml.x);
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  for (int i0 = 0; i0 < job.n_parts; i0 += 32) {
    float2 ml = make_float2(0.f, 0.f);
    if (i0 + lane < job.n_parts) ml = part.chunk_ml[at(i0 + lane)];
    const float weight = ml.y != 0.f ? exp2f(ml.x - m) : 0.f;
    l += weight * ml.y;
    for (int i = i0; i < min(i0 + 32, job.n_parts); i += 8) {
      float x[8][E];
#pragma unroll
      for (int u = 0; u < 8; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e)
          x[u][e] = i + u < job.n_parts ? part.chunk_o[at(i + u) * D + lane * E + e] : 0.f;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float a = __shfl_sync(0xffffffffu, weight, i - i0 + u);
        if (a != 0.f)
#pragma unroll
          for (int e = 0; e < E; ++e) o[e] += a * x[u][e];
      }
    }
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
  T* out = static_cast<T*>(p.out) + (long long)(job.tok + t) * p.out_stride +
           (long long)(job.head * G + g) * D + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) out[e] = Elem<T>::put(l != 0.f ? o[e] / l : 0.f);
}

// Blocks: one per (decode CTA, query head), then kUnitSlabs per chunk CTA.  Most find nothing to
// merge and leave.
constexpr int kUnitSlabs = 32;

template <typename T, int D, int G>
__global__ void __launch_bounds__(kMergeWarps * 32)
    paged_merge_kernel(const PagedAttnParams p, const PagedPartials part, const int n_decode) {
  pdl_wait();
  const int b = blockIdx.x;
  if (b < n_decode * G) {
    merge_pair<T, D, G>(p, part, b / G, b % G);
    return;
  }
  const int cta = (b - n_decode * G) / kUnitSlabs, slab = (b - n_decode * G) % kUnitSlabs;
  const PagedChunkJob job = part.chunk_jobs[cta];
  if (job.n_parts == 0) return;
  for (int i = slab * kMergeWarps + (threadIdx.x >> 5); i < job.n_tok * G;
       i += kUnitSlabs * kMergeWarps)
    merge_unit_row<T, D, G>(p, part, job, cta, i);
}

}  // namespace gqa
