// Launches of the paged operators' kernels.
#pragma once

#include <algorithm>

#include <cuda_runtime.h>

#include "gqa_paged.cuh"

namespace gqa {

// Parts of (token, KV head) pairs whose rows were split over CTAs: two slots per CTA, each
// [G][D] un-normalised outputs and [G] (m in log2 units, l), and what the merge's block of the
// same number does: all query heads of a pair of few parts, listed under the CTA that holds its
// first; else one of them, listed under one of the pair's first G CTAs each.
struct alignas(16) PagedJob {
  int tok, head;
  int cta, slot;  // of the first part
  int n_parts;    // CTAs from `cta` on (0: nothing to merge)
  int q_head;     // -1: all
};
constexpr int kFewParts = 8;  // of a pair whose query heads a warp each merges
// The same for chunks: units of some tokens, 256 rows a slot.
struct PagedChunkJob {
  int tok, n_tok, head, slot;
  int n_parts;
};
constexpr int kChunkSlotRows = 256;
constexpr int kChunkRows = 128;      // rows of a chunk's tile: token * G + head
constexpr int kMaxDecodeCtas = 512;  // of the single tokens' grid (and parts of a pair)
struct PagedPartials {
  float* o;
  float2* ml;
  PagedJob* jobs;
  int n_ctas;  // that there are slots for
  float* chunk_o;
  float2* chunk_ml;
  PagedChunkJob* chunk_jobs;
  int n_chunk_ctas;
};

// Whether no byte of n rows of a_width bytes, a_stride apart, is one of n rows of b_width, b_stride
// apart.  Rows that interleave are told apart where the strides are equal; otherwise whole extents
// are (each from its first row's start to its last row's end).
inline bool rows_apart(unsigned long long a, long long a_stride, long long a_width,
                       unsigned long long b, long long b_stride, long long b_width, int n) {
  using Wide = __int128;  // (n rows of the largest stride pass 64 bits)
  const Wide a_end = (Wide)a + (Wide)(n - 1) * a_stride + a_width;
  const Wide b_end = (Wide)b + (Wide)(n - 1) * b_stride + b_width;
  if (b >= a_end || a >= b_end) return true;
  if (a_stride != b_stride) return false;
  Wide at = ((Wide)b - (Wide)a) % a_stride;  // where b's rows start in a's
  if (at < 0) at += a_stride;
  return at >= a_width && at + b_width <= a_stride;
}

template <typename... P, typename... A>
cudaError_t launch_with_pdl(void (*kernel)(P...), dim3 grid, int threads, size_t smem,
                            cudaStream_t st, bool pdl, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

cudaError_t prepare_paged_decode();
cudaError_t launch_paged_append(const PagedAppendParams& p, int dtype, int head_dim,
                                cudaStream_t st, bool pdl);
// The attention's launches, in this order: single tokens (and, `rotate`, q of the chunks), chunks
// (max_new > 1), merge.  *grid gets the CTAs launched.
cudaError_t launch_paged_decode(const PagedAttnParams& p, const PagedPartials& part, int dtype,
                                int head_dim, int n_sm, cudaStream_t st, bool pdl, bool rotate,
                                int* grid);
cudaError_t prepare_paged_chunk16();
cudaError_t launch_paged_chunk16(const PagedAttnParams& p, const PagedPartials& part, int dtype,
                                 int head_dim, int n_sm, cudaStream_t st, int* grid);
cudaError_t prepare_paged_chunk32();
cudaError_t launch_paged_chunk32(const PagedAttnParams& p, const PagedPartials& part, int head_dim,
                                 int n_sm, cudaStream_t st, int* grid);
cudaError_t launch_paged_merge(const PagedAttnParams& p, const PagedPartials& part, int dtype,
                               int head_dim, int n_decode, int n_chunk, cudaStream_t st);

}  // namespace gqa
