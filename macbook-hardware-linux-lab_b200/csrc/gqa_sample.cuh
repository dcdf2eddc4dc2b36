// Parameters of the sampling kernel (gqa_sample.cu).
#pragma once

#include <cuda_runtime.h>

namespace gqa {

struct SampleParams {
  const void* logits;       // [n_rows] rows of vocab, logits_stride elements apart
  long long logits_stride;
  int n_rows, vocab;
  int wshift;               // weights are held in units of 2^-wshift of the largest
  const float* temperature; // [n_rows] each; null: 1 / off / off / off
  const int* top_k;
  const float* top_p;
  const float* min_p;
  const float* uniform;     // [n_rows] in [0, 1)
  int* tokens;              // [n_rows]
};

cudaError_t prepare_sample();
cudaError_t launch_sample(const SampleParams& p, int dtype, int n_sm, cudaStream_t st, bool pdl);

}  // namespace gqa
