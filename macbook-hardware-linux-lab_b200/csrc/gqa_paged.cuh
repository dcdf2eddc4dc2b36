// Shared parts of the operators over a paged KV cache (gqa_paged.cu).
//
// A paged cache is a pool of pages of 2^page_shift rows; a sequence's row r lies
// in page table[seq][r >> page_shift] at row r & (2^page_shift - 1).  Element
// (page, head, row, i) is at page * page_stride + head * head_stride +
// row * row_stride + i, so that pages may hold a head's rows together
// ([head][row][d]) or a row's heads ([row][head][d]).
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "gqa_common.cuh"

namespace gqa {

enum : int { kStatusBadPage = 1 << 4 };  // a page table entry was outside the pool

enum : int { kDtypeF32 = 0, kDtypeBf16 = 1, kDtypeF16 = 2 };

struct PagedView {
  void* k;
  void* v;
  long long page_stride, head_stride, row_stride;  // elements
  const int* table;
  long long table_stride;
  int page_shift, n_pages, max_pages;
};

// The new tokens of a call: token rows [q_starts[s], q_starts[s + 1]) are the
// last rows of sequence s, which has seq_lens[s] rows with them.  A null
// q_starts means one token per sequence, row s.
struct TokenPlan {
  const int* q_starts;
  const int* seq_lens;
  int n_seq, n_tokens;
};

struct PagedAppendParams {
  PagedView kv;
  TokenPlan plan;
  const void* qkv;
  long long qkv_stride;
  const double* turns;  // [d / 2] rotations per position: theta^(-2i/d) / (2 pi)
  int n_q, n_kv;
  int* status;
};

struct PagedAttnParams {
  PagedView kv;
  TokenPlan plan;
  const void* qkv;
  long long qkv_stride;
  void* out;
  long long out_stride;
  const double* turns;
  int n_q, n_kv;
  int max_new, max_len;
  float scale_log2;  // log2(e) / sqrt(d)
  int* status;
};

// Loads and stores of 4-byte-or-less element types as fp32.
template <typename T>
struct Elem;
template <>
struct Elem<float> {
  static __device__ __forceinline__ float get(float x) { return x; }
  static __device__ __forceinline__ float put(float x) { return x; }
};
template <>
struct Elem<__nv_bfloat16> {
  static __device__ __forceinline__ float get(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 put(float x) { return __float2bfloat16_rn(x); }
};
template <>
struct Elem<__half> {
  static __device__ __forceinline__ float get(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half put(float x) { return __float2half_rn(x); }
};

// 16 bytes of T.
template <typename T>
struct alignas(16) Vec16 {
  static constexpr int n = 16 / sizeof(T);
  T e[n];
};

// Cosine and sine of the rotation of position pos at `turns` turns a position.
// The angle is formed in 64 bits and reduced to half a turn before it is
// rounded: at position 10^5 an angle formed in fp32 is off by up to 4e-3.
__device__ __forceinline__ void rope_cos_sin(int pos, double turns, float& c, float& s) {
  double t = (double)pos * turns;
  t -= rint(t);
  sincospif(2.0f * (float)t, &s, &c);
}

// The sequence that holds token row `tok` (the last one that starts at or
// before it), by a 32-way search of the whole warp.  Every lane gets it; the
// result is in [0, n_seq) whatever q_starts holds.
__device__ __forceinline__ int find_sequence(const int* q_starts, int n_seq, int tok) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = n_seq;  // the answer is in [lo, lo + n)
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int at = lane * step;
    const bool below = at < n && q_starts[lo + at] <= tok;
    const unsigned votes = __ballot_sync(0xffffffffu, below);
    const int last = votes ? 31 - __clz(votes) : 0;
    lo += last * step;
    n = min(step, n - last * step);
  }
  return lo;
}

enum Placed : int { kPlaced, kNoSequence, kImpossible };

// Position of token row `tok` of sequence s and the sequence's new rows and
// length.  kNoSequence: the plan does not place the row in s (a row past the
// last sequence); kImpossible: the sequence's length cannot be (fewer rows than
// new ones, or more than its table has).
__host__ __device__ __forceinline__ Placed place_token(const TokenPlan& plan, const PagedView& kv,
                                                       int s, int tok, int& pos, int& n_new,
                                                       int& len) {
  int i = 0;
  n_new = 1;
  if (plan.q_starts) {
    const int b = plan.q_starts[s], e = plan.q_starts[s + 1];
    if (tok < b || tok >= e) return kNoSequence;
    if (b < 0) return kImpossible;
    i = tok - b;
    n_new = e - b;
  }
  len = plan.seq_lens[s];
  if (len < n_new || (len - 1) >> kv.page_shift >= kv.max_pages) return kImpossible;
  pos = len - n_new + i;
  return kPlaced;
}

// Pool page of row `row` of sequence s, or -1 where the table names none.
__host__ __device__ __forceinline__ int page_of(const PagedView& kv, int s, int row) {
  const int page = kv.table[(long long)s * kv.table_stride + (row >> kv.page_shift)];
  return (unsigned)page < (unsigned)kv.n_pages ? page : -1;
}

// Element offset of row `row` of KV head h in its page.
__host__ __device__ __forceinline__ long long row_offset(const PagedView& kv, int page, int h,
                                                         int row) {
  return (long long)page * kv.page_stride + (long long)h * kv.head_stride +
         (long long)(row & ((1 << kv.page_shift) - 1)) * kv.row_stride;
}

}  // namespace gqa
