// Paged KV cache: the append (the attention is in gqa_paged_decode.cu, gqa_paged_chunk.cu and
// gqa_paged_chunk32.cu).
//
// The reference keeps one contiguous cache per sequence and appends one row a
// call (kernel_attention_gqa.cl:149-194); these operators hold many sequences
// in a pool of pages and take any number of new tokens of each in one call.
#include "gqa_paged.cuh"
#include "gqa_paged_launch.cuh"

namespace gqa {

// ---------------------------------------------------------------------------
// Append: k'[i] = k[i] cos a - k[i + d/2] sin a, k'[i + d/2] = k[i] sin a +
// k[i + d/2] cos a, a = pos theta^(-2i/d); v as it is.
// ---------------------------------------------------------------------------
constexpr int kAppendThreads = 256;

// One thread per (token, KV head, 16-byte chunk of the first half): it rotates
// the chunk and its partner half a row on and copies the same two chunks of V, so
// every access is 16 bytes wide and no value passes between threads.  Bytes bound
// it: 10077 tokens of two KV heads in bf16 (20.6 MB) take 6.0 us, 2.5 of which one
// token takes too; 64 single tokens 2.5 us.
template <typename T, int D>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const PagedAppendParams p) {
  using V = Vec16<T>;
  constexpr int kChunks = D / 2 / V::n;
  // (in this order: the next kernel may read cache rows ahead of its own wait, and relies on all
  // before this one being done when it starts)
  pdl_wait();
  pdl_launch_dependents();
  const int per_token = p.n_kv * kChunks;
  const long long item = (long long)blockIdx.x * kAppendThreads + threadIdx.x;
  const long long last = (long long)p.plan.n_tokens * per_token - 1;
  const int tok = (int)(min(item, last) / per_token);
  int s = tok;
  if (p.plan.q_starts) {
    // the warp looks up its first token; its others are in that or a later sequence
    const int tok0 = __shfl_sync(0xffffffffu, tok, 0);
    s = find_sequence(p.plan.q_starts, p.plan.n_seq, tok0);
    while (s + 1 < p.plan.n_seq && p.plan.q_starts[s + 1] <= tok) ++s;
  }
  if (item > last) return;
  const int rem = (int)(item - (long long)tok * per_token);
  const int h = rem / kChunks, c = rem % kChunks;
  int pos, n_new, len;
  const Placed placed = place_token(p.plan, p.kv, s, tok, pos, n_new, len);
  if (placed == kImpossible) atomicOr(p.status, kStatusBadLength);
  if (placed != kPlaced) return;
  const int page = page_of(p.kv, s, pos);
  if (page < 0) {
    atomicOr(p.status, kStatusBadPage);
    return;
  }
  const T* k_in = static_cast<const T*>(p.qkv) + (long long)tok * p.qkv_stride +
                  (long long)(p.n_q + h) * D + c * V::n;
  const T* v_in = k_in + (long long)p.n_kv * D;
  const V k0 = *reinterpret_cast<const V*>(k_in), k1 = *reinterpret_cast<const V*>(k_in + D / 2);
  const V v0 = *reinterpret_cast<const V*>(v_in), v1 = *reinterpret_cast<const V*>(v_in + D / 2);
  V y0, y1;
#pragma unroll
  for (int e = 0; e < V::n; ++e) {
    float co, si;
    rope_cos_sin(pos, p.turns[c * V::n + e], co, si);
    const float a = Elem<T>::get(k0.e[e]), b = Elem<T>::get(k1.e[e]);
    y0.e[e] = Elem<T>::put(a * co - b * si);
    y1.e[e] = Elem<T>::put(a * si + b * co);
  }
  const long long at = row_offset(p.kv, page, h, pos) + c * V::n;
  T* k_out = static_cast<T*>(p.kv.k) + at;
  T* v_out = static_cast<T*>(p.kv.v) + at;
  *reinterpret_cast<V*>(k_out) = y0;
  *reinterpret_cast<V*>(k_out + D / 2) = y1;
  *reinterpret_cast<V*>(v_out) = v0;
  *reinterpret_cast<V*>(v_out + D / 2) = v1;
}

cudaError_t launch_paged_append(const PagedAppendParams& p, int dtype, int head_dim,
                                cudaStream_t st, bool pdl) {
  const int vec = dtype == kDtypeF32 ? 4 : 8;
  const long long items = (long long)p.plan.n_tokens * p.n_kv * (head_dim / 2 / vec);
  const dim3 grid((unsigned)((items + kAppendThreads - 1) / kAppendThreads));
  const auto go = [&](auto kernel) {
    return launch_with_pdl(kernel, grid, kAppendThreads, 0, st, pdl, p);
  };
  const bool wide = head_dim == 128;
  if (dtype == kDtypeF32)
    return wide ? go(paged_append_kernel<float, 128>) : go(paged_append_kernel<float, 64>);
  if (dtype == kDtypeBf16)
    return wide ? go(paged_append_kernel<__nv_bfloat16, 128>)
                : go(paged_append_kernel<__nv_bfloat16, 64>);
  return wide ? go(paged_append_kernel<__half, 128>) : go(paged_append_kernel<__half, 64>);
}

}  // namespace gqa
