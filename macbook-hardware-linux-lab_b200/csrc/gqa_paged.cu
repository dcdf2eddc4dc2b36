// Paged KV cache: append and attention.
//
// The reference keeps one contiguous cache per sequence and appends one row a
// call (kernel_attention_gqa.cl:149-194); these operators hold many sequences
// in a pool of pages and take any number of new tokens of each in one call.
#include <math_constants.h>

#include "gqa_paged.cuh"
#include "gqa_paged_launch.cuh"

namespace gqa {

// ---------------------------------------------------------------------------
// Append: k'[i] = k[i] cos a - k[i + d/2] sin a, k'[i + d/2] = k[i] sin a +
// k[i + d/2] cos a, a = pos theta^(-2i/d); v as it is.
// ---------------------------------------------------------------------------
constexpr int kAppendThreads = 256;

// One thread per (token, KV head, 16-byte chunk of the first half): it rotates
// the chunk and its partner half a row on and copies the same two chunks of V.
template <typename T, int D>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const PagedAppendParams p) {
  using V = Vec16<T>;
  constexpr int kChunks = D / 2 / V::n;
  pdl_launch_dependents();
  pdl_wait();
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

// ---------------------------------------------------------------------------
// Attention: out = sum_t w_t V_t / sum_t w_t, w_t = exp(q.K_t / sqrt(d) - m)
// over the rows t <= pos of the token, m the running maximum of the scores.
// ---------------------------------------------------------------------------
constexpr int kSimpleWarps = 4;

// One block per (token, KV head): its warps take the keys in turn, a lane holds
// D / 32 consecutive elements of every row, and the warps' (m, l, o) are merged
// at the end.
template <typename T, int D, int G>
__global__ void __launch_bounds__(kSimpleWarps * 32)
    paged_attn_simple_kernel(const PagedAttnParams p) {
  constexpr int E = D / 32;
  __shared__ float sq[G][D];
  __shared__ float sm[kSimpleWarps][G], sl[kSimpleWarps][G], so[kSimpleWarps][G][D];
  const int tok = blockIdx.x, h = blockIdx.y, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  pdl_wait();
  const int s = p.plan.q_starts ? find_sequence(p.plan.q_starts, p.plan.n_seq, tok) : tok;
  int pos, n_new, len;
  const Placed placed = place_token(p.plan, p.kv, s, tok, pos, n_new, len);
  if (placed == kNoSequence || (placed == kPlaced && n_new == 1)) return;
  if (placed == kImpossible || len > p.max_len || n_new > p.max_new) {
    if (threadIdx.x == 0) atomicOr(p.status, kStatusBadLength);
    return;
  }
  const T* q = static_cast<const T*>(p.qkv) + (long long)tok * p.qkv_stride +
               (long long)h * G * D;
  for (int i = threadIdx.x; i < G * (D / 2); i += blockDim.x) {
    const int g = i / (D / 2), e = i % (D / 2);
    float co, si;
    rope_cos_sin(pos, p.turns[e], co, si);
    const float a = Elem<T>::get(q[g * D + e]), b = Elem<T>::get(q[g * D + e + D / 2]);
    sq[g][e] = (a * co - b * si) * p.scale_log2;
    sq[g][e + D / 2] = (a * si + b * co) * p.scale_log2;
  }
  __syncthreads();
  float qr[G][E], o[G][E], m[G], l[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    m[g] = -CUDART_INF_F;
    l[g] = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      qr[g][e] = sq[g][lane * E + e];
      o[g][e] = 0.f;
    }
  }
  for (int t = warp; t <= pos; t += kSimpleWarps) {
    const int page = page_of(p.kv, s, t);
    if (page < 0) {
      if (lane == 0) atomicOr(p.status, kStatusBadPage);
      continue;
    }
    const long long at = row_offset(p.kv, page, h, t) + lane * E;
    float k[E], v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      k[e] = Elem<T>::get(static_cast<const T*>(p.kv.k)[at + e]);
      v[e] = Elem<T>::get(static_cast<const T*>(p.kv.v)[at + e]);
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float x = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) x = fmaf(qr[g][e], k[e], x);
#pragma unroll
      for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
      const float mn = fmaxf(m[g], x);
      const float a = mn == -CUDART_INF_F ? 1.f : exp2f(m[g] - mn);
      const float w = mn == -CUDART_INF_F ? 0.f : exp2f(x - mn);
      m[g] = mn;
      l[g] = l[g] * a + w;
#pragma unroll
      for (int e = 0; e < E; ++e) o[g][e] = o[g][e] * a + w * v[e];
    }
  }
#pragma unroll
  for (int g = 0; g < G; ++g) {
    sm[warp][g] = m[g];
    sl[warp][g] = l[g];
#pragma unroll
    for (int e = 0; e < E; ++e) so[warp][g][lane * E + e] = o[g][e];
  }
  __syncthreads();
  T* out = static_cast<T*>(p.out) + (long long)tok * p.out_stride + (long long)h * G * D;
  for (int i = threadIdx.x; i < G * D; i += blockDim.x) {
    const int g = i / D, e = i % D;
    float mm = -CUDART_INF_F;
    for (int w = 0; w < kSimpleWarps; ++w) mm = fmaxf(mm, sm[w][g]);
    float ll = 0.f, oo = 0.f;
    for (int w = 0; w < kSimpleWarps; ++w) {
      if (sl[w][g] == 0.f) continue;
      const float a = exp2f(sm[w][g] - mm);
      ll += a * sl[w][g];
      oo += a * so[w][g][e];
    }
    out[i] = Elem<T>::put(ll != 0.f ? oo / ll : 0.f);
  }
}

template <typename T>
static cudaError_t launch_simple(const PagedAttnParams& p, int head_dim, cudaStream_t st,
                                 bool pdl) {
  const dim3 grid(p.plan.n_tokens, p.n_kv);
  if (head_dim == 128)
    return launch_with_pdl(paged_attn_simple_kernel<T, 128, 6>, grid, kSimpleWarps * 32, 0, st,
                           pdl, p);
  return launch_with_pdl(paged_attn_simple_kernel<T, 64, 7>, grid, kSimpleWarps * 32, 0, st, pdl,
                         p);
}

cudaError_t launch_paged_chunks(const PagedAttnParams& p, int dtype, int head_dim,
                                cudaStream_t st, bool pdl) {
  if (dtype == kDtypeF32) return launch_simple<float>(p, head_dim, st, pdl);
  if (dtype == kDtypeBf16) return launch_simple<__nv_bfloat16>(p, head_dim, st, pdl);
  return launch_simple<__half>(p, head_dim, st, pdl);
}

}  // namespace gqa
