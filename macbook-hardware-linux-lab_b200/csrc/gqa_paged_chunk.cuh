// Shared parts of the chunk kernels of the paged attention (gqa_paged_chunk.cu in 16 bits,
// gqa_paged_chunk32.cu in fp32): units and pieces of the work, q rotated into the rows of the
// output, the merge of parts, and the matrix instruction.
#pragma once

#include <math_constants.h>

#include "gqa_paged.cuh"
#include "gqa_paged_launch.cuh"
#include "gqa_tc.cuh"

namespace gqa {

constexpr int kChunkRows = 128;  // rows of a tile: token * G + head

template <int G>
__host__ __device__ constexpr int tile_tokens() { return kChunkRows / G; }
// One piece of a CTA's share: key tiles [kt0, kt1) of a unit.
struct Piece {
  int seq, head;
  int tok, n_tok;  // the unit's first token row and its tokens
  int pos;         // position of the first
  int len;         // rows of the sequence
  int kt0, kt1;
  int slot;        // -1: the unit is whole here
};

__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(id), "r"((uint32_t)acc));
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d), "r"(a), "l"(b), "r"(id), "r"((uint32_t)acc));
}

// The new tokens of sequence s and its rows, when this kernel takes them (two or more).
__device__ __forceinline__ bool chunk_of(const PagedAttnParams& p, int s, int& tok, int& n_new,
                                         int& len) {
  tok = p.plan.q_starts[s];
  const long long n = p.plan.q_starts[s + 1] - (long long)tok;
  if (n < 2 || n > p.max_new || tok < 0 || tok + n > p.plan.n_tokens) return false;
  int pos;
  return place_token(p.plan, p.kv, s, tok, pos, n_new, len) == kPlaced && len <= p.max_len;
}

// Key tiles (of KEYS) of a unit (of U tokens) of the chunk, and of all its units.
template <int U, int KEYS>
__device__ __forceinline__ int unit_tiles(int n_new, int len, int unit) {
  return (len - n_new + min(n_new, (unit + 1) * U) + KEYS - 1) / KEYS;
}
template <int U, int KEYS>
__device__ __forceinline__ long long chunk_tiles(int n_new, int len) {
  long long sum = (len + KEYS - 1) / KEYS;  // the last unit
  unsigned x = len - n_new + U + KEYS - 1;
  const unsigned end = len + KEYS - 1;
#pragma unroll 4
  for (; x < end; x += U) sum += x / KEYS;
  return sum;
}

// q rotated into the rows of out: one thread per (token, KV head, 16-byte chunk of the
// first half of a row), all heads of the group.
template <typename T, int D, int G>
__global__ void __launch_bounds__(256) rotate_q_kernel(const PagedAttnParams p) {
  using V = Vec16<T>;
  constexpr int kChunks = D / 2 / V::n;
  pdl_wait();
  // (after the wait: what runs early beside this kernel may read all but its output)
  pdl_launch_dependents();
  const int per_token = p.n_kv * kChunks;
  const long long item = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long last = (long long)p.plan.n_tokens * per_token - 1;
  const int tok = (int)(min(item, last) / per_token);
  const int tok0 = __shfl_sync(0xffffffffu, tok, 0);
  int s = find_sequence(p.plan.q_starts, p.plan.n_seq, tok0);
  while (s + 1 < p.plan.n_seq && p.plan.q_starts[s + 1] <= tok) ++s;
  if (item > last) return;
  int first, n_new, len;
  if (!chunk_of(p, s, first, n_new, len) || tok < first || tok >= first + n_new) {
    return;  // (another kernel's sequence, or one that is reported there)
  }
  const int pos = len - n_new + tok - first;
  const int rem = (int)(item - (long long)tok * per_token);
  const int h = rem / kChunks, c = rem % kChunks;
  float co[V::n], si[V::n];
#pragma unroll
  for (int e = 0; e < V::n; ++e) rope_cos_sin(pos, p.turns[c * V::n + e], co[e], si[e]);
  const T* src = static_cast<const T*>(p.qkv) + (long long)tok * p.qkv_stride +
                 (long long)h * G * D + c * V::n;
  T* dst = static_cast<T*>(p.out) + (long long)tok * p.out_stride + (long long)h * G * D +
           c * V::n;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const V a = *reinterpret_cast<const V*>(src + g * D);
    const V b = *reinterpret_cast<const V*>(src + g * D + D / 2);
    V y0, y1;
#pragma unroll
    for (int e = 0; e < V::n; ++e) {
      const float x = Elem<T>::get(a.e[e]), y = Elem<T>::get(b.e[e]);
      y0.e[e] = Elem<T>::put(x * co[e] - y * si[e]);
      y1.e[e] = Elem<T>::put(x * si[e] + y * co[e]);
    }
    *reinterpret_cast<V*>(dst + g * D) = y0;
    *reinterpret_cast<V*>(dst + g * D + D / 2) = y1;
  }
}

// The pieces of a CTA's share, in order.
template <int U, int KEYS>
struct Walk {
  long long tile, first, last, total, n;
  int seq;
  // the sequence (n_new 0: still to be read) and the unit that holds `tile`
  int tok, n_new, len;
  int head, unit, tiles;
  long long at;  // first tile of the unit

  // This CTA's share of the tiles of all units and the unit of its first tile, by the whole
  // block.  found: two words of shared memory, scan: one per warp.
  __device__ void begin(const PagedAttnParams& p, const PagedPartials& part, long long* scan,
                        long long* found) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n_threads = blockDim.x;
    if (tid == 0) {
      part.chunk_jobs[blockIdx.x].n_parts = 0;
      found[0] = p.plan.n_seq;
    }
    const auto tiles_of = [&](int s) -> long long {
      int a, b, c;
      if (s >= p.plan.n_seq) return 0;
      return chunk_of(p, s, a, b, c) ? chunk_tiles<U, KEYS>(b, c) * p.n_kv : 0;
    };
    long long mine = 0;
    for (int s = tid; s < p.plan.n_seq; s += n_threads) {
      const long long x = tiles_of(s);
      mine += x;
      if (x == 0 && blockIdx.x == 0 &&
          p.plan.q_starts[s + 1] - (long long)p.plan.q_starts[s] > 1)
        atomicOr(p.status, kStatusBadLength);
    }
    const long long own = mine;
#pragma unroll
    for (int d = 16; d; d >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, d);
    if (lane == 0) scan[warp] = mine;
    __syncthreads();
    total = 0;
    for (int w = 0; w < n_threads / 32; ++w) total += scan[w];
    n = min((long long)gridDim.x, total);
    first = last = 0;
    if (blockIdx.x < n) {
      first = blockIdx.x * total / n;
      last = (blockIdx.x + 1) * total / n;
    }
    // the sequence of the first tile
    long long before = 0;
    for (int s0 = 0; s0 < p.plan.n_seq && first < last; s0 += n_threads) {
      const long long x = p.plan.n_seq <= n_threads ? own : tiles_of(s0 + tid);
      long long incl = x;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += y;
      }
      __syncthreads();
      if (lane == 31) scan[warp] = incl;
      __syncthreads();
      long long sum = 0;
      for (int w = 0; w < n_threads / 32; ++w) {
        if (w == warp) incl += before + sum;
        sum += scan[w];
      }
      if (incl - x <= first && first < incl) {
        found[0] = s0 + tid;
        found[1] = incl - x;
      }
      before += sum;
      if (first < before) break;
    }
    __syncthreads();
    tile = first;
    seq = (int)found[0];
    at = found[1];
    n_new = 0;
    if (seq < p.plan.n_seq && first < last && chunk_of(p, seq, tok, n_new, len)) {
      const long long per_head = chunk_tiles<U, KEYS>(n_new, len);
      head = (int)((tile - at) / per_head);
      at += head * per_head;
      unit = 0;
      tiles = unit_tiles<U, KEYS>(n_new, len, 0);
      while (tile >= at + tiles) {
        at += tiles;
        tiles = unit_tiles<U, KEYS>(n_new, len, ++unit);
      }
    }
  }

  // The next piece; false when the share is done.
  __device__ bool next(const PagedAttnParams& p, const PagedPartials& part, Piece& out) {
    if (tile >= last) return false;
    while (n_new == 0) {
      if (seq >= p.plan.n_seq) return false;
      if (!chunk_of(p, seq, tok, n_new, len)) {
        n_new = 0;
        ++seq;
        continue;
      }
      head = unit = 0;
      tiles = unit_tiles<U, KEYS>(n_new, len, 0);
    }
    out.seq = seq;
    out.head = head;
    out.tok = tok + unit * U;
    out.n_tok = min(U, n_new - unit * U);
    out.pos = len - n_new + unit * U;
    out.len = len;
    out.kt0 = (int)(tile - at);
    out.kt1 = (int)min((long long)tiles, last - at);
    const bool whole = out.kt0 == 0 && out.kt1 == tiles;
    out.slot = whole ? -1 : 2 * (int)blockIdx.x + (tile == first ? 0 : 1);
    if (!whole && out.kt0 == 0) {
      const int last_cta = (int)(((at + tiles) * n + total - 1) / total) - 1;
      part.chunk_jobs[blockIdx.x] = PagedChunkJob{out.tok, out.n_tok, head, out.slot,
                                                  last_cta - (int)blockIdx.x + 1};
    }
    tile = at + out.kt1;
    if (out.kt1 == tiles) {  // on to the next unit, head or sequence
      at += tiles;
      ++unit;
      if (unit * U >= n_new) {
        unit = 0;
        if (++head == p.n_kv) {
          n_new = 0;
          ++seq;
        }
      }
      if (n_new) tiles = unit_tiles<U, KEYS>(n_new, len, unit);
    }
    return true;
  }
};

// Merges the parts of units that crossed shares: a warp per row, blocks of 8 rows.
template <typename T, int D, int G>
__global__ void __launch_bounds__(256) paged_chunk_merge_kernel(const PagedAttnParams p,
                                                                const PagedPartials part) {
  pdl_wait();
  const PagedChunkJob job = part.chunk_jobs[blockIdx.x];
  if (job.n_parts == 0) return;
  constexpr int kTok = tile_tokens<G>(), E = D / 32;
  const int lane = threadIdx.x & 31;
  const int idx = blockIdx.y * 8 + (threadIdx.x >> 5);  // row of the unit's tokens
  const int t = idx / G, g = idx % G;
  if (t >= job.n_tok) return;
  const int row = t < kTok ? idx : kChunkRows + (t - kTok) * G + g;
  const auto at = [&](int i) {
    return (long long)(i == 0 ? job.slot : 2 * ((int)blockIdx.x + i)) * kChunkSlotRows + row;
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

}  // namespace gqa
