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

// A share's start: the sequence of its first tile.
struct WalkStart {
  int seq, tok, n_new, len;
  long long before, per_head;  // tiles of the sequences before it, and of one of its heads
};

// Equal shares of `total` tiles over n CTAs (the first few one larger), in 32 bits where that
// is enough: a 64-bit division takes some 500 clocks of every CTA's start.
struct Shares {
  long long total;
  int n;
  long long each, rest;
  __device__ static long long divide(long long a, long long b) {
    return (a | b) >> 32 ? a / b : (long long)((unsigned)a / (unsigned)b);
  }
  __device__ void set(long long tiles, int grid) {
    total = tiles;
    n = (int)min((long long)grid, tiles);
    each = n ? divide(tiles, n) : 0;
    rest = tiles - each * n;
  }
  __device__ long long first(int cta) const { return cta * each + min((long long)cta, rest); }
  __device__ int cta_of(long long tile) const {
    const long long big = rest * (each + 1);
    return (int)(tile < big ? divide(tile, each + 1) : rest + divide(tile - big, each));
  }
};

// The pieces of a CTA's share, in order.
template <int U, int KEYS>
struct Walk {
  Shares shares;
  long long tile, first, last;
  int seq;
  // the sequence (n_new 0: still to be read) and the unit that holds `tile`
  int tok, n_new, len;
  int head, unit, tiles;
  long long at;  // first tile of the unit

  // This CTA's share of the tiles of all units and the sequence of its first tile, by the
  // whole block (scan: a word of shared memory per warp); `walker` then looks up the unit.
  __device__ void begin(const PagedAttnParams& p, const PagedPartials& part, long long* scan,
                        WalkStart* start, int walker) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n_threads = blockDim.x;
    const int n_warps = n_threads / 32;
    if (tid == 0) {
      part.chunk_jobs[blockIdx.x].n_parts = 0;
      start->n_new = 0;
    }
    // (one round for up to a block of sequences: their numbers stay in registers)
    WalkStart mine{};
    const auto read = [&](int s) {
      mine.seq = s;
      mine.per_head = 0;
      if (s < p.plan.n_seq && chunk_of(p, s, mine.tok, mine.n_new, mine.len))
        mine.per_head = chunk_tiles<U, KEYS>(mine.n_new, mine.len);
      else if (s < p.plan.n_seq && blockIdx.x == 0 &&
               p.plan.q_starts[s + 1] - (long long)p.plan.q_starts[s] > 1)
        atomicOr(p.status, kStatusBadLength);
    };
    // sum of x over the block and, in `incl`, over the threads up to this one
    const auto scan_block = [&](long long x, long long& incl) {
      incl = x;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += y;
      }
      if (lane == 31) scan[warp] = incl;
      __syncthreads();
      long long w = lane < n_warps ? scan[lane] : 0, upto = w;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += y;
      }
      incl += __shfl_sync(0xffffffffu, upto - w, warp);
      return __shfl_sync(0xffffffffu, upto, 31);
    };
    long long incl, sum = 0;
    if (p.plan.n_seq <= n_threads) {
      read(tid);
      sum = scan_block(mine.per_head * p.n_kv, incl);
    } else {
      for (int s0 = 0; s0 < p.plan.n_seq; s0 += n_threads) {
        read(s0 + tid);
        sum += scan_block(mine.per_head * p.n_kv, incl);
        __syncthreads();
      }
    }
    shares.set(sum, gridDim.x);
    first = last = 0;
    if (blockIdx.x < shares.n) {
      first = shares.first(blockIdx.x);
      last = shares.first(blockIdx.x + 1);
    }
    const auto offer = [&](long long upto) {
      const long long x = mine.per_head * p.n_kv;
      if (upto - x <= first && first < upto && first < last) {
        mine.before = upto - x;
        *start = mine;
      }
    };
    if (p.plan.n_seq <= n_threads) {
      offer(incl);
    } else {
      long long before = 0;
      for (int s0 = 0; s0 < p.plan.n_seq && before <= first; s0 += n_threads) {
        read(s0 + tid);
        __syncthreads();
        const long long all = scan_block(mine.per_head * p.n_kv, incl);
        offer(before + incl);
        before += all;
      }
    }
    __syncthreads();
    if (tid != walker) return;
    tile = first;
    seq = start->seq;
    tok = start->tok;
    n_new = start->n_new;
    len = start->len;
    at = start->before;
    if (n_new == 0 || first >= last) {
      last = first;
      return;
    }
    head = (int)Shares::divide(tile - at, start->per_head);
    at += head * start->per_head;
    unit = 0;
    tiles = unit_tiles<U, KEYS>(n_new, len, 0);
    while (tile >= at + tiles) {
      at += tiles;
      tiles = unit_tiles<U, KEYS>(n_new, len, ++unit);
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
      const int last_cta = shares.cta_of(at + tiles - 1);
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
