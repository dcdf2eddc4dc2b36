// Shared parts of the chunk kernels of the paged attention (gqa_paged_chunk.cu in 16 bits,
// gqa_paged_chunk32.cu in fp32): units and pieces of the work, q rotated into the rows of the
// output, and the matrix instruction.
#pragma once

#include <math_constants.h>

#include "gqa_paged.cuh"
#include "gqa_paged_launch.cuh"
#include "gqa_tc.cuh"

namespace gqa {

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

// q of the chunks' tokens rotated into the rows of out: an item is (token, KV head, 16-byte chunk
// of the first half of a row), all heads of the group; the whole grid takes part.
template <typename T, int D, int G>
__device__ void rotate_q(const PagedAttnParams& p) {
  using V = Vec16<T>;
  constexpr int kChunks = D / 2 / V::n;
  const int per_token = p.n_kv * kChunks;
  const long long items = (long long)p.plan.n_tokens * per_token;
  const long long step = (long long)gridDim.x * blockDim.x;
  for (long long i0 = (long long)blockIdx.x * blockDim.x + threadIdx.x / 32 * 32; i0 < items;
       i0 += step) {
    const long long item = i0 + threadIdx.x % 32;
    const int tok = (int)(min(item, items - 1) / per_token);
    // the warp looks up its first token; its others are in that or a later sequence
    int s = find_sequence(p.plan.q_starts, p.plan.n_seq, __shfl_sync(0xffffffffu, tok, 0));
    while (s + 1 < p.plan.n_seq && p.plan.q_starts[s + 1] <= tok) ++s;
    int first, n_new, len;
    if (item >= items || !chunk_of(p, s, first, n_new, len) || tok < first || tok >= first + n_new)
      continue;  // (a single token, or a sequence that is reported elsewhere)
    const int pos = len - n_new + tok - first;
    const int rem = (int)(item - (long long)tok * per_token);
    const int h = rem / kChunks, c = rem % kChunks;
    const T* src = static_cast<const T*>(p.qkv) + (long long)tok * p.qkv_stride +
                   (long long)h * G * D + c * V::n;
    T* dst = static_cast<T*>(p.out) + (long long)tok * p.out_stride + (long long)h * G * D +
             c * V::n;
    // (all loads before the first store: out may be where q is, so no compiler reorders them)
    V lo[G], hi[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      lo[g] = *reinterpret_cast<const V*>(src + g * D);
      hi[g] = *reinterpret_cast<const V*>(src + g * D + D / 2);
    }
    float co[V::n], si[V::n];
#pragma unroll
    for (int e = 0; e < V::n; ++e) rope_cos_sin(pos, p.turns[c * V::n + e], co[e], si[e]);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      V y0, y1;
#pragma unroll
      for (int e = 0; e < V::n; ++e) {
        const float x = Elem<T>::get(lo[g].e[e]), y = Elem<T>::get(hi[g].e[e]);
        y0.e[e] = Elem<T>::put(x * co[e] - y * si[e]);
        y1.e[e] = Elem<T>::put(x * si[e] + y * co[e]);
      }
      *reinterpret_cast<V*>(dst + g * D) = y0;
      *reinterpret_cast<V*>(dst + g * D + D / 2) = y1;
    }
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
    if (warp != walker >> 5) return;  // (all lanes of the walker's warp find the same)
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
    // the unit, 32 at a time
    for (unit = 0;; unit += 32) {
      const int mine = unit_tiles<U, KEYS>(n_new, len, unit + lane);
      long long upto = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += y;
      }
      const unsigned past = __ballot_sync(0xffffffffu, tile < at + upto);
      const int i = past ? __ffs(past) - 1 : 31;
      const long long all = __shfl_sync(0xffffffffu, upto, i);
      tiles = __shfl_sync(0xffffffffu, mine, i);
      if (past) {
        at += all - tiles;
        unit += i;
        break;
      }
      at += all;
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

}  // namespace gqa
