// Attention of chunks of new tokens over a paged KV cache, 16-bit types, on the
// 5th-generation tensor cores.
//
// S = Q K^T and O = P V over tiles of 128 keys with the running maximum and sum of a
// softmax, causal by position.  4 G d operations a key and token against 4 d bytes a
// key: for chunks of more than a few tokens the tensor cores and the exponential unit
// bound it, not memory.
//
// Rows: the G query heads of a KV head are rows of one tile beside each other (row =
// token * G + head, 21 tokens x 6 or 18 x 7 = 126 of 128 rows), so a chunk reads
// its keys once for all of them and the causal edge is 21 tokens wide.  A unit is
// two such tiles (A and B) over the same keys: the softmax of one runs while the tensor
// cores work on the other.
//
// Work: the key tiles of all units are laid end to end and cut into equal shares, one
// per CTA, as in the decode kernel (gqa_paged_decode.cu); a unit that crosses shares
// leaves its parts in two slots per CTA, merged by a second kernel.  So a short chunk
// over a long cache uses every SM, and the triangle of a whole prompt is balanced.
//
// q is rotated for its position by the kernel before this one, which puts it where the result of the
// same token will be (every unit reads its q before it writes its output, and parts are
// merged after all units), so no workspace grows with the batch.  Rounding it to the type
// there is what the projection before it would do with a rotated q; scores and sums are
// fp32, weights are rounded to the type for the second product.
//
// Warps 0-7 / 8-15: softmax of tile A / B, two threads per row (64 keys each: with one thread a
// row, two warps a scheduler waited for their own instructions, 1800 clocks a tile against 1024
// of the exponential unit); 16: loader of K and V (TMA of the pages); 17: MMA; 18: loader of Q.
// Tensor memory: two buffers of scores (three at head_dim 64) and O_A | O_B; the P of each half of
// the keys goes over the first half of its scores.  With three buffers a tile's next scores are
// ready when its softmax is done with these, and the stream of products runs on from one unit to
// the next (four whole prompts of 1500 to 2500 tokens, f16: 96 -> 88 us; with two buffers, at
// head_dim 128, a tile's scores, softmax and product follow one another, some 4000 clocks for the
// two tiles where the tensor cores need 2048).  (One MMA warp per tile measured slower, 64 against
// 58 us for 512 tokens over 8192 rows: the products of the two interleave and both finish late.)
// Measured: 512 tokens over 8192 rows in bf16 (25 GFLOP) 41 us, 0.6 PFLOP/s.
// Every wait is bounded; a wait that runs out sets the status bit, and the CTA drains
// what it issued and returns its tensor memory.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <math_constants.h>

#include "gqa_paged_chunk.cuh"

namespace gqa {

namespace {

constexpr int kKeys = 128;
constexpr int kSoftmaxWarps = 16, kLoader = 16, kMma = 17, kQLoader = 18;
constexpr int kThreads = 19 * 32;
constexpr int kRowsTile = kChunkRows;
// Buffers of scores: what tensor memory holds beside the two outputs.
template <int D>
constexpr int kScores = D == 64 ? 3 : 2;
// Stages of K and of V, and units of which Q is held: what shared memory has room for.
template <int D>
constexpr int kStages = D == 64 ? 4 : 2;
template <int D>
constexpr int kUnitsQ = D == 64 ? 2 : 1;

template <int D, int G>
struct alignas(1024) Smem {
  uint16_t q[2 * kUnitsQ<D>][kRowsTile * D];  // [unit][tile A, B]
  uint16_t k[kStages<D>][kKeys * D];
  uint16_t v[kStages<D>][kKeys * D];
  float xch[2][2][2][kRowsTile];  // [turn][tile A, B][half of the keys][row]: maxima, sums
  Piece ring[4];
  int poison[4];         // number of the last piece of this ring place with a non-finite V
  // per key tile: its 16-row parts without a page (the softmax of a tile may still be due when
  // one of the second turn of stages after it is loaded)
  unsigned bad_rows[2 * kStages<D>];
  uint64_t item_full[4], item_empty[4];
  uint64_t q_full[2 * kUnitsQ<D>], q_empty[2 * kUnitsQ<D>];
  uint64_t k_full[kStages<D>], k_empty[kStages<D>], v_full[kStages<D>], v_empty[kStages<D>];
  // [tile][its even, odd steps]: a tile's next scores can be ready before it has looked at these
  // (never those after the next)
  uint64_t s_full[4], o_done[4], o_final[2];
  uint64_t p_full[kScores<D>], drain;  // [buffer of scores]
  long long scan[kThreads / 32];
  WalkStart start;
  Walk<2 * tile_tokens<G>(), kKeys> walk;  // (one thread's; no registers for it)
  uint32_t tmem_base;
  int err;
};

struct ChunkMaps {
  CUtensorMap q, k, v;
};

__device__ __forceinline__ uint64_t desc_k_major(uint32_t addr) { return umma_smem_desc(addr); }

// V as an operand whose rows are keys: [64-column block][key][64], 128-byte swizzle;
// leading offset between the blocks, stride offset between groups of 8 keys.
__device__ __forceinline__ uint64_t desc_mn_major(uint32_t addr) {
  uint64_t d = (uint64_t)((addr >> 4) & 0x3FFFu);
  d |= (uint64_t)((kKeys * 128) >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

template <typename T>
__host__ __device__ constexpr uint32_t idesc(int n, bool b_mn_major) {
  const uint32_t t = sizeof(T) == 2 && __is_same(T, __nv_bfloat16) ? 1u : 0u;
  return (1u << 4) | (t << 7) | (t << 10) | ((uint32_t)b_mn_major << 16) |
         ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}

__device__ __forceinline__ void tma_load4(void* dst, const CUtensorMap* map, int c0, int c1, int c2,
                                          int c3, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(smem_addr(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2),
        "r"(c3), "r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void tma_load3(void* dst, const CUtensorMap* map, int c0, int c1, int c2,
                                          uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(smem_addr(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2),
        "r"(smem_addr(bar)) : "memory");
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (__is_same(T, __nv_bfloat16)) {
    return pack_bf16(a, b);
  } else {
    const __half2 h = __floats2half2_rn(a, b);
    return reinterpret_cast<const uint32_t&>(h);
  }
}

// Weights are taken relative to m, which is held kLift below the row's reference, and the reference
// moves to the row's maximum when the weights of a tile add up to more than kMost.  fp16 ends at 2^-24
// and 2^16: with m at the reference itself, a weight below 2^-25 of it would be lost from the product
// and stay in the sum; lifted by 2^8 what is lost lies below 2^-33, and 128 keys as large as the
// reference still add up to kMost.  (Bounded by their sum, no weight passes 2^15.)  bf16 has fp32's
// range.
template <typename T>
constexpr float kLift = __is_same(T, __half) ? 8.f : 0.f;
template <typename T>
constexpr float kMost = __is_same(T, __half) ? 32768.f : 1024.f;

// Whether key tile kt holds rows past the piece's first token (at pos), which not all its rows see.
__device__ __forceinline__ bool clears_v(int pos, int kt) {
  return (kt + 1) * kKeys > pos + 1;
}

// Scores whose bit is set become -inf.
__device__ __forceinline__ void hide(float (&s)[32], unsigned hidden) {
#pragma unroll
  for (int c = 0; c < 32; ++c)
    if (hidden >> c & 1) s[c] = -CUDART_INF_F;
}

// The largest of 64 scores of this thread's row.  (Not inlined: needed on a piece's first tile
// and when a maximum moves; the loop over the tiles has to fit the instruction cache beside the
// MMA warp's.)
__device__ __noinline__ float max64(uint32_t t_s, unsigned long long hidden) {
  float top = -CUDART_INF_F;
#pragma unroll 1
  for (int c0 = 0; c0 < 64; c0 += 32) {
    float s[32];
    tmem_ld32(t_s + c0, s);
    hide(s, (unsigned)(hidden >> c0));
    float mx0 = s[0], mx1 = s[1];
#pragma unroll
    for (int c = 2; c < 30; c += 4) {
      mx0 = fmax3(mx0, s[c], s[c + 1]);
      mx1 = fmax3(mx1, s[c + 2], s[c + 3]);
    }
    top = fmax3(top, fmax3(mx0, s[30], s[31]), mx1);
  }
  return top;
}

// wait_or_abort with everything but the first look out of line, for the same reason.
__device__ __noinline__ bool wait_long(uint64_t* bar, uint32_t parity, int* err) {
  return wait_or_abort(bar, parity, err);
}
__device__ __forceinline__ bool wait_lean(uint64_t* bar, uint32_t parity, int* err) {
  return mbar_try_wait(bar, parity) || wait_long(bar, parity, err);
}

// A pair of 16-bit values with an infinity or a NaN among them.
template <typename T>
__device__ __forceinline__ bool non_finite2(uint32_t x) {
  const uint32_t e = __is_same(T, __nv_bfloat16) ? 0x7f80u : 0x7c00u;
  return (x & e) == e || ((x >> 16) & e) == e;
}
template <typename T>
__device__ __forceinline__ uint32_t drop_non_finite2(uint32_t x) {
  const uint32_t e = __is_same(T, __nv_bfloat16) ? 0x7f80u : 0x7c00u;
  if ((x & e) == e) x &= 0xffff0000u;
  if (((x >> 16) & e) == e) x &= 0xffffu;
  return x;
}

template <typename T, int D, int G>
__global__ void __launch_bounds__(kThreads, 1)
    paged_chunk_kernel(const __grid_constant__ PagedAttnParams p,
                       const __grid_constant__ PagedPartials part,
                       const __grid_constant__ ChunkMaps maps, const int hnd, const int box_rows) {
  extern __shared__ unsigned char smem_raw[];
  using S = Smem<D, G>;
  S& sm = *reinterpret_cast<S*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                ~static_cast<uintptr_t>(1023));
  constexpr int kTok = tile_tokens<G>();
  constexpr int kBlocks = D / 64;               // 64-column blocks of a row
  constexpr bool kPrefetch = kScores<D> > 2;   // of a tile's next scores before its P is ready
  constexpr int kS = kScores<D>, kSt = kStages<D>, kQ = kUnitsQ<D>;
  constexpr uint32_t kTileBytes = kKeys * D * 2;
  constexpr uint32_t kQBytes = kTok * G * D * 2;
  constexpr uint32_t kIdS = idesc<T>(128, false), kIdO = idesc<T>(D, true);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int* err = &sm.err;

  if (tid == 0) {
    for (int s = 0; s < 4; ++s) {
      mbar_init(&sm.item_full[s], 1);
      mbar_init(&sm.item_empty[s], 2 + kSoftmaxWarps);  // Q's loader, MMA and softmax warps
      mbar_init(&sm.s_full[s], 1);
      mbar_init(&sm.o_done[s], 1);
      sm.poison[s] = -1;
    }
    for (int s = 0; s < 2; ++s) mbar_init(&sm.o_final[s], 1);
    for (int s = 0; s < 2 * kQ; ++s) {
      mbar_init(&sm.q_full[s], 1);
      mbar_init(&sm.q_empty[s], 1);
    }
    for (int s = 0; s < kSt; ++s) {
      mbar_init(&sm.k_full[s], 1);
      mbar_init(&sm.k_empty[s], 1);
      mbar_init(&sm.v_full[s], 1);
      mbar_init(&sm.v_empty[s], 1);
    }
    for (int s = 0; s < kS; ++s) mbar_init(&sm.p_full[s], kSoftmaxWarps / 2);
    mbar_init(&sm.drain, 1);
    sm.err = 0;
    fence_barrier_init();
  }
  if (warp == kMma) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_addr(&sm.tmem_base)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // the two rows of a Q tile that no copy fills
  for (int i = tid; i < 2 * kQ * kBlocks * (kRowsTile - kTok * G) * 64; i += kThreads) {
    const int x = i % 64, r = i / 64 % (kRowsTile - kTok * G), b = i / 64 / (kRowsTile - kTok * G);
    sm.q[b / kBlocks][(b % kBlocks) * kRowsTile * 64 + (kTok * G + r) * 64 + x] = 0;
  }
  fence_proxy_async_smem();
  // The kernel before this one waited for all that came before it; of what it writes this one
  // uses only q: the plan, the pages and the slots can be used before it is done.
  pdl_launch_dependents();
  tc_fence_before();
  {
    Walk<2 * kTok, kKeys> walk;
    walk.begin(p, part, sm.scan, &sm.start, kLoader * 32);
    if (tid == kLoader * 32) sm.walk = walk;
  }
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;

  if (warp == kLoader) {
    // ---- loader ----
    Piece pc{};
    int kv = 0, rd = 0;
    bool ok = true;
    const CUtensorMap *km = &maps.k, *vm = &maps.v;
    for (;; ++rd) {
      const int place = rd & 3;
      if (rd >= 4) ok = wait_or_abort(&sm.item_empty[place], ((rd >> 2) - 1) & 1, err);
      if (!__all_sync(0xffffffffu, ok)) break;
      int more = 0;
      if (lane == 0) {
        more = sm.walk.next(p, part, pc);
        if (!more) pc.n_tok = 0;
        sm.ring[place] = pc;
        mbar_arrive(&sm.item_full[place]);
      }
      __syncwarp();
      more = __shfl_sync(0xffffffffu, more, 0);
      if (!more) break;
      const int seq = __shfl_sync(0xffffffffu, pc.seq, 0);
      const int head = __shfl_sync(0xffffffffu, pc.head, 0);
      const int len = __shfl_sync(0xffffffffu, pc.len, 0);
      const int kt0 = __shfl_sync(0xffffffffu, pc.kt0, 0);
      const int kt1 = __shfl_sync(0xffffffffu, pc.kt1, 0);
      const int boxes = kKeys / box_rows;
      for (int kt = kt0; kt < kt1; ++kt, ++kv) {
        const int st = kv % kSt;
        // the pages of the tile: one per lane
        int row = kt * kKeys + lane * box_rows, page = p.kv.n_pages;  // (no such page: zeros)
        bool bad = false;
        if (lane < boxes && row < len) {
          page = page_of(p.kv, seq, row);
          bad = page < 0;
          if (bad) {
            page = p.kv.n_pages;
            atomicOr(p.status, kStatusBadPage);
          }
        }
        const unsigned bad_boxes = __ballot_sync(0xffffffffu, bad);
        row &= (1 << p.kv.page_shift) - 1;
        const int c1 = hnd ? row : head, c2 = hnd ? head : row;
        const uint32_t reuse = (kv / kSt - 1) & 1;
        if (kv >= kSt) ok = wait_or_abort(&sm.k_empty[st], reuse, err);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) {
          unsigned rows16 = 0;  // 16-row parts without a page
          for (int i = 0; i < 8; ++i)
            if (bad_boxes >> (i * 16 / box_rows) & 1) rows16 |= 1u << i;
          sm.bad_rows[kv % (2 * kSt)] = rows16;
          mbar_arrive_expect_tx(&sm.k_full[st], kTileBytes);
        }
        __syncwarp();
        if (lane < boxes)
#pragma unroll
          for (int b = 0; b < kBlocks; ++b)
            tma_load4(sm.k[st] + b * kKeys * 64 + lane * box_rows * 64, km, b * 64, c1, c2, page,
                      &sm.k_full[st]);
        __syncwarp();
        if (kv >= kSt) ok = wait_or_abort(&sm.v_empty[st], reuse, err);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&sm.v_full[st], kTileBytes);
        __syncwarp();
        if (lane < boxes)
#pragma unroll
          for (int b = 0; b < kBlocks; ++b)
            tma_load4(sm.v[st] + b * kKeys * 64 + lane * box_rows * 64, vm, b * 64, c1, c2, page,
                      &sm.v_full[st]);
        __syncwarp();
      }
      if (!ok) break;
    }
    if (*err && lane == 0) {
      // Let the copies already issued land before the CTA's shared memory is handed on
      // (a phase that was never armed runs into the wait's bound).
      for (int i = max(0, kv - kSt + 1); i <= kv; ++i) {
        mbar_wait_bounded(&sm.k_full[i % kSt], (i / kSt) & 1, kWaitBudget / 16);
        mbar_wait_bounded(&sm.v_full[i % kSt], (i / kSt) & 1, kWaitBudget / 16);
      }
    }
    __syncwarp();
  } else if (warp == kQLoader) {
    // ---- loader of Q (its own warp, so that K and V of the next unit need not wait for it) ----
    int nq[2] = {0, 0};
    bool waited = false, ok = true;
    for (int rd = 0; ok; ++rd) {
      ok = __all_sync(0xffffffffu, wait_or_abort(&sm.item_full[rd & 3], (rd >> 2) & 1, err));
      if (!ok) break;
      const int n_tok = sm.ring[rd & 3].n_tok, head = sm.ring[rd & 3].head;
      const int tok = sm.ring[rd & 3].tok;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.item_empty[rd & 3]);
      if (n_tok == 0) break;
      if (!waited) pdl_wait();
      waited = true;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        if (!ok || (g == 1 && n_tok <= kTok)) break;
        const int at = nq[g] % kQ * 2 + g;
        if (nq[g] >= kQ) ok = wait_or_abort(&sm.q_empty[at], (nq[g] / kQ - 1) & 1, err);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&sm.q_full[at], kQBytes);
#pragma unroll
          for (int b = 0; b < kBlocks; ++b)
            tma_load3(sm.q[at] + b * kRowsTile * 64, &maps.q, b * 64, head * G, tok + g * kTok,
                      &sm.q_full[at]);
        }
        __syncwarp();
        ++nq[g];
      }
    }
    if (!waited) pdl_wait();  // (the grid must not end before the one whose q it stands for)
    if (*err && lane == 0)    // (as above)
      for (int g = 0; g < 2; ++g)
        for (int i = max(0, nq[g] - kQ); i < nq[g]; ++i)
          mbar_wait_bounded(&sm.q_full[i % kQ * 2 + g], (i / kQ) & 1, kWaitBudget / 16);
    __syncwarp();
  } else if (warp == kMma) {
    // ---- MMA issuer (the whole warp, one lane issues) ----
    const auto all_wait = [&](uint64_t* bar, uint32_t parity) {
      return (bool)__all_sync(0xffffffffu, wait_lean(bar, parity, &sm.err));
    };
    // (the elected lane is the same one throughout, so a commit covers all products before it)
    const auto commit = [&](uint64_t* bar) {
      if (elect_one()) umma_commit(bar);
      __syncwarp();
    };
    // Descriptors differ in their low words alone.
    const uint32_t q_low = (uint32_t)desc_k_major(smem_addr(sm.q[0]));
    const uint32_t k_low = (uint32_t)desc_k_major(smem_addr(sm.k[0]));
    const uint32_t v_low = (uint32_t)desc_mn_major(smem_addr(sm.v[0]));
    const uint32_t high = (uint32_t)(desc_k_major(0) >> 32);
    const auto desc = [&](uint32_t low) {
      uint64_t d;
      asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(low), "r"(high));
      return d;
    };
    // Steps are (key tile, A), (key tile, B), the next key tile's and so on, or those of A alone,
    // of one piece after the other.  A turn issues P V of the step kS before it, then S of its
    // own, into the buffer of scores that is free by then.  (One call site for each product: the
    // loops of all roles have to fit the instruction cache together.)
    int s_rd = 0, s_both = 0, s_steps = 0, s_at = 0, s_kv = 0;  // scores: pieces, the open one's
    int p_rd = 0, p_both = 0, p_steps = 0, p_at = 0, p_kv = 0;  // steps, key tiles before it
    int s_buf = 0, p_buf = 0, pending_a = 0, pending_b = 0, nq0 = 0, nq1 = 0;
    uint32_t p_turn = 0;              // parity of P
    uint32_t s_turn = 0, o_turn = 0;  // which of a tile's two barriers is next, a bit for each tile
    bool ok = true, more = true;
    for (;;) {
      if (more && s_at == s_steps) {
        s_kv += s_steps >> s_both;
        s_at = 0;
        ok = all_wait(&sm.item_full[s_rd & 3], (s_rd >> 2) & 1);
        if (!ok) break;
        const Piece& pc = sm.ring[s_rd & 3];
        more = pc.n_tok > 0;
        s_both = pc.n_tok > kTok;
        s_steps = (pc.kt1 - pc.kt0) << s_both;
        ++s_rd;
        ++nq0;
        nq1 += s_both;
      }
      // Scores wait for a buffer, and for the product of their tile's last scores (of those before
      // them where scores are prefetched): the barriers of a tile tell two steps apart.
      const bool full = pending_a + pending_b == kS ||
                        (s_at & s_both ? pending_b : pending_a) == (kPrefetch ? 2 : 1);
      if (full || !more) {
        if (pending_a + pending_b == 0) break;
        if (p_at == p_steps) {
          const Piece& pc = sm.ring[p_rd & 3];
          p_kv += p_steps >> p_both;
          p_at = 0;
          p_both = pc.n_tok > kTok;
          p_steps = (pc.kt1 - pc.kt0) << p_both;
        }
        const int g = p_at & p_both, v_at = p_kv + (p_at >> p_both);
        // (what the loader brings first, while the softmax is still at work)
        if (g == 0) ok = all_wait(&sm.v_full[v_at % kSt], (v_at / kSt) & 1);
        if (ok) ok = all_wait(&sm.p_full[p_buf], p_turn);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t v = v_low + (v_at % kSt) * (kKeys * D * 2 / 16);
          const uint32_t at = tmem + 128 * p_buf;
#pragma unroll
          for (int i = 0; i < kKeys / 16; ++i)
            umma_ts(tmem + 128 * kS + D * g, at + (i & 3) * 8 + (i >> 2) * 64,
                    desc(v + i * 2048 / 16), kIdO, p_at > p_both || i > 0);
          if (kPrefetch) umma_commit(&sm.o_done[2 * g + (o_turn >> g & 1)]);
          if (p_at + p_both + 1 >= p_steps) umma_commit(&sm.o_final[g]);
          if (g == p_both) umma_commit(&sm.v_empty[v_at % kSt]);
        }
        __syncwarp();
        o_turn ^= 1u << g;
        if (++p_buf == kS) {
          p_buf = 0;
          p_turn ^= 1;
        }
        --(g ? pending_b : pending_a);
        if (++p_at == p_steps) {
          if (lane == 0) mbar_arrive(&sm.item_empty[p_rd & 3]);
          ++p_rd;
        }
      }
      // (one product in a turn may not be enough, where a piece of one tile follows one of two)
      if (more && (s_at & s_both ? pending_b : pending_a) < (kPrefetch ? 2 : 1)) {
        const int g = s_at & s_both, k_at = s_kv + (s_at >> s_both);
        const int nq = (g ? nq1 : nq0) - 1, q_at = nq % kQ * 2 + g;
        if (g == 0) ok = all_wait(&sm.k_full[k_at % kSt], (k_at / kSt) & 1);
        if (ok && s_at <= s_both) ok = all_wait(&sm.q_full[q_at], (nq / kQ) & 1);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t q = q_low + q_at * (kRowsTile * D * 2 / 16);
          const uint32_t k = k_low + (k_at % kSt) * (kKeys * D * 2 / 16);
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            const uint32_t off = ((i >> 2) * (kKeys * 128) + (i & 3) * 32) / 16;
            umma_ss(tmem + 128 * s_buf, desc(q + off), desc(k + off), kIdS, i > 0);
          }
          umma_commit(&sm.s_full[2 * g + (s_turn >> g & 1)]);
          if (g == s_both) umma_commit(&sm.k_empty[k_at % kSt]);
          if (s_at + s_both + 1 >= s_steps) umma_commit(&sm.q_empty[q_at]);
        }
        __syncwarp();
        s_turn ^= 1u << g;
        if (++s_buf == kS) s_buf = 0;
        ++s_at;
        ++(g ? pending_b : pending_a);
      }
    }
    commit(&sm.drain);  // no MMA may be running when tensor memory is freed
    mbar_wait_bounded(&sm.drain, 0, kWaitBudget);
    __syncwarp();
  } else {
    // ---- softmax of tile g: row r (token r / G, head r % G), keys 64 half .. 64 half + 63 ----
    const int g = warp >> 3, half = (warp >> 2) & 1, r = (warp & 3) * 32 + lane;
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_o = tmem + lane_off + 128 * kS + D * g + D / 2 * half;  // its half of O
    const float sc = p.scale_log2;
    // The two warps of 32 rows exchange a value per row; the places alternate, so that one
    // meeting a turn is enough.  A warp that gives up arrives once more on its way out: its
    // partner meets it there at most once before its own next wait gives up too.
    const int meeting = 1 + g * 4 + (warp & 3);
    int turn = 0;
    const auto other = [&](float x) {
      float(&box)[2][kRowsTile] = sm.xch[turn++ & 1][g];
      box[half][r] = x;
      named_barrier_sync(meeting, 64);
      return box[half ^ 1][r];
    };
    // (whole 32-byte sectors: with 16-byte stores a row per thread writes each twice)
    const bool wide_out =
        (reinterpret_cast<uintptr_t>(p.out) | (uint64_t)p.out_stride * sizeof(T)) % 32 == 0;
    unsigned step = 0;  // of the MMA's steps, the first of the piece
    unsigned kv = 0;    // key tiles so far
    unsigned turns = 0;  // twice this tile's steps so far, and the parity of its pieces
    bool ok = true;
    for (int rd = 0; ok; ++rd) {
      ok = wait_lean(&sm.item_full[rd & 3], (rd >> 2) & 1, &sm.err);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const Piece& pc = sm.ring[rd & 3];  // (given back behind the piece; few registers for it)
      const int n_tok = pc.n_tok, pos = pc.pos, kt0 = pc.kt0, kt1 = pc.kt1;
      if (n_tok == 0) break;
      const int both = n_tok > kTok;
      unsigned at = step + g;
      step += (unsigned)(kt1 - kt0) << both;
      if (g > both) {  // nothing in tile B
        kv += kt1 - kt0;
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.item_empty[rd & 3]);
        continue;
      }
      const int limit = pos + min(g * kTok + r / G, n_tok - 1);  // last key of this row
      const int first_limit = pos + g * kTok;                       // of the tile's first row
      float m = -CUDART_INF_F, l = 0.f;
      for (int kt = kt0; kt < kt1; ++kt, ++kv) {
        ok = __all_sync(0xffffffffu, wait_lean(&sm.s_full[2 * g + (turns >> 1 & 1)], turns >> 2 & 1,
                                                &sm.err));
        if (!ok) break;
        tc_fence_after();
        const uint32_t t_s = tmem + lane_off + 128 * (at % kS) + 64 * half;
        const int key0 = kt * kKeys;
        const unsigned bad = sm.bad_rows[kv % (2 * kSt)];
        // Keys of this half that the row does not see: those past its own position, and rows
        // without a page.
        const bool edge = key0 + kKeys - 1 > first_limit || bad;
        unsigned long long hidden = 0;
        if (edge) {
          const int seen = limit - key0 - 64 * half + 1;
          hidden = seen >= 64 ? 0ull : ~0ull << max(seen, 0);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (bad >> (4 * half + i) & 1) hidden |= 0xffffull << (16 * i);
        }
        // Weights against the running reference, which is moved to the row's maximum (in a
        // second pass over the scores) only on the piece's first tile, or when the weights of
        // the tile add up to more than kMost in some row; the two halves of a row agree on it by
        // their sums.  No P is stored before that, as it goes over the scores.
        uint32_t pk0[16], pk1[16];
        float alpha = 1.f, sum0, sum1;
        const auto weights = [&](int c0, uint32_t (&pk)[16]) {
          float s[32];
          tmem_ld32(t_s + c0, s);
          if (edge) hide(s, (unsigned)(hidden >> c0));
          const float nm = m == -CUDART_INF_F ? 0.f : -m;
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            float x0, x1;
            ffma2(x0, x1, s[c], s[c + 1], sc, sc, nm, nm);
            const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
            fadd2(sum0, sum1, sum0, sum1, p0, p1);
            pk[c / 2] = pack2<T>(p0, p1);
          }
        };
        bool move = __any_sync(0xffffffffu, m == -CUDART_INF_F);
#pragma unroll 1
        for (int pass = 0; pass < 2; ++pass) {
          if (move) {
            const float top = max64(t_s, hidden);
            const float mn = fmaxf(m, fmaxf(top, other(top)) * sc - kLift<T>);
            alpha = mn == m ? 1.f : fast_exp2(m - mn);
            m = mn;
          }
          sum0 = sum1 = 0.f;
          weights(0, pk0);
          weights(32, pk1);
          if (move) break;
          const float sum = sum0 + sum1;
          move = __any_sync(0xffffffffu, !(sum + other(sum) <= kMost<T>));
          if (!move) break;
        }
        __syncwarp();
        tmem_st16(t_s, pk0);
        tmem_st16(t_s + 16, pk1);
        tmem_wait_st();
        l = l * alpha + (sum0 + sum1);
        if (kt != kt0 && __any_sync(0xffffffffu, alpha != 1.f)) {
          // (the scores may be ahead of the product that still adds to O)
          if (kPrefetch)
            ok = __all_sync(0xffffffffu, wait_lean(&sm.o_done[2 * g + ((turns >> 1) + 1 & 1)],
                                                   (turns >> 1) - 1 >> 1 & 1, &sm.err));
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < D / 64; ++c) {
            float v[32];
            tmem_ld32(t_o + c * 32, v);
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] *= alpha;
            tmem_st32(t_o + c * 32, v);
          }
        }
        // A weight of zero does not cancel an infinity or a NaN.  Rows of V past the
        // unit's last token are cleared; in those of its own tokens, which only some of its
        // rows see, what is not finite is cleared here and added to the rows that do see it
        // at the end.
        if (g == 0 && clears_v(pos, kt)) {
          ok = __all_sync(0xffffffffu, wait_lean(&sm.v_full[kv % kSt], (kv / kSt) & 1, &sm.err));
          if (!ok) break;
          const int own0 = max(pos + 1 - key0, 0);
          const int end = pos + n_tok - key0;
          uint4* v = reinterpret_cast<uint4*>(sm.v[kv % kSt]);
          // (chunks of the rows from own0 on)
          const int rows = kKeys - own0;
          for (int i = half * 128 + r; i < kBlocks * 8 * rows; i += 256) {
            const int row = own0 + i / 8 % rows, at = i / 8 / rows * kKeys * 8 + row * 8 + i % 8;
            if (row >= end) {
              v[at] = make_uint4(0, 0, 0, 0);
            } else {
              uint4 x = v[at];
              if (non_finite2<T>(x.x) || non_finite2<T>(x.y) || non_finite2<T>(x.z) ||
                  non_finite2<T>(x.w)) {
                x.x = drop_non_finite2<T>(x.x);
                x.y = drop_non_finite2<T>(x.y);
                x.z = drop_non_finite2<T>(x.z);
                x.w = drop_non_finite2<T>(x.w);
                v[at] = x;
                *reinterpret_cast<volatile int*>(&sm.poison[rd & 3]) = rd;
              }
            }
          }
          fence_proxy_async_smem();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_full[at % kS]);
        turns += 2;
        at += 1 + both;
      }
      if (!ok) break;
      ok = __all_sync(0xffffffffu, wait_lean(&sm.o_final[g], turns & 1, &sm.err));
      turns ^= 1;
      if (!ok) break;
      tc_fence_after();
      l += other(l);
      const bool poisoned = *reinterpret_cast<volatile int*>(&sm.poison[rd & 3]) == rd;
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
      const int t = g * kTok + r / G;
      const bool whole = pc.slot < 0, mine = r < kTok * G && t < pc.n_tok;
      T* dst = static_cast<T*>(p.out) + (long long)(pc.tok + t) * p.out_stride +
               (long long)(pc.head * G + r % G) * D + D / 2 * half;
      const long long part_at = ((long long)pc.slot * 2 + g) * kRowsTile + r;
      if (!whole && half == 0) part.chunk_ml[part_at] = make_float2(m, l);
      float* part_dst = part.chunk_o + part_at * D + D / 2 * half;
#pragma unroll 1
      for (int c = 0; c < D / 2; c += 32) {
        float o[32];
        tmem_ld32(t_o + c, o);
        if (poisoned) {
          const int k0 = max(pc.pos + 1, pc.kt0 * kKeys);
          for (int key = k0; key <= limit && key < pc.kt1 * kKeys; ++key) {
            const int page = page_of(p.kv, pc.seq, key);
            if (page < 0) continue;
            const T* row = static_cast<const T*>(p.kv.v) + row_offset(p.kv, page, pc.head, key) +
                           D / 2 * half + c;
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const float f = Elem<T>::get(row[e]);
              if (!(fabsf(f) < CUDART_INF_F)) o[e] += f;
            }
          }
        }
        uint32_t x[8];
        if (!whole) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = __float_as_uint(o[e + j]);
            st_global_32(part_dst + c + e, x);
          }
        } else if (mine) {
#pragma unroll
          for (int e = 0; e < 32; e += 16) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = pack2<T>(o[e + 2 * j] * inv, o[e + 2 * j + 1] * inv);
            if (wide_out) {
              st_global_32(dst + c + e, x);
            } else {
              *reinterpret_cast<uint4*>(dst + c + e) = make_uint4(x[0], x[1], x[2], x[3]);
              *reinterpret_cast<uint4*>(dst + c + e + 8) = make_uint4(x[4], x[5], x[6], x[7]);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.item_empty[rd & 3]);
    }
    if (!ok) {
      atomicOr(&sm.err, 1);
      asm volatile("bar.arrive %0, %1;" ::"r"(meeting), "r"(64) : "memory");
    }
  }

  tc_fence_before();
  __syncthreads();
  if (tid == 0 && sm.err) atomicOr(p.status, kStatusWaitTimeout);
  if (warp == kMma) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;"
                 ::"r"(tmem), "r"(512) : "memory");
  }
}

PFN_cuTensorMapEncodeTiled_v12000 map_encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) !=
            cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  }();
  return fn;
}

template <typename T, int D, int G>
cudaError_t launch_one(const PagedAttnParams& p, const PagedPartials& part, int n_sm,
                       cudaStream_t st, int* grid) {
  PFN_cuTensorMapEncodeTiled_v12000 encode = map_encoder();
  if (!encode) return cudaErrorNotSupported;
  ChunkMaps maps;
  const CUtensorMapDataType type = __is_same(T, __nv_bfloat16) ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                               : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const cuuint32_t ones[4] = {1, 1, 1, 1};
  const int page_rows = 1 << p.kv.page_shift;
  const int box_rows = std::min(page_rows, kKeys);
  // the dimension with the smaller stride first
  const int hnd = p.kv.row_stride <= p.kv.head_stride;
  const cuuint64_t dims[4] = {D, (cuuint64_t)(hnd ? page_rows : p.n_kv),
                              (cuuint64_t)(hnd ? p.n_kv : page_rows), (cuuint64_t)p.kv.n_pages};
  const cuuint64_t strides[3] = {
      (cuuint64_t)(hnd ? p.kv.row_stride : p.kv.head_stride) * sizeof(T),
      (cuuint64_t)(hnd ? p.kv.head_stride : p.kv.row_stride) * sizeof(T),
      (cuuint64_t)p.kv.page_stride * sizeof(T)};
  const cuuint32_t box[4] = {64, (cuuint32_t)(hnd ? box_rows : 1), (cuuint32_t)(hnd ? 1 : box_rows),
                             1};
  for (int i = 0; i < 2; ++i)
    if (encode(i ? &maps.v : &maps.k, type, 4, i ? p.kv.v : p.kv.k, dims, strides, box, ones,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return cudaErrorInvalidValue;
  const cuuint64_t qdims[3] = {D, (cuuint64_t)p.n_q, (cuuint64_t)p.plan.n_tokens};
  const cuuint64_t qstrides[2] = {D * sizeof(T), (cuuint64_t)p.out_stride * sizeof(T)};
  const cuuint32_t qbox[3] = {64, G, (cuuint32_t)tile_tokens<G>()};
  if (encode(&maps.q, type, 3, p.out, qdims, qstrides, qbox, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return cudaErrorInvalidValue;

  const long long units =
      ((long long)p.plan.n_tokens / (2 * tile_tokens<G>()) + p.plan.n_seq) * p.n_kv;
  const long long tiles = units * ((p.max_len + kKeys - 1) / kKeys);
  *grid = (int)std::min<long long>({(long long)n_sm, part.n_chunk_ctas, tiles});
  return launch_with_pdl(paged_chunk_kernel<T, D, G>, dim3(*grid), kThreads,
                         sizeof(Smem<D, G>) + 1024, st, true, p, part, maps, hnd, box_rows);
}

template <typename T, int D, int G>
cudaError_t prepare_one() {
  return cudaFuncSetAttribute((const void*)paged_chunk_kernel<T, D, G>,
                              cudaFuncAttributeMaxDynamicSharedMemorySize,
                              (int)sizeof(Smem<D, G>) + 1024);
}

}  // namespace

cudaError_t prepare_paged_chunk16() {
  cudaError_t e = prepare_one<__nv_bfloat16, 128, 6>();
  if (e == cudaSuccess) e = prepare_one<__nv_bfloat16, 64, 7>();
  if (e == cudaSuccess) e = prepare_one<__half, 128, 6>();
  if (e == cudaSuccess) e = prepare_one<__half, 64, 7>();
  return e;
}

cudaError_t launch_paged_chunk16(const PagedAttnParams& p, const PagedPartials& part, int dtype,
                                 int head_dim, int n_sm, cudaStream_t st, int* grid) {
  const bool wide = head_dim == 128;
  if (dtype == kDtypeBf16)
    return wide ? launch_one<__nv_bfloat16, 128, 6>(p, part, n_sm, st, grid)
                : launch_one<__nv_bfloat16, 64, 7>(p, part, n_sm, st, grid);
  return wide ? launch_one<__half, 128, 6>(p, part, n_sm, st, grid)
              : launch_one<__half, 64, 7>(p, part, n_sm, st, grid);
}

}  // namespace gqa
