// Attention of chunks of new tokens over a paged KV cache in fp32, on the
// 5th-generation tensor cores.
//
// Each fp32 number enters as three bf16 terms (x = h + m + l, 8 significant bits each,
// exactly), and a product of two as the six products of terms that matter (hh, hm, mh, mm,
// hl, lh).  Terms are cut off, not rounded, so they have the number's sign and what is left out
// makes a product smaller: by less than 2^-21 of it, 2^-24.5 on average.  Six bf16 matrix
// products in place of one, 279 TFLOP/s at the measured bf16 rate against some 70 of the fp32
// units.  bf16 terms rather than fp16 ones (which would do with three products) because they
// have fp32's range: no scales, and columns of V of very different size keep their digits.  The
// products of small terms are added first.  Sums of many tiles are kept in registers: the tensor cores
// add within a tile only (24 steps of 16 keys), so that how they round an addition cannot
// build up over a long cache.
//
// Rows, units and shares are as in gqa_paged_chunk.cu, with one tile of 126 rows per unit and
// 64 keys per tile (three terms of Q, K and V fill the shared memory).
//
// Warps 0-3: softmax (a row per thread, its output in registers); 4-11: read Q, K and V from
// the pages, split them and write the operands (with four warps that took twice the MMA's time);
// 12: MMA (13-15 only give their registers).  K and V have one place each: the
// next tile is read into registers while this one is worked on.  Tensor memory: two S, two P
// of three terms, one O of a single tile.
//
// Measured: 96 to 256 tokens over 500 to 2000 rows (3.8 GFLOP, six times that in bf16) 46 us; the
// softmax warps' chain of a tile bounds it, not the tensor cores (22 % busy).
#include "gqa_paged_chunk.cuh"

namespace gqa {

namespace {

constexpr int kKeys = 64;
constexpr int kOperandWarps = 8, kFirstOperand = 4, kMma = 12;
constexpr int kThreads = 512;
// Registers of a thread in each group of four warps; four groups of 128 at the launch.
constexpr int kRegsSoftmax = 232, kRegsOperands = 104, kRegsMma = 72;
static_assert(kRegsSoftmax + 2 * kRegsOperands + kRegsMma == 4 * 128, "the launch's registers");
constexpr int kRowsWarp = kKeys / kOperandWarps;  // rows of K and V of an operand warp
constexpr int kTerms = 3;
constexpr uint32_t kColS = 0, kColP = 128, kColO = 320;  // S: 2 x 64, P: 2 x 96, O: D

template <int D, int G>
struct alignas(1024) Smem {
  uint16_t q[kTerms][kChunkRows * D];
  uint16_t k[kTerms][kKeys * D];
  uint16_t v[kTerms][kKeys * D];
  uint8_t stage[4][4096];
  Piece ring[4];
  int poison[4];      // number of the last piece of this ring place with a non-finite V
  uint8_t bad[4][4];  // per key tile: its 16-row parts without a page
  uint64_t item_full[4], item_empty[4];
  uint64_t q_full, q_empty, k_full, k_empty, v_full, v_empty;
  // (P of the next tile can be ready before the MMA warp looks for this one's, which waits for V
  // first: a barrier for each of the two places)
  uint64_t s_full[2], p_full[2], o_full, o_empty, drain;
  long long scan[kThreads / 32];
  WalkStart start;
  Walk<tile_tokens<G>(), kKeys> walk;  // (one thread's; no registers for it)
  uint32_t tmem_base;
  int err;
};

// Rows of 128 bytes in 64-column blocks, 128-byte swizzle; `rows` rows a block.  lead: bytes
// between blocks (for operands read across their rows).
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead) {
  uint64_t d = (uint64_t)((addr >> 4) & 0x3FFFu);
  d |= (uint64_t)(lead >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

__host__ __device__ constexpr uint32_t idesc(int n, bool b_mn_major) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)b_mn_major << 16) |
         ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}

// x and y as three bf16 pairs: the upper halves of the number, of what is left and of what is
// left of that.  Cut off rather than rounded, each takes eight bits or more, so the three hold
// all 24 exactly; no conversion instruction is needed.
__device__ __forceinline__ void split3(float x, float y, uint32_t (&t)[kTerms]) {
#pragma unroll
  for (int i = 0; i < kTerms; ++i) {
    t[i] = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
    if (i + 1 < kTerms) {
      const float hx = __uint_as_float(__float_as_uint(x) & 0xffff0000u);
      const float hy = __uint_as_float(__float_as_uint(y) & 0xffff0000u);
      ffma2(x, y, hx, hy, -1.f, -1.f, x, y);
    }
  }
}

// Four floats of column c (a multiple of 4) of row r as three terms, at their place in an
// operand of `rows` rows.
template <int N>
__device__ __forceinline__ void put4(uint16_t (*term)[N], int rows, int r, int c, float4 x) {
  uint32_t a[kTerms], b[kTerms];
  split3(x.x, x.y, a);
  split3(x.z, x.w, b);
  const int at = (c >> 6) * rows * 64 + r * 64 + ((((c & 63) >> 3) ^ (r & 7)) << 3) + (c & 7);
#pragma unroll
  for (int i = 0; i < kTerms; ++i)
    *reinterpret_cast<uint2*>(term[i] + at) = make_uint2(a[i], b[i]);
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) < CUDART_INF_F; }

// Adds the infinities and NaN in V of the piece's keys up to `limit` to a row of output.
template <int D>
__device__ __noinline__ void add_non_finite(const PagedAttnParams& p, const Piece& pc, int limit,
                                            float* row) {
  for (int key = pc.kt0 * kKeys; key <= limit && key < pc.kt1 * kKeys; ++key) {
    const int page = page_of(p.kv, pc.seq, key);
    if (page < 0) continue;
    const float* v = static_cast<const float*>(p.kv.v) + row_offset(p.kv, page, pc.head, key);
    for (int e = 0; e < D; ++e)
      if (!finite(v[e])) row[e] += v[e];
  }
}

template <int D, int G>
__global__ void __launch_bounds__(kThreads, 1)
    paged_chunk32_kernel(const __grid_constant__ PagedAttnParams p,
                         const __grid_constant__ PagedPartials part) {
  extern __shared__ unsigned char smem_raw[];
  using S = Smem<D, G>;
  S& sm = *reinterpret_cast<S*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                ~static_cast<uintptr_t>(1023));
  constexpr int kTok = tile_tokens<G>();
  constexpr uint32_t kIdS = idesc(kKeys, false), kIdO = idesc(D, true);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int* err = &sm.err;

  if (tid == 0) {
    for (int s = 0; s < 4; ++s) {
      mbar_init(&sm.item_full[s], 1);
      mbar_init(&sm.item_empty[s], 5 + kOperandWarps);  // MMA thread, softmax, operand warps
      sm.poison[s] = -1;
    }
    mbar_init(&sm.q_full, kOperandWarps);
    mbar_init(&sm.k_full, kOperandWarps);
    mbar_init(&sm.v_full, kOperandWarps);
    mbar_init(&sm.p_full[0], 4);
    mbar_init(&sm.p_full[1], 4);
    mbar_init(&sm.o_empty, 4);
    mbar_init(&sm.q_empty, 1);
    mbar_init(&sm.k_empty, 1);
    mbar_init(&sm.v_empty, 1);
    mbar_init(&sm.s_full[0], 1);
    mbar_init(&sm.s_full[1], 1);
    mbar_init(&sm.o_full, 1);
    mbar_init(&sm.drain, 1);
    sm.err = 0;
    fence_barrier_init();
  }
  if (warp == kMma) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_addr(&sm.tmem_base)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // The kernel before this one waited for all that came before it; of what it writes this one
  // uses only q: the plan, the pages and the slots can be used before it is done.
  pdl_launch_dependents();
  tc_fence_before();
  {
    Walk<kTok, kKeys> walk;
    walk.begin(p, part, sm.scan, &sm.start, 128);
    if (tid == 128) sm.walk = walk;  // (the thread that walks)
  }
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;

  // A piece of the ring; false when another role gave up.
  const auto take = [&](int n, Piece& pc) {
    if (!wait_or_abort(&sm.item_full[n & 3], (n >> 2) & 1, err)) return false;
    pc = sm.ring[n & 3];
    return true;
  };

  if (warp >= kFirstOperand && warp < kMma) {
    // ---- operands ----
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOperands));
    const int w = warp - kFirstOperand;
    constexpr int kLanes = D / 4;          // lanes that cover a row
    constexpr int kSide = 32 / kLanes;     // rows side by side in a load
    constexpr int kLoads = kRowsWarp / kSide;  // loads of a warp's rows
    const int sub = lane / kLanes, col = lane % kLanes * 4;
    int t = 0;
    bool ok = true, waited = false;
    for (int rd = 0; ok; ++rd) {
      const int place = rd & 3;
      if (w == 0) {  // this warp hands the pieces out
        if (rd >= 4) ok = wait_or_abort(&sm.item_empty[place], ((rd >> 2) - 1) & 1, err);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) {
          if (!sm.walk.next(p, part, sm.ring[place])) sm.ring[place].n_tok = 0;
          mbar_arrive(&sm.item_full[place]);
        }
        __syncwarp();
      }
      Piece pc;
      ok = __all_sync(0xffffffffu, take(rd, pc));
      if (!ok) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.item_empty[place]);
      if (pc.n_tok == 0) break;

      // The warp's rows of a key tile: their page (-1: a bad one; n_pages: past the unit), and
      // K or V of them into registers.
      const auto page_at = [&](int kt) {
        const int row = kt * kKeys + w * kRowsWarp;
        if (kt >= pc.kt1 || row >= pc.pos + pc.n_tok) return p.kv.n_pages;
        const int page = page_of(p.kv, pc.seq, row);
        if (page < 0 && lane == 0) atomicOr(p.status, kStatusBadPage);
        return page;
      };
      const auto load = [&](const void* pool, int kt, int page, float4 (&x)[kLoads]) {
        const int row0 = kt * kKeys + w * kRowsWarp;
        const bool there = page >= 0 && page < p.kv.n_pages;
        const float* src = static_cast<const float*>(pool) +
                           (there ? row_offset(p.kv, page, pc.head, row0) : 0);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          const int r = i * kSide + sub;
          x[i] = there && row0 + r < pc.pos + pc.n_tok
                     ? __ldg(reinterpret_cast<const float4*>(src + r * p.kv.row_stride + col))
                     : make_float4(0.f, 0.f, 0.f, 0.f);
        }
      };
      const auto put_k = [&](int n, int page, const float4 (&x)[kLoads]) {
        if (n > 0 && !__all_sync(0xffffffffu, wait_or_abort(&sm.k_empty, (n - 1) & 1, err)))
          return false;
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
          put4(sm.k, kKeys, w * kRowsWarp + i * kSide + sub, col, x[i]);
        // (two warps share a 16-row part; the first half's knows its page wherever a row of the
        // part is in use, the second half's does not where the unit ends before its rows)
        static_assert(kRowsWarp == 8, "two operand warps to a 16-row part");
        if (lane == 0 && w % 2 == 0) sm.bad[n & 3][w / 2] = page < 0;
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.k_full);
        return true;
      };
      // K runs one tile ahead of V, as S runs ahead of P V; Q comes between the first K and V.
      float4 xk[kLoads], xv[kLoads];
      int page = page_at(pc.kt0), page_n = page;
      load(p.kv.k, pc.kt0, page, xk);
      load(p.kv.v, pc.kt0, page, xv);
      for (int kt = pc.kt0 - 1; kt < pc.kt1; ++kt) {
        // (here xk holds tile kt + 1 and xv tile kt, or kt + 1 at first)
        if (kt + 1 < pc.kt1) {
          ok = put_k(t + (kt >= pc.kt0), page_n, xk);
          if (!ok) break;
          page = page_n;
          page_n = page_at(kt + 2);
          load(p.kv.k, kt + 2, page_n, xk);
        }
        if (kt < pc.kt0) {
          // Q (rotated, in the rows of out)
          if (!waited) pdl_wait();
          waited = true;
          if (rd > 0) ok = wait_or_abort(&sm.q_empty, (rd - 1) & 1, err);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
#pragma unroll 1
          for (int r0 = w * 16; r0 < w * 16 + 16; r0 += kSide * 4) {
            float4 x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r = r0 + i * kSide + sub, tk = r / G;
              x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
              if (r < kTok * G && tk < pc.n_tok)
                x[i] = *reinterpret_cast<const float4*>(
                    static_cast<const float*>(p.out) + (long long)(pc.tok + tk) * p.out_stride +
                    (long long)(pc.head * G + r % G) * D + col);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) put4(sm.q, kChunkRows, r0 + i * kSide + sub, col, x[i]);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.q_full);
          continue;
        }
        // A weight of zero does not cancel an infinity or a NaN: what is not finite stays out of
        // the product, and is added at the end to the rows that see it.
        bool odd = false;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          const float4 x = xv[i];
          odd |= !(finite(x.x) && finite(x.y) && finite(x.z) && finite(x.w));
        }
        if (odd) {
          *reinterpret_cast<volatile int*>(&sm.poison[place]) = rd;
#pragma unroll
          for (int i = 0; i < kLoads; ++i) {
            float4& x = xv[i];
            x.x = finite(x.x) ? x.x : 0.f;
            x.y = finite(x.y) ? x.y : 0.f;
            x.z = finite(x.z) ? x.z : 0.f;
            x.w = finite(x.w) ? x.w : 0.f;
          }
        }
        if (t > 0) ok = wait_or_abort(&sm.v_empty, (t - 1) & 1, err);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
          put4(sm.v, kKeys, w * kRowsWarp + i * kSide + sub, col, xv[i]);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.v_full);
        load(p.kv.v, kt + 1, kt + 1 < pc.kt1 ? page : p.kv.n_pages, xv);
        ++t;
      }
    }
    if (!waited) pdl_wait();  // (the grid must not end before the one whose q it stands for)
    if (!ok) atomicOr(&sm.err, 1);
  } else if (warp >= kMma) {
    // ---- MMA issuer ----
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsMma));
    if (warp == kMma) {  // (the whole warp, one lane issues)
      const auto all_wait = [&](uint64_t* bar, uint32_t parity) {
        return (bool)__all_sync(0xffffffffu, wait_or_abort(bar, parity, err));
      };
      const auto commit = [&](uint64_t* bar) {
        if (elect_one()) umma_commit(bar);
        __syncwarp();
      };
      // Descriptors differ in their low words alone, by constants.
      const uint32_t q0 = (uint32_t)smem_desc(smem_addr(sm.q[0]), 16);
      const uint32_t k0 = (uint32_t)smem_desc(smem_addr(sm.k[0]), 16);
      const uint32_t v0 = (uint32_t)smem_desc(smem_addr(sm.v[0]), kKeys * 128);
      const uint32_t high = (uint32_t)(smem_desc(0, 0) >> 32);
      const auto desc = [&](uint32_t low) {
        uint64_t d;
        asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(low), "r"(high));
        return d;
      };
      // Pairs of terms, small products first: (2,0) (0,2) (1,1) (1,0) (0,1) (0,0), a digit each.
      // One pair unrolled: the loops of all roles have to fit the instruction cache together.
      constexpr uint32_t kA = 0x001102, kB = 0x010120;
      const auto issue_s = [&](int t) {
        const uint32_t d = tmem + kColS + 64 * (t & 1);
        if (elect_one()) {
#pragma unroll 1
          for (int i = 0; i < 24; i += 4) {
            const uint32_t q = q0 + (kA >> i & 15) * (kChunkRows * D * 2 / 16);
            const uint32_t k = k0 + (kB >> i & 15) * (kKeys * D * 2 / 16);
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks)
              umma_ss(d, desc(q + ((ks >> 2) * kChunkRows * 128 + (ks & 3) * 32) / 16),
                      desc(k + ((ks >> 2) * kKeys * 128 + (ks & 3) * 32) / 16), kIdS, i + ks > 0);
          }
          umma_commit(&sm.s_full[t & 1]);
          umma_commit(&sm.k_empty);
        }
        __syncwarp();
      };
      const auto issue_pv = [&](int t) {
        const uint32_t at = tmem + kColP + 96 * (t & 1);
        if (elect_one()) {
#pragma unroll 1
          for (int i = 0; i < 24; i += 4) {
            const uint32_t w = at + 32 * (kA >> i & 15);
            const uint32_t v = v0 + (kB >> i & 15) * (kKeys * D * 2 / 16);
#pragma unroll
            for (int ks = 0; ks < kKeys / 16; ++ks)
              umma_ts(tmem + kColO, w + ks * 8, desc(v + ks * 2048 / 16), kIdO, i + ks > 0);
          }
          umma_commit(&sm.o_full);
          umma_commit(&sm.v_empty);
        }
        __syncwarp();
      };
      const auto get = [&](int n, Piece& pc) {
        const bool good = __all_sync(0xffffffffu, take(n, pc));
        __syncwarp();
        if (good && lane == 0) mbar_arrive(&sm.item_empty[n & 3]);
        return good;
      };
      Piece pc{};
      int rd = 0, t = 0;  // pieces; tiles whose P V is issued
      bool ok = get(0, pc);
      while (ok && pc.n_tok > 0) {
        const int tiles = pc.kt1 - pc.kt0;
        // S runs one tile ahead of P V (the first of a piece follows the last P V of the one
        // before: its Q may be long in coming).
        for (int j = 0; j <= tiles; ++j) {
          if (j < tiles) {
            ok = (j > 0 || all_wait(&sm.q_full, rd & 1)) && all_wait(&sm.k_full, (t + (j > 0)) & 1);
            if (!ok) break;
            tc_fence_after();
            issue_s(t + (j > 0));
            if (j + 1 == tiles) commit(&sm.q_empty);
          }
          if (j > 0) {
            ok = all_wait(&sm.v_full, t & 1) && (t == 0 || all_wait(&sm.o_empty, (t - 1) & 1)) &&
                 all_wait(&sm.p_full[t & 1], (t >> 1) & 1);
            if (!ok) break;
            tc_fence_after();
            issue_pv(t);
            ++t;
          }
        }
        if (ok) ok = get(++rd, pc);
      }
      commit(&sm.drain);  // no MMA may be running when tensor memory is freed
      mbar_wait_bounded(&sm.drain, 0, kWaitBudget);
    }
    __syncwarp();
  } else {
    // ---- softmax: thread = row r (token r / G, head r % G) ----
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    const int r = tid;
    const uint32_t t_lane = tmem + ((uint32_t)(warp * 32) << 16);
    const float sc = p.scale_log2;
    uint8_t* stage = sm.stage[warp];
    int t = 0;
    bool ok = true;
    for (int rd = 0; ok; ++rd) {
      Piece pc;
      ok = __all_sync(0xffffffffu, take(rd, pc));
      if (!ok) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.item_empty[rd & 3]);
      if (pc.n_tok == 0) break;
      const int limit = pc.pos + min(r / G, pc.n_tok - 1);  // last key of this row
      float m = -CUDART_INF_F, l = 0.f, o[D];
#pragma unroll
      for (int e = 0; e < D; ++e) o[e] = 0.f;
      // Turn j: weights of tile j, then the product of tile j - 1 is added to the row.
      const int tiles = pc.kt1 - pc.kt0;
      for (int j = 0; j <= tiles; ++j) {
        float alpha = 1.f;
        if (j < tiles) {
          ok = __all_sync(0xffffffffu, wait_or_abort(&sm.s_full[t & 1], (t >> 1) & 1, err));
          if (!ok) break;
          tc_fence_after();
          // Keys that the row does not see: past its own position, or without a page.
          const int seen = limit - (pc.kt0 + j) * kKeys + 1;
          unsigned long long hidden = seen >= kKeys ? 0ull : ~0ull << max(seen, 0);
          const uint32_t bad = *reinterpret_cast<const uint32_t*>(sm.bad[t & 3]);
          if (bad) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (bad >> (8 * i) & 1) hidden |= 0xffffull << (16 * i);
          }
          // Sixteen scores at a time, twice: the largest, then the weights.  (A row of scores
          // beside the row of output would not fit the registers, nor all of it unrolled the
          // instruction cache.)
          const uint32_t t_s = t_lane + kColS + 64 * (t & 1), t_p = t_lane + kColP + 96 * (t & 1);
          const auto scores = [&](int c0, float (&s)[16]) {
            tmem_ld16(t_s + c0, s);
            const unsigned h = (unsigned)(hidden >> c0) & 0xffffu;
            if (__any_sync(0xffffffffu, h != 0)) {
#pragma unroll
              for (int c = 0; c < 16; ++c)
                if (h >> c & 1) s[c] = -CUDART_INF_F;
            }
          };
          float top = -CUDART_INF_F;
#pragma unroll 1
          for (int c0 = 0; c0 < kKeys; c0 += 16) {
            float s[16];
            scores(c0, s);
            float mx0 = s[0], mx1 = s[1];
#pragma unroll
            for (int c = 2; c < 14; c += 4) {
              mx0 = fmax3(mx0, s[c], s[c + 1]);
              mx1 = fmax3(mx1, s[c + 2], s[c + 3]);
            }
            top = fmax3(top, fmax3(mx0, s[14], s[15]), mx1);
          }
          const float mn = fmaxf(m, top * sc);
          alpha = mn == m ? 1.f : fast_exp2(m - mn);
          m = mn;
          const float neg = m == -CUDART_INF_F ? 0.f : -m;
          float sum0 = 0.f, sum1 = 0.f;
#pragma unroll 1
          for (int c0 = 0; c0 < kKeys; c0 += 16) {
            float s[16];
            uint32_t pk[kTerms][8];
            scores(c0, s);
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
              float x0, x1;
              ffma2(x0, x1, s[e], s[e + 1], sc, sc, neg, neg);
              const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
              fadd2(sum0, sum1, sum0, sum1, p0, p1);
              uint32_t x[kTerms];
              split3(p0, p1, x);
#pragma unroll
              for (int i = 0; i < kTerms; ++i) pk[i][e / 2] = x[i];
            }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < kTerms; ++i) tmem_st8(t_p + 32 * i + c0 / 2, pk[i]);
          }
          tmem_wait_st();
          l = l * alpha + (sum0 + sum1);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.p_full[t & 1]);
          ++t;
        }
        if (j > 0) {
          const int n = t - 1 - (j < tiles);  // the tile before
          ok = __all_sync(0xffffffffu, wait_or_abort(&sm.o_full, n & 1, err));
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < D; c += 32) {
            float v[32];
            tmem_ld32(t_lane + kColO + c, v);
#pragma unroll
            for (int e = 0; e < 32; e += 2)
              fadd2(o[c + e], o[c + e + 1], o[c + e], o[c + e + 1], v[e], v[e + 1]);
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.o_empty);
          if (__any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll
            for (int e = 0; e < D; e += 2)
              ffma2(o[e], o[e + 1], o[e], o[e + 1], alpha, alpha, 0.f, 0.f);
          }
        }
      }
      if (!ok) break;
      // Rows leave through the warp's 4 KB: written a row per thread, read back so that eight
      // lanes cover 128 bytes of a row (16-byte chunk c of row i at c ^ (i % 8)).
      const bool whole = pc.slot < 0;
      const float by = !whole ? 1.f : l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
      const long long base = (long long)pc.slot * kChunkSlotRows + warp * 32;
      if (!whole) part.chunk_ml[base + lane] = make_float2(m, l);
#pragma unroll
      for (int b = 0; b < D / 32; ++b) {
#pragma unroll
        for (int c = 0; c < 8; ++c)
          *reinterpret_cast<float4*>(stage + lane * 128 + ((c ^ (lane & 7)) << 4)) =
              make_float4(o[b * 32 + 4 * c] * by, o[b * 32 + 4 * c + 1] * by,
                          o[b * 32 + 4 * c + 2] * by, o[b * 32 + 4 * c + 3] * by);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int rr = i * 4 + (lane >> 3), c = lane & 7;
          const float4 x = *reinterpret_cast<const float4*>(stage + rr * 128 +
                                                            ((c ^ (rr & 7)) << 4));
          const int row = warp * 32 + rr, tk = row / G;
          if (!whole)
            *reinterpret_cast<float4*>(part.chunk_o + (base + rr) * D + b * 32 + c * 4) = x;
          else if (row < kTok * G && tk < pc.n_tok)
            *reinterpret_cast<float4*>(static_cast<float*>(p.out) +
                                       (long long)(pc.tok + tk) * p.out_stride +
                                       (long long)(pc.head * G + row % G) * D + b * 32 + c * 4) = x;
        }
        __syncwarp();
      }
      if (*reinterpret_cast<volatile int*>(&sm.poison[rd & 3]) == rd) {
        // what was kept out of the product, to this thread's row where it was written
        const int tk = r / G;
        float* row = whole ? static_cast<float*>(p.out) +
                                 (long long)(pc.tok + tk) * p.out_stride +
                                 (long long)(pc.head * G + r % G) * D
                           : part.chunk_o + (base + lane) * D;
        if (r < kTok * G && tk < pc.n_tok) add_non_finite<D>(p, pc, limit, row);
        __syncwarp();
      }
    }
    if (!ok) atomicOr(&sm.err, 1);
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

template <int D, int G>
cudaError_t launch_one(const PagedAttnParams& p, const PagedPartials& part, int n_sm,
                       cudaStream_t st, int* grid) {
  constexpr int kTok = tile_tokens<G>();
  const long long units = ((long long)p.plan.n_tokens / kTok + p.plan.n_seq) * p.n_kv;
  const long long tiles = units * ((p.max_len + kKeys - 1) / kKeys);
  *grid = (int)std::min<long long>({(long long)n_sm, part.n_chunk_ctas, tiles});
  return launch_with_pdl(paged_chunk32_kernel<D, G>, dim3(*grid), kThreads,
                         sizeof(Smem<D, G>) + 1024, st, true, p, part);
}

template <int D, int G>
constexpr int kSmemBytes = (int)sizeof(Smem<D, G>) + 1024;

}  // namespace

cudaError_t prepare_paged_chunk32() {
  cudaError_t e = cudaFuncSetAttribute((const void*)paged_chunk32_kernel<128, 6>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       kSmemBytes<128, 6>);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute((const void*)paged_chunk32_kernel<64, 7>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes<64, 7>);
  return e;
}

cudaError_t launch_paged_chunk32(const PagedAttnParams& p, const PagedPartials& part, int head_dim,
                                 int n_sm, cudaStream_t st, int* grid) {
  return head_dim == 128 ? launch_one<128, 6>(p, part, n_sm, st, grid)
                         : launch_one<64, 7>(p, part, n_sm, st, grid);
}

}  // namespace gqa
