// Attention of single tokens over a paged KV cache.
//
// out_h = sum_t w_t V_t / sum_t w_t, w_t = 2^(s_t - m), s_t = log2(e) q_h.K_t /
// sqrt(d), over the rows of the token's sequence; the query heads of one KV head
// share every row that is read.  The kernel streams the cache once (2 d elements a
// row and KV head against 4 G d operations), so memory bounds it.
//
// Work: the rows of all (sequence, KV head) pairs, in tiles, are laid end to end
// and cut into equal shares, one per CTA, whatever the lengths; a CTA walks the
// pieces of its share.  A pair within one share is finished there; one that crosses
// shares leaves its parts (m, l, o) in two slots per CTA, which a second kernel
// merges.  So the workspace depends on the grid alone, and a ragged batch keeps
// every SM busy to the end: 64 sequences of 255 to 8191 rows finish within one tile
// of each other.
//
// Inside a CTA each warp has its own groups of rows and its own ring of stages,
// filled by 16-byte asynchronous copies (rows past the end are filled with zeros, so
// that what stands there never meets a weight), its own softmax state, and no
// barrier until the piece is done.
//
// Measured: 64 sequences of 256 to 8192 rows in bf16 (273 MB) 50 us, 5.5 TB/s; one
// token over 32768 rows in fp32 (67 MB) 15 us, over 4096 rows 6.4 us (start and end
// of a CTA, which has one tile then).
//
// In a call with chunks the kernel also rotates their q, for the chunks' kernel after it.
#include <math_constants.h>

#include "gqa_paged_chunk.cuh"
#include "gqa_paged_merge.cuh"

namespace gqa {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kStages = 3;
constexpr int kHeads = 8;  // query heads of a KV head, padded (6 or 7 are in use)

// Rows of a warp's stage: 16 for the 16-bit types (the matrix instruction's rows),
// 8 for fp32 (the same bytes).
template <typename T>
__host__ __device__ constexpr int group_rows() { return sizeof(T) == 4 ? 8 : 16; }
template <typename T>
__host__ __device__ constexpr int tile_rows() { return kWarps * group_rows<T>(); }

template <typename T, int D>
struct Smem {
  static constexpr int kRows = group_rows<T>();
  static constexpr int kQuarter = D / 4 + 4;  // fp32 q: a quarter row, padded off the banks
  alignas(128) T k[kWarps][kStages][kRows * D];
  alignas(128) T v[kWarps][kStages][kRows * D];
  alignas(16) float q[kHeads][4 * kQuarter];
  alignas(16) float p[kWarps][8][kHeads];  // fp32: weights of a group, [row][head]
  float m[kWarps][kHeads], l[kWarps][kHeads];
  long long scan[kWarps];
  int found_seq;
  long long found_before;
};

// Rows of sequence s that this kernel attends (0: none, or not a single token) and
// its token row.
__device__ __forceinline__ int single_rows(const PagedAttnParams& p, int s, int& tok, int* bad) {
  tok = s;
  if (p.plan.q_starts) {
    tok = p.plan.q_starts[s];
    const long long n = p.plan.q_starts[s + 1] - (long long)tok;
    if (n != 1) {
      if (n < 0 || n > p.max_new) *bad |= kStatusBadLength;
      return 0;
    }
    if (tok < 0 || tok >= p.plan.n_tokens) {
      *bad |= kStatusBadLength;
      return 0;
    }
  }
  int pos, n_new, len;
  if (place_token(p.plan, p.kv, s, tok, pos, n_new, len) != kPlaced || len > p.max_len) {
    *bad |= kStatusBadLength;
    return 0;
  }
  return len;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(on ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  if constexpr (sizeof(T) == 2 && __is_same(T, __nv_bfloat16))
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// x0, x1 as a pair of T and the pair of what the rounding left.
template <typename T>
__device__ __forceinline__ void split_pair(float x0, float x1, uint32_t& hi, uint32_t& lo) {
  const T h0 = Elem<T>::put(x0), h1 = Elem<T>::put(x1);
  const T l0 = Elem<T>::put(x0 - Elem<T>::get(h0)), l1 = Elem<T>::put(x1 - Elem<T>::get(h1));
  hi = (uint32_t)reinterpret_cast<const uint16_t&>(h0) |
       (uint32_t)reinterpret_cast<const uint16_t&>(h1) << 16;
  lo = (uint32_t)reinterpret_cast<const uint16_t&>(l0) |
       (uint32_t)reinterpret_cast<const uint16_t&>(l1) << 16;
}

// The running reference of a softmax moves only when a score passes it by more than
// this (weights then stay below 2^8 of it), which saves the reduction and the rescale in almost
// every group.
constexpr float kSlack = 8.f;

// m is held kLift below the reference.  fp16 ends at 2^-24 and 2^16: with m at the reference itself, a
// weight below 2^-25 of it would be lost from the product and stay in the sum l; lifted by 2^7 (the
// largest weight is then 2^15), what is lost lies below 2^-32.  bf16 has fp32's range.
template <typename T>
constexpr float kLift = __is_same(T, __half) ? 7.f : 0.f;

// One warp's softmax state over the groups it has seen, for the 16-bit types: scores and
// outputs transposed (S^T = K Q^T with 16 rows by 8 heads, O^T = V^T P^T), so that the
// instruction's eight columns are the heads of a KV head.  q and the weights enter as two
// terms of the type each (16 bits of q and 16 of a weight for bf16): rounding them once
// would put 1.5 times the output's own rounding into the result, and the kernel waits for
// memory, not for these instructions.
template <typename T, int D, int G>
struct WarpState {
  static constexpr int kSteps = D / 16;
  uint32_t qh[kSteps][2], ql[kSteps][2];
  float o[kSteps][4];
  float m[2], l[2];

  __device__ __forceinline__ void begin(const Smem<T, D>& sm, int lane) {
    const float* row = sm.q[lane >> 2];
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int e = s * 16 + j * 8 + (lane & 3) * 2;
        split_pair<T>(row[e], row[e + 1], qh[s][j], ql[s][j]);
      }
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[s][j] = 0.f;
    m[0] = m[1] = -CUDART_INF_F;
    l[0] = l[1] = 0.f;
  }

  // Chunk c (16 bytes) of row r is stored at chunk c ^ (r % 8).
  __device__ __forceinline__ void group(Smem<T, D>& sm, int warp, int lane, int stage, int valid) {
    constexpr int kRowBytes = D * 2;
    const uint32_t k0 = smem_addr(sm.k[warp][stage]), v0 = smem_addr(sm.v[warp][stage]);
    float c[4] = {0.f, 0.f, 0.f, 0.f}, c2[4] = {0.f, 0.f, 0.f, 0.f};
    const uint32_t krow = k0 + (lane & 15) * kRowBytes;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      uint32_t a[4];
      ldmatrix4(a, krow + (((2 * s + (lane >> 4)) ^ (lane & 7)) << 4));
      mma16816<T>(c, a, qh[s][0], qh[s][1]);
      mma16816<T>(c2, a, ql[s][0], ql[s][1]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) c[j] += c2[j];
    const int r = lane >> 2;
    if (r >= valid) c[0] = c[1] = -CUDART_INF_F;
    if (r + 8 >= valid) c[2] = c[3] = -CUDART_INF_F;
    float mx0 = fmaxf(c[0], c[2]), mx1 = fmaxf(c[1], c[3]);
    if (__any_sync(0xffffffffu, mx0 > m[0] + (kSlack + kLift<T>) ||
                                      mx1 > m[1] + (kSlack + kLift<T>))) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) {
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, d));
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, d));
      }
      const float n0 = fmaxf(m[0], mx0 - kLift<T>), n1 = fmaxf(m[1], mx1 - kLift<T>);
      const float a0 = n0 == m[0] ? 1.f : fast_exp2(m[0] - n0);
      const float a1 = n1 == m[1] ? 1.f : fast_exp2(m[1] - n1);
      m[0] = n0;
      m[1] = n1;
      l[0] *= a0;
      l[1] *= a1;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        o[s][0] *= a0;
        o[s][1] *= a1;
        o[s][2] *= a0;
        o[s][3] *= a1;
      }
    }
    const float p0 = fast_exp2(c[0] - m[0]), p1 = fast_exp2(c[1] - m[1]);
    const float p2 = fast_exp2(c[2] - m[0]), p3 = fast_exp2(c[3] - m[1]);
    l[0] += p0 + p2;
    l[1] += p1 + p3;
    uint32_t h0, h1, l0, l1;
    split_pair<T>(p0, p1, h0, l0);
    split_pair<T>(p2, p3, h1, l1);
    h0 = movmatrix(h0);
    h1 = movmatrix(h1);
    l0 = movmatrix(l0);
    l1 = movmatrix(l1);
    const int vr = (lane & 7) + ((lane >> 4) << 3);
    const uint32_t vrow = v0 + vr * kRowBytes;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      uint32_t a[4];
      ldmatrix4_trans(a, vrow + (((2 * s + ((lane >> 3) & 1)) ^ (vr & 7)) << 4));
      mma16816<T>(o[s], a, h0, h1);
      mma16816<T>(o[s], a, l0, l1);
    }
  }

  // (m, l) to shared memory and o, as [head][D] floats, over the warp's own stages.
  __device__ __forceinline__ void end(Smem<T, D>& sm, int warp, int lane, float* so) {
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) {
      l[0] += __shfl_xor_sync(0xffffffffu, l[0], d);
      l[1] += __shfl_xor_sync(0xffffffffu, l[1], d);
    }
    const int h = (lane & 3) * 2;
    if (lane < 4) {
      sm.m[warp][h] = m[0];
      sm.m[warp][h + 1] = m[1];
      sm.l[warp][h] = l[0];
      sm.l[warp][h + 1] = l[1];
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int e = s * 16 + (lane >> 2);
      so[h * D + e] = o[s][0];
      so[(h + 1) * D + e] = o[s][1];
      so[h * D + e + 8] = o[s][2];
      so[(h + 1) * D + e + 8] = o[s][3];
    }
  }
};

// The fp32 state: a lane takes a quarter of one of the group's eight rows for the scores
// (q is read from shared memory, the same address in a quarter's lanes) and four columns
// of all of them for the outputs.
template <int D, int G>
struct WarpState<float, D, G> {
  static constexpr int kLanes = D / 4;       // lanes that cover a row of V
  static constexpr int kParts = 32 / kLanes; // rows of V taken at once
  float o[G][4];
  float m[G], l[G];

  __device__ __forceinline__ void begin(const Smem<float, D>&, int) {
#pragma unroll
    for (int h = 0; h < G; ++h) {
      m[h] = -CUDART_INF_F;
      l[h] = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[h][e] = 0.f;
    }
  }

  __device__ __forceinline__ void group(Smem<float, D>& sm, int warp, int lane, int stage,
                                        int valid) {
    using S = Smem<float, D>;
    const float4* k = reinterpret_cast<const float4*>(sm.k[warp][stage]);
    const float4* v = reinterpret_cast<const float4*>(sm.v[warp][stage]);
    const int r = lane & 7, quarter = lane >> 3;
    float s[G];
#pragma unroll
    for (int h = 0; h < G; ++h) s[h] = 0.f;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      const float4 x = k[r * (D / 4) + ((quarter * (D / 16) + j) ^ r)];
#pragma unroll
      for (int h = 0; h < G; ++h) {
        const float4 q = *reinterpret_cast<const float4*>(&sm.q[h][quarter * S::kQuarter + 4 * j]);
        s[h] = fmaf(q.x, x.x, fmaf(q.y, x.y, fmaf(q.z, x.z, fmaf(q.w, x.w, s[h]))));
      }
    }
    bool move = false;
#pragma unroll
    for (int h = 0; h < G; ++h) {
      s[h] += __shfl_xor_sync(0xffffffffu, s[h], 8);
      s[h] += __shfl_xor_sync(0xffffffffu, s[h], 16);
      if (r >= valid) s[h] = -CUDART_INF_F;
      move |= s[h] > m[h] + kSlack;
    }
    if (__any_sync(0xffffffffu, move)) {
#pragma unroll
      for (int h = 0; h < G; ++h) {
        float mx = s[h];
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
        mx = fmaxf(m[h], mx);
        const float a = mx == m[h] ? 1.f : exp2f(m[h] - mx);
        m[h] = mx;
        l[h] *= a;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[h][e] *= a;
      }
    }
    float w[kHeads];
#pragma unroll
    for (int h = 0; h < G; ++h) {
      w[h] = exp2f(s[h] - m[h]);
      l[h] += quarter == 0 ? w[h] : 0.f;
    }
#pragma unroll
    for (int h = G; h < kHeads; ++h) w[h] = 0.f;
    if (quarter == 0)
      *reinterpret_cast<float4*>(sm.p[warp][r]) = make_float4(w[0], w[1], w[2], w[3]);
    if (quarter == 1)
      *reinterpret_cast<float4*>(sm.p[warp][r] + 4) = make_float4(w[4], w[5], w[6], w[7]);
    __syncwarp();
    const int c = lane % kLanes;
#pragma unroll
    for (int i = 0; i < 8 / kParts; ++i) {
      const int row = i * kParts + lane / kLanes;
      const float4 x = v[row * (D / 4) + (c ^ row)];
      const float4 w0 = *reinterpret_cast<const float4*>(sm.p[warp][row]);
      const float4 w1 = *reinterpret_cast<const float4*>(sm.p[warp][row] + 4);
      const float ww[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
      for (int h = 0; h < G; ++h) {
        o[h][0] = fmaf(ww[h], x.x, o[h][0]);
        o[h][1] = fmaf(ww[h], x.y, o[h][1]);
        o[h][2] = fmaf(ww[h], x.z, o[h][2]);
        o[h][3] = fmaf(ww[h], x.w, o[h][3]);
      }
    }
    __syncwarp();
  }

  __device__ __forceinline__ void end(Smem<float, D>& sm, int warp, int lane, float* so) {
#pragma unroll
    for (int h = 0; h < G; ++h) {
#pragma unroll
      for (int d = 1; d < 8; d <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], d);
      if (kParts == 2)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[h][e] += __shfl_xor_sync(0xffffffffu, o[h][e], 16);
      if (lane == 0) {
        sm.m[warp][h] = m[h];
        sm.l[warp][h] = l[h];
      }
      if (lane < kLanes)
        *reinterpret_cast<float4*>(so + h * D + 4 * lane) =
            make_float4(o[h][0], o[h][1], o[h][2], o[h][3]);
    }
  }
};

// Inclusive sum over the block's threads of one value each, and the sum of all.
__device__ __forceinline__ long long block_scan(long long x, long long (&part)[kWarps],
                                                long long& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += y;
  }
  if (lane == 31) part[warp] = x;
  __syncthreads();
  all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w == warp) x += all;
    all += part[w];
  }
  return x;
}

template <typename T, int D, int G>
__global__ void __launch_bounds__(kThreads, 2)
    paged_decode_kernel(const PagedAttnParams p, const PagedPartials part, const int rotate) {
  extern __shared__ unsigned char smem_raw[];
  using S = Smem<T, D>;
  S& sm = *reinterpret_cast<S*>(smem_raw);
  constexpr int kRows = group_rows<T>(), kTile = tile_rows<T>();
  constexpr int kChunks = D * (int)sizeof(T) / 16;  // of a row
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_wait();
  // (after the wait: the chunks' kernel behind this one may read all but this one's output early)
  pdl_launch_dependents();
  if (rotate) rotate_q<T, D, G>(p);

  // Tiles of all pairs: a thread adds up a run of sequences, a scan over the block gives the
  // thread that holds the first tile of this CTA's share [first, last).
  const int run = (p.plan.n_seq + kThreads - 1) / kThreads;
  const int s0 = min(tid * run, p.plan.n_seq), s1 = min(s0 + run, p.plan.n_seq);
  int bad = 0;
  const auto tiles_of = [&](int s) {
    int tok;
    return (long long)((single_rows(p, s, tok, &bad) + kTile - 1) / kTile) * p.n_kv;
  };
  long long mine = 0;
#pragma unroll 4
  for (int s = s0; s < s1; ++s) mine += tiles_of(s);
  if (bad && blockIdx.x == 0) atomicOr(p.status, bad);
  long long total;
  long long before = block_scan(mine, sm.scan, total) - mine;
  const long long n = min((long long)gridDim.x, total);
  if (tid == 0) {
    part.jobs[blockIdx.x].n_parts = 0;
    sm.found_seq = p.plan.n_seq;
  }
  if (blockIdx.x >= n) return;
  const long long first = blockIdx.x * total / n, last = (blockIdx.x + 1) * total / n;
  __syncthreads();
  if (before <= first && first < before + mine) {
    int s = s0;
    for (long long x; s < s1 - 1 && before + (x = tiles_of(s)) <= first; ++s) before += x;
    sm.found_seq = s;
    sm.found_before = before;
  }
  __syncthreads();
  int seq = sm.found_seq;
  long long seq_first = sm.found_before;  // first tile of the sequence

  for (long long tile = first; tile < last && seq < p.plan.n_seq;) {
    int tok;
    const int len = single_rows(p, seq, tok, &bad);
    const int tiles = (len + kTile - 1) / kTile;
    if (tile >= seq_first + (long long)tiles * p.n_kv) {  // on to the next sequence
      seq_first += (long long)tiles * p.n_kv;
      ++seq;
      continue;
    }
    // one piece: tiles [t0, t1) of KV head h
    const int h = (int)((tile - seq_first) / tiles);
    const long long pair_first = seq_first + (long long)h * tiles;
    const int t0 = (int)(tile - pair_first);
    const int t1 = (int)min((long long)tiles, last - pair_first);
    const int r1 = min(len, t1 * kTile);
    const int row0 = t0 * kTile + warp * kRows;  // the warp's first group
    const int n_groups = row0 < r1 ? (r1 - row0 + kTile - 1) / kTile : 0;

    // Page of the warp's group `lane` of the current 32, and the rows that it has.
    int page = -1;
    const auto look_up = [&](int g0) {
      const int row = row0 + (g0 + lane) * kTile;
      page = -1;
      if (row < r1) {
        page = page_of(p.kv, seq, row);
        if (page < 0) atomicOr(p.status, kStatusBadPage);
      }
    };
    const auto issue = [&](int g) {
      const int pg = __shfl_sync(0xffffffffu, page, g & 31);
      if (g < n_groups && pg >= 0) {
        const int row = row0 + g * kTile, stage = g % kStages;
        const long long at = row_offset(p.kv, pg, h, row);
        const T* k = static_cast<const T*>(p.kv.k) + at;
        const T* v = static_cast<const T*>(p.kv.v) + at;
        const uint32_t ks = smem_addr(sm.k[warp][stage]), vs = smem_addr(sm.v[warp][stage]);
#pragma unroll
        for (int i = 0; i < kRows * kChunks / 32; ++i) {
          const int r = (i * 32 + lane) / kChunks, c = (i * 32 + lane) % kChunks;
          const bool on = row + r < r1;
          const long long src = (on ? r : 0) * p.kv.row_stride + c * (16 / (int)sizeof(T));
          const uint32_t dst = (uint32_t)(r * kChunks + (c ^ (r & 7))) << 4;
          cp_async16(ks + dst, k + src, on);
          cp_async16(vs + dst, v + src, on);
        }
      }
      cp_commit();
      return pg;
    };
    look_up(0);
    // (pages of the groups in flight, oldest first)
    int flight[kStages];
#pragma unroll
    for (int g = 0; g < kStages - 1; ++g) flight[g] = issue(g);

    const bool whole = t0 == 0 && t1 == tiles;
    if (!whole && tid == kThreads - 1) {
      // what the merge's block of this CTA's number does (the divisions while rows arrive)
      // Query heads of many parts are listed apart from one another: neighbours' blocks would
      // share an SM, whose reads then bound them (3 us more over 32768 rows).  Never under the
      // last CTA, which may list its next pair.
      static_assert(kFewParts >= G, "a CTA per query head, and one more");
      const auto cta_of = [&](long long t) { return (int)(((t + 1) * n - 1) / total); };
      const int c0 = cta_of(pair_first), n_parts = cta_of(pair_first + tiles - 1) - c0 + 1;
      const int i = (int)blockIdx.x - c0, apart = n_parts > kFewParts ? n_parts / G : 1;
      const int slot0 = 2 * c0 + (pair_first == c0 * total / n ? 0 : 1);
      if (i == 0 || (n_parts > kFewParts && i % apart == 0 && i / apart < G))
        part.jobs[blockIdx.x] =
            PagedJob{tok, h, c0, slot0, n_parts, n_parts > kFewParts ? i / apart : -1};
    }

    // q of the token, rotated for its position and scaled, while the first rows arrive
    const T* q = static_cast<const T*>(p.qkv) + (long long)tok * p.qkv_stride +
                 (long long)h * G * D;
    const auto put_q = [&](int g, int e, float x) {
      if constexpr (sizeof(T) == 4)
        sm.q[g][e / (D / 4) * S::kQuarter + e % (D / 4)] = x;
      else
        sm.q[g][e] = x;
    };
    for (int e = tid; e < D / 2; e += kThreads) {
      float co, si;
      rope_cos_sin(len - 1, p.turns[e], co, si);
#pragma unroll
      for (int g = 0; g < kHeads; ++g) {
        float a = 0.f, b = 0.f;
        if (g < G) {
          a = Elem<T>::get(q[g * D + e]);
          b = Elem<T>::get(q[g * D + e + D / 2]);
        }
        put_q(g, e, (a * co - b * si) * p.scale_log2);
        put_q(g, e + D / 2, (a * si + b * co) * p.scale_log2);
      }
    }
    __syncthreads();
    WarpState<T, D, G> st;
    st.begin(sm, lane);
    for (int g = 0; g < n_groups; ++g) {
      if (((g + kStages - 1) & 31) == 0) look_up(g + kStages - 1);
      flight[kStages - 1] = issue(g + kStages - 1);
      cp_wait<kStages - 1>();
      __syncwarp();
      const int row = row0 + g * kTile;
      if (flight[0] >= 0) st.group(sm, warp, lane, g % kStages, min(kRows, r1 - row));
      __syncwarp();
#pragma unroll
      for (int i = 0; i + 1 < kStages; ++i) flight[i] = flight[i + 1];
    }
    cp_wait<0>();
    __syncwarp();

    // Merge the warps (each puts its output over its own stages of K).
    float* so = reinterpret_cast<float*>(sm.k[warp][0]);
    static_assert(sizeof(sm.k[0]) >= sizeof(float) * kHeads * D, "room for the warp's output");
    st.end(sm, warp, lane, so);
    __syncthreads();
    const int slot = 2 * blockIdx.x + (tile == first ? 0 : 1);
    T* out = static_cast<T*>(p.out) + (long long)tok * p.out_stride + (long long)h * G * D;
    // a warp's factor for each head, by a thread each: what it weighs beside the largest maximum,
    // over the sum where the pair is whole (per element this took 4300 clocks of a piece's 9500)
    static_assert(kWarps * kHeads == 32, "one warp");
    if (warp == 0) {
      const int g = lane % kHeads, w = lane / kHeads;
      const float lw = g < G ? sm.l[w][g] : 0.f;
      const float mw = lw != 0.f ? sm.m[w][g] : -CUDART_INF_F;
      float mm = mw;
#pragma unroll
      for (int x = kHeads; x < 32; x <<= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, x));
      const float a = lw != 0.f ? exp2f(mw - mm) : 0.f;
      float ll = a * lw;
#pragma unroll
      for (int x = kHeads; x < 32; x <<= 1) ll += __shfl_xor_sync(0xffffffffu, ll, x);
      sm.m[w][g] = !whole ? a : ll != 0.f ? a / ll : 0.f;
      if (!whole && w == 0 && g < G) part.ml[slot * G + g] = make_float2(mm, ll);
    }
    __syncthreads();
    for (int i = 4 * tid; i < G * D; i += 4 * kThreads) {
      const int g = i / D;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float a = sm.m[w][g];
        const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<float*>(sm.k[w][0]) + i);
        if (a != 0.f) {  // (a warp without a row holds nothing to be added)
          o.x = fmaf(a, x.x, o.x);
          o.y = fmaf(a, x.y, o.y);
          o.z = fmaf(a, x.z, o.z);
          o.w = fmaf(a, x.w, o.w);
        }
      }
      if (whole) {
        struct alignas(4 * sizeof(T)) Four { T e[4]; };
        *reinterpret_cast<Four*>(out + i) =
            Four{Elem<T>::put(o.x), Elem<T>::put(o.y), Elem<T>::put(o.z), Elem<T>::put(o.w)};
      } else {
        *reinterpret_cast<float4*>(part.o + (long long)slot * G * D + i) = o;
      }
    }
    tile = pair_first + t1;
    __syncthreads();
  }
}

template <typename T, int D, int G>
cudaError_t prepare_one() {
  return cudaFuncSetAttribute((const void*)paged_decode_kernel<T, D, G>,
                              cudaFuncAttributeMaxDynamicSharedMemorySize,
                              (int)sizeof(Smem<T, D>));
}

template <typename T, int D, int G>
cudaError_t launch_one(const PagedAttnParams& p, const PagedPartials& part, int n_sm,
                       cudaStream_t st, bool pdl, bool rotate, int* grid) {
  const long long tiles =
      (long long)p.plan.n_seq * p.n_kv * ((p.max_len + tile_rows<T>() - 1) / tile_rows<T>());
  const long long items = (long long)p.plan.n_tokens * p.n_kv * (D / 2 / Vec16<T>::n);
  const long long want = rotate ? std::max(tiles, (items + kThreads - 1) / kThreads) : tiles;
  *grid = (int)std::min<long long>({2LL * n_sm, part.n_ctas, kMaxDecodeCtas, want});
  return launch_with_pdl(paged_decode_kernel<T, D, G>, dim3(*grid), kThreads, sizeof(Smem<T, D>),
                         st, pdl, p, part, (int)rotate);
}

template <typename T, int D, int G>
cudaError_t merge_one(const PagedAttnParams& p, const PagedPartials& part, int n_decode,
                      int n_chunk, cudaStream_t st) {
  return launch_with_pdl(paged_merge_kernel<T, D, G>, dim3(n_decode + n_chunk * kUnitSlabs),
                         kMergeWarps * 32, 0, st, true, p, part, n_decode);
}

}  // namespace

cudaError_t prepare_paged_decode() {
  cudaError_t e = prepare_one<float, 128, 6>();
  if (e == cudaSuccess) e = prepare_one<float, 64, 7>();
  if (e == cudaSuccess) e = prepare_one<__nv_bfloat16, 128, 6>();
  if (e == cudaSuccess) e = prepare_one<__nv_bfloat16, 64, 7>();
  if (e == cudaSuccess) e = prepare_one<__half, 128, 6>();
  if (e == cudaSuccess) e = prepare_one<__half, 64, 7>();
  return e;
}

cudaError_t launch_paged_decode(const PagedAttnParams& p, const PagedPartials& part, int dtype,
                                int head_dim, int n_sm, cudaStream_t st, bool pdl, bool rotate,
                                int* grid) {
  const bool wide = head_dim == 128;
  if (dtype == kDtypeF32)
    return wide ? launch_one<float, 128, 6>(p, part, n_sm, st, pdl, rotate, grid)
                : launch_one<float, 64, 7>(p, part, n_sm, st, pdl, rotate, grid);
  if (dtype == kDtypeBf16)
    return wide ? launch_one<__nv_bfloat16, 128, 6>(p, part, n_sm, st, pdl, rotate, grid)
                : launch_one<__nv_bfloat16, 64, 7>(p, part, n_sm, st, pdl, rotate, grid);
  return wide ? launch_one<__half, 128, 6>(p, part, n_sm, st, pdl, rotate, grid)
              : launch_one<__half, 64, 7>(p, part, n_sm, st, pdl, rotate, grid);
}

cudaError_t launch_paged_merge(const PagedAttnParams& p, const PagedPartials& part, int dtype,
                               int head_dim, int n_decode, int n_chunk, cudaStream_t st) {
  const bool wide = head_dim == 128;
  if (dtype == kDtypeF32)
    return wide ? merge_one<float, 128, 6>(p, part, n_decode, n_chunk, st)
                : merge_one<float, 64, 7>(p, part, n_decode, n_chunk, st);
  if (dtype == kDtypeBf16)
    return wide ? merge_one<__nv_bfloat16, 128, 6>(p, part, n_decode, n_chunk, st)
                : merge_one<__nv_bfloat16, 64, 7>(p, part, n_decode, n_chunk, st);
  return wide ? merge_one<__half, 128, 6>(p, part, n_decode, n_chunk, st)
              : merge_one<__half, 64, 7>(p, part, n_decode, n_chunk, st);
}

}  // namespace gqa
