"""The paged operators and the sampling in 64 bits (numpy), and their tolerances."""
import math

import numpy as np
import torch

THETA = 1e6
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SHAPES = {128: (6, 128), 64: (7, 64)}  # head_dim -> (q heads per KV head, head_dim)


def rotate(x, pos, d, theta=THETA):
    """x [..., heads, d] at positions pos [...]."""
    ang = np.asarray(pos, np.float64)[..., None, None] * theta ** (-2.0 * np.arange(d // 2) / d)
    c, s = np.cos(ang), np.sin(ang)
    a, b = x[..., :d // 2], x[..., d // 2:]
    return np.concatenate([a * c - b * s, a * s + b * c], axis=-1)


class Batch:
    """A paged cache with random rows and the new tokens of some sequences.

    `news` / `lens`: new tokens and rows (with them) of each sequence; the pages are handed out
    in a random order, and every element that belongs to no row is NaN."""

    def __init__(self, dtype, d, news, lens, page=16, n_kv=2, layout="hnd", seed=0, pad=0,
                 extra_rows=0, scale=1.5):
        g = np.random.default_rng(seed)
        self.dtype, self.d, self.news, self.lens, self.page = dtype, d, list(news), list(lens), page
        self.n_kv, self.layout = n_kv, layout
        self.group = SHAPES[d][0]
        self.n_q = self.group * n_kv
        self.td = DTYPES[dtype]
        counts = [-(-t // page) for t in lens]
        self.n_pages = sum(counts) + 3
        perm = g.permutation(self.n_pages)
        self.table = np.full((len(lens), max(counts + [1]) + 1), -7, np.int32)
        at = 0
        for s, n in enumerate(counts):
            self.table[s, :n] = perm[at:at + n]
            at += n
        self.starts = np.concatenate([[0], np.cumsum(self.news)]).astype(np.int32)
        self.n_tokens = int(self.starts[-1])
        width = (self.n_q + 2 * n_kv) * d
        qkv = g.standard_normal((self.n_tokens + extra_rows, width + pad))
        qkv[:, :self.n_q * d] *= scale
        self.qkv = torch.from_numpy(qkv).to(self.td)
        # cached rows, in 64 bits but holding values of the type
        self.k = [self._cast(g.standard_normal((t, n_kv, d))) for t in lens]
        self.v = [self._cast(g.standard_normal((t, n_kv, d))) for t in lens]

    def _cast(self, x):
        return torch.from_numpy(np.ascontiguousarray(x)).to(self.td).double().numpy()

    def row(self, i):
        return self.qkv[i, :(self.n_q + 2 * self.n_kv) * self.d].double().numpy().reshape(-1, self.d)

    def appended(self):
        """Caches after the append in 64 bits (K not rounded), and the bound on K's error."""
        ks, vs, tols = [], [], []
        h = torch.finfo(self.td).eps / 2
        for s, (n, t) in enumerate(zip(self.news, self.lens)):
            k, v, tol = self.k[s].copy(), self.v[s].copy(), np.zeros_like(self.k[s])
            for i in range(n):
                r = self.row(self.starts[s] + i)
                raw = r[self.n_q:self.n_q + self.n_kv]
                pos = t - n + i
                k[pos] = rotate(raw, pos, self.d)
                v[pos] = r[self.n_q + self.n_kv:]
                # fp32: the angle, its sine and cosine (2 ulp) and three operations on a and b;
                # then one rounding to the type
                both = np.abs(raw[:, :self.d // 2]) + np.abs(raw[:, self.d // 2:])
                tol[pos] = np.concatenate([both, both], -1) * 6 * 2.0 ** -24 + h * np.abs(k[pos])
            ks.append(k), vs.append(v), tols.append(tol)
        return ks, vs, tols

    def set_appended(self):
        """Puts the appended rows (rounded to the type) into the cache, as an append does."""
        ks, vs, _ = self.appended()
        self.k = [self._cast(k) for k in ks]
        self.v = [self._cast(v) for v in vs]

    def pools(self):
        shape = (self.n_pages, self.n_kv, self.page, self.d) if self.layout == "hnd" else \
            (self.n_pages, self.page, self.n_kv, self.d)
        out = []
        for rows in (self.k, self.v):
            pool = torch.full(shape, math.nan, dtype=self.td)
            for s, x in enumerate(rows):
                for t in range(x.shape[0]):
                    page, r = self.table[s, t // self.page], t % self.page
                    if not 0 <= page < self.n_pages:
                        continue
                    val = torch.from_numpy(x[t]).to(self.td)
                    if self.layout == "hnd":
                        pool[page, :, r] = val
                    else:
                        pool[page, r] = val
            out.append(pool)
        return out

    def unpool(self, pool, s):
        """Rows of sequence s as [rows, n_kv, d] in 64 bits."""
        out = np.empty((self.lens[s], self.n_kv, self.d))
        for t in range(self.lens[s]):
            p = pool[self.table[s, t // self.page]]
            r = t % self.page
            out[t] = (p[:, r] if self.layout == "hnd" else p[r]).double().numpy()
        return out

    def attend(self, skip=None):
        """Outputs [tokens, n_q, d] in 64 bits and the per-element tolerance.  skip(s, t) hides
        rows (bad pages)."""
        # Half a step of the type that q, the weights and the output are rounded to (for fp32 16
        # half steps: the rotation, a dot product's rounding errors, which grow like the square
        # root of its length, and the argument of the exponential).
        h = 2.0 ** -20 if self.dtype == "f32" else torch.finfo(self.td).eps / 2
        out = np.zeros((self.n_tokens, self.n_q, self.d))
        tol = np.zeros_like(out)
        for s, (n, t) in enumerate(zip(self.news, self.lens)):
            for i in range(n):
                at, pos = self.starts[s] + i, t - n + i
                rows = np.array([r for r in range(pos + 1) if not (skip and skip(s, r))], int)
                if rows.size == 0:
                    continue
                q = rotate(self.row(at)[:self.n_q], pos, self.d)
                for j in range(self.n_q):
                    k, v = self.k[s][rows, j // self.group], self.v[s][rows, j // self.group]
                    x = k @ q[j] / math.sqrt(self.d)
                    p = np.exp(x - x.max())
                    p /= p.sum()
                    out[at, j] = p @ v
                    # Each weight is off by the rounding of q (b: rms of a score's terms over a
                    # dot product) and of the weight itself; independent over keys, so the error
                    # adds up like the root of the squares: 6 h is 10 standard deviations of
                    # a rounding.  The last term is the output's own rounding.
                    b2 = ((k * q[j]) ** 2).sum(-1).max() / self.d
                    spread = np.sqrt((p[:, None] ** 2 * v ** 2).sum(0))
                    tol[at, j] = h * np.abs(out[at, j]) + 6 * h * math.sqrt(b2 + 2) * spread
        return out, tol + 1e-30


def sample_row(x, t, k, p, m, u):
    """The definition of gqa_sample for one row, in 64 bits."""
    x = np.asarray(x, np.float64).copy()
    x[np.isnan(x)] = -np.inf
    top = x.max()
    if top == -np.inf:
        return 0
    if not t > 0:
        return int(np.argmax(x))
    with np.errstate(invalid="ignore"):
        w = np.where(x == top, 1.0, np.exp((x - top) / t))
    if top == np.inf:
        w = (x == top).astype(np.float64)
    w[x == -np.inf] = 0
    ids = np.lexsort((np.arange(x.size), -x))
    if 0 < k < x.size:
        ids = ids[:k]
    if p < 1:
        c = np.cumsum(w[ids])
        ids = ids[:max(1, int(np.searchsorted(c, p * c[-1], side="left")) + 1)]
    ids = ids[(w[ids] >= m) | (np.arange(ids.size) == 0)]
    ids = np.sort(ids[w[ids] > 0])
    c = np.cumsum(w[ids])
    return int(ids[min(int(np.searchsorted(c, max(u, 0.0) * c[-1], side="right")), ids.size - 1)])
