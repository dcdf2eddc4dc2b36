"""Paged KV cache: append and attention against 64-bit arithmetic (tests/paged_ref.py)."""
import math

import numpy as np
import pytest

from paged_ref import THETA, Batch

pytestmark = pytest.mark.gpu

MIXED = ([1, 5, 1, 0, 40, 2, 1, 3, 21, 22], [1, 5, 200, 0, 90, 77, 33, 259, 21, 300])


def make_ctx(pkg, d, n_kv=2):
    return pkg.Context(n_heads_q=(6 if d == 128 else 7) * n_kv, n_heads_kv=n_kv, head_dim=d,
                       rope_theta=THETA)


class Run:
    """A Batch on the device."""

    def __init__(self, pkg, b, one=None):
        import torch
        self.torch, self.b = torch, b
        self.kp, self.vp = (x.cuda() for x in b.pools())
        self.table = torch.from_numpy(b.table).cuda()
        self.qkv = b.qkv.cuda()
        self.one = all(n == 1 for n in b.news) if one is None else one
        self.starts = None if self.one else torch.from_numpy(b.starts).cuda()
        self.lens = torch.tensor(b.lens, dtype=torch.int32).cuda()
        self.kv = pkg.paged_kv_of(self.kp, self.vp, self.table, layout=b.layout)
        self.n_seq = len(b.lens)

    def append(self, ctx, **kw):
        ctx.paged_append(self.kv, self.n_seq, self.b.n_tokens, self.starts, self.lens, self.qkv,
                         **kw)

    def attend(self, ctx, out=None, extra_rows=0, max_new=None, max_len=None, **kw):
        b = self.b
        if out is None:
            out = self.torch.full((b.n_tokens + extra_rows, b.n_q * b.d), 7.0, dtype=b.td).cuda()
        ctx.paged_attention(self.kv, self.n_seq, b.n_tokens, self.starts, self.lens,
                            max_new or max(b.news + [1]), max_len or max(b.lens + [1]), self.qkv,
                            out, **kw)
        return out


def check_attention(b, got, skip=None):
    want, tol = b.attend(skip)
    got = got[:b.n_tokens, :b.n_q * b.d].double().cpu().numpy().reshape(want.shape)
    bad = ~(np.abs(got - want) <= tol)  # (a NaN is bad)
    assert not bad.any(), (np.argwhere(bad)[:5].tolist(), float(np.nanmax(np.abs(got - want) / tol)))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("d,n_kv,page,layout,pad", [(128, 2, 16, "hnd", 0), (128, 1, 64, "nhd", 8),
                                                    (64, 2, 32, "nhd", 16), (64, 3, 256, "hnd", 0)])
def test_append(pkg, cuda, dtype, d, n_kv, page, layout, pad):
    b = Batch(dtype, d, *MIXED, page=page, n_kv=n_kv, layout=layout, pad=pad, extra_rows=2, seed=1)
    ks, vs, tols = b.appended()
    r = Run(pkg, b)
    before = r.kp.clone()
    with make_ctx(pkg, d, n_kv) as ctx:
        r.append(ctx)
        assert ctx.device_status() == 0
    kp, vp = r.kp.cpu(), r.vp.cpu()
    for s in range(len(b.lens)):
        assert (np.abs(b.unpool(kp, s) - ks[s]) <= tols[s]).all()
        np.testing.assert_array_equal(b.unpool(vp, s), vs[s])
    # nothing else in the pool is touched
    names = np.unique(np.concatenate([b.table[s, :-(-t // page)] for s, t in enumerate(b.lens)]))
    other = [p for p in range(b.n_pages) if p not in names]
    assert cuda.equal(r.kp[other].isnan(), before[other].isnan()) and len(other) == 3
    assert int(r.kp.isnan().sum()) == int(before.isnan().sum())


def test_append_far_position(pkg, cuda):
    """At position 900,000 an angle formed in fp32 would be off by 1e-2."""
    b = Batch("f32", 128, [1], [1], page=256, seed=2)
    pos = 900_000
    r = Run(pkg, b)
    table = cuda.zeros(1, pos // 256 + 1, dtype=cuda.int32, device="cuda")
    kv = pkg.paged_kv_of(r.kp, r.vp, table)
    lens = cuda.tensor([pos + 1], dtype=cuda.int32, device="cuda")
    with make_ctx(pkg, 128) as ctx:
        ctx.paged_append(kv, 1, 1, None, lens, r.qkv)
        assert ctx.device_status() == 0
    from paged_ref import rotate
    raw = b.row(0)[b.n_q:b.n_q + 2]
    got = r.kp[0, :, pos % 256].double().cpu().numpy()
    both = np.abs(raw[:, :64]) + np.abs(raw[:, 64:])
    assert (np.abs(got - rotate(raw, pos, 128)) <= np.concatenate([both, both], -1) * 6 * 2.0 ** -24
            ).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("d,n_kv,page,layout", [(128, 2, 16, "hnd"), (128, 1, 128, "nhd"),
                                                (64, 2, 64, "nhd"), (64, 3, 16, "hnd")])
def test_attention_mixed(pkg, cuda, dtype, d, n_kv, page, layout):
    b = Batch(dtype, d, *MIXED, page=page, n_kv=n_kv, layout=layout, pad=16, seed=3)
    b.set_appended()
    r = Run(pkg, b)
    with make_ctx(pkg, d, n_kv) as ctx:
        out = r.attend(ctx, extra_rows=1)
        assert ctx.device_status() == 0
    check_attention(b, out)
    assert (out[b.n_tokens:] == 7).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("d", [128, 64])
@pytest.mark.parametrize("lens", [[1], [2, 15, 16, 17], [63, 64, 65, 1], [1000], [4097, 3, 2500]])
def test_attention_single_tokens(pkg, cuda, dtype, d, lens):
    b = Batch(dtype, d, [1] * len(lens), lens, page=32, seed=4)
    b.set_appended()
    r = Run(pkg, b)
    with make_ctx(pkg, d) as ctx:
        out = r.attend(ctx)
        loose = r.attend(ctx, max_len=b.table.shape[1] * 32)  # a bound above every length
        assert ctx.device_status() == 0
    check_attention(b, out)
    check_attention(b, loose)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("d", [128, 64])
@pytest.mark.parametrize("news,lens", [([2], [2]), ([3], [700]), ([129], [129]), ([64], [1500]),
                                       ([150, 18, 19], [400, 18, 1100])])
def test_attention_chunks(pkg, cuda, dtype, d, news, lens):
    b = Batch(dtype, d, news, lens, page=16, seed=5)
    b.set_appended()
    r = Run(pkg, b)
    with make_ctx(pkg, d) as ctx:
        out = r.attend(ctx)
        assert ctx.device_status() == 0
    check_attention(b, out)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("d", [128, 64])
def test_large_scores(pkg, cuda, dtype, d):
    """Scores of some hundreds: one key takes all the weight, the maximum moves on the way."""
    b = Batch(dtype, d, [1, 30], [600, 300], page=16, seed=6, scale=60.0)
    b.set_appended()
    r = Run(pkg, b)
    with make_ctx(pkg, d) as ctx:
        out = r.attend(ctx)
    got = out.double().cpu().numpy()
    want, _ = b.attend()
    # The weights' errors are those of scores of this size: a score is off by at most the
    # rounding of q (half a step, on each of d terms) -- the two largest weights trade places
    # where their scores are closer than that, so only rows with a clear winner are compared.
    h = 2.0 ** -20 if dtype == "f32" else cuda.finfo(b.td).eps / 2
    clear = 0
    for s, (n, t) in enumerate(zip(b.news, b.lens)):
        from paged_ref import rotate
        for i in range(n):
            at, pos = b.starts[s] + i, t - n + i
            q = rotate(b.row(at)[:b.n_q], pos, d)
            for j in range(b.n_q):
                k = b.k[s][:pos + 1, j // b.group]
                x = np.sort(k @ q[j] / math.sqrt(d))
                err = h * np.abs(k * q[j]).sum(-1).max() / math.sqrt(d)
                if x.size == 1 or x[-1] - x[-2] > 2 * err + 12:
                    clear += 1
                    w = want[at, j]
                    # the others weigh at most pos exp(-12) together
                    assert (np.abs(got[at, j * d:(j + 1) * d] - w) <=
                            2 * h * np.abs(w) + 2 * pos * math.exp(-12) * 5).all()
    assert clear > 20


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_masked_rows_do_not_reach_the_output(pkg, cuda, dtype):
    """Infinities and NaN past the end of the sequence (all of the pool's other elements are NaN
    in Batch), and in later rows of the token's own chunk."""
    b = Batch(dtype, 128, [30, 1], [75, 40], page=16, seed=7)
    b.set_appended()
    r = Run(pkg, b)
    with make_ctx(pkg, 128) as ctx:
        clean = r.attend(ctx)
        check_attention(b, clean)
        # the last row of sequence 0 is seen by its last token alone
        page, row = int(b.table[0, 74 // 16]), 74 % 16
        for bad in (math.inf, -math.inf, math.nan):
            r.kp[page, :, row] = bad
            r.vp[page, :, row] = bad
            out = r.attend(ctx)
            keep = [t for t in range(31) if t != 29]
            assert cuda.equal(out[keep], clean[keep])


def test_bad_pages_and_lengths(pkg, cuda):
    b = Batch("f32", 128, [1, 1, 2, 1], [40, 40, 50, 20], page=16, seed=8)
    b.set_appended()
    b.table[0, 1] = -1               # rows 16..31 of sequence 0
    b.table[1, :3] = b.n_pages       # all of sequence 1
    r = Run(pkg, b)
    with make_ctx(pkg, 128) as ctx:
        out = r.attend(ctx)
        assert ctx.device_status() == pkg.gqa.STATUS_BAD_PAGE
        check_attention(b, out, skip=lambda s, t: (s == 0 and 16 <= t < 32) or s == 1)
        assert (out[1] == 0).all()
        kp = r.kp.clone()
        r.append(ctx)
        assert ctx.device_status() == pkg.gqa.STATUS_BAD_PAGE
        assert int(r.kp.isnan().sum()) == int(kp.isnan().sum())
        # lengths: below the new tokens, beyond the table, beyond max_len
        for s, n in ((2, 1), (3, b.table.shape[1] * 16 + 1), (3, 51), (3, 0), (3, -5)):
            lens = r.lens.clone()
            lens[s] = n
            out = cuda.full((5, 12 * 128), 7.0).cuda()
            ctx.paged_attention(r.kv, 4, 5, r.starts, lens, 2, 50, r.qkv, out)
            assert ctx.device_status() & pkg.gqa.STATUS_BAD_LENGTH
            rows = [2, 3] if s == 2 else [4]
            assert (out[rows] == 7).all()
            assert (out[[4] if s == 2 else [2, 3]] != 7).any()
        # more new tokens than max_new says
        out = cuda.full((5, 12 * 128), 7.0).cuda()
        ctx.paged_attention(r.kv, 4, 5, r.starts, r.lens, 1, 50, r.qkv, out)
        assert ctx.device_status() & pkg.gqa.STATUS_BAD_LENGTH
        assert (out[[2, 3]] == 7).all()


def test_rows_behind_the_last_sequence(pkg, cuda):
    """A padded batch: token rows that belong to no sequence are left alone."""
    b = Batch("bf16", 128, [3, 1], [20, 30], page=16, seed=9, extra_rows=28)
    b.set_appended()
    r = Run(pkg, b)
    with make_ctx(pkg, 128) as ctx:
        out = cuda.full((32, 12 * 128), 7.0, dtype=cuda.bfloat16).cuda()
        before = r.kp.clone()
        ctx.paged_append(r.kv, 2, 32, r.starts, r.lens, r.qkv)
        ctx.paged_attention(r.kv, 2, 32, r.starts, r.lens, 8, 64, r.qkv, out)
        assert ctx.device_status() == 0
        assert int(r.kp.isnan().sum()) == int(before.isnan().sum())
    check_attention(b, out)
    assert (out[4:] == 7).all()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_output_in_place(pkg, cuda, dtype):
    b = Batch(dtype, 64, [40, 1, 3], [300, 1200, 5], page=16, seed=10)
    b.set_appended()
    r = Run(pkg, b)
    with make_ctx(pkg, 64) as ctx:
        plain = r.attend(ctx)
        r.attend(ctx, out=r.qkv)
    assert cuda.equal(r.qkv[:, :14 * 64], plain)
    assert cuda.equal(r.qkv[:, 14 * 64:].cpu(), b.qkv[:, 14 * 64:])


def test_matches_the_contiguous_decode(pkg, cuda):
    """fp32: one step of three sequences as decode_batched makes it over contiguous caches."""
    lens = [40, 300, 129]
    b = Batch("f32", 128, [1] * 3, lens, page=16, seed=11)
    r = Run(pkg, b)
    with make_ctx(pkg, 128) as ctx:
        kc = [cuda.zeros(2, 4096, 128, device="cuda") for _ in lens]
        vc = [cuda.zeros(2, 4096, 128, device="cuda") for _ in lens]
        for s, n in enumerate(lens):
            kc[s][:, :n - 1] = cuda.from_numpy(b.k[s][:-1]).float().cuda().transpose(0, 1)
            vc[s][:, :n - 1] = cuda.from_numpy(b.v[s][:-1]).float().cuda().transpose(0, 1)
        ptr = [cuda.tensor([x.data_ptr() for x in c], dtype=cuda.int64, device="cuda")
               for c in (kc, vc)]
        want = cuda.empty(3, 1536, device="cuda")
        ctx.decode_batched(3, *ptr, r.qkv, 2048, r.lens, 512, want, 1536)
        r.append(ctx)
        got = r.attend(ctx)
        assert ctx.device_status() == 0
    # both within the bound of the 64-bit value (the decode's angles are fp32: pos 300 * 2^-24
    # turns of a radian, below the bound's 16 half steps times the scores)
    b.set_appended()
    check_attention(b, got)
    check_attention(b, want)


def test_prefill_then_decode_with_sampling(pkg, cuda):
    """A run of the operators as a server makes it: a prompt in two chunks, then single tokens,
    beside a running sequence; every output against 64 bits over the cache as it then is."""
    for dtype in ("f32", "bf16"):
        b = Batch(dtype, 128, [33 + 20 + 1 + 1, 4], [55, 104], page=16, seed=12)
        ks, vs, tols = b.appended()
        r = Run(pkg, b)
        want = None
        with make_ctx(pkg, 128) as ctx:
            out = cuda.zeros(b.n_tokens, b.n_q * 128, dtype=b.td, device="cuda")
            step_in = [0, 0]
            for take in ([33, 1], [20, 1], [1, 1], [1, 1]):
                rows = [b.starts[s] + step_in[s] + i for s in (0, 1) for i in range(take[s])]
                qkv = r.qkv[rows].contiguous()
                starts = cuda.tensor([0, take[0], sum(take)], dtype=cuda.int32, device="cuda")
                step_in = [a + c for a, c in zip(step_in, take)]
                lens = [b.lens[s] - b.news[s] + step_in[s] for s in (0, 1)]
                d_lens = cuda.tensor(lens, dtype=cuda.int32, device="cuda")
                o = cuda.empty(len(rows), b.n_q * 128, dtype=b.td, device="cuda")
                args = (r.kv, 2, len(rows), starts if max(take) > 1 else None, d_lens)
                ctx.paged_append(*args, qkv)
                ctx.paged_attention(*args, max(take), max(lens), qkv, o)
                out[rows] = o
                # a logit row made of the outputs: the greedy token is its largest
                tok = cuda.empty(len(rows), dtype=cuda.int32, device="cuda")
                zero = cuda.zeros(len(rows), device="cuda")
                ctx.sample(len(rows), b.n_q * 128, o, zero, None, None, None, zero, tok)
                assert cuda.equal(tok.long(), o.float().argmax(dim=1))
            assert ctx.device_status() == 0
        kp = r.kp.cpu()
        for s in (0, 1):
            assert (np.abs(b.unpool(kp, s) - ks[s]) <= tols[s]).all()
        b.set_appended()
        check_attention(b, out)


def test_streams_and_graphs(pkg, cuda):
    b = Batch("bf16", 128, [30, 1, 1], [90, 500, 40], page=16, seed=13)
    b.set_appended()
    r = Run(pkg, b)
    with make_ctx(pkg, 128) as ctx:
        want = r.attend(ctx)
        side = cuda.cuda.Stream()
        side.wait_stream(cuda.cuda.current_stream())
        out = cuda.zeros_like(want)
        r.attend(ctx, out=out, stream=side)
        side.synchronize()
        assert cuda.equal(out, want)
        graph = cuda.cuda.CUDAGraph()
        out2 = cuda.zeros_like(want)
        with cuda.cuda.graph(graph):
            r.append(ctx)
            r.attend(ctx, out=out2)
        # an eager call that needs a larger workspace, between capture and replay
        big = Batch("bf16", 128, [1] * 8, [3000] * 8, page=16, seed=14)
        rb = Run(pkg, big)
        rb.attend(ctx)
        for _ in range(3):
            out2.zero_()
            graph.replay()
            cuda.cuda.synchronize()
            assert cuda.equal(out2, want)
        assert ctx.device_status() == 0
        del graph


def test_refusals(pkg, cuda):
    b = Batch("f16", 128, [1, 1], [20, 30], page=16, seed=15)
    r = Run(pkg, b)
    out = cuda.zeros(2, 12 * 128, dtype=cuda.float16, device="cuda")
    bad = pytest.raises(pkg.GqaError)
    with make_ctx(pkg, 128) as ctx:
        ok = (r.kv, 2, 2, None, r.lens)
        with bad:
            ctx.paged_append(*ok, r.qkv.float())                       # another type
        with bad:
            ctx.paged_append(*ok, r.qkv.cpu())                         # another device
        with bad:
            ctx.paged_append(r.kv, 2, 2, None, r.lens.long(), r.qkv)   # lengths not int32
        with bad:
            ctx.paged_append(r.kv, 2, 1, None, r.lens, r.qkv)          # not one token each
        with bad:
            ctx.paged_append(r.kv, 3, 3, None, r.lens, r.qkv)          # more sequences than tables
        with bad:
            ctx.paged_append(*ok, r.qkv, qkv_stride=100)               # rows overlap
        with bad:
            ctx.paged_append(*ok, r.qkv.data_ptr() + 2, qkv_stride=2048)  # not 16-byte aligned
        with bad:
            ctx.paged_attention(*ok, 2, 30, r.qkv, out)                # max_new without q_starts
        with bad:
            ctx.paged_attention(*ok, 1, 0, r.qkv, out)
        with bad:
            ctx.paged_attention(*ok, 1, 30, r.qkv, r.qkv[:, 8:], out_stride=2048)  # overlap
        for field, value in (("dtype", 3), ("page_size", 8), ("page_size", 48), ("n_pages", 0),
                             ("max_pages", 0), ("table_stride", 1), ("row_stride", 64),
                             ("row_stride", 132), ("page_stride", 0), ("k_pages", None),
                             ("v_pages", r.kv.v_pages + 2), ("page_table", None)):
            kv = pkg.paged_kv_of(r.kp, r.vp, r.table)
            setattr(kv, field, value)
            with bad:
                ctx.paged_append(kv, 2, 2, None, r.lens.data_ptr(), r.qkv.data_ptr(),
                                 qkv_stride=2048)
        with bad:
            pkg.paged_kv_of(r.kp, r.vp.float(), r.table)
        with bad:
            pkg.paged_kv_of(r.kp, r.vp, r.table.long())
        with bad:
            pkg.paged_kv_of(r.kp, r.vp, r.table, layout="dhn")
        ctx.paged_append(r.kv, 0, 0, None, None, None)                 # nothing to do
        ctx.paged_attention(r.kv, 2, 0, None, r.lens, 1, 30, r.qkv, out)
    with make_ctx(pkg, 64) as ctx, bad:
        ctx.paged_append(r.kv, 2, 2, None, r.lens, r.qkv)              # heads of another size


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
def test_padded_pages(pkg, cuda, dtype, layout):
    """Pages, heads and rows with gaps between them, which are not touched."""
    b = Batch(dtype, 128, [40, 1, 2], [70, 90, 33], page=32, n_kv=2, layout=layout, seed=16)
    ks, vs, tols = b.appended()
    r = Run(pkg, b)
    wide = []
    for x in (r.kp, r.vp):
        w = cuda.full((x.shape[0], x.shape[1] + 1, x.shape[2] + 3, 128 + 8), 7.0, dtype=b.td,
                      device="cuda")
        w[:, :x.shape[1], :x.shape[2], :128] = x
        wide.append(w)
    view = [w[:, :x.shape[1], :x.shape[2], :128] for w, x in zip(wide, (r.kp, r.vp))]
    r.kv = pkg.paged_kv_of(*view, r.table, layout=layout)
    with make_ctx(pkg, 128) as ctx:
        r.append(ctx)
        out = r.attend(ctx)
        assert ctx.device_status() == 0
    for w, v in zip(wide, view):
        v_bits = v.clone()
        v.fill_(7.0)
        assert (w == 7).all()
        v.copy_(v_bits)
    kp, vp = (v.cpu() for v in view)
    for s in range(3):
        assert (np.abs(b.unpool(kp, s) - ks[s]) <= tols[s]).all()
        np.testing.assert_array_equal(b.unpool(vp, s), vs[s])
    b.set_appended()
    check_attention(b, out)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_more_sequences_than_threads(pkg, cuda, dtype):
    """700 sequences, some of them empty or not advanced, single tokens and chunks."""
    g = np.random.default_rng(17)
    news = g.choice([0, 1, 1, 1, 2, 5], 700).tolist()
    news[:3], news[-2:] = [0, 0, 1], [30, 0]
    lens = [n + int(t) for n, t in zip(news, g.integers(0, 40, 700))]
    b = Batch(dtype, 64, news, lens, page=16, n_kv=1, seed=18)
    b.set_appended()
    r = Run(pkg, b)
    before = r.kp.clone()
    with make_ctx(pkg, 64, 1) as ctx:
        out = r.attend(ctx)
        r.append(ctx)
        assert ctx.device_status() == 0
    check_attention(b, out)
    kp = r.kp.cpu()
    for s in range(0, 700, 13):
        assert (np.abs(b.unpool(kp, s) - b.k[s]) <=
                cuda.finfo(b.td).eps * np.abs(b.k[s]) + 1e-5).all()
    assert int(r.kp.isnan().sum()) == int(before.isnan().sum())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d,n_kv", [(128, 2), (64, 8)])
def test_long_beside_short(pkg, cuda, dtype, d, n_kv):
    """Single tokens whose rows many CTAs share beside some that one CTA holds."""
    b = Batch(dtype, d, [1] * 6, [9000, 20, 5000, 1, 700, 6001], page=64, n_kv=n_kv, seed=19)
    b.set_appended()
    r = Run(pkg, b)
    with make_ctx(pkg, d, n_kv) as ctx:
        out = r.attend(ctx)
        assert ctx.device_status() == 0
    check_attention(b, out)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_output_rows_apart(pkg, cuda, dtype):
    """Rows of the output 16 bytes off a sector's start; what lies between them stays."""
    b = Batch(dtype, 128, [50, 1, 300], [50, 400, 330], page=16, seed=20)
    b.set_appended()
    r = Run(pkg, b)
    pad = 16 // b.qkv.element_size()
    wide = cuda.full((b.n_tokens, b.n_q * 128 + pad), 7.0, dtype=b.td, device="cuda")
    with make_ctx(pkg, 128) as ctx:
        r.attend(ctx, out=wide[:, :b.n_q * 128])
        want = r.attend(ctx)
        assert ctx.device_status() == 0
    check_attention(b, wide)
    assert (wide[:, b.n_q * 128:] == 7).all()
    assert cuda.equal(wide[:, :b.n_q * 128], want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_offsets_past_32_bits(pkg, cuda, dtype):
    """Pages that lie more than 2^31 elements into their pools."""
    b = Batch(dtype, 128, [20, 1], [60, 100], page=16, seed=21)
    ks, vs, tols = b.appended()
    r = Run(pkg, b)
    far = 2 ** 31 // (2 * 16 * 128)
    pools = []
    for x in (r.kp, r.vp):
        w = cuda.empty(far + b.n_pages, 2, 16, 128, dtype=b.td, device="cuda")
        w[far:] = x
        pools.append(w)
    table = r.table + far
    r.kv = pkg.paged_kv_of(*pools, table)
    with make_ctx(pkg, 128) as ctx:
        r.append(ctx)
        out = r.attend(ctx)
        # entry -7 of Batch became a page of the pool; no row of the sequences is in it
        assert ctx.device_status() == 0
    kp, vp = (w[far:].cpu() for w in pools)
    for s in range(2):
        assert (np.abs(b.unpool(kp, s) - ks[s]) <= tols[s]).all()
        np.testing.assert_array_equal(b.unpool(vp, s), vs[s])
    b.set_appended()
    check_attention(b, out)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_overlapped_launches(pkg, cuda, dtype):
    """GQA_OPT_PDL off and on: a chain of calls, each of which needs the one before it."""
    b = Batch(dtype, 128, [40, 1, 1], [90, 500, 40], page=16, seed=22)
    outs = []
    for pdl in (0, 1):
        r = Run(pkg, b)
        with make_ctx(pkg, 128) as ctx:
            ctx.set_option(pkg.gqa.GQA_OPT_PDL, pdl)
            for _ in range(20):
                # the output is the next call's qkv (q | the same k and v)
                r.append(ctx)
                r.attend(ctx, out=r.qkv)
            tok = cuda.empty(b.n_tokens, dtype=cuda.int32, device="cuda")
            u = cuda.full((b.n_tokens,), 0.5, device="cuda")
            ctx.sample(b.n_tokens, b.n_q * 128, r.qkv, None, None, None, None, u, tok)
            assert ctx.device_status() == 0
        outs.append((r.kp, r.vp, r.qkv, tok))
    for x, y in zip(*outs):
        assert cuda.equal(cuda.nan_to_num(x.float(), 9.0), cuda.nan_to_num(y.float(), 9.0))


def test_two_contexts_at_once(pkg, cuda):
    """Two contexts on two streams do not share a workspace."""
    bs = [Batch("bf16", 128, [60, 1, 1], [800, 3000, 40], page=16, seed=23 + i) for i in (0, 1)]
    runs = []
    for b in bs:
        b.set_appended()
        runs.append(Run(pkg, b))
    streams = [cuda.cuda.Stream() for _ in bs]
    ctxs = [make_ctx(pkg, 128) for _ in bs]
    outs = [cuda.zeros(b.n_tokens, b.n_q * 128, dtype=b.td, device="cuda") for b in bs]
    cuda.cuda.synchronize()
    for _ in range(20):
        for r, st, ctx, out in zip(runs, streams, ctxs, outs):
            r.attend(ctx, out=out, stream=st)
    cuda.cuda.synchronize()
    for b, ctx, out in zip(bs, ctxs, outs):
        assert ctx.device_status() == 0
        check_attention(b, out)
        ctx.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("d", [128, 64])
def test_units_of_one_and_two_tiles(pkg, cuda, dtype, d):
    """Chunks that end in one tile or in two, in a mixed order, many of them per CTA; every run
    gives the same bits."""
    g = np.random.default_rng(24)
    tok = 128 // {128: 6, 64: 7}[d]
    news = g.choice([2, 5, tok, tok + 1, 2 * tok - 1, 2 * tok, 2 * tok + 1, 3 * tok, 4 * tok + 1],
                    120).tolist()
    lens = [n + int(t) for n, t in zip(news, g.choice([0, 0, 3, 90, 128, 300, 700], 120))]
    b = Batch(dtype, d, news, lens, page=64, n_kv=4, seed=25)
    b.set_appended()
    r = Run(pkg, b)
    with make_ctx(pkg, d, 4) as ctx:
        out = r.attend(ctx)
        for _ in range(10):
            assert cuda.equal(r.attend(ctx), out)
        assert ctx.device_status() == 0
    check_attention(b, out)


def test_tensors_too_small_for_their_stride(pkg, cuda):
    """Rows that would lie past a tensor's end are refused; tensors of other shapes that hold them
    are taken."""
    b = Batch("f32", 128, [1, 1, 1], [20, 30, 40], page=16, seed=26)
    b.set_appended()
    r = Run(pkg, b)
    out = cuda.zeros(3, 12 * 128, device="cuda")
    logits = cuda.zeros(3, 100, device="cuda")
    u = cuda.zeros(3, device="cuda")
    tok = cuda.zeros(3, dtype=cuda.int32, device="cuda")
    with make_ctx(pkg, 128) as ctx:
        args = (r.kv, 3, 3, None, r.lens)
        bad = pytest.raises(pkg.GqaError)
        with bad:
            ctx.paged_append(*args, r.qkv, qkv_stride=4096)
        with bad:
            ctx.paged_append(*args, r.qkv[:2].reshape(-1))
        with bad:
            ctx.paged_attention(*args, 1, 40, r.qkv, out[:2].reshape(-1))
        with bad:
            ctx.paged_attention(*args, 1, 40, r.qkv, out, out_stride=2048)
        with bad:
            ctx.sample(3, 100, logits, None, None, None, None, u, tok, logits_stride=128)
        with bad:
            ctx.sample(3, 100, logits, None, None, None, None, u[:2], tok)
        want = r.attend(ctx)
        heads = cuda.zeros(3, 12, 128, device="cuda")
        ctx.paged_attention(*args, 1, 40, r.qkv.reshape(-1), heads)
        assert cuda.equal(heads.reshape(3, -1), want)
        wide = cuda.zeros(3, 2048, device="cuda")
        ctx.paged_attention(*args, 1, 40, r.qkv, wide[:, :1536], out_stride=2048)
        assert cuda.equal(wide[:, :1536], want)
        assert ctx.device_status() == 0


def test_empty_batches(pkg, cuda):
    """Steps in which no sequence brings a token, as tensors of no rows."""
    b = Batch("bf16", 128, [1, 1], [20, 30], page=16, seed=27)
    r = Run(pkg, b)
    before = r.kp.clone()
    starts = cuda.zeros(3, dtype=cuda.int32, device="cuda")
    none = r.qkv[:0]
    out = cuda.empty(0, 12 * 128, dtype=b.td, device="cuda")
    with make_ctx(pkg, 128) as ctx:
        ctx.paged_append(r.kv, 2, 0, starts, r.lens, none)
        ctx.paged_attention(r.kv, 2, 0, starts, r.lens, 1, 30, none, out)
        ctx.paged_append(r.kv, 0, 0, None, r.lens[:0], none)
        empty = cuda.empty(0, device="cuda")
        ctx.sample(0, 100, cuda.empty(0, 100, device="cuda"), empty, None, None, None, empty,
                   r.lens[:0])
        assert ctx.device_status() == 0
    assert cuda.equal(r.kp.isnan(), before.isnan())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_graphs_replayed_with_other_lengths(pkg, cuda, dtype):
    """Two captured graphs of one context, replayed in turn while the plan in device memory (which
    sequences bring how many tokens, lengths, pages) changes under them."""
    plans = [([30, 1, 1, 0], [90, 500, 40, 0]), ([1, 1, 28, 2], [1, 900, 700, 2]),
             ([8, 8, 8, 8], [8, 8, 300, 1000]), ([1, 1, 1, 1], [64, 1, 1024, 17])]
    batches = [Batch(dtype, 128, *p, page=16, seed=30 + i) for i, p in enumerate(plans)]
    for b in batches:
        b.set_appended()
    runs = [Run(pkg, b, one=False) for b in batches]
    n_pages = max(b.n_pages for b in batches)
    cols = max(b.table.shape[1] for b in batches)
    kp, vp = (cuda.zeros(n_pages, 2, 16, 128, dtype=batches[0].td, device="cuda") for _ in "kv")
    table = cuda.zeros(4, cols, dtype=cuda.int32, device="cuda")
    lens = cuda.zeros(4, dtype=cuda.int32, device="cuda")
    starts = cuda.zeros(5, dtype=cuda.int32, device="cuda")
    qkv = cuda.zeros(32, batches[0].qkv.shape[1], dtype=batches[0].td, device="cuda")
    outs = [cuda.zeros(32, 12 * 128, dtype=batches[0].td, device="cuda") for _ in range(2)]
    kv = pkg.paged_kv_of(kp, vp, table)
    with make_ctx(pkg, 128) as ctx:
        graphs = []
        for out in outs:
            g = cuda.cuda.CUDAGraph()
            with cuda.cuda.graph(g):
                ctx.paged_append(kv, 4, 32, starts, lens, qkv)
                ctx.paged_attention(kv, 4, 32, starts, lens, 32, 1024, qkv, out)
            graphs.append(g)
        for turn in range(8):
            b, r = batches[turn % 4], runs[turn % 4]
            kp[:b.n_pages], vp[:b.n_pages] = r.kp, r.vp
            table[:, :b.table.shape[1]] = r.table
            lens.copy_(r.lens)
            starts.copy_(r.starts)
            qkv[:b.n_tokens] = r.qkv
            out = outs[turn % 2]
            out.fill_(7.0)
            graphs[turn % 2].replay()
            cuda.cuda.synchronize()
            assert ctx.device_status() == 0
            check_attention(b, out)
            assert (out[b.n_tokens:] == 7).all()
        del graphs
