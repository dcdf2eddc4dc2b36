"""Sampling against its definition in 64 bits (tests/paged_ref.py): tokens have to be equal."""
import math

import numpy as np
import pytest

from paged_ref import DTYPES, sample_row

pytestmark = pytest.mark.gpu


def run(pkg, torch, x, t, k, p, m, u, **kw):
    """x [rows, vocab] tensor; the settings as lists or None."""
    rows, vocab = x.shape[0], kw.pop("vocab", x.shape[1])
    dev = lambda v, ty: None if v is None else torch.tensor(v, dtype=ty).cuda()  # noqa: E731
    tok = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    with pkg.Context() as ctx:
        ctx.sample(rows, vocab, x.cuda(), dev(t, torch.float32), dev(k, torch.int32),
                   dev(p, torch.float32), dev(m, torch.float32), dev(u, torch.float32), tok, **kw)
        assert ctx.device_status() == 0
    got = tok.cpu().numpy()
    f = lambda v, i, d: d if v is None else float(np.float32(v[i]))  # noqa: E731
    want = [sample_row(x[i, :vocab].double().numpy(), f(t, i, 1.0), 0 if k is None else k[i],
                       f(p, i, 1.0), f(m, i, 0.0), f(u, i, 0.0)) for i in range(rows)]
    np.testing.assert_array_equal(got, want)
    return got


def settings(rows, vocab, seed):
    g = np.random.default_rng(seed)
    t = np.where(g.random(rows) < 0.1, 0.0, 0.3 + 1.2 * g.random(rows))
    k = np.where(g.random(rows) < 0.5, 0, g.integers(1, vocab + 2, rows))
    k[::5] = np.minimum(40, vocab)
    p = np.where(g.random(rows) < 0.4, 1.0, g.random(rows))
    m = np.where(g.random(rows) < 0.6, 0.0, 0.2 * g.random(rows))
    u = g.random(rows)
    return [v.tolist() for v in (t, k.astype(int), p, m, u)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (40, 33), (64, 1000), (24, 4097),
                                        (9, 50257), (5, 151936)])
def test_random_rows(pkg, cuda, dtype, rows, vocab):
    g = np.random.default_rng(vocab)
    x = cuda.from_numpy(g.standard_normal((rows, vocab)) * 3).to(DTYPES[dtype])
    run(pkg, cuda, x, *settings(rows, vocab, rows))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_spread_rows(pkg, cuda, dtype):
    """Rows from nearly flat to one token far above the rest, with strides that are not dense."""
    g = np.random.default_rng(5)
    vocab = 5003
    width = [1e-3, 0.1, 1, 5, 20, 100] * 6
    x = np.stack([g.standard_normal(vocab + 13) * w for w in width])
    x = cuda.from_numpy(x).to(DTYPES[dtype]).cuda()
    st = settings(len(width), vocab, 6)
    got = run(pkg, cuda, x.cpu()[:, :vocab].contiguous(), *st)
    tok = cuda.empty(len(width), dtype=cuda.int32, device="cuda")
    dev = [cuda.tensor(v, dtype=cuda.int32 if i == 1 else cuda.float32).cuda()
           for i, v in enumerate(st)]
    with pkg.Context() as ctx:
        ctx.sample(len(width), vocab, x, *dev, tok)
    np.testing.assert_array_equal(tok.cpu().numpy(), got)


@pytest.mark.parametrize("levels", [1, 2, 7])
def test_ties_go_to_the_lowest_id(pkg, cuda, levels):
    """A few distinct logits: every border falls among ties."""
    g = np.random.default_rng(levels)
    rows, vocab = 48, 777
    x = cuda.from_numpy(g.integers(0, levels, (rows, vocab)).astype(np.float32))
    st = settings(rows, vocab, 7)
    # cumulative weights of exact ties can meet top_p times their total exactly; a top_p that is
    # no multiple of a tie's share keeps the border inside a token in any arithmetic
    st[2] = [min(1.0, v) if v == 1 else 0.05 + 0.9 * v for v in st[2]]
    run(pkg, cuda, x, *st)


def test_signed_zeros_tie(pkg, cuda):
    x = cuda.zeros(4, 50)
    x[:, ::2] = -0.0
    run(pkg, cuda, x, [1.0] * 4, [1, 2, 3, 10], None, None, [0.0, 0.99, 0.5, 0.95])


def test_uniform_at_its_ends(pkg, cuda):
    x = cuda.randn(6, 300, generator=cuda.Generator().manual_seed(1))
    u = [0.0, 1 - 2.0 ** -24, 2.0 ** -24, 0.5, 1.0, -0.0]
    run(pkg, cuda, x, [1.0] * 6, None, None, None, u)
    run(pkg, cuda, x, None, [300] * 6, [1.0] * 6, [0.0] * 6, u)


def test_filters_at_their_ends(pkg, cuda):
    x = cuda.randn(8, 500, generator=cuda.Generator().manual_seed(2))
    u = [0.0, 0.3, 0.6, 0.9] * 2
    run(pkg, cuda, x, None, [1] * 8, None, None, u)
    run(pkg, cuda, x, None, [-3] * 8, None, None, u)
    run(pkg, cuda, x, None, [500, 501, 499, 2] * 2, None, None, u)
    run(pkg, cuda, x, None, None, [0.0, -1.0, 1e-30, 0.9999999] * 2, None, u)
    run(pkg, cuda, x, None, None, None, [1.0, 2.0, 1e-30, -1.0] * 2, u)
    run(pkg, cuda, x, [1e-30, 1e30, 1e-3, 100.0] * 2, None, [0.5] * 8, None, u)
    run(pkg, cuda, x, [0.0, -1.0, math.nan, 0.0] * 2, [3] * 8, None, None, u)


def test_infinities_and_nan(pkg, cuda):
    g = cuda.Generator().manual_seed(3)
    x = cuda.randn(12, 400, generator=g)
    x[0] = -math.inf
    x[1, 1:] = -math.inf
    x[2, ::3] = -math.inf
    x[3, 50] = math.inf
    x[4, 50:60] = math.inf
    x[5, ::2] = math.nan
    x[6] = math.nan
    x[7, 10] = math.nan
    x[8, :] = cuda.finfo(cuda.float32).min
    x[9, 5:] = cuda.finfo(cuda.float32).min
    x[10, 7] = cuda.finfo(cuda.float32).max
    u = [0.7] * 12
    for k, p, m in ((None, None, None), ([300] * 12, None, None), (None, [0.9] * 12, None),
                    ([5] * 12, [0.5] * 12, [0.1] * 12)):
        run(pkg, cuda, x, [0.8] * 12, k, p, m, u)
    run(pkg, cuda, x, [0.0] * 12, None, None, None, u)


@pytest.mark.parametrize("vocab", [3000, 60001, 500000])
def test_top_k_beyond_the_weighted(pkg, cuda, vocab):
    """A top_k that takes in every logit with a weight, on one CTA and on clusters of them, and
    a vocabulary of which a part stays in memory."""
    g = np.random.default_rng(10)
    x = cuda.from_numpy(g.standard_normal((12, vocab)).astype(np.float32) * 3)
    u = g.random(12).tolist()
    for p, m in ((None, None), ([0.8] * 12, None), (None, [0.01] * 12)):
        run(pkg, cuda, x, [0.02] * 6 + [0.9] * 6, [2500] * 11 + [vocab - 1], p, m, u)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_largest_vocabulary_off_alignment(pkg, cuda, dtype):
    """Rows that start off a 16-byte boundary, at the limit of the vocabulary."""
    g = cuda.Generator().manual_seed(4)
    vocab = pkg.gqa.SAMPLE_MAX_VOCAB
    x = (cuda.randn(3, vocab + 3, generator=g) * 2).to(DTYPES[dtype]).cuda()
    u = cuda.tensor([0.999999, 0.5, 0.25], device="cuda")
    p = cuda.tensor([1.0, 0.9, 1.0], device="cuda")
    k = cuda.tensor([0, 0, 5000], dtype=cuda.int32, device="cuda")
    tok = cuda.empty(3, dtype=cuda.int32, device="cuda")
    with pkg.Context() as ctx:
        ctx.sample(3, vocab, x[:, 1:], None, k, p, None, u, tok)
    want = [sample_row(x[i, 1:vocab + 1].double().cpu().numpy(), 1.0, int(k[i]), float(p[i]), 0.0,
                       float(u[i])) for i in range(3)]
    np.testing.assert_array_equal(tok.cpu().numpy(), want)


def test_high_temperature(pkg, cuda):
    """All logits within a few steps of the exponent: the steps are cut again by the logits."""
    g = np.random.default_rng(11)
    x = cuda.from_numpy(g.standard_normal((10, 40000)).astype(np.float32))
    u = g.random(10).tolist()
    t = [100.0, 1e4, 1e30, 300.0, 50.0] * 2
    run(pkg, cuda, x, t, [20000, 7] * 5, None, None, u)
    run(pkg, cuda, x, t, None, [0.5, 0.9] * 5, None, u)
    run(pkg, cuda, x, t, [30000, 600] * 5, [0.7, 0.1] * 5, None, u)
    run(pkg, cuda, cuda.zeros(10, 40000), t, [20000, 7] * 5, [0.37, 0.71] * 5, None, u)


def test_distribution(pkg, cuda):
    """Evenly spaced uniform numbers give each token its share, to one number each way."""
    rows = 4096
    x = cuda.tensor([[0.0, 1.0, 2.0, -1.0, 0.5]]).expand(rows, 5).contiguous()
    u = ((np.arange(rows) + 0.5) / rows).tolist()
    got = run(pkg, cuda, x, [1.0] * rows, None, None, None, u)
    w = np.exp(x[0].double().numpy())
    assert (np.abs(np.bincount(got, minlength=5) - rows * w / w.sum()) <= 1).all()


def test_agrees_with_the_greedy_pick(pkg, cuda):
    """Temperature 0 gives the token that gqa_lm_head picks from the same logits."""
    g = np.random.default_rng(9)
    vocab = 1000
    q6k = g.integers(0, 256, (vocab * 6, 210), dtype=np.uint8)
    q6k[:, 208:] = np.frombuffer(np.float16(0.01).tobytes(), np.uint8)
    with pkg.Context() as ctx:
        packed = cuda.empty(ctx.lm_head_packed_bytes(vocab), dtype=cuda.uint8, device="cuda")
        ctx.lm_head_pack(cuda.from_numpy(q6k).cuda(), vocab, packed)
        state = cuda.randn(1536, device="cuda")
        gamma = cuda.ones(1536, device="cuda")
        logits = cuda.empty(1, vocab, device="cuda")
        pick = cuda.empty(1, dtype=cuda.int32, device="cuda")
        ctx.lm_head(packed, vocab, gamma, state, logits, pick)
        tok = cuda.empty(1, dtype=cuda.int32, device="cuda")
        zero = cuda.zeros(1, device="cuda")
        ctx.sample(1, vocab, logits, zero, None, None, None, zero, tok)
        assert int(tok) == int(pick) == int(logits.argmax())


def test_streams_and_graphs(pkg, cuda):
    x = cuda.randn(5, 3000, device="cuda")
    u = cuda.rand(5, device="cuda")
    k = cuda.full((5,), 50, dtype=cuda.int32, device="cuda")
    p = cuda.full((5,), 0.9, device="cuda")
    want, tok = (cuda.empty(5, dtype=cuda.int32, device="cuda") for _ in range(2))
    with pkg.Context() as ctx:
        ctx.sample(5, 3000, x, None, k, p, None, u, want)
        side = cuda.cuda.Stream()
        side.wait_stream(cuda.cuda.current_stream())
        ctx.sample(5, 3000, x, None, k, p, None, u, tok, stream=side)
        side.synchronize()
        assert cuda.equal(tok, want)
        graph = cuda.cuda.CUDAGraph()
        with cuda.cuda.graph(graph):
            ctx.sample(5, 3000, x, None, k, p, None, u, tok)
        for _ in range(2):
            tok.fill_(-1)
            graph.replay()
            cuda.cuda.synchronize()
            assert cuda.equal(tok, want)
        del graph


def test_refusals(pkg, cuda):
    x = cuda.randn(4, 100, device="cuda")
    u = cuda.rand(4, device="cuda")
    tok = cuda.empty(4, dtype=cuda.int32, device="cuda")
    bad = pytest.raises(pkg.GqaError)
    with pkg.Context() as ctx:
        none = (None, None, None, None)
        with bad:
            ctx.sample(5, 100, x, *none, u, tok)                       # more rows than there are
        with bad:
            ctx.sample(4, 101, x, *none, u, tok)
        with bad:
            ctx.sample(4, 0, x, *none, u, tok)
        with bad:
            ctx.sample(4, pkg.gqa.SAMPLE_MAX_VOCAB + 1, x.data_ptr(), *none, u, tok,
                       dtype=pkg.gqa.F32)
        with bad:
            ctx.sample(4, 100, x.double(), *none, u, tok)
        with bad:
            ctx.sample(4, 100, x, *none, u.cpu(), tok)
        with bad:
            ctx.sample(4, 100, x, *none, None, tok)
        with bad:
            ctx.sample(4, 100, x, *none, u, tok.long())
        with bad:
            ctx.sample(4, 100, x, *none, u[:3], tok)
        with bad:
            ctx.sample(4, 100, x, None, u, None, None, u, tok)         # top_k not int32
        with bad:
            ctx.sample(4, 100, x, *none, u, tok, logits_stride=99)
        with bad:
            ctx.sample(4, 50, x[:, ::2], *none, u, tok)                # not dense
        with bad:
            ctx.sample(4, 100, x.data_ptr() + 2, *none, u, tok, logits_stride=100,
                       dtype=pkg.gqa.F32)
        ctx.sample(0, 100, x, *none, u, tok)                           # nothing to do


@pytest.mark.parametrize("rows,vocab", [(1100, 501), (513, 30000)])
def test_rows_that_take_turns(pkg, cuda, rows, vocab):
    """More rows than run at once, of every kind of settings: each is written once, by itself."""
    g = np.random.default_rng(rows)
    x = cuda.from_numpy(g.standard_normal((rows, vocab)) * 2).float()
    st = settings(rows, vocab, 30)
    st[1][1::7] = [vocab // 2] * len(st[1][1::7])
    run(pkg, cuda, x, *st)
    alike = [[1.0] * rows, [0] * rows, [1.0] * rows, [0.0] * rows, g.random(rows).tolist()]
    run(pkg, cuda, x, *alike)
