"""A key that takes nearly all the weight, and a long tail of keys whose small weights add up."""
import math

import numpy as np
import pytest

from paged_ref import Batch
from test_paged_gpu import Run, make_ctx

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [128, 64])
@pytest.mark.parametrize("score", [16.0, 17.6, 19.0])
def test_small_weights_add_up(pkg, cuda, dtype, d, score):
    """V is 0 at the dominant key and 64 at all others, which score 0: an output is 64 times the
    tail's share.  Weights of e^-16 to e^-19 of the largest lie below fp16's smallest numbers."""
    n_seq, rows, n_kv = 120, 300, 4
    news = [2] * (n_seq // 2) + [1] * (n_seq // 2)
    b = Batch(dtype, d, news, [rows] * n_seq, page=64, n_kv=n_kv, seed=60)
    # only the slowest pair of a head turns, by less than 1e-3 over these rows
    e, width = d // 2 - 1, b.n_q * d
    b.qkv[:] = 0
    b.qkv[:, e:width:d] = 8.0
    b.qkv[:, width + n_kv * d:] = 64.0
    for s in range(n_seq):
        at = (0, 130, 290)[s % 3]
        b.k[s][:] = 0
        b.k[s][at, :, e] = score * math.sqrt(d) / 8.0
        b.k[s] = b._cast(b.k[s])
        b.v[s][:] = 64
        b.v[s][at] = 0
    b.set_appended()
    want, _ = b.attend()
    r = Run(pkg, b)
    with make_ctx(pkg, d, n_kv) as ctx:
        got = r.attend(ctx).double().cpu().numpy().reshape(want.shape)
        assert ctx.device_status() == 0
    # A tail's weight w is off by half of fp16's smallest step at 2^7 (single tokens) or 2^8
    # times its value, all alike; chunks round it and q (half a step each, the latter times the
    # score); single tokens hold both in two terms (half a step squared).  The output is rounded
    # once, and fp32 sums of 300 terms are off by less than 2^-14.
    h = cuda.finfo(b.td).eps / 2
    w = math.exp(-float(b.k[0].max()) * 8.0 / math.sqrt(d))
    low = 0.0 if dtype == "bf16" else 1.0
    for s, n in enumerate(news):
        at = slice(b.starts[s], b.starts[s + 1])
        own = low * 2.0 ** -33 / w + h + 1.01 * math.expm1(score * h) if n > 1 else \
            low * 2.0 ** -32 / w + (1 + score) * h * h
        tol = want[at] * (own + 2.0 ** -14 + h) + (2.0 ** -25 if dtype == "f16" else 0)
        assert (np.abs(got[at] - want[at]) <= tol).all(), (s, got[at][0, 0, 0], want[at][0, 0, 0])
