"""Attention over page tables with entries outside the pool: their rows are not attended, wherever
they lie in a chunk's key tiles and units, and every run gives the same bits."""
import numpy as np
import pytest

from paged_ref import Batch
from test_paged_gpu import Run, check_attention, make_ctx

pytestmark = pytest.mark.gpu

# (new tokens, rows, rows whose page's entry is bad).  Chunks that end 1..8 and 9..15 rows into a
# 16-row part whose entry is bad, bad entries first, in the middle and last, all of them, one under
# the end of a unit (21 or 18 tokens: rows 90 + 21 and 90 + 18), and single tokens.
CASES = [(10, 21, [20]), (12, 28, [27]), (2, 17, [16]), (7, 24, [16]), (30, 75, [0]),
         (25, 100, [50]), (5, 40, range(40)), (60, 150, [111]), (60, 150, [107]), (43, 133, [129]),
         (2, 300, [299]), (1, 90, [89]), (1, 40, [3]), (150, 400, [130, 270, 399]), (4, 4, []),
         (70, 70, [33])]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("d", [128, 64])
@pytest.mark.parametrize("page,layout", [(16, "hnd"), (64, "nhd"), (256, "hnd")])
def test_bad_entries_in_chunks(pkg, cuda, dtype, d, page, layout):
    b = Batch(dtype, d, [c[0] for c in CASES], [c[1] for c in CASES], page=page, layout=layout,
              seed=40)
    b.set_appended()
    bad = [{r // page for r in c[2]} for c in CASES]
    for s, pages in enumerate(bad):
        for i, p in enumerate(sorted(pages)):
            b.table[s, p] = (-1, b.n_pages, 2 ** 31 - 1, -2 ** 31)[(s + i) % 4]
    r = Run(pkg, b)
    with make_ctx(pkg, d) as ctx:
        out = r.attend(ctx)
        assert ctx.device_status() == pkg.gqa.STATUS_BAD_PAGE
        for _ in range(10):
            assert cuda.equal(r.attend(ctx), out)
    check_attention(b, out, skip=lambda s, t: t // page in bad[s])
    none = [t for s, c in enumerate(CASES) for t in range(b.starts[s], b.starts[s + 1])
            if all(row // page in bad[s] for row in range(c[1] - c[0] + t - b.starts[s] + 1))]
    assert len(none) >= 5 and (out[none] == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("length", [17, 20, 24, 25, 31])
def test_last_entry_bad_many_times(pkg, cuda, dtype, length):
    """Many chunks alike, all of which end in a page without an entry: what the last rows weigh
    does not depend on which warp is faster."""
    n = 96
    b = Batch(dtype, 128, [9] * n, [length] * n, page=16, n_kv=4, seed=41)
    b.set_appended()
    b.table[:, 1] = -1
    r = Run(pkg, b)
    with make_ctx(pkg, 128, 4) as ctx:
        out = r.attend(ctx)
        for _ in range(20):
            assert cuda.equal(r.attend(ctx), out)
        assert ctx.device_status() == pkg.gqa.STATUS_BAD_PAGE
    check_attention(b, out, skip=lambda s, t: t >= 16)
