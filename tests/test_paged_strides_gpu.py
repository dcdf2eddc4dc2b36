"""Strides of the pools and of the calls' rows: any order of pages, heads and rows, and the largest."""
import pytest

from paged_ref import Batch
from test_paged_gpu import Run, check_attention, make_ctx

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("order", [(1, 0, 2, 3), (1, 2, 0, 3), (2, 0, 1, 3), (2, 1, 0, 3)])
def test_any_order_of_pages_heads_and_rows(pkg, cuda, dtype, order):
    """Pools whose memory holds [head][page][row], [head][row][page], [row][page][head] and
    [row][head][page]."""
    b = Batch(dtype, 128, [40, 1, 2], [70, 90, 33], page=32, n_kv=2, seed=80)
    b.set_appended()
    r = Run(pkg, b)
    with make_ctx(pkg, 128) as ctx:
        r.append(ctx)
        want = r.attend(ctx)
        back = sorted(range(4), key=lambda i: order[i])
        kp, vp = (x.permute(order).contiguous().permute(back) for x in (r.kp, r.vp))
        assert kp.shape == r.kp.shape and kp.stride() != r.kp.stride()
        r.kv = pkg.paged_kv_of(kp, vp, r.table)
        assert cuda.equal(r.attend(ctx), want)
        r.append(ctx)
        assert ctx.device_status() == 0
        assert cuda.equal(kp.nan_to_num(9.0), r.kp.nan_to_num(9.0))
    check_attention(b, want)


def test_strides_beyond_the_largest_are_refused(pkg, cuda):
    """Before any launch: a call in place would otherwise have turned its q already."""
    b = Batch("bf16", 128, [3, 1], [20, 30], page=16, seed=81)
    b.set_appended()
    r = Run(pkg, b)
    q = r.qkv.clone()
    ptr = (r.starts.data_ptr(), r.lens.data_ptr())
    with make_ctx(pkg, 128) as ctx:
        for field in ("page_stride", "head_stride", "row_stride", "table_stride"):
            for stride in (1 << 39, 1 << 40, 1 << 62):
                kv = pkg.paged_kv_of(r.kp, r.vp, r.table)
                setattr(kv, field, stride)
                with pytest.raises(pkg.GqaError) as e:
                    ctx.paged_attention(kv, 2, 4, *ptr, 3, 30, q.data_ptr(), q.data_ptr(),
                                        qkv_stride=2048, out_stride=2048)
                assert e.value.code == pkg.gqa.GQA_ERR_INVALID_ARG
        for kw in ({"qkv_stride": 1 << 39, "out_stride": 2048},
                   {"qkv_stride": 2048, "out_stride": 1 << 39},
                   {"qkv_stride": 1 << 62, "out_stride": 1 << 62}):
            with pytest.raises(pkg.GqaError):
                ctx.paged_attention(r.kv, 2, 4, *ptr, 3, 30, q.data_ptr(), q.data_ptr(), **kw)
        tok = cuda.zeros(2, dtype=cuda.int32, device="cuda")
        u = cuda.zeros(2, device="cuda")
        with pytest.raises(pkg.GqaError):
            ctx.sample(2, 100, q.data_ptr(), None, None, None, None, u, tok,
                       logits_stride=1 << 39, dtype=pkg.gqa.BF16)
        assert ctx.device_status() == 0
    assert cuda.equal(q, r.qkv)
