"""Where the rows of out may lie beside those of qkv: any place that no row of qkv covers."""
import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

from paged_ref import Batch

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(REPO, "macbook-hardware-linux-lab_b200", "csrc")

SOURCE = r"""
#include "gqa_paged_launch.cuh"
extern "C" int apart(unsigned long long a, long long as, long long aw, unsigned long long b,
                     long long bs, long long bw, int n) {
  return gqa::rows_apart(a, as, aw, b, bs, bw, n);
}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    d = tmp_path_factory.mktemp("overlap")
    src, lib = str(d / "overlap.cu"), str(d / "overlap.so")
    with open(src, "w") as f:
        f.write(SOURCE)
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-shared",
                    "-Xcompiler", "-fPIC", "-I", CSRC, "-I", os.path.join(REPO, "include"), "-o",
                    lib, src], check=True)
    fn = ctypes.CDLL(lib).apart
    ull, ll = ctypes.c_ulonglong, ctypes.c_longlong
    fn.argtypes = [ull, ll, ll, ull, ll, ll, ctypes.c_int]
    return fn


def test_against_the_bytes(host):
    """Every pair of places of a few rows, against the sets of bytes that they cover.  Rows of
    different strides may be refused although they do not touch, never the other way round."""
    g = np.random.default_rng(0)
    told = 0
    for _ in range(4000):
        n = int(g.integers(1, 6))
        aw, bw = (int(g.integers(1, 12)) for _ in "ab")
        stride_a = aw + int(g.integers(0, 16))
        stride_b = stride_a if g.random() < 0.6 else bw + int(g.integers(0, 16))
        if stride_b < bw:
            continue
        a, b = 200, 200 + int(g.integers(-90, 90))
        cover = [{s + i * st + j for i in range(n) for j in range(w)}
                 for s, st, w in ((a, stride_a, aw), (b, stride_b, bw))]
        want = not (cover[0] & cover[1])
        got = bool(host(a, stride_a, aw, b, stride_b, bw, n))
        assert want or not got
        if stride_a == stride_b and n > 1 and abs(b - a) < (n - 1) * stride_a:
            assert got == want  # (beside each other over their whole length)
            told += want
    assert told > 100


def test_extents_end_with_the_last_row(host):
    # the padding behind the last row belongs to neither
    assert host(0, 100, 30, 330, 100, 30, 4) == 1
    assert host(330, 100, 30, 0, 100, 30, 4) == 1
    assert host(0, 100, 30, 329, 50, 30, 4) == 0
    # one row: its stride does not matter
    assert host(0, 1 << 39, 30, 30, 1 << 39, 30, 1) == 1
    # sizes beyond 64 bits
    far = 1 << 46
    assert host(far, (1 << 40) - 16, 4096, far + 4096, (1 << 40) - 16, 4096, 1 << 24) == 1
    assert host(far, (1 << 40) - 16, 4096, far + 4080, (1 << 40) - 16, 4096, 1 << 24) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("first", ["qkv", "out"])
def test_rows_beside_each_other(pkg, cuda, dtype, first):
    """qkv and out as columns of one buffer, and as columns whose padding reaches past it."""
    from test_paged_gpu import Run, check_attention, make_ctx
    b = Batch(dtype, 128, [40, 1, 3], [90, 300, 20], page=16, seed=70)
    b.set_appended()
    r = Run(pkg, b)
    wide, own = b.qkv.shape[1], b.n_q * 128
    buf = cuda.full((b.n_tokens, wide + own), 7.0, dtype=b.td, device="cuda")
    at = (0, wide) if first == "qkv" else (own, 0)
    qkv, out = buf[:, at[0]:at[0] + wide], buf[:, at[1]:at[1] + own]
    qkv.copy_(r.qkv)
    with make_ctx(pkg, 128) as ctx:
        want = r.attend(ctx)
        args = (r.kv, r.n_seq, b.n_tokens, r.starts, r.lens, max(b.news), max(b.lens))
        ctx.paged_attention(*args, qkv, out)
        assert cuda.equal(out, want) and cuda.equal(qkv, r.qkv)
        check_attention(b, out)
        # rows that share a column stay refused
        with pytest.raises(pkg.GqaError):
            ctx.paged_attention(*args, qkv, buf[:, 8:8 + own], out_stride=wide + own)
        assert ctx.device_status() == 0
