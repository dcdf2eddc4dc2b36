"""Where the paged operators' kernels place tokens and look for rows (csrc/gqa_paged.cuh): the same
functions, compiled for the host, against the definitions in include/gqa.h; and the calls that need
no device to be refused."""
import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(REPO, "macbook-hardware-linux-lab_b200", "csrc")

SOURCE = r"""
#include "gqa_paged.cuh"
using namespace gqa;
static PagedView view(const int* table, long long table_stride, int shift, int n_pages,
                      int max_pages) {
  PagedView v{};
  v.table = table;
  v.table_stride = table_stride;
  v.page_shift = shift;
  v.n_pages = n_pages;
  v.max_pages = max_pages;
  return v;
}
extern "C" int place(const int* starts, const int* lens, int n_seq, int n_tokens, int shift,
                     int max_pages, int s, int tok, int* out) {
  return place_token(TokenPlan{starts, lens, n_seq, n_tokens}, view(nullptr, 0, shift, 1, max_pages),
                     s, tok, out[0], out[1], out[2]);
}
extern "C" int page(const int* table, long long table_stride, int shift, int n_pages, int s,
                    int row) {
  return page_of(view(table, table_stride, shift, n_pages, 1 << 20), s, row);
}
extern "C" long long offset(long long ps, long long hs, long long rs, int shift, int page, int h,
                            int row) {
  PagedView v = view(nullptr, 0, shift, 1, 1);
  v.page_stride = ps;
  v.head_stride = hs;
  v.row_stride = rs;
  return row_offset(v, page, h, row);
}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    d = tmp_path_factory.mktemp("plan")
    src, lib = str(d / "plan.cu"), str(d / "plan.so")
    with open(src, "w") as f:
        f.write(SOURCE)
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-shared",
                    "-Xcompiler", "-fPIC", "-I", CSRC, "-I", os.path.join(REPO, "include"), "-o",
                    lib, src], check=True)
    h = ctypes.CDLL(lib)
    h.offset.restype = ctypes.c_longlong
    h.offset.argtypes = [ctypes.c_longlong] * 3 + [ctypes.c_int] * 4
    h.page.argtypes = [ctypes.c_void_p, ctypes.c_longlong] + [ctypes.c_int] * 4
    return h


def ints(x):
    return np.ascontiguousarray(x, np.int32)


def place(host, starts, lens, shift, max_pages, s, tok):
    out = ints([-1, -1, -1])
    starts = None if starts is None else ints(starts)
    lens = ints(lens)
    n_tokens = int(starts[-1]) if starts is not None else len(lens)
    rc = host.place(ctypes.c_void_p(None if starts is None else starts.ctypes.data),
                    ctypes.c_void_p(lens.ctypes.data), len(lens), n_tokens, shift, max_pages, s,
                    tok, ctypes.c_void_p(out.ctypes.data))
    return (rc, *out.tolist())


PLACED, NO_SEQUENCE, IMPOSSIBLE = 0, 1, 2


def test_positions(host):
    starts, lens = [0, 3, 3, 4], [10, 7, 1]
    for s, (n, t) in enumerate(zip(np.diff(starts), lens)):
        for tok in range(-1, 6):
            got = place(host, starts, lens, 4, 8, s, tok)
            if starts[s] <= tok < starts[s + 1]:
                assert got == (PLACED, t - n + tok - starts[s], n, t)
            else:
                assert got[0] == NO_SEQUENCE
    for s in range(3):  # one token each
        assert place(host, None, lens, 4, 8, s, s) == (PLACED, lens[s] - 1, 1, lens[s])


def test_lengths_that_cannot_be(host):
    for length, want in ((3, PLACED), (2, IMPOSSIBLE), (0, IMPOSSIBLE), (-5, IMPOSSIBLE),
                         (128, PLACED), (129, IMPOSSIBLE), (2 ** 31 - 1, IMPOSSIBLE),
                         (-2 ** 31, IMPOSSIBLE)):
        assert place(host, [0, 3], [length], 4, 8, 0, 1)[0] == want
    assert place(host, None, [0], 4, 8, 0, 0)[0] == IMPOSSIBLE
    assert place(host, [-2, 1], [3], 4, 8, 0, 0)[0] == IMPOSSIBLE
    assert place(host, [3, 0], [3], 4, 8, 0, 1)[0] == NO_SEQUENCE  # (not ascending)


@pytest.mark.parametrize("shift", [4, 5, 6, 7, 8])
def test_pages(host, shift):
    g = np.random.default_rng(shift)
    table = ints(g.integers(-3, 12, (4, 9)))
    table[0, :3] = [-1, 9, 2 ** 31 - 1]
    for s in range(4):
        for row in [0, 1, (1 << shift) - 1, 1 << shift, (2 << shift) + 3, (7 << shift) - 1]:
            e = int(table[s, row >> shift])
            assert host.page(table.ctypes.data, 9, shift, 9, s, row) == (e if 0 <= e < 9 else -1)


def test_offsets(host):
    # [page][head][row] and [page][row][head], padded, and past 32 bits
    for ps, hs, rs in ((2 * 16 * 128, 16 * 128, 128), (16 * 3 * 72, 72, 3 * 72),
                       (2 ** 33 + 8, 2 ** 20, 136)):
        for page, h, row in ((0, 0, 0), (5, 1, 17), (70000, 1, 1023), (2 ** 31 - 1, 1, 15)):
            want = page * ps + h * hs + row % 16 * rs
            if want < 2 ** 60:  # (no memory holds the others)
                assert host.offset(ps, hs, rs, 4, page, h, row) == want


def test_null_arguments_are_refused(pkg):
    lib = pkg.gqa.lib()
    kv = pkg.gqa.PagedKV()
    assert lib.gqa_paged_append(None, None, ctypes.byref(kv), 1, 1, None, None, None, 0) != 0
    assert lib.gqa_paged_attention(None, None, ctypes.byref(kv), 1, 1, None, None, 1, 1, None, 0,
                                   None, 0) != 0
    assert lib.gqa_sample(None, None, 1, 1, 0, None, 1, None, None, None, None, None, None) != 0


def test_views_are_refused_without_a_device(pkg):
    import torch
    k = torch.zeros(4, 2, 16, 128)
    table = torch.zeros(1, 4, dtype=torch.int32)
    for args, kw in (((k, k, table), {}),                       # not on a device
                     ((k[0], k[0], table), {}),
                     ((k, k.double(), table), {}),
                     ((k, k, table), {"layout": "dhn"})):
        with pytest.raises((pkg.GqaError, ValueError)):
            pkg.paged_kv_of(*args, **kw)
