"""Overlapped launches (GQA_OPT_PDL): a kernel that lets the next one start early has waited for
those before it, since the decode kernels read cache rows before their own wait."""
import os
import re

import numpy as np
import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(REPO, "macbook-hardware-linux-lab_b200", "csrc")


@pytest.mark.parametrize("name", ["gqa_paged.cu", "gqa_paged_decode.cu"])
def test_waits_before_it_lets_the_next_start(name):
    """(The chunks' kernels are followed by the merge alone, which waits at once and lets nothing
    start early.)"""
    with open(os.path.join(CSRC, name)) as f:
        calls = re.findall(r"\b(pdl_wait|pdl_launch_dependents)\(\);", f.read())
    assert calls == ["pdl_wait", "pdl_launch_dependents"]
    for name in ("gqa_paged_merge.cuh", "gqa_sample.cu"):
        with open(os.path.join(CSRC, name)) as f:
            assert "pdl_launch_dependents" not in f.read()


@pytest.mark.gpu
def test_append_between_contiguous_calls(pkg, cuda):
    """Row pos written by rope_kv_append, then a paged append, then the layer call that attends
    rows [0, pos + 1] of the contiguous cache: bits equal with overlapped launches off and on."""
    steps, t_max = 60, 128
    g = np.random.default_rng(50)
    rows = cuda.from_numpy(g.standard_normal((2 * steps, 2048))).float().cuda()
    table = cuda.arange(64, dtype=cuda.int32, device="cuda").view(8, 8)
    lens = cuda.full((8,), 100, dtype=cuda.int32, device="cuda")
    outs = []
    for pdl in (0, 1):
        kc, vc = (cuda.zeros(2, t_max, 128, device="cuda") for _ in "kv")
        kp, vp = (cuda.zeros(64, 2, 16, 128, device="cuda") for _ in "kv")
        qkv, out = rows.clone(), cuda.zeros(steps, 1536, device="cuda")
        with pkg.Context(t_max=t_max) as ctx:
            ctx.set_option(pkg.gqa.GQA_OPT_PDL, pdl)
            kv, paged = pkg.kv_of(kc, vc), pkg.paged_kv_of(kp, vp, table)
            cuda.cuda.synchronize()
            for i in range(steps):
                q = qkv[2 * i]
                ctx.rope_kv_append(kv, q, q[1536:], q[1792:], 2 * i)
                ctx.paged_append(paged, 8, 8, None, lens, rows[:8])
                ctx.layer_attention_out(kv, qkv[2 * i + 1], 2 * i + 1, 2 * i + 2, out[i])
            assert ctx.device_status() == 0
        outs.append((kc, vc, kp, vp, out))
    for x, y in zip(*outs):
        assert cuda.equal(x, y)
