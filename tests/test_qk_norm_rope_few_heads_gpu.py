"""qk_norm_rope of few heads and many tokens on the B200.  Bounds: see test_packed_ops_gpu.py."""
from __future__ import annotations

import pytest
import torch
from test_packed_ops_gpu import DEV, UNIT, assert_within, check_rope, randn, rotated

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hk", [(1, 0), (0, 3), (2, 1), (4, 1), (5, 5), (8, 2), (10, 1)])
@pytest.mark.parametrize("d,axes", [(128, [16, 56, 56]), (64, [64]), (96, [32, 64]), (256, [256]), (128, [64]), (40, [8, 32]), (128, [])])
@pytest.mark.parametrize("interleaved", [True, False])
def test_few_heads(engine, hq, hk, d, axes, interleaved):
    t = 1024 + 37 * hq
    q, k = randn((t, hq, d), 1, 2.0, torch.bfloat16), randn((t, hk, d), 2, 2.0, torch.bfloat16)
    pos = randn((t, len(axes)), 5).abs() * 100
    norms = 1 + randn((d,), 6, 0.2), 1 + randn((d,), 7, 0.2)
    got = engine.qk_norm_rope(q, k, pos, axes, q_norm=norms[0], k_norm=norms[1], interleaved=interleaved)
    torch.cuda.synchronize()
    for g, x, w in zip(got, (q, k), norms):
        assert g.shape == x.shape
        if x.numel():
            want, size = rotated(x, w, pos, axes, 10000.0, interleaved, 1e-6)
            u = UNIT[torch.bfloat16]
            assert_within(g, want, 2.0 ** -17 * size * (1 + u) + u * want.abs())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("norms", [(True, True), (True, False), (False, True), (False, False)])
def test_few_heads_types_and_norms(engine, dtype, out_dtype, norms):
    t, d = 5000, 128
    q, k = randn((t, 3, d), 1, 2.0, dtype), randn((t, 2, d), 2, 2.0, dtype)
    qn, kn = (1 + randn((d,), 6 + i, 0.2) if on else None for i, on in enumerate(norms))
    check_rope(engine, q, k, randn((t, 2), 5) * 1000, [64, 64], True, qn, kn, out_dtype)


@pytest.mark.parametrize("interleaved", [True, False])
def test_few_heads_in_place_views(engine, interleaved):
    """Views of a fused projection, written over."""
    t, d = 3001, 64
    qkv = randn((t, 8, d), 3, 1.0, torch.bfloat16)
    before = qkv.clone()
    pos = randn((t, 1), 4) * 50
    want = engine.qk_norm_rope(before[:, :4], before[:, 4:6], pos, [64], interleaved=interleaved)
    engine.qk_norm_rope(qkv[:, :4], qkv[:, 4:6], pos, [64], interleaved=interleaved, q_out=qkv[:, :4], k_out=qkv[:, 4:6])
    torch.cuda.synchronize()
    assert torch.equal(qkv[:, :4], want[0]) and torch.equal(qkv[:, 4:6], want[1])
    assert torch.equal(qkv[:, 6:], before[:, 6:])


def test_few_heads_zero_rows(engine):
    q = torch.zeros((2000, 2, 128), dtype=torch.float16, device=DEV)
    q[7, 1] = 1
    qo, ko = engine.qk_norm_rope(q, q[:, :0], torch.ones((2000, 1), device=DEV), [128], q_norm=torch.ones(128, device=DEV))
    torch.cuda.synchronize()
    assert ko.numel() == 0 and bool((qo[:7] == 0).all()) and bool(qo[7, 1].any()) and not bool(qo[7, 0].any())
