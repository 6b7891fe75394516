"""The packed operators give the same bits for the same inputs, whatever ran before."""
from __future__ import annotations

import pytest
import torch
from test_packed_ops_gpu import DEV, offsets, qkv, randn, weight

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lq,lk,hq,hk,d", [([1] * 48, [8000, 1, 700, 33, 16, 4097] * 8, 32, 8, 128), ([700, 210, 539], None, 32, 8, 128),
                                           ([700, 210, 539], None, 27, 9, 64), ([240, 100, 7, 239], None, 33, 11, 128),
                                           ([300, 5], None, 2, 2, 128)])
def test_attention_packed(engine, lq, lk, hq, hk, d):
    lk = lq if lk is None else lk
    q, k, v = qkv(sum(lq), sum(lk), hq, hk, d, torch.bfloat16, 1)
    first = engine.attention_packed(q, k, v, offsets(lq), offsets(lk), causal=True)
    for _ in range(20):
        assert torch.equal(engine.attention_packed(q, k, v, offsets(lq), offsets(lk), causal=True), first)


@pytest.mark.parametrize("m,n,k", [(3, 700, 512), (40, 2000, 2600), (300, 513, 640), (600, 512, 8000)])
def test_gemm_s8(engine, m, n, k):
    wq, ws = weight(n, k, 2)
    x = randn((m, k), 3, 1.0, torch.bfloat16)
    first = engine.gemm_s8(x, wq, ws, epilogue="gelu")
    for _ in range(20):
        assert torch.equal(engine.gemm_s8(x, wq, ws, epilogue="gelu"), first)


@pytest.mark.parametrize("tokens,heads", [(64, 32), (2000, 3)])
def test_qk_norm_rope(engine, tokens, heads):
    q, pos, w = randn((tokens, heads, 128), 4, 1.0, torch.bfloat16), randn((tokens, 1), 5) * 100, 1 + randn((128,), 6, 0.1)
    first = engine.qk_norm_rope(q, q, pos, [128], w, w)
    for _ in range(20):
        again = engine.qk_norm_rope(q, q, pos, [128], w, w)
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])


@pytest.mark.parametrize("rows,cols", [(37, 1000), (300, 5120), (3, 20000)])
def test_quantize_s8(engine, rows, cols):
    x = randn((rows, cols), 7)
    first = engine.quantize_s8(x)
    for _ in range(20):
        again = engine.quantize_s8(x)
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])
