"""attention_packed on the B200 with more tiles than SMs: every way of pairing tiles, several items per block.
Bounds: see test_packed_ops_gpu.py.
"""
from __future__ import annotations

import pytest
import torch
from test_packed_ops_gpu import check_attention, qkv

pytestmark = pytest.mark.gpu

SHORT = [1, 127, 128, 129, 0, 255, 256, 257, 60, 300, 2, 40]  # 256 tokens on average at most
LONG = [300, 700, 1000, 513, 0, 640, 1]


@pytest.mark.parametrize("lens", [SHORT, LONG])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("hq,hk,d,dtype", [(24, 24, 128, torch.bfloat16), (23, 23, 64, torch.float16), (24, 8, 128, torch.bfloat16),
                                           (32, 8, 64, torch.bfloat16), (40, 2, 128, torch.float16), (25, 5, 64, torch.bfloat16)])
def test_self(engine, lens, causal, hq, hk, d, dtype):
    t = sum(lens)
    check_attention(engine, *qkv(t, t, hq, hk, d, dtype, t + hq), lens, lens, causal)


@pytest.mark.parametrize("lq,lk", [(SHORT, SHORT[::-1]), (LONG, [20, 900, 0, 1200, 5, 640, 300]), ([40] * 9, [700] * 9)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("hq,hk,d", [(33, 33, 128), (32, 4, 128), (64, 64, 64)])
def test_other_keys(engine, lq, lk, causal, hq, hk, d):
    check_attention(engine, *qkv(sum(lq), sum(lk), hq, hk, d, torch.bfloat16, hq), lq, lk, causal)


@pytest.mark.parametrize("heads", [1, 2, 5])
@pytest.mark.parametrize("causal", [False, True])
def test_one_long_sequence_of_few_heads(engine, heads, causal):
    n = 3001
    check_attention(engine, *qkv(n, n, heads, 1, 128, torch.bfloat16, heads), [n], [n], causal)


@pytest.mark.parametrize("hq,hk,d", [(24, 24, 128), (23, 23, 64), (32, 8, 128)])
@pytest.mark.parametrize("lq,lk", [([2000, 300, 1500, 400, 900], [0, 500, 0, 800, 10]), ([3000, 3000, 20], [100, 0, 3000]),
                                   ([200] * 8 + [30], [0] * 8 + [70]), ([400] * 6, [0] * 6)])
def test_many_rows_without_keys(engine, hq, hk, d, lq, lk):
    check_attention(engine, *qkv(sum(lq), sum(lk), hq, hk, d, torch.bfloat16, hq), lq, lk, True)


@pytest.mark.parametrize("hq,hk,d,scale", [(3, 3, 64, 1), (4, 2, 128, 1), (2, 1, 64, 6)])
@pytest.mark.parametrize("causal", [False, True])
def test_more_sequences_than_are_sorted(engine, hq, hk, d, scale, causal):
    """Thousands of sequences, taken as they come; empty ones among them."""
    g = torch.Generator().manual_seed(hq)
    lq = (torch.randint(0, 60, (2500,), generator=g) * scale).tolist()
    lk = (torch.randint(0, 60, (2500,), generator=g) * torch.randint(0, 2, (2500,), generator=g)).tolist()
    check_attention(engine, *qkv(sum(lq), sum(lk), hq, hk, d, torch.bfloat16, hq), lq, lk, causal)
