"""The packed operators on the B200 with elements past 2^31 from a buffer's start: long caches, wide row strides.
Bounds: see test_packed_ops_gpu.py.
"""
from __future__ import annotations

import pytest
import torch
from test_packed_ops_gpu import DEV, attend, assert_within, check_gemm, check_rope, offsets, randn, weight, F64, UNIT

pytestmark = pytest.mark.gpu
ROWS, FAR = 2 ** 21 + 4000, 2 ** 21 + 100  # rows of 8 heads of 128: row FAR begins past element 2^31


@pytest.mark.parametrize("lq", [[1, 1], [150, 300]])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_packed_far_into_a_cache(engine, lq, causal):
    k, v = (torch.empty((ROWS, 8, 128), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    used, starts = [500, 3000], [64, FAR]
    for b in range(2):
        for t, seed in ((k, 1), (v, 2)):
            t[starts[b]:starts[b] + used[b]] = randn((used[b], 8, 128), seed + b, 1.0, torch.bfloat16)
    q = randn((sum(lq), 16, 128), 9, 1.5, torch.bfloat16)
    cu_k = torch.tensor([64, FAR, ROWS], dtype=torch.int32, device=DEV)
    lens = torch.tensor(used, dtype=torch.int32, device=DEV)
    out = engine.attention_packed(q, k, v, offsets(lq), cu_k, k_lens=lens, causal=causal)
    torch.cuda.synchronize()
    engine.check_device_error()
    want, a = attend(q, k, v, lq, used, causal, 128 ** -0.5, starts)
    u = UNIT[q.dtype]
    assert_within(out, want, (1.1 * u + 1e-4) * a * (1 + u) + u * want.abs() + 1e-6)


def far_rows(rows, cols, dtype, seed):
    """[rows, cols] with 2^24 elements from row to row: from row 128 on past 2^31."""
    t = torch.empty((rows, 2 ** 24), dtype=dtype, device=DEV)[:, :cols]
    t.copy_(randn((rows, cols), seed, 1.0, dtype))
    return t


@pytest.mark.parametrize("interleaved", [True, False])
def test_qk_norm_rope_wide_strides(engine, interleaved):
    t = 140
    q, k = (far_rows(t, h * 128, torch.bfloat16, h).unflatten(1, (h, 128)) for h in (4, 2))
    check_rope(engine, q, k, randn((t, 3), 5).abs() * 100, [16, 56, 56], interleaved, None, None, torch.bfloat16)
    check_rope(engine, q, k, randn((t, 1), 5).abs() * 100, [66], interleaved, None, None, torch.float32)


@pytest.mark.parametrize("m,k", [(140, 520), (133, 20000)])
def test_gemm_s8_wide_strides(engine, m, k):
    wq, ws = weight(130, k, 4)
    x = far_rows(m, k, torch.bfloat16, 6)
    check_gemm(engine, x, None, wq, ws, None, torch.float32, "none")
    out = torch.empty((m, 2 ** 24), dtype=torch.bfloat16, device=DEV)[:, :130]
    engine.gemm_s8(x, wq, ws, out=out)
    codes, xs = engine.quantize_s8(x)
    torch.cuda.synchronize()
    assert torch.equal(out, engine.gemm_s8(codes, wq, ws, x_scale=xs, out_dtype=torch.bfloat16))


@pytest.mark.parametrize("m", [2, 40, 200])
def test_gemm_s8_weight_with_wide_rows(engine, m):
    """Weight rows 2^24 bytes apart: channel 128 on past 2^31."""
    k = 2048
    wq, ws = weight(200, k, 4)
    far = torch.empty((200, 2 ** 24), dtype=torch.int8, device=DEV)[:, :k]
    far.copy_(wq)
    x = randn((m, k), 5, 1.0, torch.bfloat16)
    got, want = engine.gemm_s8(x, far, ws), engine.gemm_s8(x, wq, ws)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
