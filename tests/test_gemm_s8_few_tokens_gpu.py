"""gemm_s8 for a few tokens on the B200: the launch that quantises and multiplies, the product whose K axis a cluster
of blocks shares out, and the sizes at which one gives way to the next.  Bounds: see test_packed_ops_gpu.py.
"""
from __future__ import annotations

import pytest
import torch
from test_packed_ops_gpu import DEV, F64, assert_within, check_gemm, quantized, randn, weight

pytestmark = pytest.mark.gpu


# Up to 8 tokens and 16384 values in all (their number rounded up to a power of two), and just past it.
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 5, 16384), (1, 40, 16385), (2, 33, 8192), (2, 7, 8200), (3, 100, 4096),
                                   (3, 17, 4097), (4, 31, 513), (5, 64, 2047), (7, 48, 63), (8, 1030, 2048), (8, 20, 65),
                                   (1, 9000, 130), (6, 7300, 72)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_one_launch(engine, m, n, k, dtype):
    wq, ws = weight(n, k, m + n + k)
    x = randn((m, k), k + m, 1.0, dtype)
    check_gemm(engine, x, None, wq, ws, randn((n,), 3, 0.1), dtype, "none")


@pytest.mark.parametrize("offset", [0, 1, 4, 8])
@pytest.mark.parametrize("m,k", [(1, 1001), (5, 300), (8, 2048)])
def test_one_launch_views(engine, offset, m, k):
    """Tokens at any alignment and row stride, into a strided output."""
    wq, ws = weight(50, k, 5)
    x = randn((m, k + 21), 6, 1.0, torch.bfloat16)[:, offset:offset + k]
    buf = torch.full((m, 64), 7.0, device=DEV)
    engine.gemm_s8(x, wq, ws, out=buf[:, 3:53])
    torch.cuda.synchronize()
    assert torch.equal(buf[:, 3:53], engine.gemm_s8(x.contiguous(), wq, ws))
    assert bool((buf[:, :3] == 7).all()) and bool((buf[:, 53:] == 7).all())


# K shared out among 1 to 8 blocks per 128 channels; channels, tokens and K past the tiles' edges.
@pytest.mark.parametrize("m,n,k", [(9, 1, 1000), (9, 129, 2048), (16, 300, 4099), (17, 128, 5000), (31, 1000, 3000),
                                   (33, 2600, 1600), (64, 5120, 3072), (64, 19000, 3080), (100, 257, 4800), (127, 640, 6100),
                                   (128, 384, 6144), (128, 20000, 6144), (100, 257, 4799)])
@pytest.mark.parametrize("given", ["codes", "bf16", "f32"])
def test_shared_k(engine, m, n, k, given):
    wq, ws = weight(n, k, m + n + k)
    x, xs = randn((m, k), k, 1.0, torch.float32 if given == "f32" else torch.bfloat16), None
    if given == "codes":
        x, xs = engine.quantize_s8(x)
    check_gemm(engine, x, xs, wq, ws, randn((n,), 3, 0.1, torch.bfloat16), torch.bfloat16, "none")


@pytest.mark.parametrize("m,n,k", [(129, 300, 3200), (200, 512, 10000), (257, 100, 4200), (400, 700, 6500), (1000, 130, 6001)])
@pytest.mark.parametrize("given", ["codes", "bf16"])
def test_shared_k_blocks_of_tokens(engine, m, n, k, given):
    wq, ws = weight(n, k, m + n + k)
    x, xs = randn((m, k), k, 1.0, torch.bfloat16), None
    if given == "codes":
        x, xs = engine.quantize_s8(x)
    check_gemm(engine, x, xs, wq, ws, randn((n,), 3, 0.1), torch.float16, "silu")


@pytest.mark.parametrize("m,n,k", [(130, 261, 304), (700, 1003, 160), (1500, 2307, 64)])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_rows_of_odd_width(engine, m, n, k, out_dtype):
    """Output rows without the alignment of wide stores, whole and as a view that leaves its neighbours alone."""
    wq, ws = weight(n, k, m)
    x = randn((m, k), 9, 1.0, torch.bfloat16)
    check_gemm(engine, x, None, wq, ws, randn((n,), 3, 0.1), out_dtype, "gelu")
    buf = torch.full((m, n + 11), 7.0, dtype=out_dtype, device=DEV)
    engine.gemm_s8(x, wq, ws, out=buf[:, 5:5 + n])
    torch.cuda.synchronize()
    assert torch.equal(buf[:, 5:5 + n], engine.gemm_s8(x, wq, ws, out_dtype=out_dtype))
    assert bool((buf[:, :5] == 7).all()) and bool((buf[:, 5 + n:] == 7).all())


@pytest.mark.parametrize("m,k", [(3, 700), (40, 2600)])
@pytest.mark.parametrize("epilogue", ["none", "gelu", "silu"])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_epilogues(engine, m, k, epilogue, out_dtype):
    wq, ws = weight(200, k, m)
    ws = ws * 0.1  # sums of some units
    check_gemm(engine, randn((m, k), 9, 1.0, torch.float16), None, wq, ws, randn((200,), 3), out_dtype, epilogue)


@pytest.mark.parametrize("m,k", [(3, 700), (40, 2600)])
def test_gated_residual(engine, m, k):
    n = 300
    wq, ws = weight(n, k, 8)
    x = randn((m, k), 9, 1.0, torch.bfloat16)
    gate, res = randn((n,), 10), randn((m, n), 12)
    out = res.clone()
    engine.gemm_s8(x, wq, ws, out=out, epilogue="gated_residual", gate=gate)
    torch.cuda.synchronize()
    codes, xs = quantized(x)
    g = gate.to(F64)
    prod = (codes @ wq.to(F64).T) * xs[:, None] * ws.to(F64)
    want = res.to(F64) + g * prod
    e = 2.0 ** -24
    assert_within(out, want, g.abs() * 8 * e * prod.abs() + 2 * e * want.abs())
    with pytest.raises(engine.B2GError, match="needs a gate"):
        engine.gemm_s8(x, wq, ws, out=out, epilogue="gated_residual")


@pytest.mark.parametrize("m,n,k", [(300, 301, 600), (300, 130, 5000)])
def test_gated_residual_of_many_tokens(engine, m, n, k):
    """Rows of odd width; K shared out over blocks of tokens."""
    wq, ws = weight(n, k, 8)
    x, xs = engine.quantize_s8(randn((m, k), 9, 1.0, torch.bfloat16))
    gate, res = randn((n,), 10), randn((m, n), 12)
    out = res.clone()
    engine.gemm_s8(x, wq, ws, out=out, epilogue="gated_residual", gate=gate, x_scale=xs)
    torch.cuda.synchronize()
    g = gate.to(F64)
    prod = (x.to(F64) @ wq.to(F64).T) * xs.to(F64)[:, None] * ws.to(F64)
    want = res.to(F64) + g * prod
    e = 2.0 ** -24
    assert_within(out, want, g.abs() * 8 * e * prod.abs() + 2 * e * want.abs())


@pytest.mark.parametrize("m,k", [(4, 900), (20, 1100), (130, 1100)])
def test_rows_of_any_size(engine, m, k):
    """A row of zeros, rows near both ends of the type's range, a row with an infinity: the others are right."""
    wq, ws = weight(70, k, 4)
    x = randn((m, k), 3, 1.0, torch.bfloat16)
    x[0] = 0
    x[1] *= 2.0 ** 120
    x[2] *= 2.0 ** -125
    x[3, 7] = float("inf")
    out = engine.gemm_s8(x, wq, ws)
    torch.cuda.synchronize()
    codes, unit = quantized(x)
    prod = (codes @ wq.to(F64).T) * unit[:, None] * ws.to(F64)
    keep = [i for i in range(m) if i != 3]
    # (2 subnormals of the row's scale, times the codes' sum and the channel's)
    small = 2 * 2.0 ** -149 * (codes @ wq.to(F64).T).abs() * ws.to(F64) + 2.0 ** -148
    assert_within(out[keep], prod[keep], (10 * 2.0 ** -24 * prod.abs() + small)[keep])
    assert bool(torch.isnan(out[3]).all())


@pytest.mark.parametrize("dtype,big", [(torch.bfloat16, 3.0e38), (torch.float32, 3.3e38), (torch.float16, 65504.0)])
def test_quantize_rows_at_the_top_of_the_range(engine, dtype, big):
    x = torch.tensor([[big, big / 2, -big / 4, big / 254, 0.0, -big]], device=DEV).to(dtype)
    q, s = engine.quantize_s8(x)
    torch.cuda.synchronize()
    want, unit = quantized(x)
    assert torch.equal(q.to(F64), want) if dtype != torch.float32 else float((q.to(F64) - want).abs().max()) <= 1
    assert_within(s, unit, unit * 2.0 ** -24)


def test_every_pair_of_16_bit_magnitudes(engine):
    """Codes of every bf16 value in one binade against every maximum in the next: all the exact halves."""
    low = torch.arange(128, 256, device=DEV, dtype=torch.float32) / 256
    tops = torch.arange(128, 256, device=DEV, dtype=torch.float32) / 128
    x = torch.cat([low * 2.0 ** -i for i in range(8)] + [tops.new_zeros(1)])[None].repeat(128, 1)
    x[:, -1] = tops
    for scale in (1.0, 2.0 ** 60, 2.0 ** -60):
        b = (x * scale).to(torch.bfloat16)
        q, _ = engine.quantize_s8(b)
        torch.cuda.synchronize()
        assert torch.equal(q.to(F64), quantized(b)[0])


def test_repeated_in_a_graph(engine):
    """Each way replays with new contents."""
    for m, k in ((1, 512), (24, 2048), (200, 512)):
        wq, ws = weight(260, k, 2)
        x = randn((m, k), 1, 1.0, torch.bfloat16)
        engine.gemm_s8(x, wq, ws)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = engine.gemm_s8(x, wq, ws)
        for seed in (5, 6):
            x.copy_(randn((m, k), seed, 1.0, torch.bfloat16))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, engine.gemm_s8(x, wq, ws))
