"""Packed-batch operators on the B200 against their definitions in 64 bits: the 8-bit integer linear
layer, the per-head norm with multi-axis rotation, attention over packed sequences.

Tolerances are bounds, per element.  With u the unit roundoff of a type (half its epsilon: 2^-8 bf16,
2^-11 fp16) and e = 2^-24 that of fp32:
  quantize_s8       16-bit inputs: codes equal.  x * 127 is exact and the quotient correctly rounded;
                    a quotient of 16-bit values is a half-integer or at least 2^-20 of itself away
                    from one.  F32: two roundings of a quotient <= 127, so within 0.5 + 2^-16 of it.
  gemm_s8           the integer sum is exact; conversion, two scales and the bias are 4 roundings; an
                    activation adds at most 2^-16 of the result (the argument of its exponential is
                    rounded at up to 100 units) and has a slope of at most 1.2.
  qk_norm_rope      D roundings in the sum of squares (half of them in its root), the angle to 2^-23 of
                    a turn: 2^-17 of the pair's length in all.
  attention_packed  P rounded to the operands' type (u sum p |v| / sum p), the scores' fp32
                    sums of D products of a few units (1e-4 of the same), the output's rounding.
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F64 = torch.float64
UNIT = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}


def randn(shape, seed, scale=1.0, dtype=torch.float32):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def assert_within(got, want, bound, what=""):
    """|got - want| <= bound everywhere (NaN where and only where `want` has it)."""
    got = got.to(F64)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    over = ((got - want).abs() - bound).nan_to_num(0.0)
    at = int(over.argmax())
    assert float(over.max()) <= 0, (what, at, float(got.flatten()[at]), float(want.flatten()[at]),
                                    float(bound.expand_as(want).flatten()[at]))


# ---------------------------------------------------------------------------- 8-bit integers
def quantized(x):
    """The definition in 64 bits: (codes, scales)."""
    x = x.to(F64)
    top = x.abs().amax(1)
    safe = torch.where(top > 0, top, 1.0)
    return torch.round(x * 127 / safe[:, None]), torch.where(top > 0, top / 127, 1.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 5120), (3, 7), (37, 1000), (9, 1032), (5, 4099), (64, 8192),
                                       (2, 16384), (3, 16400)])
def test_quantize_s8(engine, dtype, rows, cols):
    x = randn((rows, cols), rows + cols, 3.0, dtype)
    x[0, 0] = x.abs().max() * 2
    x[0, cols // 2:] *= 0.25
    x[rows - 1, cols // 2] = x[rows - 1].abs().max() / 2  # a quotient of 63.5
    if rows > 2:
        x[1] = 0
    q, s = engine.quantize_s8(x)
    torch.cuda.synchronize()
    wq, ws = quantized(x)
    assert torch.equal(s, ws.float())
    if dtype == torch.float32:
        top = x.to(F64).abs().amax(1, keepdim=True).clamp_min(1e-300)
        assert float((q.to(F64) - x.to(F64) * 127 / top).abs().max()) <= 0.5 + 2.0 ** -16
    else:
        assert torch.equal(q.to(F64), wq)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_s8_strides_and_small_numbers(engine, dtype):
    """Odd row strides and starts, an output with its own stride, rows of subnormal size."""
    base = randn((6, 301), 5, 1.0, dtype)
    x = base[:, 3:256]
    x[2] *= 1e-38
    x[3] = 0
    x[3, 100] = 1e-40
    buf = torch.full((6, 260), 77, dtype=torch.int8, device=DEV)
    q, s = engine.quantize_s8(x, out=buf[:, 1:254])
    torch.cuda.synchronize()
    wq, ws = quantized(x)
    assert float((s.to(F64) - ws).abs().max()) <= 2.0 ** -24 and bool((s > 0).all())
    assert float((q.to(F64) - wq).abs().max()) <= (0 if dtype == torch.bfloat16 else 1)
    assert bool((buf[:, 0] == 77).all()) and bool((buf[:, 254:] == 77).all())


def test_quantize_s8_nonfinite_rows(engine):
    x = randn((4, 64), 6, 1.0, torch.bfloat16)
    x[1, 5] = float("inf")
    x[2, 6] = float("nan")
    q, s = engine.quantize_s8(x)
    w = randn((16, 64), 7, 30.0).round().clamp(-127, 127).to(torch.int8)
    y = engine.gemm_s8(x, w, torch.ones(16, device=DEV))
    torch.cuda.synchronize()
    assert torch.isnan(s).tolist() == [False, True, True, False]
    assert int(q[1:3].abs().max()) == 0
    assert torch.isnan(y).all(1).tolist() == [False, True, True, False]


def weight(n, k, seed):
    """int8 [n, k] with rows padded to 16 bytes; the padding holds anything."""
    w = randn((n, (k + 15) // 16 * 16), seed, 40.0).round().clamp(-127, 127).to(torch.int8)
    return w[:, :k], 0.01 * torch.exp(0.3 * randn((n,), seed + 1))


def act(y, epilogue):
    if epilogue == "gelu":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    return y / (1 + torch.exp(-y)) if epilogue == "silu" else y


def check_gemm(engine, x, xs, wq, ws, bias, out_dtype, epilogue):
    out = engine.gemm_s8(x, wq, ws, bias, out_dtype=out_dtype, epilogue=epilogue, x_scale=xs)
    torch.cuda.synchronize()
    engine.check_device_error()
    codes, unit = (x.to(F64), xs.to(F64)) if xs is not None else quantized(x)
    if xs is None and x.dtype == torch.float32:  # (its codes are allowed a little)
        q, s = engine.quantize_s8(x)
        codes, unit = q.to(F64), s.to(F64)
    prod = (codes @ wq.to(F64).T) * unit[:, None] * ws.to(F64)
    b = bias.to(F64) if bias is not None else 0.0
    want = act(prod + b, epilogue)
    e = 2.0 ** -24
    lin = 5 * e * (prod.abs() + (prod + b).abs())
    bound = 1.2 * lin + (0 if epilogue == "none" else 2.0 ** -16) * want.abs() + 1e-30
    u = UNIT[out_dtype]
    assert_within(out, want, bound * (1 + u) + u * want.abs() + (2.0 ** -25 if out_dtype == torch.float16 else 0))


@pytest.mark.parametrize("m,n,k", [(1, 5120, 5120), (1, 17, 1), (3, 250, 33), (8, 512, 1000), (9, 1000, 512), (16, 96, 4099),
                                   (17, 300, 272), (33, 129, 77), (128, 128, 128), (100, 513, 640), (300, 257, 1025),
                                   (344, 5120, 5120), (520, 2050, 384)])
@pytest.mark.parametrize("given", ["codes", "bf16"])
def test_gemm_s8_sizes(engine, m, n, k, given):
    wq, ws = weight(n, k, m + n + k)
    x = randn((m, k), k, 1.0, torch.bfloat16)
    xs = None
    if given == "codes":
        x, xs = engine.quantize_s8(x)
    check_gemm(engine, x, xs, wq, ws, randn((n,), 3, 0.1), torch.float32, "none")


@pytest.mark.parametrize("m", [2, 12, 65, 300])
@pytest.mark.parametrize("epilogue", ["none", "gelu", "silu"])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bias", [None, torch.float32, torch.bfloat16])
def test_gemm_s8_epilogues(engine, m, epilogue, out_dtype, bias):
    n, k = 328, 416
    wq, ws = weight(n, k, m)
    x = randn((m, k), 9, 1.0, torch.float32 if out_dtype == torch.float32 else out_dtype)
    check_gemm(engine, x, None, wq, ws, None if bias is None else randn((n,), 3, 0.1, bias), out_dtype, epilogue)


@pytest.mark.parametrize("variant", [0, 1, 2])
def test_gemm_s8_tile_variants(engine, variant):
    """Every tile shape, with more tiles than CTAs and ragged edges; a forced split is ignored."""
    engine.set_gemm_variant(variant, 2)
    try:
        wq, ws = weight(9001, 700, 4)
        check_gemm(engine, randn((1100, 700), 5, 1.0, torch.bfloat16), None, wq, ws, None, torch.bfloat16, "none")
    finally:
        engine.set_gemm_variant(-1, 0)


@pytest.mark.parametrize("m", [5, 130])
def test_gemm_s8_gated_residual(engine, m):
    n, k = 260, 304
    wq, ws = weight(n, k, 8)
    x, xs = engine.quantize_s8(randn((m, k), 9))
    gate, bias, res = randn((n,), 10), randn((n,), 11), randn((m, n), 12)
    out = res.clone()
    engine.gemm_s8(x, wq, ws, bias, out=out, epilogue="gated_residual", gate=gate, x_scale=xs)
    torch.cuda.synchronize()
    prod = (x.to(F64) @ wq.to(F64).T) * xs.to(F64)[:, None] * ws.to(F64)
    y = prod + bias.to(F64)
    e = 2.0 ** -24
    want = res.to(F64) + gate.to(F64) * y
    assert_within(out, want, gate.to(F64).abs() * 6 * e * (prod.abs() + y.abs()) + 2 * e * want.abs())


def test_gemm_s8_extreme_codes_are_exact(engine):
    """All codes at +-127 (and -128) over a long K: the 32-bit sums do not overflow or round."""
    for m in (4, 200):
        k = 131071
        x = torch.full((m, (k + 15) // 16 * 16), -128, dtype=torch.int8, device=DEV)[:, :k]
        w = torch.full((32, (k + 15) // 16 * 16), -128, dtype=torch.int8, device=DEV)[:, :k]
        w[1::2] = 127
        one = torch.ones(m, device=DEV)
        out = engine.gemm_s8(x, w, torch.ones(32, device=DEV), x_scale=one)
        torch.cuda.synchronize()
        want = torch.where(torch.arange(32, device=DEV) % 2 == 0, 128.0 * 128 * k, -128.0 * 127 * k).to(F64)
        assert_within(out, want.expand(m, 32), want.abs() * 2.0 ** -24)


def test_gemm_s8_views_and_streams(engine):
    """Strided x and output rows, on a stream of the caller's, twice at once on two streams."""
    m, n, k = 70, 192, 256
    wq, ws = weight(n, k, 20)
    big = randn((m, 2 * k + 8), 21, 1.0, torch.bfloat16)
    buf = torch.zeros((m, n + 40), device=DEV)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i, st in enumerate(streams):
        x = big[:, i * (k + 8):i * (k + 8) + k]
        outs.append((x, engine.gemm_s8(x, wq, ws, stream=st)))
    engine.gemm_s8(big[:, :k], wq, ws, out=buf[:, 20:20 + n], stream=streams[0])
    torch.cuda.synchronize()
    for x, out in outs:
        assert torch.equal(out, engine.gemm_s8(x.contiguous(), wq, ws))
    assert torch.equal(buf[:, 20:20 + n], outs[0][1])
    assert not buf[:, :20].any() and not buf[:, 20 + n:].any()


# ---------------------------------------------------------------------------- norm and rotation
def rotated(x, w, pos, axes, theta, interleaved, eps):
    """The definition in 64 bits and each pair's length."""
    x = x.to(F64)
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.to(F64)
    y, size, rot, p = x.clone(), x.abs(), sum(axes), 0
    for a, width in enumerate(axes):
        for j in range(width // 2):
            lo, hi = (2 * p, 2 * p + 1) if interleaved else (p, p + rot // 2)
            ang = pos[:, a].to(F64) * float(theta) ** (-2 * j / width)
            c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
            y[..., lo] = x[..., lo] * c - x[..., hi] * s
            y[..., hi] = x[..., lo] * s + x[..., hi] * c
            size[..., lo] = size[..., hi] = torch.hypot(x[..., lo], x[..., hi])
            p += 1
    return y, size


def check_rope(engine, q, k, pos, axes, interleaved, qn, kn, out_dtype, theta=10000.0, **kw):
    got = engine.qk_norm_rope(q, k, pos, axes, q_norm=qn, k_norm=kn, interleaved=interleaved, out_dtype=out_dtype,
                              theta=theta, **kw)
    torch.cuda.synchronize()
    for g, x, w in zip(got, (q, k), (qn, kn)):
        want, size = rotated(x, w, pos, axes, theta, interleaved, 1e-6)
        u = UNIT[out_dtype]
        assert_within(g, want, 2.0 ** -17 * size * (1 + u) + u * want.abs() + (2.0 ** -25 if out_dtype == torch.float16 else 0))


@pytest.mark.parametrize("d,axes", [(128, [16, 56, 56]), (128, [128]), (64, [16, 24, 24]), (96, [32, 64]), (256, [256]),
                                    (128, [64]), (80, [10, 30, 40]), (66, [22, 22, 22]), (128, []), (8, [2, 2, 2, 2])])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("tokens", [1, 7, 700])
def test_qk_norm_rope_layouts(engine, d, axes, interleaved, tokens):
    hq, hk = 6, 2
    qkv = randn((tokens, (hq + 2 * hk) * d), d + tokens, 2.0, torch.bfloat16)
    q, k = qkv[:, :hq * d].view(tokens, hq, d), qkv[:, hq * d:(hq + hk) * d].view(tokens, hk, d)
    pos = randn((tokens, len(axes)), 5).abs() * 100
    check_rope(engine, q, k, pos, axes, interleaved, 1 + randn((d,), 6, 0.2), 1 + randn((d,), 7, 0.2), torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("norms", ["both", "q", "none"])
def test_qk_norm_rope_types(engine, dtype, out_dtype, norms):
    q, k = randn((50, 24, 128), 1, 1.0, dtype), randn((50, 24, 128), 2, 1.0, dtype)
    pos = torch.randint(0, 64, (50, 3), device=DEV).float()
    qn = 1 + randn((128,), 3, 0.2) if norms != "none" else None
    kn = 1 + randn((128,), 4, 0.2) if norms == "both" else None
    check_rope(engine, q, k, pos, [16, 56, 56], True, qn, kn, out_dtype)


@pytest.mark.parametrize("interleaved", [True, False])
def test_qk_norm_rope_far_positions(engine, interleaved):
    """Angles of a million radians, fractional, negative and zero positions; other bases."""
    pos = torch.tensor([[0.0], [-3.5], [8191.25], [1e6 + 1], [16777215.0]], device=DEV)
    q, k = randn((5, 3, 64), 1, 1.0, torch.float32), randn((5, 1, 64), 2, 1.0, torch.float32)
    for theta in (10000.0, 500000.0, 3.0):
        check_rope(engine, q, k, pos, [64], interleaved, None, None, torch.float32, theta)


def test_qk_norm_rope_zero_rows_and_few_heads(engine):
    q, k = randn((3000, 1, 128), 1, 1.0, torch.bfloat16), torch.zeros((3000, 1, 128), dtype=torch.bfloat16, device=DEV)
    pos = torch.arange(3000, device=DEV).float()[:, None].repeat(1, 2)
    w = 1 + randn((128,), 3, 0.2)
    check_rope(engine, q, k, pos, [64, 64], True, w, w, torch.bfloat16)


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("d,start", [(128, 0), (64, 0), (96, 3)])
def test_qk_norm_rope_in_place_and_odd_starts(engine, interleaved, d, start):
    """In place over views of the projection; the rest of the buffer is untouched."""
    t, h = 33, 4
    buf = randn((t, 3 * h * d + 5), 4, 1.0, torch.bfloat16)
    was = buf.clone()
    q, k = (b[:, start + i * h * d:start + (i + 1) * h * d].unflatten(1, (h, d)) for i, b in ((0, buf), (1, buf)))
    pos, w = randn((t, 1), 5).abs() * 50, 1 + randn((d,), 6, 0.2)
    want = engine.qk_norm_rope(q.contiguous(), k.contiguous(), pos, [d], w, w, interleaved=interleaved)
    got = engine.qk_norm_rope(q, k, pos, [d], w, w, interleaved=interleaved, q_out=q, k_out=k)
    torch.cuda.synchronize()
    assert got[0].data_ptr() == q.data_ptr()
    for g, x in zip(got, want):
        assert float((g.float() - x.float()).abs().max()) <= 2.0 ** -8 * float(x.float().abs().max())
    assert torch.equal(buf[:, start + 2 * h * d:], was[:, start + 2 * h * d:]) and torch.equal(buf[:, :start], was[:, :start])


def test_qk_norm_rope_equals_the_projection_epilogue(engine):
    """On the values the fused qkv projection rotates by a table, the same result to its rounding."""
    t, h, d = 40, 3, 128
    x, w = randn((t, 256), 1, 1.0, torch.bfloat16), randn((3 * h * d, 256), 2, 0.05, torch.bfloat16)
    qn, kn = 1 + randn((d,), 3, 0.2), 1 + randn((d,), 4, 0.2)
    pos = torch.randint(0, 40, (t, 3), device=DEV).float()
    ang = torch.cat([pos[:, a:a + 1].to(F64) * 10000.0 ** (-torch.arange(0, n, 2, device=DEV, dtype=F64) / n)
                     for a, n in enumerate((16, 56, 56))], 1)
    pe = torch.stack([ang.cos(), -ang.sin(), ang.sin(), ang.cos()], -1).float().contiguous()
    out = torch.empty((t, 3 * h * d), dtype=torch.bfloat16, device=DEV)
    engine.gemm_qkv_rope([dict(x=x, w=w, bias=torch.zeros(3 * h * d, device=DEV), out=out, pe=pe, q_norm=qn, k_norm=kn)], h)
    flat = engine.gemm(x, w, out_dtype=torch.float32).view(t, 3, h, d)
    q, k = engine.qk_norm_rope(flat[:, 0], flat[:, 1], pos, [16, 56, 56], qn, kn, out_dtype=torch.bfloat16)
    torch.cuda.synchronize()
    for got, ref in ((q, out[:, :h * d]), (k, out[:, h * d:2 * h * d])):
        ref = ref.reshape(t, h, d).to(F64)
        assert_within(got, ref, 2.0 ** -7 * ref.abs() + 1e-4)


# ---------------------------------------------------------------------------- packed attention
def offsets(lens):
    return torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device=DEV)


def attend(q, k, v, lq, lk, causal, scale, starts_k=None):
    """The definition in 64 bits: (out, sum p |v| / sum p) per element."""
    group = q.shape[1] // k.shape[1]
    y, a = torch.zeros(q.shape, dtype=F64, device=DEV), torch.zeros(q.shape, dtype=F64, device=DEV)
    q0 = k0 = 0
    for b, (n, m) in enumerate(zip(lq, lk)):
        k0 = starts_k[b] if starts_k is not None else k0
        if n and m:
            qs, ks, vs = (t.to(F64).transpose(0, 1) for t in (q[q0:q0 + n], k[k0:k0 + m], v[k0:k0 + m]))
            s = qs @ ks.repeat_interleave(group, 0).transpose(1, 2) * scale
            if causal:
                s.masked_fill_(torch.arange(m, device=DEV) > torch.arange(n, device=DEV)[:, None] + m - n, -math.inf)
            p = torch.exp(s - s.amax(-1, keepdim=True).nan_to_num(neginf=0.0))
            tot = p.sum(-1, keepdim=True)
            p = torch.where(tot > 0, p / torch.where(tot > 0, tot, 1.0), 0.0)
            vs = vs.repeat_interleave(group, 0)
            y[q0:q0 + n], a[q0:q0 + n] = (p @ vs).transpose(0, 1), (p @ vs.abs()).transpose(0, 1)
        q0, k0 = q0 + n, k0 + m
    return y, a


def check_attention(engine, q, k, v, lq, lk, causal, scale=None, **kw):
    cu_q, cu_k = offsets(lq), offsets(lk)
    out = engine.attention_packed(q, k, v, cu_q, cu_k, causal=causal, scale=scale, **kw)
    torch.cuda.synchronize()
    engine.check_device_error()
    want, a = attend(q, k, v, lq, lk, causal, q.shape[2] ** -0.5 if scale is None else scale)
    u = UNIT[q.dtype]
    n = sum(lq)
    assert_within(out[:n], want[:n], ((1.1 * u + 1e-4) * a * (1 + u) + u * want.abs() + 1e-6)[:n])
    return out


def qkv(tq, tk, hq, hk, d, dtype, seed):
    return (randn((tq, hq, d), seed, 1.5, dtype), randn((tk, hk, d), seed + 1, 1.0, dtype),
            randn((tk, hk, d), seed + 2, 1.0, dtype))


LENGTHS = [[1], [5, 0, 3], [127, 128, 129], [256, 1, 255, 257], [300, 700, 20], [64] * 9, [0, 0, 33, 0], [1000]]


@pytest.mark.parametrize("lens", LENGTHS)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("hq,hk,d,dtype", [(3, 3, 128, torch.bfloat16), (8, 2, 128, torch.bfloat16),
                                           (6, 2, 64, torch.float16), (4, 4, 64, torch.bfloat16),
                                           (2, 1, 128, torch.float16)])
def test_attention_packed_self(engine, lens, causal, hq, hk, d, dtype):
    t = sum(lens)
    check_attention(engine, *qkv(t, t, hq, hk, d, dtype, t), lens, lens, causal)


@pytest.mark.parametrize("lq,lk", [([1, 1, 1], [1, 700, 33]), ([1] * 5, [0, 1, 16, 17, 5000]), ([2, 1, 3], [900, 0, 2]),
                                   ([4, 4], [4000, 3]), ([1], [20000]), ([5, 17, 0, 1], [100, 100, 100, 100]),
                                   ([200, 3, 150], [90, 400, 0]), ([130], [2000]), ([1, 300], [300, 1])])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("hq,hk,d,dtype", [(8, 2, 128, torch.bfloat16), (3, 3, 64, torch.float16),
                                           (16, 1, 64, torch.bfloat16), (24, 1, 128, torch.float16)])
def test_attention_packed_other_keys(engine, lq, lk, causal, hq, hk, d, dtype):
    """Queries against caches or another text: single tokens, fewer keys than queries (causal rows
    that see nothing are 0), empty sequences on either side."""
    check_attention(engine, *qkv(sum(lq), sum(lk), hq, hk, d, dtype, sum(lk)), lq, lk, causal)


@pytest.mark.parametrize("lq", [[1, 1, 1], [60, 200, 9]])
def test_attention_packed_cache_lengths(engine, lq):
    """Sequences at slots of a cache, filled to k_lens; the room left holds NaN and infinities."""
    slots, used = [512, 512, 512], [512, 130, 47]
    q, k, v = qkv(sum(lq), sum(slots), 4, 2, 128, torch.bfloat16, 3)
    for b, n in enumerate(used):
        k[512 * b + n:512 * (b + 1)] = float("nan")
        v[512 * b + n:512 * (b + 1)] = float("inf")
    for causal in (False, True):
        out = engine.attention_packed(q, k, v, offsets(lq), offsets(slots), causal=causal,
                                      k_lens=torch.tensor(used, dtype=torch.int32, device=DEV))
        torch.cuda.synchronize()
        want, a = attend(q, k, v, lq, used, causal, 128 ** -0.5, starts_k=[0, 512, 1024])
        u = UNIT[q.dtype]
        assert_within(out, want, (1.1 * u + 1e-4) * a * (1 + u) + u * want.abs() + 1e-6)


def test_attention_packed_neighbours_do_not_leak(engine):
    """A sequence of NaN between two others touches neither."""
    lens = [100, 60, 200]
    for hq, hk in ((2, 2), (4, 2)):
        q, k, v = qkv(360, 360, hq, hk, 128, torch.bfloat16, 8)
        clean = engine.attention_packed(q, k, v, offsets(lens))
        for t in (q, k, v):
            t[100:160] = float("nan")
        out = engine.attention_packed(q, k, v, offsets(lens))
        torch.cuda.synchronize()
        assert torch.equal(out[:100], clean[:100]) and torch.equal(out[160:], clean[160:])
        assert torch.isnan(out[100:160]).all()


def test_attention_packed_rising_scores(engine):
    """Later keys with far larger scores: the running maximum rises (and the sums are rescaled) at
    nearly every block; and scores of a few hundred units."""
    n = 1000
    q, k, v = qkv(n, n, 2, 2, 128, torch.bfloat16, 9)
    q[:, :, 0], k[:, :, 0] = 8.0, torch.linspace(0, 100, n, device=DEV).to(torch.bfloat16)[:, None]
    for causal in (False, True):
        check_attention(engine, q, k, v, [n], [n], causal)
        check_attention(engine, q, k, v, [400, 600], [400, 600], causal, scale=0.3)


def test_attention_packed_views_rows_outside_and_streams(engine):
    """Views of one projection, an output view with its own strides, rows of no sequence, a stream."""
    h, d, t = 3, 64, 200
    buf = randn((t, 3 * h * d + 8), 10, 1.0, torch.bfloat16)
    q, k, v = (buf[:, 8 + i * h * d:8 + (i + 1) * h * d].unflatten(1, (h, d)) for i in range(3))
    out = torch.full((t, h, 2 * d), 9.0, dtype=torch.bfloat16, device=DEV)
    cu = torch.tensor([10, 60, 190], dtype=torch.int32, device=DEV)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    engine.attention_packed(q, k, v, cu, out=out[:, :, d:], stream=st)
    torch.cuda.synchronize()
    want, a = attend(q[10:190], k[10:190], v[10:190], [50, 130], [50, 130], False, d ** -0.5)
    u = UNIT[q.dtype]
    assert_within(out[10:190, :, d:], want, (1.1 * u + 1e-4) * a * (1 + u) + u * want.abs() + 1e-6)
    assert bool((out[:, :, :d] == 9).all()) and bool((out[:10] == 9).all()) and bool((out[190:] == 9).all())


@pytest.mark.parametrize("lq", [1, 90])
def test_attention_packed_bad_offsets_stay_inside(engine, lq):
    """Offsets past the buffers, falling and negative: clamped, and what they name is computed."""
    q, k, v = qkv(2 * lq, 300, 2, 2, 64, torch.bfloat16, 11)
    guard = torch.full((2 * lq + 64, 2, 64), 5.0, dtype=torch.bfloat16, device=DEV)
    cu_q = torch.tensor([-7, lq, 10 ** 9], dtype=torch.int32, device=DEV)
    cu_k = torch.tensor([-3, 150, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    engine.attention_packed(q, k, v, cu_q, cu_k, out=guard[:2 * lq])
    torch.cuda.synchronize()
    engine.check_device_error()
    want, a = attend(q, k, v, [lq, lq], [150, 150], False, 0.125)
    u = UNIT[q.dtype]
    assert_within(guard[:2 * lq], want, (1.1 * u + 1e-4) * a * (1 + u) + u * want.abs() + 1e-6)
    assert bool((guard[2 * lq:] == 5).all())
    engine.attention_packed(q, k, v, cu_q.flip(0).contiguous(), cu_k, out=guard[:2 * lq])  # no sequence at all
    torch.cuda.synchronize()
    engine.check_device_error()


def test_attention_packed_no_keys_no_rows(engine):
    q, k, v = qkv(4, 0, 2, 2, 64, torch.bfloat16, 12)
    out = engine.attention_packed(q, k, v, offsets([1, 3]), offsets([0, 0]))
    torch.cuda.synchronize()
    assert out.shape == q.shape and not out.any()
    none = engine.attention_packed(q[:0], q, q, offsets([0]), offsets([4]))
    assert none.shape == (0, 2, 64)


def test_attention_packed_replays_with_other_lengths(engine):
    """The offsets are read by the kernels: a captured graph follows them."""
    t = 300
    q, k, v = qkv(t, t, 4, 2, 128, torch.bfloat16, 13)
    cu, out = offsets([300, 0]), torch.empty_like(q)
    engine.attention_packed(q, k, v, cu, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        engine.attention_packed(q, k, v, cu, out=out, causal=True)
    for lens in ([300, 0], [120, 180], [1, 299]):
        cu.copy_(offsets(lens))
        g.replay()
        torch.cuda.synchronize()
        want, a = attend(q, k, v, lens, lens, True, 128 ** -0.5)
        u = UNIT[q.dtype]
        assert_within(out, want, (1.1 * u + 1e-4) * a * (1 + u) + u * want.abs() + 1e-6)
    engine.check_device_error()
