"""Low-rank adapters of a packed batch's requests on the B200 against their definition in 64 bits.

Tolerances per element, with u the unit roundoff of y's type and e = 2^-24 that of fp32.  A sum of n products in fp32 on the
tensor cores is off by at most n 2 e times the sum of the products' magnitudes (each step may truncate):
  t        K 2 e (|x| |a|^T)
  delta    s (that, and t's representation: 2^-17 of it in bf16 or 2^-21 of the row's largest in fp16) |b|^T, and
           (2 R + 8) 2 e (s |t| |b|^T)
  out      delta's, times the gate or the activation's largest slope 1.13; 2^-16 of it for the exponential, whose argument is
           rounded at up to 100 units; the output's rounding
Whole numbers whose products stay below 2^16 come out exactly.
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F64 = torch.float64
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
UNIT = {t: torch.finfo(t).eps / 2 for t in (BF16, F16, F32)}


def randn(shape, seed, scale=1.0, dtype=F32):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def ints(values):
    return torch.tensor(list(values), dtype=torch.int32, device=DEV)


def offsets(lens):
    return ints([0] + list(torch.tensor(lens).cumsum(0)))


def plain(x, a, b, y, lens, ids, scale, epilogue, gate):
    """The definition in 64 bits: (out, bound)."""
    e2, K, R = 2.0 ** -23, a.shape[2], a.shape[1]
    delta, off = torch.zeros(y.shape, dtype=F64, device=DEV), torch.zeros(y.shape, dtype=F64, device=DEV)
    at = 0
    for n, i in zip(lens, ids):
        if 0 <= i < a.shape[0] and n:
            xs, A, B = x[at:at + n].to(F64), a[i].to(F64), b[i].to(F64)
            s = 1.0 if scale is None else float(scale[i])
            t = xs @ A.T
            t_off = K * e2 * (xs.abs() @ A.abs().T)
            t_off = t_off + (2.0 ** -17 * t.abs() if x.dtype == BF16 else 2.0 ** -21 * t.abs().amax(1, keepdim=True))
            delta[at:at + n] = s * (t @ B.T)
            off[at:at + n] = abs(s) * (t_off @ B.abs().T + (2 * R + 8) * e2 * (t.abs() @ B.abs().T))
        at += n
    z = y.to(F64)
    if epilogue == "gated_residual":
        out, off = z + gate.to(F64) * delta, gate.to(F64).abs() * off
    else:
        z = z + delta
        out = {"none": z, "gelu": torch.nn.functional.gelu(z, approximate="tanh"), "silu": z * torch.sigmoid(z)}[epilogue]
        off = 1.13 * off
        if epilogue != "none":
            off = off + 2.0 ** -16 * out.abs() + 1e-30
    u = UNIT[y.dtype]
    return out, off * (1 + u) + (u + 2 * e2) * out.abs() + 2 * e2 * y.to(F64).abs() + 1e-7 * (y.dtype == F16)


def assert_within(got, want, bound, what=""):
    got = got.to(F64)
    over = ((got - want).abs() - bound)
    assert bool(torch.isfinite(got).all()), what
    at = int(over.argmax())
    assert float(over.max()) <= 0, (what, at, float(got.flatten()[at]), float(want.flatten()[at]), float(bound.flatten()[at]))


def inputs(lens, K, N, R, adapters, dtype, y_dtype, seed):
    m = sum(lens)
    return (randn((m, K), seed, 1.0, dtype), randn((adapters, R, K), seed + 1, K ** -0.5, dtype),
            randn((adapters, N, R), seed + 2, 0.3, dtype), randn((m, N), seed + 3, 1.0, y_dtype))


def ids_of(lens, adapters, seed):
    g = torch.Generator().manual_seed(seed)
    return [int(i) for i in torch.randint(-1, adapters + 1, (len(lens),), generator=g)]


def check(engine, lens, K, N, R, adapters=3, dtype=BF16, y_dtype=BF16, epilogue="none", seed=0, ids=None, scaled=True):
    x, a, b, y = inputs(lens, K, N, R, adapters, dtype, y_dtype, seed)
    ids = ids_of(lens, adapters, seed) if ids is None else ids
    scale = torch.exp(randn((adapters,), seed + 4)) if scaled else None
    gate = randn((N,), seed + 5) if epilogue == "gated_residual" else None
    kept = y.clone()
    got = engine.lora(x, a, b, y, offsets(lens), ids=ints(ids), scale=scale, epilogue=epilogue, gate=gate)
    torch.cuda.synchronize()
    engine.check_device_error()
    assert torch.equal(y, kept) and got.dtype == y.dtype
    want, bound = plain(x, a, b, y, lens, ids, scale, epilogue, gate)
    assert_within(got, want, bound, (lens, ids))


LENGTHS = [[1], [1] * 9, [5, 0, 17, 1], [33, 64, 1, 40], [127, 128, 129], [300, 0, 700, 20], [900, 50], [0, 0, 3, 0]]


@pytest.mark.parametrize("lens", LENGTHS)
@pytest.mark.parametrize("R", [8, 16, 24, 32, 56, 64, 128])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_lora_lengths_and_ranks(engine, lens, R, dtype):
    check(engine, lens, 256, 320, R, dtype=dtype, y_dtype=dtype, seed=sum(lens) + R, ids=[i % 3 for i in range(len(lens))])


@pytest.mark.parametrize("lens", [[3, 1, 6], [40, 70, 9], [300, 150]])
@pytest.mark.parametrize("epilogue", ["none", "gelu", "silu", "gated_residual"])
@pytest.mark.parametrize("dtype,y_dtype", [(BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
def test_lora_epilogues_and_types(engine, lens, epilogue, dtype, y_dtype):
    check(engine, lens, 520, 264, 16, dtype=dtype, y_dtype=y_dtype, epilogue=epilogue, seed=len(epilogue))
    check(engine, lens, 520, 264, 16, dtype=dtype, y_dtype=y_dtype, epilogue=epilogue, seed=7, scaled=False)


@pytest.mark.parametrize("lens", [[2, 7], [60, 33], [200, 130]])
@pytest.mark.parametrize("K,N", [(8, 1), (24, 7), (40, 257), (1000, 513), (4104, 30), (15360, 100)])
@pytest.mark.parametrize("y_dtype", [BF16, F32])
def test_lora_odd_sizes(engine, lens, K, N, y_dtype):
    check(engine, lens, K, N, 40, y_dtype=y_dtype, seed=K + N)


@pytest.mark.parametrize("lens", [[700, 130, 90], [40, 3, 60]])
@pytest.mark.parametrize("y_dtype", [BF16, F32])
@pytest.mark.parametrize("R", [16, 64, 128])
@pytest.mark.parametrize("epilogue", ["none", "silu"])
def test_lora_wide_layers_with_and_without_adapters(engine, lens, y_dtype, R, epilogue):
    """Many steps along N; a request without an adapter, whose rows are copied, between two with one."""
    for _ in range(3):
        check(engine, lens, 64, 9000, R, y_dtype=y_dtype, epilogue=epilogue, seed=R, ids=[0, -1, 2])
        check(engine, lens, 64, 9000, R, y_dtype=y_dtype, epilogue=epilogue, seed=R, ids=[-1, 1, 9])


@pytest.mark.parametrize("lens", [[1, 2, 1, 0], [30, 60, 3], [260, 129]])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("R", [8, 64, 128])
def test_lora_whole_numbers_are_exact(engine, lens, dtype, R):
    g = torch.Generator(device=DEV).manual_seed(R)
    def draw(*s):
        return torch.randint(-2, 3, s, generator=g, device=DEV)
    m = sum(lens)
    x, a, b = draw(m, 1024).to(dtype), draw(2, R, 1024).to(dtype), draw(2, 520, R).to(dtype)
    y = 100.0 * draw(m, 520).float()
    got = engine.lora(x, a, b, y, offsets(lens), ids=ints([i % 2 for i in range(len(lens))]))
    torch.cuda.synchronize()
    want, _ = plain(x, a, b, y, lens, [i % 2 for i in range(len(lens))], None, "none", None)
    assert torch.equal(got.to(F64), want)


@pytest.mark.parametrize("lens", [[2, 5, 3], [40, 9, 60], [200, 70, 140]])
@pytest.mark.parametrize("epilogue", ["none", "gelu", "gated_residual"])
@pytest.mark.parametrize("start,width", [(0, 264), (3, 131)])
def test_lora_in_place_on_part_of_a_buffer(engine, lens, epilogue, start, width):
    """y and out a part of a wider buffer, x a part of another, b rows of a fused projection's adapter; rows and columns
    beside them, and rows of no request, stay as they were."""
    rows = sum(lens) + 11
    wide = randn((rows, 600), 1, 1.0, BF16)
    wide_x = randn((rows, 512), 2, 1.0, BF16)
    x, y = wide_x[:, 128:384], wide[:, start:start + width]
    a, b = randn((3, 16, 256), 3, 0.06, BF16), randn((3, 500, 16), 4, 0.3, BF16)[:, 100:100 + width]
    gate = randn((width,), 5) if epilogue == "gated_residual" else None
    kept, ids = wide.clone(), [2, -1, 0]
    got = engine.lora(x, a, b, y, offsets(lens), ids=ints(ids), epilogue=epilogue, gate=gate, out=y)
    torch.cuda.synchronize()
    assert got is y
    n = sum(lens)
    want, bound = plain(x[:n], a, b, kept[:n, start:start + width], lens, ids, None, epilogue, gate)
    assert_within(wide[:n, start:start + width], want, bound)
    assert torch.equal(wide[n:], kept[n:]) and torch.equal(wide[:, :start], kept[:, :start])
    assert torch.equal(wide[:, start + width:], kept[:, start + width:])


@pytest.mark.parametrize("lens", [[1, 3], [50, 40], [300, 20]])
def test_lora_one_down_for_several_ups(engine, lens):
    """lora_down's t serves the parts of a fused projection; together they are lora over all of it, bit for bit."""
    x, a, b, y = inputs(lens, 384, 640, 32, 2, BF16, BF16, 3)
    cu, ids = offsets(lens), ints([1, 0])
    t = engine.lora_down(x, a, cu, ids=ids)
    parts = [engine.lora_up(t, b[:, s], y[:, s].contiguous(), cu, ids=ids) for s in (slice(0, 256), slice(256, 640))]
    whole = engine.lora(x, a, b, y, cu, ids=ids)
    torch.cuda.synchronize()
    assert t.shape == (sum(lens), 32) and t.dtype == F32
    want = torch.cat([x[:lens[0]].to(F64) @ a[1].to(F64).T, x[lens[0]:].to(F64) @ a[0].to(F64).T])
    mass = torch.cat([x[:lens[0]].to(F64).abs() @ a[1].to(F64).abs().T, x[lens[0]:].to(F64).abs() @ a[0].to(F64).abs().T])
    assert_within(t, want, 384 * 2.0 ** -23 * mass)
    assert torch.equal(torch.cat(parts, 1), whole)


@pytest.mark.parametrize("lens", [[1, 2, 4], [100, 60, 200]])
def test_lora_rows_do_not_leak(engine, lens):
    """A request of NaN and infinities between two others, and adapters of NaN that nobody uses, touch neither."""
    x, a, b, y = inputs(lens, 256, 300, 16, 3, BF16, F32, 5)
    cu, ids = offsets(lens), ints([0, 2, 0])
    clean = engine.lora(x, a, b, y, cu, ids=ids)
    lo, hi = lens[0], lens[0] + lens[1]
    x[lo:hi] = float("nan")
    x[lo, 5] = float("inf")
    a[1], b[1] = float("nan"), float("inf")
    out = engine.lora(x, a, b, y, cu, ids=ids)
    torch.cuda.synchronize()
    assert torch.equal(out[:lo], clean[:lo]) and torch.equal(out[hi:], clean[hi:])
    assert bool(torch.isnan(out[lo + 1:hi]).all())


@pytest.mark.parametrize("size", [1e-6, 1e4])
def test_lora_f16_far_from_one(engine, size):
    """t = x a^T may leave fp16's range, its product with b need not."""
    lens = [3, 200]
    x, a, b, y = inputs(lens, 512, 72, 16, 2, F16, F32, 9)
    a = (a.float() * min(size, 300.0)).to(F16) if size > 1 else (a.float() * 0.02).to(F16)
    x = (x.float() * (size / 300.0 if size > 1 else 0.01)).to(F16)
    got = engine.lora(x, a, b, y, offsets(lens))
    torch.cuda.synchronize()
    want, bound = plain(x, a, b, y, lens, [0, 1], None, "none", None)
    assert_within(got, want, bound)


def test_lora_bad_offsets_and_no_adapters(engine):
    x, a, b, y = inputs([40], 64, 48, 8, 2, BF16, BF16, 1)
    wild = torch.tensor([-50, 2 ** 30, 7, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    for rows in (40, 2):
        engine.lora(x[:rows], a, b, y[:rows], wild, ids=ints([2 ** 31 - 1, -2 ** 31, 1]))
    few = engine.lora(x, a[:0], b[:0], y, offsets([30, 10]), epilogue="silu")
    some = engine.lora(x, a, b, y, offsets([30, 10]), ids=ints([-1, 5]), epilogue="silu")
    none = engine.lora(x[:0], a, b, y[:0], offsets([0]))
    torch.cuda.synchronize()
    engine.check_device_error()
    assert torch.equal(few, some) and none.shape == (0, 48)
    z = y.to(F64)
    assert_within(few, z * torch.sigmoid(z), 2.0 ** -8 * z.abs() + 2.0 ** -15 * z.abs() + 1e-30)


@pytest.mark.parametrize("lens", [[1, 1, 1], [100, 30, 200]])
def test_lora_replays_with_other_requests_and_repeats(engine, lens):
    """A captured call follows offsets and adapters changed afterwards; on another stream; bit for bit the same each time."""
    x, a, b, y = inputs(lens, 256, 200, 16, 3, BF16, BF16, 2)
    cu, ids, out = offsets(lens), ints([0, 1, 2]), torch.empty_like(y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    engine.lora(x, a, b, y, cu, ids=ids, out=out, epilogue="gelu", stream=side)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        engine.lora(x, a, b, y, cu, ids=ids, out=out, epilogue="gelu")
    n = sum(lens)
    for new, which in (([0, 1, 2], lens), ([2, -1, 0], [n, 0, 0]), ([1, 1, 1], [0, n - 1, 1])):
        ids.copy_(ints(new))
        cu.copy_(offsets(which))
        graph.replay()
        first = out.clone()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(first, out)
        want, bound = plain(x, a, b, y, which, new, None, "gelu", None)
        assert_within(first, want, bound)


def test_lora_past_32_bits_of_elements(engine):
    """y of more than 2^31 elements: the last rows are reached."""
    rows, N = 70000, 32768
    x = randn((rows, 64), 1, 1.0, BF16)
    a, b = randn((2, 8, 64), 2, 0.1, BF16), randn((2, N, 8), 3, 0.3, BF16)
    y = torch.zeros((rows, N), dtype=BF16, device=DEV)
    lens = [rows - 300, 300]
    engine.lora(x, a, b, y, offsets(lens), out=y)
    torch.cuda.synchronize()
    for lo, i in ((0, 0), (rows - 300, 1), (rows - 2, 1)):
        part = slice(lo, lo + 2)
        want, bound = plain(x[part], a, b, torch.zeros((2, N), dtype=BF16, device=DEV), [2], [i], None, "none", None)
        assert_within(y[part], want, bound)


@pytest.mark.parametrize("lens", [[3, 1, 6], [40, 70, 9], [500, 40, 390]])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("R", [16, 64, 128])
def test_lora_rows_of_zeros_with_large_scales(engine, lens, dtype, R):
    x, a, b, y = inputs(lens, 128, 264, R, 3, dtype, F32, R)
    x[::2] = 0
    scale = torch.tensor([1.0, 8.0, 4096.0], device=DEV)
    got = engine.lora(x, a, b, y, offsets(lens), scale=scale)
    assert torch.equal(got[::2], y[::2])
    want, bound = plain(x, a, b, y, lens, [0, 1, 2], scale, "none", None)
    assert_within(got, want, bound)


@pytest.mark.parametrize("lens", [[1, 3, 2], [40, 70, 9], [500, 40, 390]])
@pytest.mark.parametrize("R", [16, 128])
def test_lora_one_matrix_for_all_adapters(engine, lens, R):
    """Adapters that share A or B, and differ in their scale: views with a stride of 0; and others apart by part of a row."""
    x, a, b, y = inputs(lens, 128, 264, R, 3, BF16, BF16, R)
    scale = torch.tensor([0.5, 1.0, 2.0], device=DEV)
    one_a, one_b = a[:1].expand(3, R, 128), b[:1].expand(3, 264, R)
    woven_a = a.transpose(0, 1).contiguous().transpose(0, 1)
    woven_b = b.transpose(0, 1).contiguous().transpose(0, 1)
    for va, vb in ((one_a, b), (a, one_b), (one_a, one_b), (woven_a, woven_b)):
        got = engine.lora(x, va, vb, y, offsets(lens), scale=scale)
        want, bound = plain(x, va, vb, y, lens, [0, 1, 2], scale, "none", None)
        assert_within(got, want, bound)
        assert torch.equal(got, engine.lora(x, va.contiguous(), vb.contiguous(), y, offsets(lens), scale=scale))
