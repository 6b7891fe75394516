"""attention_packed on the B200: each way of pairing tiles, with more tiles than SMs, against what neighbours, the room left
in a cache and the largest scores hold.  Bounds: see test_packed_ops_gpu.py.
"""
from __future__ import annotations

import pytest
import torch
from test_packed_ops_gpu import DEV, UNIT, assert_within, attend, check_attention, offsets, qkv

pytestmark = pytest.mark.gpu

# (hq, hk, longest sequence): an even group shares its key head's stages; an odd one takes two tiles of a head, or, where
# there are at most 256 queries per sequence, two heads.
WAYS = {"heads of a group": (32, 8, 700), "tiles of a head": (27, 9, 700), "heads apart": (33, 11, 240)}
ways = pytest.mark.parametrize("way", WAYS)
widths = pytest.mark.parametrize("d,dtype", [(128, torch.bfloat16), (64, torch.float16)])
causes = pytest.mark.parametrize("causal", [False, True])


def lengths(way, lens):
    """Parts of the longest sequence as lengths; checks that they are taken the way they are meant to be."""
    hq, hk, longest = WAYS[way]
    lens = [int(longest * x) for x in lens]
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert (sum(lens) // 128 + len(lens)) * hq > sms and sum(lens) > 16 * len(lens)
    if (hq // hk) % 2:
        assert (sum(lens) > 256 * len(lens)) == (way == "tiles of a head")
    return hq, hk, lens


def within(out, q, k, v, lq, lk, causal, scale=None, starts=None, scores=1e-4):
    want, a = attend(q, k, v, lq, lk, causal, q.shape[2] ** -0.5 if scale is None else scale, starts)
    u = UNIT[q.dtype]
    assert_within(out, want, (1.1 * u + scores) * a * (1 + u) + u * want.abs() + 1e-6)


@ways
@widths
@causes
def test_neighbours_do_not_leak(engine, way, d, dtype, causal):
    """Sequences of NaN and of infinities between others, whose last blocks reach into them."""
    hq, hk, lens = lengths(way, [1.0, 0.41, 0.77, 0.13, 1.0, 0.55])
    t = sum(lens)
    q, k, v = qkv(t, t, hq, hk, d, dtype, 8)
    cu = offsets(lens)
    clean = engine.attention_packed(q, k, v, cu, causal=causal)
    ends = cu.tolist()
    bad = [1, 3]
    for x in (q, k, v):
        x[ends[1]:ends[2]] = float("nan")
        x[ends[3]:ends[4]] = float("inf")
    out = engine.attention_packed(q, k, v, cu, causal=causal)
    torch.cuda.synchronize()
    engine.check_device_error()
    for b in range(len(lens)):
        rows = slice(ends[b], ends[b + 1])
        if b in bad:
            assert torch.isnan(out[rows]).all()
        else:
            assert torch.equal(out[rows], clean[rows])
            within(out[rows], q[rows], k[rows], v[rows], [lens[b]], [lens[b]], causal)


@ways
@widths
@causes
def test_room_left_in_a_cache(engine, way, d, dtype, causal):
    """k_lens short of the slots, by less and by more than a block; the room holds NaN and infinities."""
    hq, hk, lq = lengths(way, [1.0, 0.3, 0.62, 0.99, 0.45, 0.7])
    slots, used = [768] * 6, [768, 130, 47, 0, 641, 512]
    q, k, v = qkv(sum(lq), sum(slots), hq, hk, d, dtype, 3)
    for b, n in enumerate(used):
        k[768 * b + n:768 * (b + 1)] = float("nan")
        v[768 * b + n:768 * (b + 1)] = float("inf") if b % 2 else float("nan")
    out = engine.attention_packed(q, k, v, offsets(lq), offsets(slots), causal=causal,
                                  k_lens=torch.tensor(used, dtype=torch.int32, device=DEV))
    torch.cuda.synchronize()
    engine.check_device_error()
    within(out, q, k, v, lq, used, causal, starts=[768 * b for b in range(6)])


@ways
@widths
@causes
def test_rising_scores(engine, way, d, dtype, causal):
    """Later keys with far larger scores: the running maximum rises, and the sums are rescaled, at nearly every block.

    The products sum up to 900 in steps of 16, at most 8 additions and a scaling of 2^-14 each; a score's error counts twice, in
    a key's weight and in the weights' sum."""
    hq, hk, lens = lengths(way, [1.0, 0.9, 0.2, 1.0, 0.8, 0.6])
    t = sum(lens)
    q, k, v = qkv(t, t, hq, hk, d, dtype, 9)
    q[:, :, 0] = 8.0
    k[:, :, 0] = torch.cat([torch.linspace(0, 100, n, device=DEV) for n in lens]).to(dtype)[:, None]
    cu = offsets(lens)
    for scale in (d ** -0.5, 0.3):
        out = engine.attention_packed(q, k, v, cu, causal=causal, scale=scale)
        torch.cuda.synchronize()
        engine.check_device_error()
        within(out, q, k, v, lens, lens, causal, scale, scores=1e-4 + 2 * 9 * 2.0 ** -14 * scale)


@ways
@widths
def test_offsets_outside_the_buffers(engine, way, d, dtype):
    """Offsets past the buffers and negative ones are clamped; nothing past the output is written."""
    hq, hk, lens = lengths(way, [1.0] * 6)
    t = sum(lens)
    q, k, v = qkv(t, t, hq, hk, d, dtype, 11)
    guard = torch.full((t + 64, hq, d), 5.0, dtype=dtype, device=DEV)
    cu = offsets(lens)
    cu[0], cu[-1] = -7, 10 ** 9
    engine.attention_packed(q, k, v, cu, out=guard[:t])
    torch.cuda.synchronize()
    engine.check_device_error()
    within(guard[:t], q, k, v, lens, lens, False)
    assert bool((guard[t:] == 5).all())


@ways
@widths
@causes
def test_rows_of_no_sequence_stay(engine, way, d, dtype, causal):
    """Rows before the first and after the last sequence are not written."""
    hq, hk, lens = lengths(way, [0.9, 0.5, 0.21, 1.0, 0.8, 0.66])
    t = sum(lens)
    q, k, v = qkv(t + 150, t + 150, hq, hk, d, dtype, 12)
    out = torch.full((t + 150, hq, 2 * d), 9.0, dtype=dtype, device=DEV)
    engine.attention_packed(q, k, v, offsets(lens) + 10, causal=causal, out=out[:, :, d:])
    torch.cuda.synchronize()
    engine.check_device_error()
    rows = slice(10, 10 + t)
    within(out[rows, :, d:], q[rows], k[rows], v[rows], lens, lens, causal)
    assert bool((out[:, :, :d] == 9).all()) and bool((out[:10] == 9).all()) and bool((out[10 + t:] == 9).all())


@ways
@widths
def test_replays_with_other_lengths(engine, way, d, dtype):
    hq, hk, lens = lengths(way, [1.0, 0.9, 0.2, 1.0, 0.8, 0.6])
    t = sum(lens)
    q, k, v = qkv(t, t, hq, hk, d, dtype, 13)
    cu, out = offsets(lens), torch.empty_like(q)
    engine.attention_packed(q, k, v, cu, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        engine.attention_packed(q, k, v, cu, out=out, causal=True)
    for other in (lens, lens[::-1], [t, 0, 0, 0, 0, 0], [0, 1, 129, 0, t - 131, 1]):
        cu.copy_(offsets(other))
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        engine.check_device_error()
        within(out, q, k, v, other, other, True)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hk,lens", [(32, 8, [700, 210, 539]), (27, 9, [700, 210, 539]), (33, 11, [240, 100, 200, 239]),
                                        (2, 2, [300, 5]), (8, 2, [1] * 5)])
@causes
def test_head_major_buffers(engine, hq, hk, lens, d, causal):
    """Heads apart by more than tokens are: [heads, tokens, d] seen as [tokens, heads, d]."""
    t = sum(lens)
    q, k, v = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in qkv(t, t, hq, hk, d, torch.bfloat16, 14))
    assert q.stride(1) > q.stride(0)
    out = torch.empty((hq, t, d), dtype=torch.bfloat16, device=DEV).transpose(0, 1)
    got = check_attention(engine, q, k, v, lens, lens, causal, out=out)
    assert got.data_ptr() == out.data_ptr()


@pytest.mark.parametrize("hq,hk,d", [(32, 8, 128), (9, 3, 64)])
@pytest.mark.parametrize("lq,lk", [([1] * 40 + [900], [300] * 40 + [900]), ([1] * 200 + [2000], [50] * 200 + [2000]),
                                   ([1, 700, 1, 1, 300, 2], [4000, 700, 1, 0, 900, 2])])
def test_prompts_and_single_tokens_in_one_call(engine, hq, hk, d, lq, lk):
    check_attention(engine, *qkv(sum(lq), sum(lk), hq, hk, d, torch.bfloat16, 15), lq, lk, True)
