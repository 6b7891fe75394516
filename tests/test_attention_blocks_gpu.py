"""Means of key blocks, the choice of blocks and attention over chosen blocks on the B200, against their definitions
in 64 bits.

Tolerances per element, with u the unit roundoff of a type (half its epsilon) and e = 2^-24 that of fp32:
  block_means       a lane adds 32 keys in turn, four such sums are added, one division: 36 roundings of e of sum |k| / n
  select_blocks     equal.  The inputs make scores either exactly equal (ties) or far apart beside 2^-52
  attention_blocks  P rounded to the operands' type (u sum p |v| / sum p), the scores' fp32 sums of D products of a
                    few units (1e-4 of the same), the output's rounding
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F64 = torch.float64
UNIT = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}
BLOCK = 128


def randn(shape, seed, scale=1.0, dtype=torch.float32):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def assert_within(got, want, bound, what=""):
    got = got.to(F64)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    over = ((got - want).abs() - bound).nan_to_num(0.0)
    at = int(over.argmax())
    assert float(over.max()) <= 0, (what, at, float(got.flatten()[at]), float(want.flatten()[at]))


def ints(values):
    return torch.tensor(list(values), dtype=torch.int32, device=DEV)


def offsets(lens):
    return ints([0] + list(torch.tensor(lens).cumsum(0)))


def ceil(n):
    return -(-n // BLOCK)


# ---------------------------------------------------------------------------- means
def means_of(k, room, lens):
    """The definition: (means, bound) with a row for every block that there is room for."""
    rows = k.shape[0] // BLOCK + len(room)
    m, a = (torch.zeros((rows, *k.shape[1:]), dtype=F64, device=DEV) for _ in range(2))
    at = k0 = 0
    for n, have in zip(room, lens):
        for j in range(ceil(have)):
            x = k[k0 + j * BLOCK:k0 + min(have, (j + 1) * BLOCK)].to(F64)
            m[at + j], a[at + j] = x.mean(0), x.abs().mean(0)
        at += ceil(n)
        k0 += n
    return m, 36 * 2.0 ** -24 * a + 1e-38


@pytest.mark.parametrize("lens", [[1], [127, 128, 129], [0, 300, 0, 5], [1000, 1, 257], [0], [3] * 40])
@pytest.mark.parametrize("hk,d,dtype", [(1, 64, torch.bfloat16), (8, 128, torch.float16), (3, 128, torch.bfloat16), (24, 64, torch.float16)])
def test_block_means(engine, lens, hk, d, dtype):
    qkv = randn((sum(lens), 3, hk, d), sum(lens), 1.0, dtype)
    k = qkv[:, 1]
    got = engine.block_means(k, offsets(lens))
    torch.cuda.synchronize()
    want, bound = means_of(k, lens, lens)
    assert got.shape == want.shape and got.dtype == torch.float32
    assert_within(got, want, bound)


def test_block_means_of_caches_and_steps(engine):
    """Caches with room left (whose rows hold NaN); then steps that write a few keys update the kept means alone."""
    room, lens, hk, d = [512, 256, 128, 384], [130, 0, 128, 255], 2, 128
    k = randn((sum(room), hk, d), 1, 1.0, torch.bfloat16)
    starts = [0, 512, 768, 896]
    for s, n, r in zip(starts, lens, room):
        k[s + n:s + r] = float("nan")
    cu = offsets(room)
    means = engine.block_means(k, cu, k_lens=ints(lens))
    for step, more in enumerate(([1, 1, 0, 1], [3, 200, 0, 2], [1, 1, 0, 1])):
        grown = [n + m for n, m in zip(lens, more)]
        for s, n, g in zip(starts, lens, grown):
            k[s + n:s + g] = randn((g - n, hk, d), 5 + step, 1.0, torch.bfloat16)
        kept = means.clone()
        assert engine.block_means(k, cu, k_lens=ints(grown), since=ints(lens), out=means) is means
        torch.cuda.synchronize()
        want, bound = means_of(k, room, grown)
        assert_within(means, want, bound, step)
        # Blocks in front of the new keys, and those of sequences without any, are as they were.
        at = 0
        for n, r, m in zip(lens, room, more):
            untouched = ceil(r) if m == 0 else n // BLOCK
            assert torch.equal(means[at:at + untouched], kept[at:at + untouched])
            at += ceil(r)
        lens = grown


def test_block_means_writes_its_rows_only(engine):
    lens = [200, 140]
    k = randn((340, 2, 64), 3, 1.0, torch.bfloat16)
    buf = torch.full((9, 2, 64), 7.0, device=DEV)
    engine.block_means(k, offsets(lens), out=buf[1:7])
    short = torch.full((4, 2, 64), 7.0, device=DEV)
    engine.block_means(k, offsets(lens), out=short[:3])  # the last block has no row
    torch.cuda.synchronize()
    want, bound = means_of(k, lens, lens)
    assert_within(buf[1:5], want, bound)
    assert bool((buf[0] == 7).all()) and bool((buf[7:] == 7).all()) and bool((buf[5:7] == 0).all())
    assert torch.equal(short[:3], buf[1:4]) and bool((short[3] == 7).all())


# ---------------------------------------------------------------------------- choice
def sight(lq, lk, causal, tile):
    """Keys that the first and the last query of a tile see."""
    last = min(lq, (tile + 1) * BLOCK) - 1
    return tuple(max(0, min(lk, i + 1 + lk - lq)) if causal else lk for i in (tile * BLOCK, last))


def choice(q, means, lq, lk, room, top, first, last, causal, words, tiles):
    """The definition, with sums of 64 bits and a sort."""
    hk, group = means.shape[1], q.shape[1] // means.shape[1]
    out = torch.zeros((tiles, hk, words), dtype=torch.int64)
    tile = q0 = at = 0
    for n, m, r in zip(lq, lk, room):
        for t in range(ceil(n)):
            lo, hi = sight(n, m, causal, t)
            nb = min(ceil(hi), 32 * words)
            sure = [j for j in range(nb) if j < first or j >= nb - last or min((j + 1) * BLOCK, hi) > lo]
            summed = q[q0 + t * BLOCK:q0 + min(n, (t + 1) * BLOCK)].to(F64).unflatten(1, (hk, group)).sum((0, 2))
            score = torch.einsum("hd,bhd->hb", summed, means[at:at + nb].to(F64)).nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf).tolist()
            for h in range(hk):
                free = sorted((j for j in range(nb) if j not in sure), key=lambda j: (-score[h][j], j))[:top]  # noqa: B023
                for j in sure + free:
                    out[tile, h, j // 32] |= 1 << j % 32
            tile += 1
        q0 += n
        at += ceil(r)
    return torch.where(out >= 1 << 31, out - (1 << 32), out).int().to(DEV)


def check_choice(engine, lq, lk, room, hq, hk, d, dtype, top, first, last, causal, seed=0, q=None, means=None):
    rows = sum(room) // BLOCK + len(room)
    q = randn((sum(lq), hq, d), seed, 1.0, dtype) if q is None else q
    means = randn((rows, hk, d), seed + 1) if means is None else means
    got = engine.select_blocks(q, means, offsets(lq), top, cu_k=offsets(room), k_lens=ints(lk), first=first, last=last,
                               causal=causal, max_k=max(room))
    torch.cuda.synchronize()
    words = -(-ceil(max(room)) // 32)
    assert got.shape == (sum(lq) // BLOCK + len(lq), hk, words)
    assert torch.equal(got, choice(q, means, lq, lk, room, top, first, last, causal, words, got.shape[0]))


@pytest.mark.parametrize("lq,lk", [([1], [1]), ([1, 1, 1], [0, 700, 5000]), ([300, 0, 129], [300, 0, 129]), ([40, 1000], [900, 1000]),
                                   ([260], [100]), ([2, 5], [9000, 4097])])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("hq,hk,d,dtype", [(3, 3, 128, torch.bfloat16), (8, 2, 64, torch.float16), (6, 1, 128, torch.float16)])
@pytest.mark.parametrize("top,first,last", [(3, 1, 1), (0, 0, 0), (7, 0, 2), (100, 4, 0)])
def test_select_blocks(engine, lq, lk, causal, hq, hk, d, dtype, top, first, last):
    check_choice(engine, lq, lk, [n + 200 for n in lk], hq, hk, d, dtype, top, first, last, causal, sum(lk))


@pytest.mark.parametrize("lk,top", [(60000, 40), (140000, 300), (140000, 5000)])
def test_select_blocks_long_caches(engine, lk, top):
    """More blocks than are ranked by counting: the threshold is searched."""
    check_choice(engine, [1, 130], [lk, 40000], [lk, 40000], 4, 2, 64, torch.bfloat16, top, 1, 1, True)


@pytest.mark.parametrize("lens", [[4100, 300, 129], [500] * 9, [3000, 0, 1700]])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("hq,hk,d,dtype", [(24, 24, 128, torch.bfloat16), (48, 24, 64, torch.float16)])
def test_select_blocks_many_tiles(engine, lens, causal, hq, hk, d, dtype):
    """Four tiles a CTA, of one sequence and of two, the last ones of none."""
    check_choice(engine, lens, lens, lens, hq, hk, d, dtype, 5, 1, 1, causal, sum(lens))
    check_choice(engine, lens, [max(0, n - 150) for n in lens], lens, hq, hk, d, dtype, 2, 0, 0, causal, sum(lens))


@pytest.mark.parametrize("blocks", [20, 600])
@pytest.mark.parametrize("top", [1, 6, 19, 64])
def test_select_blocks_ties_and_odd_scores(engine, blocks, top):
    """Whole numbers, many of them equal; zeros of both signs; infinities and NaN in the means."""
    g = torch.Generator(device=DEV).manual_seed(blocks + top)
    q = torch.randint(-1, 2, (1, 2, 64), generator=g, device=DEV).to(torch.bfloat16)
    q[:, :, 0] = 1
    means = torch.zeros((blocks + 1, 1, 64), device=DEV)
    means[:, 0, 0] = torch.randint(-2, 3, (blocks + 1,), generator=g, device=DEV).float()
    means[3, 0, 0] = float("inf")
    means[5, 0, 0] = float("nan")
    means[6, 0, 0] = -float("inf")
    means[8, 0, 0] = -0.0
    check_choice(engine, [1], [blocks * BLOCK], [blocks * BLOCK], 2, 1, 64, torch.bfloat16, top, 0, 0, False, q=q, means=means)


def test_select_blocks_few_words_bad_offsets_and_views(engine):
    """Blocks past the words are never chosen; offsets outside the buffers are clamped; q from a fused projection."""
    lens = [40 * BLOCK, 3 * BLOCK]
    qkv = randn((sum(lens), 3, 2, 64), 3, 1.0, torch.bfloat16)
    q, means = qkv[:, 0], engine.block_means(qkv[:, 1], offsets(lens))
    few = torch.full((50, 2, 1), 7, dtype=torch.int32, device=DEV)
    assert engine.select_blocks(q, means, offsets(lens), 40, out=few[:49]) .data_ptr() == few.data_ptr()
    torch.cuda.synchronize()
    assert bool((few[:40] == -1).all()) and bool((few[40:43] == 7).all()) and bool((few[43:49] == 0).all())
    assert bool((few[49] == 7).all())
    wild = torch.tensor([-50, 2 ** 30, 77, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    engine.select_blocks(q, means, wild, 4)
    engine.block_means(qkv[:, 1], wild)
    engine.block_means(qkv[:, 1], wild, k_lens=ints([2 ** 31 - 1, -4, 9]), since=ints([-9, 2 ** 30, 5]), out=means)
    chosen = engine.select_blocks(q, means, offsets(lens), 4)
    for rows in (q, q[:5]):
        engine.attention_blocks(rows, qkv[:, 1], qkv[:, 2], chosen, wild)
        engine.attention_blocks(rows, qkv[:, 1], qkv[:, 2], chosen[:2], wild, causal=True, k_lens=ints([2 ** 31 - 1, -4, 9]))
    torch.cuda.synchronize()
    engine.check_device_error()


# ---------------------------------------------------------------------------- attention
def attend(q, k, v, chosen, lq, lk, causal, scale, starts_k=None):
    """The definition in 64 bits: (out, sum p |v| / sum p) per element; chosen: truth values [tile, key head, block]."""
    group = q.shape[1] // k.shape[1]
    y, a = torch.zeros(q.shape, dtype=F64, device=DEV), torch.zeros(q.shape, dtype=F64, device=DEV)
    q0 = k0 = tile = 0
    for b, (n, m) in enumerate(zip(lq, lk)):
        k0 = starts_k[b] if starts_k is not None else k0
        if n and m:
            qs, ks, vs = (t.to(F64).transpose(0, 1) for t in (q[q0:q0 + n], k[k0:k0 + m], v[k0:k0 + m]))
            s = qs @ ks.repeat_interleave(group, 0).transpose(1, 2) * scale
            mine = chosen[tile:tile + ceil(n)].repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 2)[..., :m]
            mine = torch.nn.functional.pad(mine, (0, m - mine.shape[-1]))
            s.masked_fill_(~mine.transpose(0, 1).repeat_interleave(group, 0), -math.inf)
            if causal:
                s.masked_fill_(torch.arange(m, device=DEV) > torch.arange(n, device=DEV)[:, None] + m - n, -math.inf)
            p = torch.exp(s - s.amax(-1, keepdim=True).nan_to_num(neginf=0.0))
            tot = p.sum(-1, keepdim=True)
            p = torch.where(tot > 0, p / torch.where(tot > 0, tot, 1.0), 0.0)
            vs = vs.repeat_interleave(group, 0)
            y[q0:q0 + n], a[q0:q0 + n] = (p @ vs).transpose(0, 1), (p @ vs.abs()).transpose(0, 1)
        q0, k0, tile = q0 + n, k0 + m, tile + ceil(n)
    return y, a


def pack(bits):
    bits = torch.nn.functional.pad(bits, (0, -bits.shape[-1] % 32))
    w = (bits.unflatten(-1, (-1, 32)).long() << torch.arange(32, device=DEV)).sum(-1)
    return (w - ((w >> 31) << 32)).int()


def random_choice(lq, lk, hk, seed, share=0.4, extra=0):
    """Truth values [tiles, hk, blocks], blocks out of sight among them; some tiles choose nothing."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    shape = (max(1, sum(map(ceil, lq))), hk, ceil(max(lk)) + extra)
    bits = torch.rand(shape, generator=g, device=DEV) < share
    return bits & (torch.rand(shape[:2], generator=g, device=DEV) < 0.85)[..., None]


def check_attention(engine, q, k, v, bits, lq, lk, causal, scale=None, room=None, **kw):
    starts = None if room is None else [0] + list(torch.tensor(room).cumsum(0))
    out = engine.attention_blocks(q, k, v, pack(bits), offsets(lq), cu_k=offsets(lk if room is None else room), causal=causal,
                                  scale=scale, **kw)
    torch.cuda.synchronize()
    engine.check_device_error()
    want, a = attend(q, k, v, bits, lq, lk, causal, q.shape[2] ** -0.5 if scale is None else scale, starts)
    u = UNIT[q.dtype]
    n = sum(lq)
    assert_within(out[:n], want[:n], ((1.1 * u + 1e-4) * a * (1 + u) + u * want.abs() + 1e-6)[:n])
    return out


def qkv(tq, tk, hq, hk, d, dtype, seed):
    return (randn((tq, hq, d), seed, 1.5, dtype), randn((tk, hk, d), seed + 1, 1.0, dtype),
            randn((tk, hk, d), seed + 2, 1.0, dtype))


HEADS = [(3, 3, 128, torch.bfloat16), (8, 2, 128, torch.bfloat16), (6, 2, 64, torch.float16), (4, 4, 64, torch.bfloat16),
         (2, 1, 128, torch.float16)]


@pytest.mark.parametrize("lens", [[1], [5, 0, 3], [127, 128, 129], [256, 1, 255, 257], [300, 700, 20], [64] * 9, [0, 0, 33, 0],
                                  [1000], [4200, 600]])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("hq,hk,d,dtype", HEADS)
def test_attention_blocks_self(engine, lens, causal, hq, hk, d, dtype):
    t = sum(lens)
    check_attention(engine, *qkv(t, t, hq, hk, d, dtype, t), random_choice(lens, lens, hk, t, extra=3), lens, lens, causal)


@pytest.mark.parametrize("lq,lk", [([1, 1, 1], [1, 700, 33]), ([1] * 5, [0, 1, 16, 17, 5000]), ([2, 1, 3], [900, 0, 2]),
                                   ([4, 4], [4000, 3]), ([1], [40000]), ([5, 17, 0, 1], [100, 100, 100, 100]),
                                   ([200, 3, 150], [90, 400, 0]), ([130], [2000]), ([1, 300], [300, 1]), ([150, 1] + [0] * 12, [800, 500] + [0] * 12)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("hq,hk,d,dtype", [(8, 2, 128, torch.bfloat16), (3, 3, 64, torch.float16),
                                           (16, 1, 64, torch.bfloat16), (24, 1, 128, torch.float16)])
def test_attention_blocks_other_keys(engine, lq, lk, causal, hq, hk, d, dtype):
    """Queries against caches or another text, few and many of them."""
    check_attention(engine, *qkv(sum(lq), sum(lk), hq, hk, d, dtype, sum(lk)), random_choice(lq, lk, hk, sum(lk), extra=1), lq, lk, causal)


@pytest.mark.parametrize("lq", [[1, 1, 1], [60, 200, 9]])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_blocks_caches_and_unchosen_values(engine, lq, causal):
    """The room left in a cache and the blocks that nobody chose hold NaN and infinities."""
    room, used = [512, 512, 512], [512, 130, 47]
    q, k, v = qkv(sum(lq), sum(room), 4, 2, 128, torch.bfloat16, 3)
    bits = random_choice(lq, used, 2, 5, share=0.7)
    bits[..., 1] = False
    for b, n in enumerate(used):
        for t, what in ((k, float("nan")), (v, float("inf"))):
            t[512 * b + n:512 * (b + 1)] = what
            t[512 * b + 128:512 * b + 256] = what
    kept = [t.clone() for t in (q, k, v)]
    for t in (k, v):  # the oracle's masked scores stay finite
        t.nan_to_num_(0.0, 0.0)
    want, a = attend(q, k, v, bits, lq, used, causal, 128 ** -0.5, [0, 512, 1024])
    out = engine.attention_blocks(*kept, pack(bits), offsets(lq), cu_k=offsets(room), causal=causal, k_lens=ints(used))
    torch.cuda.synchronize()
    u = UNIT[q.dtype]
    assert_within(out, want, (1.1 * u + 1e-4) * a * (1 + u) + u * want.abs() + 1e-6)


@pytest.mark.parametrize("hq,hk,d", [(4, 4, 128), (8, 2, 64)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens", [[700, 129, 1, 0, 300], [1] * 8])
def test_all_blocks_chosen_is_attention_packed(engine, hq, hk, d, causal, lens):
    """Same tiles, same order of keys: every bit set gives what attention_packed gives."""
    q, k, v = qkv(sum(lens), sum(lens), hq, hk, d, torch.bfloat16, 4)
    bits = torch.full((sum(map(ceil, lens)), hk, 1), -1, dtype=torch.int32, device=DEV)
    got = engine.attention_blocks(q, k, v, bits, offsets(lens), causal=causal)
    want = engine.attention_packed(q, k, v, offsets(lens), causal=causal)
    torch.cuda.synchronize()
    u = UNIT[q.dtype]
    assert float((got.to(F64) - want.to(F64)).abs().max()) <= 4 * u * float(v.abs().max())


def test_attention_blocks_rising_scores(engine):
    """Scores that grow by thousands from block to block: the maximum in use is raised again and again."""
    lens, hq = [600, 1200], 2
    for d in (64, 128):
        q, k, v = qkv(1800, 1800, hq, hq, d, torch.bfloat16, 6)
        k *= torch.arange(1800, device=DEV)[:, None, None].to(torch.bfloat16) / 100
        for lq in (lens, [1, 1]):
            n = sum(lq)
            check_attention(engine, q[:n], k, v, random_choice(lq, lens, hq, d, share=0.6), lq, lens, False, scale=1.0)


def test_attention_blocks_views_rows_outside_and_streams(engine):
    """Parts of one buffer, an output of its own strides, rows of no sequence untouched, another stream."""
    lens, hq, hk, d = [300, 150], 4, 2, 128
    total = sum(lens) + 40
    buf = randn((total, (hq + 2 * hk) * d), 7, 1.0, torch.bfloat16)
    q = buf[:, :hq * d].view(total, hq, d)
    k = buf[:, hq * d:(hq + hk) * d].view(total, hk, d)
    v = buf[:, (hq + hk) * d:].view(total, hk, d)
    bits = random_choice(lens, lens, hk, 9, share=0.8)
    out = torch.full((total, hq, 2 * d), 3.0, dtype=torch.bfloat16, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    engine.attention_blocks(q, k, v, pack(bits), offsets(lens), causal=True, out=out[..., :d], stream=side)
    side.synchronize()
    want, a = attend(q, k, v, bits, lens, lens, True, d ** -0.5)
    u = UNIT[q.dtype]
    n = sum(lens)
    assert_within(out[:n, :, :d], want[:n], ((1.1 * u + 1e-4) * a * (1 + u) + u * want.abs() + 1e-6)[:n])
    assert bool((out[n:] == 3).all()) and bool((out[..., d:] == 3).all())


@pytest.mark.parametrize("lq", [[1, 1, 1], [300, 20, 129]])
def test_attention_blocks_replays_with_other_lengths_and_choices(engine, lq):
    """A captured run of the three operators follows offsets, lengths and queries changed after the capture."""
    room = [1024, 640, 384]
    q, k, v = qkv(sum(lq), sum(room), 4, 2, 64, torch.bfloat16, 13)
    cu_q, cu_k, lens = offsets(lq), offsets(room), ints([1000, 640, 129])
    out, means = torch.empty_like(q), torch.empty((19, 2, 64), device=DEV)

    def step():
        engine.block_means(k, cu_k, k_lens=lens, out=means)
        chosen = engine.select_blocks(q, means, cu_q, 2, cu_k=cu_k, k_lens=lens, first=1, last=1, causal=True, max_k=1024)
        engine.attention_blocks(q, k, v, chosen, cu_q, cu_k=cu_k, k_lens=lens, causal=True, out=out)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for new_lens, new_cu in (([1000, 640, 129], lq), ([77, 0, 384], lq), ([513, 600, 1], [lq[0] - 1, lq[1] + 1, lq[2]])):
        lens.copy_(ints(new_lens))
        cu_q.copy_(offsets(new_cu))
        q.copy_(randn(q.shape, new_lens[0], 1.5, torch.bfloat16))
        graph.replay()
        got = out.clone()
        step()
        torch.cuda.synchronize()
        assert torch.equal(got, out), (new_lens, new_cu)


def test_the_three_together(engine):
    """Means, choice and attention of a packed batch against the definitions in 64 bits."""
    lens, hq, hk, d = [900, 130, 2100], 4, 2, 128
    q, k, v = qkv(sum(lens), sum(lens), hq, hk, d, torch.bfloat16, 17)
    means = engine.block_means(k, offsets(lens))
    chosen = engine.select_blocks(q, means, offsets(lens), 3, first=1, causal=True, max_k=2100)
    tiles = sum(map(ceil, lens))
    want = choice(q, means.float(), lens, lens, lens, 3, 1, 0, True, 1, chosen.shape[0])
    assert torch.equal(chosen, want)
    bits = (chosen[:tiles, ..., None] >> torch.arange(32, device=DEV)).bitwise_and(1).flatten(2).bool()
    out = engine.attention_blocks(q, k, v, chosen, offsets(lens), causal=True)
    torch.cuda.synchronize()
    y, a = attend(q, k, v, bits[..., :ceil(2100)], lens, lens, True, d ** -0.5)
    u = UNIT[q.dtype]
    assert_within(out, y, (1.1 * u + 1e-4) * a * (1 + u) + u * y.abs() + 1e-6)


def test_attention_blocks_repeats_bit_for_bit(engine):
    for lq, lk in (([1] * 4, [5000] * 4), ([700, 300], [700, 300])):
        q, k, v = qkv(sum(lq), sum(lk), 8, 2, 128, torch.bfloat16, 23)
        bits = pack(random_choice(lq, lk, 2, 3))
        runs = [engine.attention_blocks(q, k, v, bits, offsets(lq), cu_k=offsets(lk), causal=True) for _ in range(5)]
        torch.cuda.synchronize()
        assert all(torch.equal(runs[0], r) for r in runs[1:])


def test_no_rows_no_keys(engine):
    q, k, v = qkv(4, 0, 2, 2, 64, torch.bfloat16, 1)
    cu_q, cu_k = offsets([1, 3]), offsets([0, 0])
    means = engine.block_means(k, cu_k)
    chosen = engine.select_blocks(q, means, cu_q, 3, cu_k=cu_k, first=1, last=1)
    assert float(engine.attention_blocks(q, k, v, chosen, cu_q, cu_k=cu_k).float().abs().max()) == 0
    none = engine.attention_blocks(q, *qkv(300, 300, 2, 2, 64, torch.bfloat16, 2)[1:], chosen[:0], cu_q, cu_k=offsets([200, 100]))
    assert float(none.float().abs().max()) == 0
    empty = offsets([])
    assert engine.block_means(k, empty).shape[0] == 0
    assert engine.attention_blocks(q[:0], k, v, chosen[:0], empty).shape == (0, 2, 64)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("hq,hk,d,dtype", [(8, 4, 128, torch.bfloat16), (4, 4, 64, torch.float16)])
def test_attention_blocks_many_short_sequences(engine, causal, hq, hk, d, dtype):
    """Hundreds of sequences with few queries: more pairs of sequence and key head than one line holds."""
    lq = [(1, 2, 0, 1, 17)[i % 5] for i in range(300)]
    lk = [(40, 1, 300, 0, 130)[i % 5] for i in range(300)]
    check_attention(engine, *qkv(sum(lq), sum(lk), hq, hk, d, dtype, 31), random_choice(lq, lk, hk, 32, extra=1), lq, lk, causal)


@pytest.mark.parametrize("lq", [[1, 1], [150, 90]])
def test_blocks_past_32_bits_of_elements(engine, lq):
    """Keys and values whose rows lie far apart in one buffer of more than 2^31 elements."""
    lk, hq, hk, d, ld = [700, 400], 4, 2, 128, 1 << 21
    buf = torch.empty(sum(lk) * ld, dtype=torch.bfloat16, device=DEV)
    k = buf.as_strided((sum(lk), hk, d), (ld, d, 1))
    v = buf.as_strided((sum(lk), hk, d), (ld, d, 1), hk * d)
    q, near_k, near_v = qkv(sum(lq), sum(lk), hq, hk, d, torch.bfloat16, 33)
    k.copy_(near_k)
    v.copy_(near_v)
    means = engine.block_means(k, offsets(lk))
    assert torch.equal(means, engine.block_means(near_k, offsets(lk)))
    chosen = engine.select_blocks(q, means, offsets(lq), 2, cu_k=offsets(lk), last=1)
    got = engine.attention_blocks(q, k, v, chosen, offsets(lq), cu_k=offsets(lk))
    assert torch.equal(got, engine.attention_blocks(q, near_k, near_v, chosen, offsets(lq), cu_k=offsets(lk)))


def test_blocks_on_several_streams_at_once(engine):
    """Calls side by side on four streams, and two captured graphs replayed side by side: workspaces of their own."""
    lq, lk, hq, hk, d = [1] * 6, [3000, 20, 700, 1500, 0, 4000], 8, 2, 128
    cu_q, cu_k = offsets(lq), offsets(lk)
    sets = [qkv(6, sum(lk), hq, hk, d, torch.bfloat16, 40 + i) for i in range(4)]

    def run(i, stream=None):
        q, k, v = sets[i]
        means = engine.block_means(k, cu_k, stream=stream)
        chosen = engine.select_blocks(q, means, cu_q, 4, cu_k=cu_k, first=1, last=1, stream=stream)
        return engine.attention_blocks(q, k, v, chosen, cu_q, cu_k=cu_k, stream=stream)

    want = [run(i) for i in range(4)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    for _ in range(20):
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(run(i))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run(i))
        graphs.append(graph)
    for _ in range(20):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("n,hq,hk", [(64, 8, 8), (130, 4, 4), (64, 16, 8)])
def test_attention_blocks_many_long_caches(engine, causal, n, hq, hk):
    """Single queries to many caches, of which most are in use: heads of their own go to tiles, groups to rows."""
    lq, lk = [1 + (i == 3) for i in range(n)], [1300 - 11 * (i % 30) for i in range(n)]
    check_attention(engine, *qkv(sum(lq), sum(lk), hq, hk, 128, torch.bfloat16, n), random_choice(lq, lk, hk, 32), lq, lk, causal)


@pytest.mark.parametrize("lq", [8, 9, 16, 17])
@pytest.mark.parametrize("hq,hk", [(2, 2), (4, 2), (8, 1)])
def test_attention_blocks_between_the_forms(engine, lq, hq, hk):
    lens, lk = [lq] * 5, [700, 3, 130, 0, 1024]
    check_attention(engine, *qkv(5 * lq, sum(lk), hq, hk, 64, torch.float16, lq), random_choice(lens, lk, hk, lq), lens, lk, True)
