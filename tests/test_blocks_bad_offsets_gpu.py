"""Offsets that jump back and forth (0, n, 0, n, ..): every other sequence holds the same rows, so that sums over the sequences
in front of one (blocks, tiles) exceed 32 bits, or the rows that there are.  Nothing outside the buffers is read or written: what
lies past the rows of the means counts as not there.
"""
from __future__ import annotations

import pytest
import torch

from test_attention_blocks_gpu import BLOCK, DEV, F64, UNIT, assert_within, attend, ceil, choice, ints, offsets, qkv, randn

pytestmark = pytest.mark.gpu
MANY = 65536              # sequences
ROOM = (1 << 16) + 64     # blocks of every other one: 2^31 in front of the last ones


def back_and_forth(n, batch):
    return torch.arange(batch + 1, device=DEV).remainder(2).mul(n).int()


def test_block_means_where_the_blocks_in_front_pass_32_bits(engine):
    n, rows = ROOM * BLOCK, 4
    k = torch.zeros((n, 1, 64), dtype=torch.bfloat16, device=DEV)
    k[:rows * BLOCK] = randn((rows * BLOCK, 1, 64), 1, 1.0, torch.bfloat16)
    since = torch.full((MANY,), n - 1, dtype=torch.int32, device=DEV)
    since[0] = 0
    buf = torch.full((3 * rows, 1, 64), 7.0, device=DEV)
    engine.block_means(k, back_and_forth(n, MANY), since=since, out=buf[rows:2 * rows])
    torch.cuda.synchronize()
    x = k[:rows * BLOCK].to(F64).unflatten(0, (rows, BLOCK))
    assert_within(buf[rows:2 * rows], x.mean(1), 36 * 2.0 ** -24 * x.abs().mean(1))
    assert bool((buf[:rows] == 7).all()) and bool((buf[2 * rows:] == 7).all())


def test_select_blocks_where_the_blocks_in_front_pass_32_bits(engine):
    top, sight = 3, 32
    q, means = randn((MANY, 1, 64), 2, 1.0, torch.bfloat16), randn((ROOM, 1, 64), 3)
    got = engine.select_blocks(q, means, torch.arange(MANY + 1, dtype=torch.int32, device=DEV), top, max_k=sight * BLOCK,
                               cu_k=back_and_forth(ROOM * BLOCK, MANY))
    torch.cuda.synchronize()
    assert got.shape == (MANY // BLOCK + MANY, 1, 1)
    assert torch.equal(got[:1], choice(q[:1], means, [1], [sight * BLOCK], [sight * BLOCK], top, 0, 0, False, 1, 1))
    # No row of the means: equal scores, of which the first are taken.  No key, no tile: nothing.
    assert bool((got[2:MANY:2] == (1 << top) - 1).all())
    assert bool((got[1:MANY:2] == 0).all()) and bool((got[MANY:] == 0).all())


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("hq,hk,d", [(4, 2, 64), (3, 3, 128)])
@pytest.mark.parametrize("chosen_rows", [12, 500])
def test_attention_over_the_same_rows_again_and_again(engine, causal, hq, hk, d, chosen_rows):
    """More tiles than rows have room for, each of which gives the same; those without a row of `chosen` see nothing, and
    in the other call there are none."""
    n, batch = 700, 64
    q, k, v = qkv(n, n, hq, hk, d, torch.bfloat16, 5)
    bits = torch.full((chosen_rows, hk, 1), -1, dtype=torch.int32, device=DEV)
    cu = back_and_forth(n, batch)
    packed = engine.attention_packed(q, k, v, cu, causal=causal)
    got = engine.attention_blocks(q, k, v, bits, cu, causal=causal)
    torch.cuda.synchronize()
    engine.check_device_error()
    every = torch.ones((ceil(n), hk, ceil(n)), dtype=torch.bool, device=DEV)
    want, a = attend(q, k, v, every, [n], [n], causal, d ** -0.5)
    u = UNIT[q.dtype]
    bound = (1.1 * u + 1e-4) * a * (1 + u) + u * want.abs() + 1e-6
    assert_within(packed, want, bound)
    if chosen_rows > batch // 2 * ceil(n):
        assert_within(got, want, bound)


def test_offsets_out_of_the_buffers_and_back(engine):
    """Clamped, and over again: no sequence's rows are outside, whatever the others are."""
    q, k, v = qkv(300, 300, 4, 2, 64, torch.bfloat16, 7)
    wild = ints([0, 2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, -5, 300, 100, 299] * 40 + [0])
    means = engine.block_means(k, wild)
    chosen = engine.select_blocks(q, means, wild, 2, first=1, causal=True, max_k=300)
    buf = torch.full((500, 4, 64), 3.0, dtype=torch.bfloat16, device=DEV)
    engine.attention_blocks(q, k, v, chosen, wild, causal=True, out=buf[100:400])
    engine.attention_blocks(q, k, v, chosen, wild, cu_k=offsets([1] * 320), out=buf[100:400])
    torch.cuda.synchronize()
    engine.check_device_error()
    assert bool((buf[:100] == 3).all()) and bool((buf[400:] == 3).all())
