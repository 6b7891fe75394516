"""The packed single-stream block with each request's own adapter and with attention over chosen key blocks: the further
operators run together as a user runs them, against the block's formulas in 64 bits with one sequence at a time.

Tolerance of the update (relative L2 norm): that of the block without them (tests/test_packed_block.py), 3 %, and one more
rounding to bf16, 2^-8: with adapters the MLP half leaves its product before the GELU.
"""
from __future__ import annotations

import pytest
import torch

import blocks
import packed
from test_packed_block import F64, inputs, quantised

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
RANK, MANY = 24, 3


def adapters_of(gen):
    def make(*shape, scale):
        return (blocks._randn(gen, shape) * scale).to(torch.bfloat16)

    return packed.AdaptersS8(make(MANY, RANK, 3072, scale=3072 ** -0.5), make(MANY, 21504, RANK, scale=0.4),
                             make(MANY, RANK, 15360, scale=15360 ** -0.5), make(MANY, 3072, RANK, scale=0.4),
                             torch.tensor([0.5, 1.0, 2.0], device=DEV))


def plain_block(w, x_mod, x, gate, positions, low=None, visible=None):
    """One sequence in 64 bits.  low: its adapter's (A1, B1, A2, B2, scale); visible [heads, rows, rows]: keys that a
    query sees."""
    H, D = blocks.HEADS, blocks.DHEAD
    y = quantised(x_mod.to(F64)) @ quantised(w.linear1_w.to(F64)).T + w.linear1_b.to(F64)
    if low:
        y = y + low[4] * (x_mod.to(F64) @ low[0].to(F64).T) @ low[1].to(F64).T
    q, k, v = y[:, :3 * blocks.HIDDEN].unflatten(1, (3, H, D)).unbind(1)
    mlp = torch.nn.functional.gelu(y[:, 3 * blocks.HIDDEN:], approximate="tanh")
    angle = torch.cat([positions[:, i:i + 1].to(F64) * 10000.0 ** (-torch.arange(0, d, 2, dtype=F64, device=x.device) / d)
                       for i, d in enumerate(packed.AXES)], 1)[:, None]

    def norm_rope(t, scale):
        t = t * torch.rsqrt(t.pow(2).mean(2, keepdim=True) + 1e-6) * scale.to(F64)
        a, b = t[..., ::2], t[..., 1::2]
        return torch.stack([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()], 3).flatten(2)

    s = torch.einsum("ihd,jhd->hij", norm_rope(q, w.q_norm), norm_rope(k, w.k_norm)) * D ** -0.5
    if visible is not None:
        s = s.masked_fill(~visible, -torch.inf)
    attn = torch.einsum("hij,jhd->ihd", torch.softmax(s, 2), v).flatten(1)
    cat = torch.cat([attn, mlp], 1)
    out = quantised(cat) @ quantised(w.linear2_w.to(F64)).T + w.linear2_b.to(F64)
    if low:
        out = out + low[4] * (cat @ low[2].to(F64).T) @ low[3].to(F64).T
    return gate.to(F64) * out


def check(w, batch, x_mod, x, gate, got, adapters=None, ids=None, masks=None):
    ends = batch.offsets.tolist()
    for i, (a, b) in enumerate(zip(ends, ends[1:])):
        low = None
        if adapters and 0 <= ids[i] < MANY:
            low = (adapters.linear1_a[ids[i]], adapters.linear1_b[ids[i]], adapters.linear2_a[ids[i]], adapters.linear2_b[ids[i]],
                   float(adapters.scale[ids[i]]))
        want = plain_block(w, x_mod[a:b], x[a:b], gate, batch.positions[a:b], low, masks[i] if masks else None)
        err = (got[a:b].to(F64) - x[a:b].to(F64) - want).norm() / want.norm()
        assert float(err) <= 0.03 + 2.0 ** -8, (a, b, float(err))


def test_block_with_adapters(engine):
    w, batch, x_mod, x, gate = inputs(DEV)
    adapters, ids = adapters_of(torch.Generator(device=DEV).manual_seed(9)), [1, -1, 0, 2, 7]
    got = x.clone()
    packed.single_block(packed.quantize_single(w), x_mod, got, gate, batch, packed.Scratch(x.shape[0] + 9, DEV), adapters,
                        torch.tensor(ids, dtype=torch.int32, device=DEV))
    check(w, batch, x_mod, x, gate, got, adapters, ids)


def test_block_without_an_adapter_keeps_its_result(engine):
    """Nobody has an adapter: the block's own update, but for the MLP half's rounding before the GELU."""
    w, batch, x_mod, x, gate = inputs(DEV)
    adapters = adapters_of(torch.Generator(device=DEV).manual_seed(9))
    w8, scratch = packed.quantize_single(w), packed.Scratch(x.shape[0], DEV)
    plain, got = x.clone(), x.clone()
    packed.single_block(w8, x_mod, plain, gate, batch, scratch)
    packed.single_block(w8, x_mod, got, gate, batch, scratch, adapters, torch.full((5,), -1, dtype=torch.int32, device=DEV))
    torch.cuda.synchronize()
    assert float((got - plain).norm() / (plain - x).norm()) <= 0.014 + 2 * 2.0 ** -8  # (codes that the rounding moves: 1.4 %)


@pytest.mark.parametrize("with_adapters", [False, True])
def test_block_with_chosen_key_blocks(engine, with_adapters):
    """Attention over few blocks.  The choice is taken again from the rotated q and k that the block leaves."""
    import b2g

    w, batch, x_mod, x, gate = inputs(DEV)
    batch = packed.pack([(200, 20, 25), (3, 5, 7), (130, 1, 1)], DEV)
    n = int(batch.offsets[-1])
    gen = torch.Generator(device=DEV).manual_seed(3)
    x_mod = blocks._randn(gen, (n, blocks.HIDDEN)).to(torch.bfloat16)
    x = blocks._randn(gen, (n, blocks.HIDDEN))
    adapters, ids = (adapters_of(gen), [2, 0, -1]) if with_adapters else (None, None)
    got, scratch = x.clone(), packed.Scratch(n, DEV)
    choice = packed.Choice(top=1, first=1, last=1, max_k=700)
    packed.single_block(packed.quantize_single(w), x_mod, got, gate, batch, scratch, adapters,
                        torch.tensor(ids, dtype=torch.int32, device=DEV) if ids else None, choice)
    q, k, _ = scratch.qkv.unbind(1)
    chosen = b2g.select_blocks(q, b2g.block_means(k, batch.offsets), batch.offsets, 1, first=1, last=1, max_k=700)
    bits = (chosen[..., None] >> torch.arange(32, device=DEV)).bitwise_and(1).flatten(2).bool()  # [tile, head, block]
    masks, tile, ends = [], 0, batch.offsets.tolist()
    for a, b in zip(ends, ends[1:]):
        tiles, rows = -(-(b - a) // 128), b - a
        mine = bits[tile:tile + tiles].repeat_interleave(128, 0)[:rows].repeat_interleave(128, 2)[..., :rows]
        masks.append(mine.transpose(0, 1))
        tile += tiles
    assert int(bits[:tile].sum(2).max()) == 3 and not bool(masks[0].all())
    check(w, batch, x_mod, x, gate, got, adapters, ids, masks)


def test_block_options_are_the_same_in_a_graph(engine):
    w, batch, x_mod, x, gate = inputs(DEV)
    adapters, ids = adapters_of(torch.Generator(device=DEV).manual_seed(9)), torch.tensor([1, -1, 0, 2, 0], dtype=torch.int32, device=DEV)
    w8, scratch, choice = packed.quantize_single(w), packed.Scratch(x.shape[0], DEV), packed.Choice(top=1, first=1, max_k=300)
    eager, replayed = x.clone(), x.clone()
    packed.single_block(w8, x_mod, eager, gate, batch, scratch, adapters, ids, choice)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        packed.single_block(w8, x_mod, replayed, gate, batch, scratch, adapters, ids, choice)
    replayed.copy_(x)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(eager, replayed)
