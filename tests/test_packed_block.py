"""The packed single-stream block (packed.py): 8-bit linear layers, norm with rotation and packed attention
run together, against the block's formulas in 64 bits with one sequence at a time.

Tolerance of the update (relative L2 norm), for both sides quantise the same values of x_mod to the same codes: q, k, v,
the rotated q and k, P and the concat buffer are each rounded to bf16 once, at most 2^-8 of themselves: 4 such
roundings on the way of any value, 1.6 %.  Where rounding moves a value of the concat buffer across a half, its code
changes by one step: with a normal row (maximum 4 sigma, step 0.033 sigma) and a shift of 0.006 sigma a share
of 0.006 / 0.033 of the codes does, an rms error of sqrt(0.006 * 0.033) sigma = 1.4 %.  Together 3 %.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import blocks
import model
import packed

F64 = torch.float64
REQUESTS = [(5, 3, 7), (1, 1, 1), (77, 16, 12), (0, 1, 130), (3, 9, 9)]


def test_pack_positions_are_those_of_the_rope_table():
    txt, rows, cols = 7, 6, 4
    batch = packed.pack([(3, 2, 5), (txt, rows, cols)], "cpu")
    assert batch.offsets.tolist() == [0, 13, 13 + txt + rows * cols]
    assert batch.positions.dtype == torch.float32 and batch.positions.shape == (13 + txt + rows * cols, 3)
    table = model.rope_table(rows * model.PATCH, cols * model.PATCH, txt).reshape(-1, 64, 4)
    first = np.cumsum([0] + [d // 2 for d in packed.AXES[:-1]])  # pair 0 of an axis turns by the position itself
    pos = batch.positions[13:].numpy()
    np.testing.assert_allclose(table[:, first, 0], np.cos(pos), atol=2**-20)
    np.testing.assert_allclose(table[:, first, 2], np.sin(pos), atol=2**-20)


def quantised(x):
    top = x.abs().amax(1, keepdim=True)
    return torch.round(x * 127 / top) * (top / 127)


def plain_block(w, x_mod, x, gate, positions):
    """One sequence in 64 bits; w: the bf16 block's weights."""
    H, D = blocks.HEADS, blocks.DHEAD
    y = quantised(x_mod.to(F64)) @ quantised(w.linear1_w.to(F64)).T + w.linear1_b.to(F64)
    q, k, v = y[:, :3 * blocks.HIDDEN].unflatten(1, (3, H, D)).unbind(1)
    mlp = torch.nn.functional.gelu(y[:, 3 * blocks.HIDDEN:], approximate="tanh")
    angle = torch.cat([positions[:, i:i + 1].to(F64) * 10000.0 ** (-torch.arange(0, d, 2, dtype=F64, device=x.device) / d)
                       for i, d in enumerate(packed.AXES)], 1)[:, None]

    def norm_rope(t, scale):
        t = t * torch.rsqrt(t.pow(2).mean(2, keepdim=True) + 1e-6) * scale.to(F64)
        a, b = t[..., ::2], t[..., 1::2]
        return torch.stack([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()], 3).flatten(2)

    q, k = norm_rope(q, w.q_norm), norm_rope(k, w.k_norm)
    p = torch.softmax(torch.einsum("ihd,jhd->hij", q, k) * D ** -0.5, 2)
    attn = torch.einsum("hij,jhd->ihd", p, v).flatten(1)
    out = quantised(torch.cat([attn, mlp], 1)) @ quantised(w.linear2_w.to(F64)).T + w.linear2_b.to(F64)
    return x.to(F64) + gate.to(F64) * out


def inputs(dev):
    gen = torch.Generator(device=dev).manual_seed(5)
    w = blocks.random_single(gen, dev)
    batch = packed.pack(REQUESTS, dev)
    rows = int(batch.offsets[-1])
    x_mod = blocks._randn(gen, (rows, blocks.HIDDEN)).to(torch.bfloat16)
    return w, batch, x_mod, blocks._randn(gen, (rows, blocks.HIDDEN)), blocks._randn(gen, blocks.HIDDEN)


@pytest.mark.gpu
def test_single_block(engine):
    dev = "cuda:0"
    w, batch, x_mod, x, gate = inputs(dev)
    got = x.clone()
    scratch = packed.Scratch(x.shape[0] + 9, dev)
    packed.single_block(packed.quantize_single(w), x_mod, got, gate, batch, scratch)
    ends = batch.offsets.tolist()
    for a, b in zip(ends, ends[1:]):
        want = plain_block(w, x_mod[a:b], x[a:b], gate, batch.positions[a:b]) - x[a:b].to(F64)
        err = (got[a:b].to(F64) - x[a:b].to(F64) - want).norm() / want.norm()
        assert float(err) <= 0.03, (a, b, float(err))


@pytest.mark.gpu
def test_single_block_is_the_same_in_a_graph(engine):
    dev = "cuda:0"
    w, batch, x_mod, x, gate = inputs(dev)
    w8, scratch = packed.quantize_single(w), packed.Scratch(x.shape[0], dev)
    eager, replayed = x.clone(), x.clone()
    packed.single_block(w8, x_mod, eager, gate, batch, scratch)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        packed.single_block(w8, x_mod, replayed, gate, batch, scratch)
    replayed.copy_(x)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(eager, replayed)
