"""A single-stream block over a packed batch: requests of different prompt lengths and image sizes in one
pass, with 8-bit integer weights.

The blocks of blocks.py run one sequence of [txt; img] rows, or halves of equal length, on one RoPE
table.  Here a batch is the concatenation of any number of sequences (`pack`): row offsets say where each begins, and
every row carries its own positions.  The block is that of the reference's single_block_forward
(chroma.cuh:1101-1157), its linear layers in the form of the reference's quantised path
(cublas_ops.cuh:294-352: weights with a scale per channel, activations with a scale per token):

    codes = quantize_s8(x_mod)                              once, for both halves of linear1
    q, k, v  = gemm_s8(codes, W1[0:9216])                    bf16
    cat[mlp] = gelu(gemm_s8(codes, W1[9216:]))               the GELU in the epilogue, into the concat buffer
    q, k     = qk_norm_rope(q, k, positions)                 in place
    cat[attn] = attention_packed(q, k, v, offsets)           into the concat buffer
    x       += gate * gemm_s8(cat, W2)                       quantised per token in the call

q, k and v leave their projection in bf16, the type that the attention takes, so that the rotation can write over its inputs
and qkv is held once; q and k are thus rounded before the norm and again after the rotation, where the epilogue of the
bf16 block's projection rounds them once, at the end.  In F32 they would be written and read as 4 bytes a value: for
1536 rows 38 MB more of traffic.  The rounding is at most 2^-8 of a value; the operands' 8 bits leave an rms of 1.3 % (two
roundings with a step of 4 sigma / 127).
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

import b2g
from blocks import DHEAD, HEADS, HIDDEN, MLP, SingleWeights

AXES = [16, 56, 56]  # values of a head turned by each coordinate: index, row, column


@dataclass
class SingleWeightsS8:
    linear1_q: torch.Tensor  # int8 [21504, 3072]
    linear1_s: torch.Tensor  # f32 [21504]
    linear1_b: torch.Tensor
    q_norm: torch.Tensor     # f32 [128]
    k_norm: torch.Tensor
    linear2_q: torch.Tensor  # int8 [3072, 15360]
    linear2_s: torch.Tensor  # f32 [3072]
    linear2_b: torch.Tensor


def quantize_single(w: SingleWeights) -> SingleWeightsS8:
    """The block's weights with 8 bits, done once when they are loaded."""
    return SingleWeightsS8(*b2g.quantize_s8(w.linear1_w), w.linear1_b, w.q_norm, w.k_norm,
                           *b2g.quantize_s8(w.linear2_w), w.linear2_b)


@dataclass
class Packed:
    """Where the sequences of a batch lie, on the device."""
    offsets: torch.Tensor    # int32 [batch + 1]
    positions: torch.Tensor  # f32 [rows, 3]


def pack(requests: list[tuple[int, int, int]], dev) -> Packed:
    """The layout of requests (txt tokens, rows of patches, columns of patches): txt tokens at the origin,
    patch (y, x) at (0, y, x), as in the reference's tables (rope.cuh:84-124)."""
    offsets, positions = [0], []
    for txt, rows, cols in requests:
        yx = torch.cartesian_prod(torch.arange(rows), torch.arange(cols)).reshape(-1, 2)
        positions.append(torch.nn.functional.pad(yx.float(), (1, 0, txt, 0)))
        offsets.append(offsets[-1] + txt + rows * cols)
    return Packed(torch.tensor(offsets, dtype=torch.int32, device=dev), torch.cat(positions).to(dev))


class Scratch:
    """Activations of a block over up to `rows` packed rows, allocated once."""

    def __init__(self, rows: int, dev):
        self.codes = torch.empty((rows, HIDDEN), dtype=torch.int8, device=dev)
        self.scales = torch.empty(rows, dtype=torch.float32, device=dev)
        self.qkv = torch.empty((rows, 3, HEADS, DHEAD), dtype=torch.bfloat16, device=dev)
        self.cat = torch.empty((rows, HIDDEN + MLP), dtype=torch.bfloat16, device=dev)


def single_block(w: SingleWeightsS8, x_mod: torch.Tensor, x: torch.Tensor, gate: torch.Tensor, batch: Packed,
                 s: Scratch) -> None:
    """Updates x [rows, 3072] (F32 residual stream of all sequences) in place from the modulated x_mod
    (bf16, fp16 or F32)."""
    n = x.shape[0]
    codes, scales = b2g.quantize_s8(x_mod, out=s.codes[:n], scales=s.scales[:n])
    qkv, cat = s.qkv[:n], s.cat[:n]
    b2g.gemm_s8(codes, w.linear1_q[:3 * HIDDEN], w.linear1_s[:3 * HIDDEN], w.linear1_b[:3 * HIDDEN],
                out=qkv.view(n, 3 * HIDDEN), x_scale=scales)
    b2g.gemm_s8(codes, w.linear1_q[3 * HIDDEN:], w.linear1_s[3 * HIDDEN:], w.linear1_b[3 * HIDDEN:],
                out=cat[:, HIDDEN:], epilogue="gelu", x_scale=scales)
    q, k, v = qkv.unbind(1)
    b2g.qk_norm_rope(q, k, batch.positions, AXES, q_norm=w.q_norm, k_norm=w.k_norm, q_out=q, k_out=k)
    b2g.attention_packed(q, k, v, batch.offsets, out=cat[:, :HIDDEN].unflatten(1, (HEADS, DHEAD)))
    b2g.gemm_s8(cat, w.linear2_q, w.linear2_s, w.linear2_b, out=x, epilogue="gated_residual", gate=gate)
