"""CPU checks of what the packed single-stream block refuses before its first launch: nothing of x is updated then."""
from __future__ import annotations

from dataclasses import replace

import pytest
import torch

import b2g
import packed

BF16 = torch.bfloat16


def adapters(**kw):
    good = packed.AdaptersS8(torch.zeros(2, 8, 3072, dtype=BF16), torch.zeros(2, 21504, 8, dtype=BF16),
                             torch.zeros(2, 16, 15360, dtype=BF16), torch.zeros(2, 3072, 16, dtype=BF16))
    return replace(good, **kw)


@pytest.mark.parametrize("given,x_type,word", [
    (adapters(), torch.float16, "x_mod must be BF16"),
    (adapters(), torch.float32, "x_mod must be BF16"),
    (adapters(linear1_b=torch.zeros(2, 21504, 8, dtype=torch.float16)), BF16, "linear1 must be BF16"),
    (adapters(linear1_a=torch.zeros(2, 8, 3072, dtype=torch.float16), linear1_b=torch.zeros(2, 21504, 8, dtype=torch.float16)),
     torch.float16, "x_mod must be BF16"),
    (adapters(linear2_a=torch.zeros(2, 16, 15360)), BF16, "linear2 must be BF16"),
    (adapters(linear2_a=torch.zeros(2, 16, 12288, dtype=BF16)), BF16, "linear2 must be .adapters, rank, 15360"),
    (adapters(linear2_b=torch.zeros(2, 3072, 8, dtype=BF16)), BF16, "linear2 must be .adapters, rank, 15360"),
    (adapters(linear2_b=torch.zeros(1, 3072, 16, dtype=BF16)), BF16, "linear2 must be .adapters, rank, 15360"),
    (adapters(linear2_a=torch.zeros(2, 12, 15360, dtype=BF16), linear2_b=torch.zeros(2, 3072, 12, dtype=BF16)), BF16,
     "rank of linear2"),
    (adapters(linear2_a=torch.zeros(2, 15360, 16, dtype=BF16).transpose(1, 2)), BF16, "linear2 need 16-byte aligned rows"),
    (adapters(linear2_b=torch.zeros(2, 3072, 20, dtype=BF16)[..., :16]), BF16, "linear2 need 16-byte aligned rows"),
    (adapters(linear1_a=torch.zeros(8 * 3072 * 2 + 4, dtype=BF16)[4:].view(2, 8, 3072)), BF16, "linear1 need 16-byte aligned rows"),
])
def test_adapters_that_the_block_cannot_take(given, x_type, word):
    batch = packed.pack([(3, 1, 1)], "cpu")
    with pytest.raises(b2g.B2GError, match=f"single_block: .*{word}"):
        packed.single_block(None, torch.zeros(4, 3072, dtype=x_type), torch.zeros(4, 3072), torch.zeros(3072), batch, None, given)
