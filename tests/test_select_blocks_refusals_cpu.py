"""CPU checks of select_blocks: how many words a choice has, where nobody says how long a sequence may be."""
from __future__ import annotations

import pytest
import torch

import b2g


@pytest.mark.parametrize("rows", [8193, 20000])
@pytest.mark.parametrize("batch", [1, 2])
def test_many_keys_without_max_k(rows, batch):
    """More than 2^20 keys, or room for them, which no one sequence need have: the refusal names the argument that says so."""
    q, means = torch.zeros(2, 1, 64, dtype=torch.bfloat16), torch.zeros(rows, 1, 64)
    cu = torch.arange(batch + 1, dtype=torch.int32)
    with pytest.raises(b2g.B2GError, match="select_blocks: max_k"):
        b2g.select_blocks(q, means, cu, 4)
    for kw in (dict(max_k=4096), dict(out=torch.zeros(2, 1, 4, dtype=torch.int32))):  # (these get as far as the device)
        with pytest.raises(b2g.B2GError, match="CUDA tensors"):
            b2g.select_blocks(q, means, cu, 4, **kw)
    with pytest.raises(b2g.B2GError, match="CUDA tensors"):
        b2g.select_blocks(q, means[:8192], cu, 4)
