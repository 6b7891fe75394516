"""quantize_s8 at the ends of its sizes: rows without a value, the longest row."""
from __future__ import annotations

import pytest
import torch
from test_packed_ops_gpu import DEV

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows", [1, 7, 300])
def test_rows_without_values(engine, dtype, rows):
    """No value is other than zero: scale 1."""
    given = torch.full((rows,), 7.0, device=DEV)
    codes, scales = engine.quantize_s8(torch.empty((rows, 0), dtype=dtype, device=DEV), scales=given)
    torch.cuda.synchronize()
    assert codes.shape == (rows, 0) and scales is given and bool((scales == 1).all())
    assert bool((engine.quantize_s8(torch.empty((rows, 0), dtype=dtype, device=DEV))[1] == 1).all())
