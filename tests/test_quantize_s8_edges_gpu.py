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


def test_the_longest_row(engine):
    """2^31 - 16 values, the most that a row may have: all of them, and nothing before or behind."""
    cols, room = 2 ** 31 - 16, 64
    x = torch.empty((1, cols), dtype=torch.bfloat16, device=DEV)
    x.normal_(generator=torch.Generator(device=DEV).manual_seed(1))
    x[0, cols - 5] = 9.0
    buf = torch.full((1, cols + 2 * room), 77, dtype=torch.int8, device=DEV)
    codes, scales = engine.quantize_s8(x, out=buf[:, room:room + cols])
    torch.cuda.synchronize()
    engine.check_device_error()
    assert float(scales[0]) == float(torch.tensor(9.0) / 127)
    for at in range(0, cols, 2 ** 26):
        part = slice(at, min(cols, at + 2 ** 26))
        assert torch.equal(codes[0, part].double(), torch.round(x[0, part].double() * 127 / 9.0)), at
    assert bool((buf[0, :room] == 77).all()) and bool((buf[0, room + cols:] == 77).all())
