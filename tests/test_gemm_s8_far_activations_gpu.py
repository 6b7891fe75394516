"""GELU and SiLU of the 8-bit integer linear layer at both ends of F32's range, in each of its kernels: one launch,
the shared K axis, the tiles (output rows with and without the alignment of wide stores).

Bounds.  y is within lin = 10 * 2^-24 |y| of its 64-bit value (see test_packed_ops_gpu.py).  Below -100 both functions are closer
to 0 than 1e-39, whatever y's error, so that the outputs are 0 to 1e-30.  Above 100 they are y to 1e-30: lin and the division's
2^-22.  Between, 1.2 lin and 2^-16 of the result for the exponential's argument.
"""
from __future__ import annotations

import pytest
import torch
from test_packed_ops_gpu import F64, UNIT, act, quantized, randn, weight

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,k", [(4, 900), (20, 1100), (130, 1100)])
@pytest.mark.parametrize("n", [70, 72])
@pytest.mark.parametrize("epilogue", ["gelu", "silu"])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
def test_rows_of_any_size(engine, m, k, n, epilogue, out_dtype):
    wq, ws = weight(n, k, 4)
    x = randn((m, k), 3, 1.0, torch.bfloat16)
    x[0] *= 2.0 ** 120
    x[1] *= 2.0 ** 100
    x[2] *= 2.0 ** -110
    out = engine.gemm_s8(x, wq, ws, out_dtype=out_dtype, epilogue=epilogue)
    torch.cuda.synchronize()
    codes, unit = quantized(x)
    y = (codes @ wq.to(F64).T) * unit[:, None] * ws.to(F64)
    assert bool((y[:2] < -1e25).any()) and bool((y[:2] > 1e25).any())
    want = torch.where(y < -100, 0.0, torch.where(y > 100, y, act(y.clamp(-100, 100), epilogue)))
    lin = 10 * 2.0 ** -24 * y.abs()
    bound = torch.where(y < -100, 0.0, torch.where(y > 100, lin + 2.0 ** -22 * y, 1.2 * lin + 2.0 ** -16 * want.abs()))
    u = UNIT[out_dtype]
    over = (out.to(F64) - want).abs() - (bound * (1 + u) + u * want.abs() + 1e-30)
    at = int(over.argmax())
    assert float(over.max()) <= 0, (float(out.flatten()[at]), float(want.flatten()[at]), float(y.flatten()[at]))
