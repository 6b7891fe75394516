"""qk_norm_rope's angles on the B200 up to the largest positions that its bound is given for: 2^24, theta from 1 on.

An angle is right to 2^-22 of a turn, 2 pi 2^-22 of the pair's length; the cosine and sine add an ulp or two (2^-22) and the
two products and their sum 3 roundings of at most sqrt(2) times the length: 2.0e-6 in all.  The 64-bit angle itself is off by
2^24 * 2^-52 at most.
"""
from __future__ import annotations

import pytest
import torch
from test_packed_ops_gpu import DEV, assert_within, randn, rotated

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("theta", [10000.0, 500000.0, 3.0, 1.0])
@pytest.mark.parametrize("d", [64, 66, 128, 256])
@pytest.mark.parametrize("tokens,heads", [(300, 6), (2000, 3)])
@pytest.mark.parametrize("interleaved", [True, False])
def test_far_positions(engine, theta, d, tokens, heads, interleaved):
    """Spread over 2^18 to 2^24 on both sides of 0, the ends among them."""
    size = torch.exp2(18 + 6 * torch.rand(tokens, generator=torch.Generator().manual_seed(d))).to(DEV)
    pos = torch.where(randn((tokens,), 3) < 0, -size, size)
    pos[0], pos[1], pos[2] = 2.0 ** 24, -2.0 ** 24, 2.0 ** 24 - 1
    q, k = randn((tokens, heads, d), 1), randn((tokens, 1, d), 2)
    got = engine.qk_norm_rope(q, k, pos[:, None].contiguous(), [d], theta=theta, interleaved=interleaved)
    torch.cuda.synchronize()
    for g, x in zip(got, (q, k)):
        want, length = rotated(x, None, pos[:, None], [d], theta, interleaved, 1e-6)
        assert_within(g, want, 2.0e-6 * length)
