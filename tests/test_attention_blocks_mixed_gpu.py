"""A prompt among single tokens and among empty places of a batch: one form takes the whole call, by the average number of
queries.  Definition and tolerances: test_attention_blocks_gpu.py.
"""
from __future__ import annotations

import pytest
import torch

from test_attention_blocks_gpu import check_attention, qkv, random_choice

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("singles,empty,prompt", [(95, 0, 512), (10, 53, 200), (0, 31, 250), (40, 0, 900)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("hq,hk,d,dtype", [(8, 2, 64, torch.bfloat16), (3, 3, 128, torch.float16), (24, 1, 64, torch.float16)])
@pytest.mark.parametrize("at", ["front", "middle"])
def test_a_prompt_among_others(engine, singles, empty, prompt, causal, hq, hk, d, dtype, at):
    lq = [1] * singles + [0] * empty
    lk = [37 * (i % 40) + 1 for i in range(singles)] + [0] * empty
    place = 0 if at == "front" else len(lq) // 2
    lq.insert(place, prompt)
    lk.insert(place, prompt + 130)
    t = singles + prompt
    check_attention(engine, *qkv(t, sum(lk), hq, hk, d, dtype, t), random_choice(lq, lk, hk, t, extra=1), lq, lk, causal)
