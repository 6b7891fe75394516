"""A prompt among single tokens and among empty places of a batch: one form takes the whole call, by the average number of
queries.  Definition and tolerances: test_attention_blocks_gpu.py.
"""
from __future__ import annotations

import pytest
import torch

from test_attention_blocks_gpu import check_attention, offsets, qkv, random_choice

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


def timed(run):
    """us a replay, the best of some."""
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    best = float("inf")
    for _ in range(5):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        graph.replay()
        b.record()
        torch.cuda.synchronize()
        best = min(best, 1e3 * a.elapsed_time(b))
    return best


def test_a_long_prompt_among_single_tokens_is_found_in_linear_time(engine):
    """Thousands of tiles of one sequence on the line: right, and no more than ten or so times what the prompt and the single
    tokens take apart (tiles looked for one by one, from the sequence's first for each: 95 times)."""
    singles, prompt, hq, d = 1000, 7000, 8, 128
    lq, lk = [1] * singles + [prompt], [256] * singles + [prompt]
    q, k, v = qkv(singles + prompt, sum(lk), hq, 1, d, torch.bfloat16, 3)
    bits = random_choice(lq, lk, 1, 4, share=0.35)
    check_attention(engine, q, k, v, bits, lq, lk, True)
    tiles = torch.full((len(bits), 1, 2), -1, dtype=torch.int32, device=q.device)

    def run(a, b):  # sequences a to b
        qs, ks = slice(sum(lq[:a]), sum(lq[:b])), slice(sum(lk[:a]), sum(lk[:b]))
        cu_q, cu_k = offsets(lq[a:b]), offsets(lk[a:b])
        args = q[qs], k[ks], v[ks], tiles[a:], cu_q, cu_k
        return timed(lambda: engine.attention_blocks(*args, causal=True))

    apart, together = run(0, singles) + run(singles, singles + 1), run(0, singles + 1)
    assert together <= 30 * apart, (together, apart)
