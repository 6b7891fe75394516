"""Low-rank adapters on both sides of the sizes at which the kernels for few and for many rows change over, and many calls side
by side.  Definition and tolerances: test_lora_gpu.py.
"""
from __future__ import annotations

import pytest
import torch

from test_lora_gpu import BF16, DEV, F16, F32, check, inputs, ints, offsets

pytestmark = pytest.mark.gpu


def spread(rows, batch):
    """Uneven requests: batch of them, rows in all, one empty where there is room for it."""
    lens = [rows // batch + (1 if i < rows % batch else 0) for i in range(batch)]
    if batch > 2 and lens[0] > 1:
        lens[1] += lens[0] - 1
        lens[2] += 1
        lens[0] = 0
    return lens


# up: 768 rows, or 32 a request (64 beyond rank 64); down: 32 a request (16 beyond rank 32), or (rows / 16 + requests) rank 2600
@pytest.mark.parametrize("rows,batch,R", [(768, 1, 16), (2591, 1, 16), (1280, 40, 16), (1280, 40, 64), (2560, 40, 128), (640, 40, 128),
                                          (640, 40, 40), (303, 1, 128)])
@pytest.mark.parametrize("more", [0, 1])
@pytest.mark.parametrize("dtype,y_dtype,epilogue", [(BF16, BF16, "gelu"), (F16, F32, "gated_residual"), (BF16, F32, "none")])
def test_both_sides_of_the_forms(engine, rows, batch, R, more, dtype, y_dtype, epilogue):
    lens = spread(rows + more, batch)
    check(engine, lens, 320, 328, R, adapters=5, dtype=dtype, y_dtype=y_dtype, epilogue=epilogue, seed=rows + R)


@pytest.mark.parametrize("lens", [[1] * 6, [40, 9, 60], [700, 5, 260]])
def test_lora_on_several_streams_at_once(engine, lens):
    """Calls side by side on four streams, and captured graphs replayed side by side, give what each gives alone."""
    cu, ids = offsets(lens), ints([i % 3 for i in range(len(lens))])
    sets = [inputs(lens, 512, 640, 32, 3, BF16, BF16, 10 + i) for i in range(4)]

    def run(i):
        x, a, b, y = sets[i]
        t = engine.lora_down(x, a, cu, ids=ids)
        part = engine.lora_up(t, b[:, :256], y[:, :256], cu, ids=ids)
        return engine.lora(x, a, b, y, cu, ids=ids, epilogue="silu"), part

    want = [run(i) for i in range(4)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]

    def same(got):
        torch.cuda.synchronize()
        return all(torch.equal(g, w) for gs, ws in zip(got, want) for g, w in zip(gs, ws))

    for _ in range(20):
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(run(i))
        assert same(got)
    graphs, outs = [], []
    for i in range(4):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run(i))
        graphs.append(graph)
    for _ in range(20):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        assert same(outs)
    engine.check_device_error()


@pytest.mark.parametrize("lens,n", [([1, 3], 264), ([900, 40], 9216)])
def test_lora_in_place_on_column_ranges_with_one_down(engine, lens, n):
    """A fused projection as a block runs it: one t, both parts of the columns updated in place in buffers that are wider."""
    rows, k, R, wide = sum(lens), 256, 24, n + 512
    x, a, b, y = inputs(lens, k, 2 * n, R, 2, BF16, BF16, 4)
    cu, ids = offsets(lens), ints([1, 0])
    want = engine.lora(x, a, b, y, cu, ids=ids)
    left, right = torch.full((rows, n), 5.0, dtype=BF16, device=DEV), torch.full((rows, wide), 5.0, dtype=BF16, device=DEV)
    left.copy_(y[:, :n])
    part = right[:, 512:]
    part.copy_(y[:, n:])
    t = engine.lora_down(x, a, cu, ids=ids)
    engine.lora_up(t, b[:, :n], left, cu, ids=ids, out=left)
    engine.lora_up(t, b[:, n:], part, cu, ids=ids, out=part)
    torch.cuda.synchronize()
    assert torch.equal(torch.cat([left, part], 1), want) and bool((right[:, :512] == 5).all())
