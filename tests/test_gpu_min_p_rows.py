"""Sampling with min-p: rows that are masked, and rows beside others."""
import math

import pytest
import torch

from easy_gpt.cpp_amd import kernels

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, I32 = torch.float32, torch.int32


def operands(rows, temperature, top_k, top_p, min_p, seed=1):
    full = lambda v, dt=F32: torch.full((rows,), v, dtype=dt, device=DEV)
    u = torch.rand((rows,), generator=torch.Generator().manual_seed(seed)).to(DEV)
    return full(temperature), full(top_k, I32), full(top_p), u, full(0, I32), full(min_p)


def microseconds(f, calls=10):
    """Of a call, replayed from a graph of several: the least of five."""
    f()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(calls):
            f()
    graph.replay()
    best = math.inf
    for _ in range(5):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        graph.replay()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b) / calls * 1e3)
    return best


@pytest.mark.parametrize("cuts", [(0.8, 50, 0.95, 0.1), (1.0, 0, 1.0, 0.05), (0.7, 0, 0.9, 0.02), (0.0, 0, 1.0, 0.1)], ids=str)
@pytest.mark.parametrize("mask", [-math.inf, -1e9])
def test_masked_rows_take_no_longer(mask, cuts):
    # Five sixths of the vocabulary masked, whole pieces of the row among them: nothing there is listed, and the row is not walked for it.  (Walked rows
    # take two to ten times as long.)
    rows, vocab = 64, 151936
    x = torch.randn((rows, vocab), generator=torch.Generator().manual_seed(2)).to(DEV) * 2.5
    masked = x.clone()
    masked[:, vocab // 6 :] = mask
    k = kernels.backend()
    t, top_k, top_p, u, out, min_p = operands(rows, *cuts)
    run = lambda logits: lambda: k.sample(logits, t, top_k, top_p, u, out, min_p=min_p)
    whole, here = microseconds(run(x)), microseconds(run(masked))
    run(masked)()
    got = out.tolist()
    short = x[:, : vocab // 6].contiguous()
    run(short)()
    assert got == out.tolist()                               # (the tokens of the row without what is masked)
    print(f"cuts {cuts} mask {mask}: {here:.1f} us, unmasked {whole:.1f}")
    assert here < 1.4 * whole
