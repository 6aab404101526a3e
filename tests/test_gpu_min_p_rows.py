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


def border_uniforms(x, temperature, top_k, g):
    """For every row a uniform number that falls, to the last bit or next to it, on the running sum of the tokens that top-k leaves."""
    w = torch.exp((x - x.max(1, keepdim=True).values) / temperature)
    if top_k:
        w = torch.where(w >= torch.topk(w, top_k).values[:, -1:], w, torch.zeros_like(w))
    share = torch.cumsum(w.double(), 1)
    share /= share[:, -1:]
    return share.gather(1, torch.randint(0, x.shape[1] - 1, (x.shape[0], 1), generator=g).to(x.device))[:, 0].float()


@pytest.mark.parametrize("vocab,top_k", [(700, 0), (700, 20), (5000, 20), (5000, 0), (40000, 50), (40000, 0)])
def test_a_request_has_the_tokens_that_it_has_without_a_neighbour_with_min_p(monkeypatch, vocab, top_k):
    from easy_gpt.cpp_amd.sampling import Sampler, SamplingParams, sampler

    rows, g = 512, torch.Generator().manual_seed(vocab + top_k)
    x = (torch.randn((rows, vocab), generator=g) * 1.5).to(DEV)
    u = border_uniforms(x, 0.9, top_k, g).cpu().numpy()

    def uniforms(params, serials, counts, out):
        out[:] = u

    monkeypatch.setattr(sampler, "fill_uniforms", uniforms)
    plain = [SamplingParams(temperature=0.9, top_k=top_k, top_p=1.0 if r % 3 else 0.9) for r in range(rows)]
    with_one = [SamplingParams(temperature=0.9, top_k=top_k, top_p=p.top_p, min_p=0.05) if r in (3, 200) else p for r, p in enumerate(plain)]
    s, numbers = Sampler(DEV), list(range(rows))
    alone, beside = s.sample(x, plain, numbers, numbers), s.sample(x, with_one, numbers, numbers)
    assert [r for r in numbers if alone[r] != beside[r] and r not in (3, 200)] == []
    # and the two have the tokens that they have among their like
    among = s.sample(x, [SamplingParams(temperature=0.9, top_k=top_k, top_p=p.top_p, min_p=0.05) for p in plain], numbers, numbers)
    assert beside[3] == among[3] and beside[200] == among[200]


@pytest.mark.parametrize("top_k,top_p", [(0, 0.95), (0, 1.0), (50, 0.95)])
def test_a_neighbour_with_min_p_costs_its_own_time(monkeypatch, top_k, top_p):
    # 64 rows of 151,936, one of them with min-p: the kernels of the other 63 and those of one row (7 to 20 us) behind each other
    from easy_gpt.cpp_amd.sampling import Sampler, SamplingParams

    rows, vocab = 64, 151936
    x = (torch.randn((rows, vocab), generator=torch.Generator().manual_seed(3)) * 2.5).to(DEV)
    k, asked = kernels.backend(), []
    sample = type(k).sample
    monkeypatch.setattr(k, "sample", lambda *a, **kw: asked.append((a, kw)) or sample(k, *a, **kw), raising=False)
    one = SamplingParams(temperature=1.0, top_k=top_k, top_p=top_p)
    other = SamplingParams(temperature=1.0, top_k=top_k, top_p=top_p, min_p=0.05)
    s, numbers = Sampler(DEV), list(range(rows))
    s.sample(x, [one] * rows, numbers, numbers)
    s.sample(x, [one] * 20 + [other] + [one] * 43, numbers, numbers)
    alone, beside = (microseconds(lambda: sample(k, *a, **kw)) for a, kw in asked)
    print(f"top-k {top_k} top-p {top_p}: {alone:.1f} us, beside one with min-p {beside:.1f}")
    assert beside < 1.05 * alone + 20


def test_mixed_calls_are_refused_without_min_p():
    with pytest.raises(ValueError):
        kernels.backend().sample(torch.zeros((2, 9), device=DEV), *operands(2, 1.0, 0, 1.0, 0.1)[:5], mixed=True)


@pytest.mark.parametrize("vocab", [700, 5000, 32766, 40000, 151936])
def test_tokens_on_the_border_of_top_p_are_kept_by_the_exact_mass(monkeypatch, vocab):
    # Logits that fall along the row, a top_p that is the running share of one of them to the last bits, and a draw of the last token that is kept: which one that is follows
    # from sums in integers, as the kernels without min-p have it, however the row is cut.  (A min_p below all of those tokens.)
    rows, g = 192, torch.Generator().manual_seed(vocab)
    x = torch.sort(torch.randn((rows, vocab), generator=g) * 2.5, descending=True).values.to(DEV)
    w = torch.exp(x - x[:, :1]).double()
    share = torch.cumsum(w, 1) / w.sum(1, keepdim=True)
    last = (w >= 2e-3).sum(1)
    at = (torch.rand((rows,), generator=g).to(DEV) * (last - 1)).long()
    top_p = share.gather(1, at[:, None])[:, 0].float()
    k = kernels.backend()
    temperature, top_k, _, u, out, min_p = operands(rows, 1.0, 0, 1.0, 1e-3)
    u.fill_(0.99999994)
    k.sample(x, temperature, top_k, top_p, u, out)
    want = out.tolist()
    assert sum(abs(a - b) <= 1 for a, b in zip(want, at.tolist())) == rows
    for pieces in (None, 3, 8, 17) if vocab < 32769 else (None, 5, 8, 17, 40) if vocab > 100000 else (None, 3, 8, 17):
        with monkeypatch.context() as m:
            if pieces is not None and vocab > 1024:
                m.setattr(k, "_sample_pieces", lambda *a: pieces, raising=False)
            k.sample(x, temperature, top_k, top_p, u, out, min_p=min_p)
        got = out.tolist()
        assert [(r, a, b) for r, (a, b) in enumerate(zip(got, want)) if a != b] == [], pieces
