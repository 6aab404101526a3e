"""Steps of drafted tokens on the GPU: every node's logits are the plain model's behind its path, from a graph and kernel by kernel; what
a step keeps is read by the next; generation with drafts."""
import random

import pytest
import torch

import helpers as H
import plain_qwen2
from conftest import TINY
from easy_gpt.cpp_amd.engine import DraftEntry, Engine, StepEntry
from easy_gpt.cpp_amd.generate import LLM

pytestmark = pytest.mark.gpu


def random_tree(rng, root, n, vocab):
    parents = [-1] + [rng.randrange(max(0, i - 5), i) for i in range(1, n)]
    return [root] + [rng.randrange(vocab) for _ in range(n - 1)], parents


def path_of(parents, node):
    path = []
    while node >= 0:
        path.append(node)
        node = parents[node]
    return path[::-1]


@pytest.mark.parametrize("graphs", [True, False], ids=["graphs", "eager"])
@pytest.mark.parametrize("name,dtype", [("A", "float32"), ("C", "float32"), ("C", "bfloat16"), ("D", "bfloat16"), ("D", "float32"), ("E", "bfloat16")])
def test_every_node_s_logits_and_what_is_kept(tiny_models, name, dtype, graphs):
    cfg_json = TINY[name][0]
    vocab = cfg_json["vocab_size"]
    cfg, w = plain_qwen2.read_model(tiny_models[name], round_to_bf16=dtype == "bfloat16")
    tol = H.FP32_TOL if dtype == "float32" else H.BF16_TOL_RANDOM
    rng = random.Random(7)
    reqs = {f"r{i}": [rng.randrange(vocab) for _ in range(n)] for i, n in enumerate((5, 33, 50))}
    eng = Engine.from_dir(tiny_models[name], dtype=dtype, page_size=16, max_tokens=1024, max_requests=4, use_graphs=graphs)
    known = {}
    for rid, p in reqs.items():
        eng.add_request(rid)
        eng.step([StepEntry(rid, p[:-1], [])])
        known[rid] = list(p)
    for round_ in range(5):                                  # (a shape's graph is captured behind its first visit and replayed from then on)
        sizes = [4, 16, 9] if round_ < 3 else [1, 20, 3]
        entries = [DraftEntry(rid, *random_tree(rng, known[rid][-1], n, vocab)) for rid, n in zip(known, sizes)]
        want = []
        for e in entries:
            for i in range(len(e.tokens)):
                path = path_of(e.parents, i)
                want.append(plain_qwen2.forward_logits(cfg, w, known[e.request_id][:-1] + [e.tokens[j] for j in path])[-1])
        # behind every node the token of one of its children, where it has any: a path from the root to a leaf is taken
        chosen, at = [], 0
        for e in entries:
            for i in range(len(e.tokens)):
                kids = [j for j in range(len(e.tokens)) if e.parents[j] == i]
                chosen.append(e.tokens[rng.choice(kids)] if kids else rng.randrange(vocab))
        seen = {}

        def choose(logits):
            seen["logits"] = logits.double().cpu()
            return torch.tensor(chosen, dtype=torch.int32, device="cuda")

        new = eng.step_drafts(entries, choose)
        eng.cache.check()
        for row, ref in zip(seen["logits"], want):
            assert float((row - ref).abs().max()) <= tol * float(ref.abs().max()), (round_, float((row - ref).abs().max() / ref.abs().max()))
        for e, got in zip(entries, new):
            path, here, base = [], 0, at
            while True:
                path.append(here)
                nxt = [j for j in range(here + 1, len(e.tokens)) if e.parents[j] == here and e.tokens[j] == chosen[base + here]]
                if not nxt:
                    break
                here = nxt[0]
            assert got == [chosen[base + j] for j in path]
            at += len(e.tokens)
            known[e.request_id] += got
            assert eng.cache.requests[e.request_id].num_tokens == len(known[e.request_id]) - 1
    logits = eng.step([StepEntry(rid, [known[rid][-1]], [0]) for rid in known]).double().cpu()
    for row, rid in zip(logits, known):
        ref = plain_qwen2.forward_logits(cfg, w, known[rid])[-1]
        assert float((row - ref).abs().max()) <= tol * float(ref.abs().max()), rid


@pytest.mark.parametrize("name,dtype", [("A", "float32"), ("C", "float32"), ("D", "bfloat16"), ("E", "bfloat16")])
def test_generation_with_drafts(tiny_models, name, dtype):
    vocab = TINY[name][0]["vocab_size"]
    cfg, w = plain_qwen2.read_model(tiny_models[name], round_to_bf16=dtype == "bfloat16")
    tol = 2e-5 if dtype == "float32" else 1e-2
    rng = random.Random(2)
    prompts = [[rng.randrange(vocab) for _ in range(n)] * 3 for n in (4, 9, 2)]
    llm = LLM(tiny_models[name], dtype=dtype, cache_tokens=2048, draft_nodes=12)
    outs = llm.generate(prompts, max_new_tokens=40, greedy=True, ignore_eos=True)
    stats = llm.last_stats
    assert stats.drafted > 0 and stats.generated == 120
    for p, out in zip(prompts, outs):
        logits = plain_qwen2.forward_logits(cfg, w, p + out)
        for i, tok in enumerate(out):
            row = logits[len(p) + i - 1]
            assert float(row.max() - row[tok]) <= tol * float(row.abs().max()), (i, tok)
    # sampled: the numbers that draw a token are the same, so in 32 bits the tokens are
    if dtype == "float32":
        sampled = [LLM(tiny_models[name], dtype=dtype, cache_tokens=2048, draft_nodes=n).generate(prompts, max_new_tokens=24, temperature=0.7, top_k=0, top_p=1.0,
                                                                                                  min_p=0.05, ignore_eos=True) for n in (0, 12)]
        assert sampled[0] == sampled[1]


def test_drafts_of_more_tokens_than_a_graph_takes(tiny_models):
    eng = Engine.from_dir(tiny_models["D"], dtype="bfloat16", page_size=16, max_tokens=4096, max_requests=8)
    rng = random.Random(3)
    known = {}
    for i in range(6):
        eng.add_request(i)
        known[i] = [rng.randrange(650) for _ in range(10 + 7 * i)]
        eng.step([StepEntry(i, known[i][:-1], [])])
    rows = {}
    entries = [DraftEntry(i, *random_tree(rng, known[i][-1], 64, 650)) for i in known]

    def choose(kind):
        def f(logits):
            rows[kind] = logits.clone()
            return torch.full((logits.shape[0],), 649, dtype=torch.int32, device="cuda")
        return f

    for e in entries:
        e.tokens[1:] = [t % 649 for t in e.tokens[1:]]       # (nothing but the roots is taken)
    new = eng.step_drafts(entries, choose("all"))
    assert new == [[649]] * 6 and not eng._draft_plans
    # the same trees one request at a time, from a graph: the rows agree
    other = Engine.from_dir(tiny_models["D"], dtype="bfloat16", page_size=16, max_tokens=4096, max_requests=8)
    for i, e in enumerate(entries):
        other.add_request(i)
        other.step([StepEntry(i, known[i][:-1], [])])
        assert other.step_drafts([e], choose("one")) == [[649]]
        part = rows["all"][64 * i : 64 * i + 64].double()
        assert float((rows["one"].double() - part).abs().max()) <= 2 * H.BF16_TOL_RANDOM * float(part.abs().max())
    assert other._draft_plans
