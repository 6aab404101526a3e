"""Drafted tokens through the engine and the scheduler on the CPU, with the tests' slow stand-in for the kernels: the tokens are those
of decoding one by one, and the books of the cache close."""
import random

import pytest
import torch

import helpers as H
import plain_drafts as plain
from conftest import TINY
from emulated_kernels import EmulatedKernels
from easy_gpt.cpp_amd import kernels
from easy_gpt.cpp_amd.cache import OutOfPages
from easy_gpt.cpp_amd.engine import DraftEntry, Engine, PromptLookup, StepEntry
from easy_gpt.cpp_amd.engine.scheduler import Request, Scheduler, SchedulerConfig
from easy_gpt.cpp_amd.generate import LLM
from easy_gpt.cpp_amd.sampling import Sampler, SamplingParams


class DraftKernels(EmulatedKernels):
    def tree_attention(self, qkv, out, k_cache, v_cache, block_table, q_start, q_len, kv_len, visible, nq, nkv, hd, page_size, scale, max_q_len, max_kv_len,
                       window=0, positions=None):
        assert int(q_len.max()) <= max_q_len <= 64 and int(kv_len.max()) <= max_kv_len
        got, _ = plain.tree_attention(qkv, k_cache, v_cache, block_table, q_start, q_len, kv_len, visible, nq, nkv, hd, page_size, scale, window, positions)
        there = ~got.isnan().any(1)
        out[there] = got[there].to(out.dtype)

    def accept_drafts(self, tokens, parents, sampled, q_start, q_len):
        return tuple(torch.tensor(v, dtype=torch.int32) for v in plain.accept_drafts(tokens, parents, sampled, q_start, q_len))

    def keep_drafts(self, k_cache, v_cache, block_table, start, path, count):
        k, v = plain.keep_drafts(k_cache, v_cache, block_table, start, path, count)
        k_cache.copy_(k), v_cache.copy_(v)

    def sample(self, logits, temperature, top_k, top_p, uniform, out, min_p=None):
        for r in range(logits.shape[0]):
            out[r] = plain.sample_row(logits[r].tolist(), float(temperature[r]), int(top_k[r]), float(top_p[r]), float(uniform[r]),
                                      0.0 if min_p is None else float(min_p[r]))


@pytest.fixture(autouse=True)
def emulated_backend():
    kernels.use_backend(DraftKernels())
    yield
    kernels.use_backend(None)


def engine_of(folder, **kw):
    kw = {"page_size": 4, "max_tokens": 256, "max_requests": 4, **kw}
    return Engine.from_dir(folder, dtype="float32", device="cpu", **kw)


def argmax_of(logits):
    return logits.argmax(1).int()


def greedy_by_steps(eng, rid, prompt, n):
    """n tokens one by one, the last one not in the cache."""
    eng.add_request(rid)
    out = [int(eng.step([StepEntry(rid, prompt, [len(prompt) - 1])]).argmax())]
    while len(out) < n:
        out.append(int(eng.step([StepEntry(rid, [out[-1]], [0])]).argmax()))
    return out


# --------------------------------------------------------------------------------------------------------------- drafter
def test_lookup_proposes_what_followed():
    d = PromptLookup(longest=3, branches=2)
    d.extend([1, 2, 3, 4, 5, 1, 2, 3])
    assert d.propose(8, 4) == ([3, 4, 5, 1, 2], [-1, 0, 1, 2, 3])
    assert d.propose(3, 4) == ([3, 4, 5], [-1, 0, 1])
    assert d.propose(8, 1) == ([3, 4], [-1, 0])
    assert d.propose(8, 0) == ([3], [-1]) and d.propose(1, 5) == ([3], [-1])
    d.extend([9, 1, 2, 3])
    tokens, parents = d.propose(8, 2)                        # the latest place first, then the one before it
    assert tokens == [3, 9, 1, 4, 5] and parents == [-1, 0, 1, 0, 3]


def test_lookup_shares_what_two_places_have_in_common_and_falls_back_to_shorter_runs():
    d = PromptLookup(longest=2, branches=3)
    d.extend([7, 1, 2, 8, 1, 2, 9, 1, 2, 8])
    tokens, parents = d.propose(16, 3)
    assert tokens[0] == 8 and tokens[1:4] == [1, 2, 9] and parents[:4] == [-1, 0, 1, 2]
    d = PromptLookup(longest=3)
    d.extend([5, 6, 7, 6])
    assert d.propose(9, 2) == ([6, 7, 6], [-1, 0, 1])
    d = PromptLookup()
    d.extend([5])
    assert d.propose(9, 2) == ([5], [-1])
    d.extend([5, 5, 5])
    tokens, parents = d.propose(9, 4)
    assert all(t == 5 for t in tokens) and parents == list(range(-1, len(tokens) - 1))


def test_lookup_trees_are_trees():
    rng = random.Random(1)
    for _ in range(200):
        d = PromptLookup(longest=rng.randint(1, 4), branches=rng.randint(1, 5))
        d.extend([rng.randrange(4) for _ in range(rng.randint(1, 80))])
        n, deep = rng.randint(1, 64), rng.randint(0, 12)
        tokens, parents = d.propose(n, deep)
        depth, _ = kernels.draft_masks(parents)
        assert 1 <= len(tokens) <= n and max(depth) <= deep and tokens[0] == d.tokens[-1]
        pairs = [(p, t) for p, t in zip(parents[1:], tokens[1:])]
        assert len(set(pairs)) == len(pairs)                 # no child of a node twice


# ---------------------------------------------------------------------------------------------------------------- engine
@pytest.mark.parametrize("name", ["A", "B", "C"])
def test_drafts_that_agree_are_taken_whatever_stands_beside_them(tiny_models, name):
    vocab = TINY[name][0]["vocab_size"]
    prompts = H.make_requests(vocab, [7, 30, 19], seed=5)
    eng = engine_of(tiny_models[name])
    truth = {rid: greedy_by_steps(eng, rid, p, 12) for rid, p in prompts.items()}
    for rid in prompts:
        eng.finish(rid)
    rng = random.Random(6)
    outs = {}
    for rid, p in prompts.items():
        eng.add_request(rid)
        outs[rid] = [int(eng.step([StepEntry(rid, p, [len(p) - 1])]).argmax())]
    while min(len(o) for o in outs.values()) < 12:
        entries, expect = [], []
        for rid, o in outs.items():
            # the true continuation for a while, with wrong tokens beside it, in an order of its own
            left = truth[rid][len(o) :]
            good = rng.randint(0, max(0, len(left) - 1)) if left else 0
            tokens, parents, node = [o[-1]], [-1], 0
            for t in left[:good]:
                for _ in range(rng.randint(0, 2)):
                    tokens.append((t + rng.randint(1, 5)) % vocab)
                    parents.append(node)
                tokens.append(t)
                parents.append(node)
                node = len(tokens) - 1
            entries.append(DraftEntry(rid, tokens, parents))
            expect.append(good + 1)
        new = eng.step_drafts(entries, argmax_of)
        eng.cache.check()
        for e, got, n in zip(entries, new, expect):
            if len(outs[e.request_id]) < 12:
                assert len(got) >= n
            outs[e.request_id] += got
            rc = eng.cache.requests[e.request_id]
            assert rc.num_tokens == len(prompts[e.request_id]) + len(outs[e.request_id]) - 1
            assert all(t == -(-rc.num_tokens // 4) for t in rc.table_lens)
    for rid, o in outs.items():
        assert o[:12] == truth[rid], rid
    # and what was kept in the cache is what decoding one by one would have left there: the next step's logits are the plain model's
    ref = H.plain_rows(tiny_models[name], {rid: prompts[rid] + outs[rid][:-1] + [3] for rid in prompts})
    logits = eng.step([StepEntry(rid, [3], [0]) for rid in prompts])
    for row, rid in zip(logits, prompts):
        want = ref[rid][-1]
        # (float32 against 64 bits, as other steps here are compared)
        assert float((row.double() - want).abs().max()) <= 1e-6 * float(want.abs().max())
    for rid in prompts:
        eng.finish(rid)
    assert eng.cache.free_pages() == [p.num_pages for p in eng.cache.pools]


def test_step_drafts_refuses_what_it_cannot_check(tiny_models):
    eng = engine_of(tiny_models["A"], num_pages=6, max_tokens=None)
    eng.add_request("a")
    eng.step([StepEntry("a", [1, 2, 3], [])])
    before = eng.cache.free_pages()
    for error, entry in ((ValueError, DraftEntry("a", [], [])), (ValueError, DraftEntry("a", [1, 2], [-1])), (ValueError, DraftEntry("a", [1, 2], [-1, 1])),
                         (KeyError, DraftEntry("z", [1], [-1])), (IndexError, DraftEntry("a", [512], [-1])),
                         (OutOfPages, DraftEntry("a", [1] * 30, [-1] + [0] * 29))):
        with pytest.raises(error):
            eng.step_drafts([entry], argmax_of)
        assert eng.cache.free_pages() == before and eng.cache.requests["a"].num_tokens == 3
        eng.cache.check()
    with pytest.raises(ValueError, match="twice"):
        eng.step_drafts([DraftEntry("a", [1], [-1]), DraftEntry("a", [1], [-1])], argmax_of)
    with pytest.raises(ValueError, match="choose"):
        eng.step_drafts([DraftEntry("a", [1, 2], [-1, 0])], lambda logits: logits.argmax(1))
    assert eng.cache.free_pages() == before and eng.cache.requests["a"].num_tokens == 3

    def fails(logits):
        raise RuntimeError("no")

    with pytest.raises(RuntimeError, match="no"):
        eng.step_drafts([DraftEntry("a", [1, 2], [-1, 0])], fails)
    assert eng.cache.free_pages() == before
    eng.cache.check()
    assert eng.step_drafts([], argmax_of) == []
    # places in the cache beyond max_position_embeddings are fine, positions are not
    eng = engine_of(tiny_models["A"], max_tokens=512)
    eng.add_request("a")
    eng.step([StepEntry("a", [1] * 126, [])])
    with pytest.raises(ValueError, match="max_position"):
        eng.step_drafts([DraftEntry("a", [1, 2, 3], [-1, 0, 1])], argmax_of)
    assert len(eng.step_drafts([DraftEntry("a", [1, 2, 3, 4, 5], [-1, 0, 0, 0, 0])], argmax_of)[0]) >= 1


def test_models_with_other_mixers_refuse_drafts():
    import os
    import tempfile

    import nebanex_models

    cfg, seed, rows, rank = nebanex_models.CONFIGS["A"]
    with tempfile.TemporaryDirectory() as d:
        nebanex_models.write_model(os.path.join(d, "m"), cfg, seed, rows, rank)
        eng = engine_of(os.path.join(d, "m"))
    assert not eng.supports_drafts
    eng.add_request("a")
    with pytest.raises(RuntimeError, match="drafted"):
        eng.step_drafts([DraftEntry("a", [1], [-1])], argmax_of)


# ------------------------------------------------------------------------------------------------------------- scheduler
def repeating_prompts(vocab, seed):
    rng = random.Random(seed)
    out = []
    for n in (6, 11, 3, 8, 5):
        part = [rng.randrange(vocab) for _ in range(n)]
        out.append(part * 3 + part[: rng.randint(1, n)])
    return out


@pytest.mark.parametrize("name,sampling", [("A", dict(greedy=True)), ("C", dict(greedy=True)), ("A", dict(temperature=0.02, top_k=0, top_p=1.0, min_p=0.05)),
                                           ("B", dict(temperature=0.9, top_k=20, top_p=0.95, min_p=0.01))], ids=str)
def test_scheduled_tokens_are_those_without_drafts(tiny_models, name, sampling):
    prompts = repeating_prompts(TINY[name][0]["vocab_size"], 3)
    results = []
    for nodes in (0, 6, 16):
        eng = engine_of(tiny_models[name], max_tokens=400)
        sched = Scheduler(eng, SchedulerConfig(max_active=4, draft_nodes=nodes), eos_token_id=-1)
        reqs = [sched.add(Request(i, p, SamplingParams(seed=9, **sampling), 14 + i)) for i, p in enumerate(prompts)]
        sched.run()
        assert all(r.status == "finished" and r.finish_reason == "length" for r in reqs)
        assert eng.cache.free_pages() == [p.num_pages for p in eng.cache.pools]
        eng.cache.check()
        results.append([r.output for r in reqs])
        if nodes:
            assert sched.stats.drafted > 0 and sched.stats.generated == sum(14 + i for i in range(5))
            assert sched.stats.decode_tokens + sched.stats.prompt_tokens >= sched.stats.generated
    assert results[0] == results[1] == results[2]


def test_drafts_save_steps_where_text_repeats(tiny_models):
    # greedy decoding of a tiny model runs into a cycle, which the lookup foresees
    steps = {}
    for nodes in (0, 8):
        eng = engine_of(tiny_models["A"], max_tokens=400)
        sched = Scheduler(eng, SchedulerConfig(draft_nodes=nodes), eos_token_id=-1)
        r = sched.add(Request(0, [5, 6, 7], SamplingParams(greedy=True), 80))
        sched.run()
        steps[nodes] = (sched.stats.steps, r.output, sched.stats.accepted)
    assert steps[0][1] == steps[8][1]
    if len(set(steps[0][1][-30:])) < 20:
        assert steps[8][2] > 0 and steps[8][0] < steps[0][0]


def test_ends_of_requests_inside_a_path(tiny_models):
    # an end token in the middle of an accepted path ends the request there; few pages cut the trees and preempt as without drafts
    prompts = repeating_prompts(512, 7)
    base = None
    for nodes in (0, 12):
        eng = engine_of(tiny_models["A"], num_pages=26, max_tokens=None)
        sched = Scheduler(eng, SchedulerConfig(max_active=4, draft_nodes=nodes), eos_token_id=-1)
        reqs = [sched.add(Request(i, p, SamplingParams(greedy=True), 20)) for i, p in enumerate(prompts)]
        sched.run()
        outs = [r.output for r in reqs]
        base = base or outs
        assert outs == base
        assert eng.cache.free_pages() == [26]
    eos = base[0][9]
    ends = []
    for nodes in (0, 12):
        eng = engine_of(tiny_models["A"], max_tokens=400)
        sched = Scheduler(eng, SchedulerConfig(max_active=4, draft_nodes=nodes), eos_token_id=eos)
        reqs = [sched.add(Request(i, p, SamplingParams(greedy=True), 20)) for i, p in enumerate(prompts)]
        sched.run()
        ends.append([(r.output, r.finish_reason) for r in reqs])
    assert ends[0] == ends[1] and ends[0][0][1] == "eos"


def test_requests_reach_the_last_position(tiny_models):
    outs = []
    for nodes in (0, 16):
        eng = engine_of(tiny_models["A"], max_tokens=400)
        sched = Scheduler(eng, SchedulerConfig(draft_nodes=nodes), eos_token_id=-1)
        r = sched.add(Request(0, [3, 4, 5] * 30, SamplingParams(greedy=True), 200))
        sched.run()
        outs.append((r.output, r.finish_reason))
    assert outs[0] == outs[1] and outs[0][1] == "max_position"


def test_options(tiny_models):
    from easy_gpt.cpp_amd.cli import CliError, parse_args

    for bad in (dict(draft_nodes=65), dict(draft_nodes=-1)):
        with pytest.raises(ValueError):
            SchedulerConfig(**bad)
    for bad in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError):
            SamplingParams(min_p=bad)
    o = parse_args(["--min-p", "0.1", "--draft-nodes", "16", "1 2"])
    assert o.min_p == 0.1 and o.draft_nodes == 16
    for bad in (["--min-p", "2"], ["--min-p", "x"], ["--draft-nodes", "65"], ["--draft-nodes"]):
        with pytest.raises(CliError):
            parse_args([*bad, "1"][: len(bad) + (len(bad) > 1)])
    outs = []
    for nodes in (0, 8):
        llm = LLM(tiny_models["A"], dtype="float32", device="cpu", cache_tokens=512, draft_nodes=nodes)
        outs.append(llm.generate([[1, 2, 3] * 4, [9, 8]], max_new_tokens=10, temperature=0.5, min_p=0.1, ignore_eos=True))
    assert outs[0] == outs[1]
