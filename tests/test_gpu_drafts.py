"""Attention for trees of drafted tokens, min-p sampling, the walk over accepted tokens and the move of their keys and values, against
64-bit arithmetic, and the refusals of their entry points."""
import math
import random

import pytest
import torch

import plain_drafts as plain
from easy_gpt.cpp_amd import kernels

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


def run_tree(c, out=None):
    if out is None:
        out = torch.full((c["qkv"].shape[0], c["nq"] * c["hd"]), math.nan, dtype=c["qkv"].dtype, device=DEV)
    lens, kvs = c["q_len"].tolist(), c["kv_len"].tolist()
    kernels.backend().tree_attention(c["qkv"], out, c["k_cache"], c["v_cache"], c["block_table"], c["q_start"], c["q_len"], c["kv_len"], c["visible"],
                                     c["nq"], c["nkv"], c["hd"], c["page_size"], c["scale"], max(lens), max(kvs), window=c["window"],
                                     positions=c["positions"])
    return out


def expected(c):
    names = ("qkv", "k_cache", "v_cache", "block_table", "q_start", "q_len", "kv_len", "visible", "nq", "nkv", "hd", "page_size", "scale",
             "window", "positions")
    return plain.tree_attention(*(c[n] for n in names))


def check_tree(c, got=None):
    want, spread = expected(c)
    got = (run_tree(c) if got is None else got).cpu().to(torch.float64)
    nobody = want.isnan()
    assert bool(got[nobody].isnan().all())
    err, tol = (got - want).abs()[~nobody], plain.tree_tolerance(c, spread, want)[~nobody]
    assert bool((err <= tol).all()), (float((err / tol).max()), float(err.max()))


# head layouts (nq, nkv, hd) and page sizes: those of the matrix-core kernel (features and keys that fill 16 bytes), and others
HEADS = [(14, 2, 64), (6, 1, 128), (4, 2, 16), (3, 1, 32), (8, 8, 48), (5, 5, 80), (2, 2, 96), (4, 1, 256), (16, 1, 64), (4, 2, 20), (2, 1, 33), (3, 3, 7)]


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_trees_of_any_heads(heads, dtype):
    rng = random.Random(sum(heads))
    c, _ = plain.tree_case(rng, [9, 1, 16, 2], [37, 0, 100, 15], *heads, 16, dtype, DEV)
    check_tree(c)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("page", [1, 5, 8, 16, 32, 48, 64, 256])
def test_trees_in_pages_of_any_size(page, dtype):
    c, _ = plain.tree_case(random.Random(page), [7, 30], [61, 200], 6, 2, 64, page, dtype, DEV)
    check_tree(c)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nodes", [1, 2, 4, 5, 9, 17, 33, 63, 64])
def test_trees_of_any_size(nodes, hd):
    # rows of a request: from less than a block of 32 to several workgroups of 256
    c, _ = plain.tree_case(random.Random(nodes), [nodes, max(1, nodes // 3)], [129, 16 * nodes], 14, 2, hd, 16, BF16, DEV)
    check_tree(c)


@pytest.mark.parametrize("before", [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 255, 256, 257, 511, 513, 1023, 2049])
def test_trees_behind_any_number_of_tokens(before):
    # the tree's first key at every place of a tile of keys, of a page and of a range of keys
    c, _ = plain.tree_case(random.Random(before), [13, 6], [before, max(0, before - 3)], 4, 2, 64, 16, BF16, DEV)
    check_tree(c)


@pytest.mark.parametrize("dtype,hd", [(BF16, 128), (F32, 64), (F32, 128), (BF16, 256)])
def test_trees_behind_long_contexts(dtype, hd):
    c, _ = plain.tree_case(random.Random(hd), [24, 3], [5000, 900], 4, 2, hd, 16, dtype, DEV)
    check_tree(c)


@pytest.mark.parametrize("dtype,hd,page", [(BF16, 64, 16), (F32, 64, 16), (BF16, 128, 32), (BF16, 20, 16)])
@pytest.mark.parametrize("window", [1, 2, 17, 64, 100, 1000])
def test_trees_with_a_window(window, dtype, hd, page):
    c, _ = plain.tree_case(random.Random(window), [20, 64, 1], [333, 150, 40], 4, 2, hd, page, dtype, DEV, window=window)
    check_tree(c)


@pytest.mark.parametrize("dtype,hd", [(BF16, 64), (BF16, 128), (F32, 64), (BF16, 20)])
def test_pages_behind_a_window_are_not_read(dtype, hd):
    c, _ = plain.tree_case(random.Random(5), [20, 7], [333, 150], 4, 2, hd, 16, dtype, DEV, window=50)
    c["block_table"][0, : (333 - 50) // 16] = -1
    c["block_table"][1, : (150 - 50) // 16] = -1
    check_tree(c)


@pytest.mark.parametrize("dtype,hd", [(BF16, 64), (BF16, 128), (F32, 64), (F32, 20)])
def test_rows_that_see_nothing_are_zeros(dtype, hd):
    c, _ = plain.tree_case(random.Random(6), [6, 40], [0, 0], 4, 2, hd, 16, dtype, DEV)
    c["visible"][:] = torch.tensor([0 if i % 3 == 0 else 1 << (i % 6) for i in range(46)], device=DEV)
    c["visible"][1] = -1 << 40                               # only nodes that the request does not have
    check_tree(c)
    got = run_tree(c)
    assert not bool(got[0].any()) and not bool(got[1].any())


@pytest.mark.parametrize("dtype,hd", [(BF16, 64), (BF16, 128), (F32, 64), (BF16, 20)])
def test_visibility_is_any_set_of_nodes(dtype, hd):
    c, _ = plain.tree_case(random.Random(7), [64, 64], [50, 7], 4, 2, hd, 16, dtype, DEV)
    rng = random.Random(8)
    c["visible"][:] = torch.tensor([rng.getrandbits(64) - (1 << 63) for _ in range(128)], dtype=torch.int64, device=DEV)
    check_tree(c)


@pytest.mark.parametrize("dtype,hd", [(BF16, 64), (BF16, 128), (F32, 64), (F32, 128), (BF16, 20)])
@pytest.mark.parametrize("number", [math.inf, -math.inf, math.nan])
def test_numbers_that_a_row_does_not_see_do_not_reach_it(number, dtype, hd):
    # node 3 of 12 holds no finite numbers: the rows that do not see it are as if it held others, the rest are what the formula gives
    c, _ = plain.tree_case(random.Random(9), [12, 5], [45, 20], 4, 2, hd, 16, dtype, DEV)
    place = 45 + 3
    page = int(c["block_table"][0, place // 16])
    c["v_cache"][page, :, : hd // 2, place % 16] = number
    c["k_cache"][page, 1, place % 16, 0] = number
    sees = [b >> 3 & 1 for b in c["visible"].tolist()[:12]] + [0] * 5
    assert 0 < sum(sees) < 12
    got = run_tree(c).cpu()
    clean = dict(c, v_cache=c["v_cache"].clone(), k_cache=c["k_cache"].clone())
    clean["v_cache"][page, :, :, place % 16] = 0.5
    clean["k_cache"][page, :, place % 16] = 0.5
    want, spread = expected(clean)
    tol = plain.tree_tolerance(clean, spread, want)
    for row, sees_it in enumerate(sees):
        if not sees_it:
            assert bool(((got[row].double() - want[row]).abs() <= tol[row]).all()), row
        else:
            mine, full = got[row].float(), expected(c)[0][row]
            # (a finite key: heads 0 and 1 see the number in the first half of the features)
            for h in range(4):
                part, ref = mine[h * hd : (h + 1) * hd], full[h * hd : (h + 1) * hd]
                assert bool((part.isfinite() == ref.isfinite()).all()), (row, h)


@pytest.mark.parametrize("dtype,hd", [(BF16, 64), (F32, 64), (BF16, 20)])
def test_infinities_before_the_tree_are_every_row_s(dtype, hd):
    c, _ = plain.tree_case(random.Random(10), [9], [70], 2, 1, hd, 16, dtype, DEV)
    page = int(c["block_table"][0, 1])
    c["v_cache"][page, 0, 3, 5] = math.inf
    got = run_tree(c).cpu().float().view(9, 2, hd)
    assert bool((got[:, :, 3] == math.inf).all())
    assert bool(got[:, :, :3].isfinite().all()) and bool(got[:, :, 4:].isfinite().all())


@pytest.mark.parametrize("dtype,hd", [(BF16, 64), (F32, 64), (BF16, 20)])
def test_large_and_negative_scales(dtype, hd):
    for scale in (0.0, -0.2, 3.0):
        c, _ = plain.tree_case(random.Random(11), [9, 4], [70, 3], 4, 2, hd, 16, dtype, DEV)
        c["scale"] = scale
        check_tree(c)


@pytest.mark.parametrize("dtype,hd", [(BF16, 64), (BF16, 128), (BF16, 256), (F32, 64), (BF16, 20)])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_so_large_that_one_key_has_all_the_weight(sign, dtype, hd):
    # Scores of up to 2^39 times the scale, all exact in 24 bits: products of powers of two and an integer up to 15.  Equal ones are equal, others lie 2^28 hd scale
    # and more below, where a weight is zero: the greatest ones' values in equal shares, whose rounding and sums alone count.
    c, _ = plain.tree_case(random.Random(hd), [9, 33], [500, 3000], 4, 2, hd, 16, dtype, DEV)
    g = torch.Generator().manual_seed(hd)
    steps = torch.randint(0, 16, c["k_cache"].shape[:3], generator=g).to(DEV)
    c["k_cache"][:] = (steps * 2.0 ** 14)[..., None].to(dtype)
    signs = torch.randint(0, 2, (42, 4, 1), generator=g).to(DEV) * 2 - 1
    c["qkv"][:, : 4 * hd] = (signs * 2.0 ** 14).expand(42, 4, hd).reshape(42, 4 * hd).to(dtype)
    c["scale"] *= sign
    want, spread = expected(c)
    share = 2.0 ** -20 + 2 * 3033 * 2.0 ** -24 + (2.0 ** -8 if dtype == BF16 else 0.0)
    tol = share * spread + torch.finfo(dtype).eps / 2 * want.abs() * (1 + share) + 1e-30
    err = (run_tree(c).cpu().double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("dtype,hd", [(BF16, 64), (F32, 64), (BF16, 20)])
def test_rows_of_no_request_stay_and_requests_may_be_empty(dtype, hd):
    c, _ = plain.tree_case(random.Random(12), [4, 0, 17, 0], [33, 20, 64, 0], 4, 2, hd, 16, dtype, DEV, parents=None, extra_rows=9)
    out = torch.full((30, 4 * hd), 7.0, dtype=dtype, device=DEV)
    run_tree(c, out)
    assert bool((out[21:] == 7.0).all())
    want, spread = expected(c)
    tol = plain.tree_tolerance(c, spread, want)
    assert bool(((out.cpu().double() - want).abs() <= tol)[:21].all())


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_many_ragged_requests(dtype):
    rng = random.Random(13)
    lens = [rng.randint(0, 24) for _ in range(70)]
    befores = [rng.randint(0, 300) for _ in range(70)]
    lens[5], befores[5] = 64, 1500
    c, _ = plain.tree_case(rng, lens, befores, 4, 2, 64, 16, dtype, DEV)
    check_tree(c)


@pytest.mark.parametrize("loose", [False, True], ids=["bounds", "loose_bounds"])
@pytest.mark.parametrize("heads", [(14, 2, 64), (6, 1, 128), (4, 1, 256)], ids=str)
def test_uneven_contexts_are_cut_by_what_they_are(heads, loose):
    # one long context beside short and empty ones, in more requests than a wavefront has lanes and in few: parts of every length; and bounds far
    # above what there is, as a captured step has them
    rng = random.Random(21)
    for b in (2, 5, 131):
        lens = [rng.choice([0, 1, 2, 5, 11]) for _ in range(b)]
        befores = [rng.choice([0, 1, 15, 64, 127, 300]) for _ in range(b)]
        lens[b // 2], befores[b // 2] = 13, 1777
        lens[-1], befores[-1] = 3, 640
        c, _ = plain.tree_case(rng, lens, befores, *heads, 16, BF16, DEV)
        if loose:
            c["block_table"] = torch.cat([c["block_table"], torch.full((b, 200), -1, dtype=torch.int32, device=DEV)], 1)
        out = torch.full((c["qkv"].shape[0], c["nq"] * c["hd"]), math.nan, dtype=BF16, device=DEV)
        kernels.backend().tree_attention(c["qkv"], out, c["k_cache"], c["v_cache"], c["block_table"], c["q_start"], c["q_len"], c["kv_len"], c["visible"],
                                         *heads, 16, c["scale"], 64 if loose else 13, c["block_table"].shape[1] * 16 if loose else int(c["kv_len"].max()))
        check_tree(c, out)


def test_a_chain_is_a_prompt_portion():
    # every node sees all before it: what paged_attention does with those tokens
    c, _ = plain.tree_case(random.Random(14), [40, 12], [130, 6], 6, 2, 64, 16, BF16, DEV, parents=[list(range(-1, 39)), list(range(-1, 11))])
    c["k_cache"].nan_to_num_(0.0), c["v_cache"].nan_to_num_(0.0)
    got = run_tree(c)
    other = torch.empty_like(got)
    kernels.backend().paged_attention(c["qkv"], other, c["k_cache"], c["v_cache"], c["block_table"], c["q_start"], c["q_len"], c["kv_len"], 6, 2, 64, 16,
                                      c["scale"], 0, 40, 170)
    want, spread = expected(c)
    tol = plain.tree_tolerance(c, spread, want)
    assert bool(((got.cpu().double() - want).abs() <= tol).all())
    assert bool(((other - got).cpu().double().abs() <= 2 * tol).all())


def test_trees_in_a_cache_that_passes_32_bits():
    # pages beyond 4 GiB of keys: 2 heads of 128 in bfloat16, 8 KiB a page of 16 tokens
    pages = (1 << 32) // (2 * 16 * 128 * 2) + 40
    small, _ = plain.tree_case(random.Random(15), [6], [100], 4, 2, 128, 16, BF16, DEV)
    k = torch.empty((pages, 2, 16, 128), dtype=BF16, device=DEV)
    v = torch.empty((pages, 2, 128, 16), dtype=BF16, device=DEV)
    n = small["k_cache"].shape[0]
    k[-n:], v[-n:] = small["k_cache"], small["v_cache"]
    big = dict(small, k_cache=k, v_cache=v, block_table=small["block_table"] + (pages - n))
    assert torch.equal(run_tree(big), run_tree(small))
    path = torch.full((1, 64), -1, dtype=torch.int32, device=DEV)
    path[0, :3] = torch.tensor([0, 2, 5], device=DEV)
    count, start = torch.tensor([3], dtype=torch.int32, device=DEV), torch.tensor([100], dtype=torch.int32, device=DEV)
    kernels.backend().keep_drafts(k, v, big["block_table"], start, path, count)
    want = plain.keep_drafts(small["k_cache"], small["v_cache"], small["block_table"], start, path, count)
    assert torch.equal(k[-n:].view(torch.int16), want[0].view(torch.int16)) and torch.equal(v[-n:].view(torch.int16), want[1].view(torch.int16))


def test_trees_replayed_from_a_graph_and_on_two_streams():
    c, _ = plain.tree_case(random.Random(16), [16, 3], [3000, 700], 4, 2, 64, 16, BF16, DEV)
    eager = run_tree(c)
    out = torch.empty_like(eager)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run_tree_static(c, out)
    second = torch.cuda.CUDAGraph()
    out2 = torch.empty_like(eager)
    with torch.cuda.graph(second):
        run_tree_static(c, out2)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for i in range(4):
        out.zero_(), out2.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(a):
            graph.replay()
        with torch.cuda.stream(b):
            second.replay()
        again = run_tree(c)
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(out2, eager) and torch.equal(again, eager)
        c["qkv"].mul_(1.25)
        torch.cuda.synchronize()
        eager = run_tree(c)
        torch.cuda.synchronize()


def run_tree_static(c, out):
    kernels.backend().tree_attention(c["qkv"], out, c["k_cache"], c["v_cache"], c["block_table"], c["q_start"], c["q_len"], c["kv_len"], c["visible"],
                                     c["nq"], c["nkv"], c["hd"], c["page_size"], c["scale"], 16, 3016)


def test_attention_refusals():
    k = kernels.backend()
    c, _ = plain.tree_case(random.Random(17), [4], [20], 4, 2, 64, 16, BF16, DEV)
    good = [c[n] for n in ("qkv",)] + [torch.empty((4, 256), dtype=BF16, device=DEV)] + [c[n] for n in (
        "k_cache", "v_cache", "block_table", "q_start", "q_len", "kv_len", "visible")] + [4, 2, 64, 16, 0.125, 4, 24]
    k.tree_attention(*good)
    def refused(error, at, value, **more):
        with pytest.raises(error):
            k.tree_attention(*good[:at], value, *good[at + 1 :], **more)
    refused(TypeError, 0, c["qkv"].half())
    refused(ValueError, 0, c["qkv"][:, :-1])
    refused(TypeError, 0, c["qkv"].cpu())
    refused(TypeError, 0, None)
    refused(ValueError, 0, c["qkv"][0])
    refused(TypeError, 1, None)
    refused(TypeError, 2, None)
    refused(ValueError, 2, c["k_cache"][:-1])
    refused(TypeError, 3, [])
    refused(TypeError, 4, None)
    refused(TypeError, 8, None)
    refused(TypeError, 1, good[1].float())
    refused(ValueError, 1, good[1][:3])
    refused(TypeError, 2, c["k_cache"].float())
    refused(ValueError, 3, c["v_cache"].transpose(2, 3))
    refused(TypeError, 4, c["block_table"].long())
    refused(ValueError, 4, c["block_table"][0])
    refused(ValueError, 5, c["q_start"].repeat(2))
    refused(TypeError, 8, c["visible"].int())
    refused(ValueError, 8, c["visible"][:-1])
    refused(ValueError, 9, 3)
    refused(ValueError, 11, 0)
    refused(ValueError, 11, 257)
    refused(ValueError, 14, 65)
    refused(ValueError, 15, 33)                              # the table holds 32
    refused(ValueError, 15, 24, window=8)                    # no positions
    refused(ValueError, 15, 24, window=-1)


# ------------------------------------------------------------------------------------------------------------- sampling
def sample(x, temperature, top_k, top_p, uniform, min_p):
    r = x.shape[0]
    row = lambda v, dt=F32: (v if torch.is_tensor(v) else torch.full((r,), v)).to(dt).to(DEV)
    out = torch.empty(r, dtype=torch.int32, device=DEV)
    kernels.backend().sample(x.to(DEV), row(temperature), row(top_k, torch.int32), row(top_p), row(uniform), out,
                             min_p=None if min_p is None else row(min_p))
    return out.tolist()


def far_from_borders(x, temperature, top_k, top_p, u, min_p, slack=3e-5):
    """Whether no cut and no draw of the row lies so near a border that float32 may take the other side: the weights are off by some 2^-18
    relatively at most (an argument below 2^7 rounded twice, an exponential; the greatest are exactly 1), running sums of them by as much again.  Tokens that may fall
    on either side of min_p move the sums by their mass."""
    w = torch.exp((x.double() - x.double().max()) / temperature)
    order = torch.sort(w, descending=True).values
    kept = torch.ones_like(w, dtype=torch.bool)
    if 0 < top_k < len(w):
        if abs(float(order[top_k - 1] / order[top_k]) - 1) < slack and float(order[top_k - 1]) != float(order[top_k]):
            return False
        kept = w >= order[top_k - 1]
    if top_p < 1:
        run = torch.cumsum(torch.sort(torch.where(kept, w, torch.zeros_like(w)), descending=True).values, 0)
        if bool(((run / run[-1] - top_p).abs() < slack).any()):
            return False
        line = order[int((run < top_p * run[-1]).sum())]
        kept = kept & (w >= line)
    either = torch.zeros_like(kept)
    if min_p > 0:
        either = kept & ((w / min_p - 1).abs() < slack) & (w < 1)
        kept = kept & (w >= min_p)
    run = torch.cumsum(torch.where(kept, w, torch.zeros_like(w)), 0)
    slack += 2 * float(w[either].sum() / run[-1])
    return not bool(((run / run[-1] - u).abs()[kept & (run < run[-1])] < slack).any())


@pytest.mark.parametrize("vocab", [1, 2, 5, 300, 1024, 1025, 5000, 8191, 8192, 20000, 151936])
@pytest.mark.parametrize("cuts", [(0, 1.0, 0.05), (0, 1.0, 0.5), (0, 1.0, 1e-6), (0, 0.9, 0.02), (0, 0.3, 0.02), (20, 0.95, 0.1), (200, 1.0, 0.01), (20, 1.0, 0.0),
                                  (0, 0.99, 1e-6), (5, 0.5, 1.0)], ids=str)
def test_min_p_against_64_bits(vocab, cuts):
    top_k, top_p, min_p = cuts
    g = torch.Generator().manual_seed(vocab + top_k)
    rows = 6
    checked = 0
    for temperature in (0.4, 1.3):
        x = torch.randn((rows, vocab), generator=g) * 2.5
        x[0] = x[0] * 0.01                                   # nearly flat: everything may be kept
        x[1, vocab // 2] += 12.0                             # one that stands out
        u = torch.randint(0, 1 << 24, (rows,), generator=g).float() / float(1 << 24)
        got = sample(x, temperature, top_k, top_p, u, min_p)
        t, p, m = (float(torch.tensor(v, dtype=F32)) for v in (temperature, top_p, min_p))
        for r in range(rows):
            if vocab > 20000 and r > 2:
                continue
            if far_from_borders(x[r], t, top_k, p, float(u[r]), m):
                assert got[r] == plain.sample_row(x[r].tolist(), t, top_k, p, float(u[r]), m), (r, temperature)
                checked += 1
    assert checked >= (3 if vocab < 20000 else 1)


@pytest.mark.parametrize("vocab", [700, 9000, 40000])
def test_min_p_keeps_what_it_says(vocab):
    # every uniform number falls on a kept token, the kept ones alone, and each of them is reached
    g = torch.Generator().manual_seed(3)
    x = torch.randn((1, vocab), generator=g) * 2.0
    w = torch.exp(x.double() - x.double().max())[0]
    kept = set(torch.nonzero(w >= 0.2).flatten().tolist())
    border = int(((w / 0.2 - 1).abs() < 1e-5).sum())
    assert border == 0 and len(kept) < 200
    n = 1024
    u = (torch.arange(n).float() + 0.5) / n
    got = set(sample(x.expand(n, vocab).contiguous(), 1.0, 0, 1.0, u, 0.2))
    assert got <= kept and len(got) >= len(kept) // 2


@pytest.mark.parametrize("vocab", [100, 9000])
def test_min_p_ends_of_its_range(vocab):
    g = torch.Generator().manual_seed(4)
    x = torch.randn((5, vocab), generator=g)
    u = torch.rand((5,), generator=g)
    best = x.argmax(1).tolist()
    assert sample(x, 0.9, 0, 1.0, u, 1.0) == best
    assert sample(x, 0.9, 0, 1.0, u, 2.0) == best
    plain_draw = sample(x, 0.9, 0, 1.0, u, None)
    assert sample(x, 0.9, 0, 1.0, u, 0.0) == plain_draw
    assert sample(x, 0.9, 0, 1.0, u, -1.0) == plain_draw
    assert sample(x, 0.9, 0, 1.0, u, math.nan) == plain_draw
    assert sample(x, 0.0, 0, 1.0, u, 0.3) == best
    tied = torch.zeros((2, vocab))
    tied[:, [3, 50, 77]] = 4.0
    got = sample(tied, 0.5, 0, 1.0, torch.tensor([0.4, 0.9]), 1.0)
    assert got == [50, 77]


@pytest.mark.parametrize("vocab", [100, 9000, 40000])
def test_min_p_with_infinities_and_rows_of_nothing_but_nan(vocab):
    x = torch.randn((4, vocab), generator=torch.Generator().manual_seed(5))
    x[0, 7] = math.inf
    x[1] = math.nan
    x[2, ::2] = -math.inf
    x[3, 5:50] = math.nan
    x[3, 60] = 9.0
    for cuts in ((0, 1.0, 0.05), (0, 0.9, 0.05), (20, 0.9, 0.05)):
        got = sample(x, 0.8, cuts[0], cuts[1], torch.tensor([0.5] * 4), cuts[2])
        assert got[0] == 7 and got[1] == 0 and got[2] % 2 == 1 and not (5 <= got[3] < 50), (cuts, got)


@pytest.mark.parametrize("vocab", [1500, 3000, 40000])
def test_min_p_among_logits_that_hardly_differ(vocab):
    # differences below what an exponential or a reciprocal tells from nothing: all weigh the same, every cut leaves all of them
    g = torch.Generator().manual_seed(12)
    x = torch.randint(0, 9, (4, vocab), generator=g).float() * 1e-39
    x[1] *= 1e30                                             # (and one whose differences are no smaller than that: 1e-9)
    x[2] = 1e6 + torch.randint(0, 2, (vocab,), generator=g).float() * 0.0625
    u = torch.tensor([0.3, 0.3, 0.0, 0.77])
    for cuts in ((20, 0.9, 0.5), (20, 1.0, 0.0), (1000, 0.5, 0.1)):
        got = sample(x, 1.0, *cuts[:2], u, cuts[2])
        assert got[0] == int(float(u[0]) * vocab) and got[3] == int(float(u[3]) * vocab), (cuts, got)      # (of the uniform numbers in 32 bits)
        top = torch.nonzero(x[2] == x[2].max()).flatten().tolist()
        if cuts[0] <= len(top):
            assert got[2] == top[0], (cuts, got)
        assert got[1] == int(float(u[1]) * vocab), (cuts, got)   # (weights of 1 and 1 - 1e-9 are the same in 32 bits)


def test_rows_of_any_number_of_pieces_agree(monkeypatch):
    # rows that begin between 16 bytes, pieces of a few tokens and of as many as they may have: the tokens are the same
    g = torch.Generator().manual_seed(9)
    n, vocab = 12, 70001
    x = torch.randn((n, vocab), generator=g) * 2.5
    x[3] *= 0.01
    x[5, 100:60000] = -math.inf
    x[6, 69000:] = math.nan
    u = torch.rand((n,), generator=g)
    k = kernels.backend()
    for cuts in ((0, 1.0, 0.05), (50, 0.9, 0.05), (300, 1.0, 0.0), (0, 0.8, 0.01), (1000, 0.9, 1e-6)):
        want = sample(x, 0.9, cuts[0], cuts[1], u, cuts[2])
        for r in range(n):
            if r not in (3, 5, 6) and far_from_borders(x[r], float(torch.tensor(0.9, dtype=F32)), cuts[0], float(torch.tensor(cuts[1], dtype=F32)), float(u[r]),
                                                       float(torch.tensor(cuts[2], dtype=F32))):
                assert want[r] == plain.sample_row(x[r].tolist(), float(torch.tensor(0.9, dtype=F32)), cuts[0], float(torch.tensor(cuts[1], dtype=F32)), float(u[r]),
                                                   float(torch.tensor(cuts[2], dtype=F32))), (cuts, r)
        for pieces in (3, 4, 9, 17, 40, 100, 1024):
            with monkeypatch.context() as m:
                m.setattr(k, "_sample_pieces", lambda *a: pieces, raising=False)
                got = sample(x, 0.9, cuts[0], cuts[1], u, cuts[2])
            assert got == want, (cuts, pieces)
        one = x[:, :32765].contiguous()
        want = sample(one, 0.9, cuts[0], cuts[1], u, cuts[2])
        for pieces in (2, 13):
            with monkeypatch.context() as m:
                m.setattr(k, "_sample_pieces", lambda *a: pieces, raising=False)
                got = sample(one, 0.9, cuts[0], cuts[1], u, cuts[2])
            assert got == want, (cuts, pieces)


@pytest.mark.parametrize("vocab", [650, 32768, 32766, 151936])
def test_min_p_replayed_from_a_graph_and_on_another_stream(vocab):
    n, k = 6, kernels.backend()
    g = torch.Generator().manual_seed(11)
    xs = [(torch.randn((n, vocab), generator=g) * 2.5).to(DEV) for _ in range(3)]
    full = lambda v, dt=F32: torch.full((n,), v, dtype=dt, device=DEV)
    x, temp, top_k, top_p, min_p, u = xs[0].clone(), full(0.8), full(30, torch.int32), full(0.9), full(0.03), torch.rand((n,), generator=g).to(DEV)

    def eager(x):
        out = torch.empty(n, dtype=torch.int32, device=DEV)
        k.sample(x, temp, top_k, top_p, u, out, min_p=min_p)
        return out.tolist()

    want = [eager(v) for v in xs]
    side, out = torch.cuda.Stream(), torch.empty(n, dtype=torch.int32, device=DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        k.sample(x, temp, top_k, top_p, u, out, min_p=min_p)
    side.synchronize()
    assert out.tolist() == want[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        k.sample(x, temp, top_k, top_p, u, out, min_p=min_p)
    for v, w in list(zip(xs, want)) * 2:
        x.copy_(v)
        out.fill_(-1)
        graph.replay()
        assert eager(xs[1]) == want[1]
        assert out.tolist() == w


def test_rows_of_one_call_have_cuts_of_their_own():
    g = torch.Generator().manual_seed(6)
    n, vocab = 40, 30000
    x = torch.randn((n, vocab), generator=g) * 2.5
    u = torch.rand((n,), generator=g)
    rng = random.Random(6)
    temp = torch.tensor([rng.choice([0.0, 0.5, 1.0]) for _ in range(n)])
    k = torch.tensor([rng.choice([0, 1, 30, 300]) for _ in range(n)])
    p = torch.tensor([rng.choice([1.0, 0.5, 0.95]) for _ in range(n)])
    m = torch.tensor([rng.choice([0.0, 1e-6, 0.03, 0.4]) for _ in range(n)])
    together = sample(x, temp, k, p, u, m)
    for r in range(n):
        assert together[r] == sample(x[r : r + 1], float(temp[r]), int(k[r]), float(p[r]), float(u[r]), float(m[r]))[0], r


# ---------------------------------------------------------------------------------------------------- the walk, the move
def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def walk_case(rng, lens, vocab=6):
    tokens, parents, sampled = [], [], []
    for n in lens:
        par = plain.random_tree(rng, n, rng.choice([1, 3, 8, 64])) if n else []
        tokens += [rng.randrange(vocab) for _ in range(n)]
        sampled += [rng.randrange(vocab) for _ in range(n)]
        parents += par
    return i32(tokens), i32(parents), i32(sampled), i32([sum(lens[:r]) for r in range(len(lens))]), i32(lens)


@pytest.mark.parametrize("vocab", [1, 2, 6])
@pytest.mark.parametrize("lens", [[1], [64], [0, 5, 0, 63, 2], [7] * 300], ids=["one", "full", "empty", "many"])
def test_accepted_drafts(lens, vocab):
    rng = random.Random(len(lens) * 10 + vocab)
    for _ in range(6):
        c = walk_case(rng, lens, vocab)
        path, count, accepted = kernels.backend().accept_drafts(*c)
        want = plain.accept_drafts(*c)
        assert path.tolist() == want[0] and count.tolist() == want[1] and accepted.tolist() == want[2]


def test_accept_takes_the_lowest_of_equal_children_and_any_order_of_requests():
    # root 0 with children 1, 2, 3 (tokens 5, 9, 9), node 4 behind 3, node 5 behind 2
    tokens, parents = [0, 5, 9, 9, 8, 8], [-1, 0, 0, 0, 3, 2]
    sampled = [9, 0, 8, 8, 1, 7]
    path, count, accepted = kernels.backend().accept_drafts(i32(tokens * 2), i32(parents * 2), i32(sampled * 2), i32([6, 0]), i32([6, 6]))
    for r in range(2):
        assert path[r, :4].tolist() == [0, 2, 5, -1] and int(count[r]) == 3 and accepted[r, :4].tolist() == [9, 8, 7, -1]


@pytest.mark.parametrize("dtype,nkv,dk,dv,page,slabs", [(BF16, 2, 64, 64, 16, 3), (F32, 2, 64, 64, 16, 2), (BF16, 3, 20, 12, 10, 2), (F32, 1, 7, 9, 5, 1), (BF16, 8, 128, 128, 64, 0)])
def test_kept_drafts(dtype, nkv, dk, dv, page, slabs):
    rng = random.Random(nkv + dk)
    g = torch.Generator().manual_seed(dk)
    befores, lens = [0, 33, 5, 160], [64, 20, 1, 9]
    need = [-(-(a + b) // page) for a, b in zip(befores, lens)]
    ids = list(range(sum(need) + 2))
    rng.shuffle(ids)
    table, at = [], 0
    for n in need:
        table.append(ids[at : at + n] + [-1] * (max(need) - n))
        at += n
    lead = (slabs,) if slabs else ()
    k = torch.randn((*lead, len(ids), nkv, page, dk), generator=g).to(dtype).to(DEV)
    v = torch.randn((*lead, len(ids), nkv, dv, page), generator=g).to(dtype).to(DEV)
    for kind in range(5):
        paths = []
        for n in lens:
            inner = sorted(rng.sample(range(1, n), rng.randint(0, n - 1)))
            inner = [[], list(range(1, n)), list(range(2, n)), inner, inner[-3:]][kind]
            paths.append([0] + inner)
        path = i32([p + [-1] * (64 - len(p)) for p in paths])
        count = i32([len(p) for p in paths])
        start, tab = i32(befores), i32(table)
        want = plain.keep_drafts(k, v, tab, start, path, count)
        kernels.backend().keep_drafts(k, v, tab, start, path, count)
        assert torch.equal(k, want[0]) and torch.equal(v, want[1]), kind


def test_keep_touches_nothing_it_cannot_place():
    k, v = torch.randn((2, 6, 1, 16, 8), device=DEV), torch.randn((2, 6, 1, 8, 16), device=DEV)
    k0, v0 = k.clone(), v.clone()
    table = i32([[2, -1], [4, 9]])                           # no second page; a page that the cache does not have
    path = i32([[0, 20, 21], [0, 18, 22]])
    kernels.backend().keep_drafts(k, v, table, i32([0, 0]), path, i32([3, 3]))
    assert torch.equal(k, k0) and torch.equal(v, v0)
    kernels.backend().keep_drafts(k, v, table, i32([0, 0]), path, i32([0, -5]))
    kernels.backend().keep_drafts(k, v, table, i32([31, 40]), i32([[0, 3], [0, 2]]), i32([2, 2]))      # behind the table's end
    assert torch.equal(k, k0) and torch.equal(v, v0)


@pytest.mark.parametrize("far", [2 ** 31 - 1, 2 ** 31 - 5, -(2 ** 31), -1])
def test_starts_far_from_everything_are_nobody_s(far):
    # (a start to which a node's number cannot be added in 32 bits)
    k, v = torch.randn((2, 6, 1, 16, 8), device=DEV), torch.randn((2, 6, 1, 8, 16), device=DEV)
    k0, v0 = k.clone(), v.clone()
    kernels.backend().keep_drafts(k, v, i32([[2, 3], [4, 5]]), i32([far, far]), i32([[0, 20, 21], [0, 18, 22]]), i32([3, 3]))
    assert torch.equal(k, k0) and torch.equal(v, v0)
    path, count, accepted = kernels.backend().accept_drafts(i32([1, 2, 3]), i32([-1, 0, 1]), i32([2, 3, 9]), i32([far, 0]), i32([40, 3]))
    assert accepted[1].tolist()[:4] == [2, 3, 9, -1] and count[1] == 3 and path[1].tolist()[:4] == [0, 1, 2, -1]
    assert bool((accepted[0] == -1).all())
    for hd, dtype in ((64, BF16), (20, F32)):
        c, _ = plain.tree_case(random.Random(31), [6, 9], [40, 900], 4, 2, hd, 16, dtype, DEV)
        whole = run_tree(c)
        c["q_start"][0 if far < 0 else 1] = far                  # (starts ascend)
        got = run_tree(c)
        there = slice(6, 15) if far < 0 else slice(0, 6)
        nobody = slice(0, 6) if far < 0 else slice(6, 15)
        assert torch.equal(got[there], whole[there]), (hd, dtype)
        assert far < 0 or bool(got[nobody].isnan().all())


def test_walk_and_move_refusals():
    k = kernels.backend()
    tok, par, sam, qs, ql = walk_case(random.Random(1), [5, 3])
    for bad in ((tok.long(), par, sam, qs, ql), (tok, par[:-1], sam, qs, ql), (tok, par, sam, qs[:1], ql), (tok.cpu(), par, sam, qs, ql)):
        with pytest.raises((TypeError, ValueError)):
            k.accept_drafts(*bad)
    kc, vc = torch.zeros((2, 4, 1, 16, 8), device=DEV), torch.zeros((2, 4, 1, 8, 16), device=DEV)
    good = (kc, vc, i32([[0, 1]]), i32([3]), i32([[0, 2]]), i32([2]))
    k.keep_drafts(*good)
    for at, bad in ((0, kc.half()), (0, kc[0]), (1, vc.transpose(3, 4)), (1, vc[:, :3].contiguous()), (2, i32([0, 1])), (3, i32([3, 4])), (4, i32([0, 2])),
                    (4, i32([[0, 2]] * 2)), (5, i32([2]).long())):
        with pytest.raises((TypeError, ValueError)):
            k.keep_drafts(*good[:at], bad, *good[at + 1 :])
    with pytest.raises((TypeError, ValueError)):
        k.sample(torch.zeros((2, 9), device=DEV), *(torch.ones(2, device=DEV),), i32([0, 0]), torch.ones(2, device=DEV), torch.zeros(2, device=DEV), i32([0, 0]),
                 min_p=torch.zeros(3, device=DEV))


def test_a_check_of_drafted_tokens_as_a_server_runs_it():
    """Attention, sampling of every node, the walk and the move behind each other on one stream, from a graph as well as eagerly: the kept keys and
    values are those of the accepted tokens, and a next step's attention reads them."""
    rng, nkv, hd, page, vocab = random.Random(20), 2, 64, 16, 50
    lens, befores = [16, 5, 1], [100, 31, 7]
    c, parents = plain.tree_case(rng, lens, befores, 6, nkv, hd, page, BF16, DEV)
    t = sum(lens)
    g = torch.Generator().manual_seed(21)
    w = torch.randn((6 * hd, vocab), generator=g).to(DEV)
    tokens = torch.randint(0, vocab, (t,), generator=g, dtype=torch.int32).to(DEV)
    par, start = i32([p for tree in parents for p in tree]), i32(befores)
    u = torch.rand((t,), generator=g).to(DEV)
    full = lambda x, dt=F32: torch.full((t,), x, dtype=dt, device=DEV)
    cuts = (full(0.9), full(0, torch.int32), full(1.0))
    min_p, out, sampled = full(0.02), torch.empty((t, 6 * hd), dtype=BF16, device=DEV), torch.empty(t, dtype=torch.int32, device=DEV)
    k0, v0 = c["k_cache"].clone(), c["v_cache"].clone()
    k = kernels.backend()

    def step():
        run_args = (c["qkv"], out, c["k_cache"], c["v_cache"], c["block_table"], c["q_start"], c["q_len"], c["kv_len"], c["visible"], 6, nkv, hd, page,
                    c["scale"], 16, 116)
        k.tree_attention(*run_args)
        logits = out.float() @ w
        k.sample(logits, cuts[0], cuts[1], cuts[2], u, sampled, min_p=min_p)
        path, count, accepted = k.accept_drafts(tokens, par, sampled, c["q_start"], c["q_len"])
        k.keep_drafts(c["k_cache"], c["v_cache"], c["block_table"], start, path, count)
        return path, count, accepted

    step()
    tokens.copy_(tokens)
    # drafts that agree with the model for a while: what it sampled behind a node becomes the token of a child
    said = sampled.tolist()
    at = 0
    for n, tree in zip(lens, parents):
        for i in range(1, n):
            if rng.random() < 0.8:
                tokens[at + i] = said[at + tree[i]]
        at += n
    c["k_cache"].copy_(k0), c["v_cache"].copy_(v0)
    path, count, accepted = step()
    torch.cuda.synchronize()
    want = plain.accept_drafts(tokens, par, sampled, c["q_start"], c["q_len"])
    assert path.tolist() == want[0] and count.tolist() == want[1] and accepted.tolist() == want[2]
    assert max(want[1]) > 2
    kw, vw = plain.keep_drafts(k0, v0, c["block_table"], start, path, count)
    bits = lambda x: x.view(torch.int16)
    assert torch.equal(bits(c["k_cache"]), bits(kw)) and torch.equal(bits(c["v_cache"]), bits(vw))
    eager = out.clone()
    graph = torch.cuda.CUDAGraph()
    c["k_cache"].copy_(k0), c["v_cache"].copy_(v0)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        path_g, count_g, accepted_g = step()
    for _ in range(3):
        c["k_cache"].copy_(k0), c["v_cache"].copy_(v0)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(path_g, path) and torch.equal(count_g, count) and torch.equal(accepted_g, accepted)
        assert torch.equal(bits(c["k_cache"]), bits(kw)) and torch.equal(bits(c["v_cache"]), bits(vw))
