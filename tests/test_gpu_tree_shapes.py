"""Attention for trees of drafted tokens in every shape of the matrix-core kernel, with the keys of a request in one part and in several, against
64-bit arithmetic."""
import math
import random

import pytest
import torch

import plain_drafts as plain
from easy_gpt.cpp_amd import kernels

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32
# (type, head size) and the shapes that the kernel has for it: 10 * (blocks of 32 rows to a workgroup) + wavefronts that share a block's keys
SHAPES = [(BF16, 64, 14), (BF16, 64, 22), (BF16, 64, 41), (BF16, 128, 14), (BF16, 128, 22), (BF16, 128, 81), (BF16, 256, 11), (BF16, 256, 21),
          (BF16, 256, 41), (F32, 64, 14), (F32, 64, 22), (F32, 128, 22), (F32, 128, 41), (F32, 256, 21)]
every_shape = pytest.mark.parametrize("dtype,hd,shape", SHAPES, ids=lambda v: str(v).replace("torch.", ""))
in_parts = pytest.mark.parametrize("parts", [1, 5])


def run_shape(monkeypatch, c, shape, parts, out=None):
    """The call, with this shape and at most so many parts of a request's keys, all of them used."""
    k = kernels.backend()
    if out is None:
        out = torch.full((c["qkv"].shape[0], c["nq"] * c["hd"]), math.nan, dtype=c["qkv"].dtype, device=DEV)
    lens, rows = c["q_len"].tolist(), 32 * (shape // 10)
    blocks = sum(-(-n * (c["nq"] // c["nkv"]) // rows) for n in lens) * c["nkv"]
    asked = []
    with monkeypatch.context() as m:
        m.setattr(k, "_tree_shape", lambda *a: asked.append(a) or (shape, parts, blocks * parts), raising=False)
        k.tree_attention(c["qkv"], out, c["k_cache"], c["v_cache"], c["block_table"], c["q_start"], c["q_len"], c["kv_len"], c["visible"], c["nq"], c["nkv"],
                         c["hd"], c["page_size"], c["scale"], max(lens), max(c["kv_len"].tolist()), window=c["window"], positions=c["positions"])
    assert asked                                             # (the kernel that has shapes)
    return out


def expected(c):
    names = ("qkv", "k_cache", "v_cache", "block_table", "q_start", "q_len", "kv_len", "visible", "nq", "nkv", "hd", "page_size", "scale",
             "window", "positions")
    return plain.tree_attention(*(c[n] for n in names))


def exact_scores_tolerance(c, spread, want):
    """Where scores are exact, what is left is an exponential (2^-21, its argument's rounding included), sums over the L weights, the rounding of bfloat16's
    weights to 2^-8 and that of the result."""
    bf16 = c["qkv"].dtype == BF16
    share = 2.0 ** -20 + 2 * int(c["kv_len"].max()) * 2.0 ** -24 + (2.0 ** -8 if bf16 else 0.0)
    return share * spread + torch.finfo(c["qkv"].dtype).eps / 2 * want.abs() * (1 + share) + 1e-30


def within(got, want, tol):
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("sign", [1, -1])
@in_parts
@every_shape
def test_large_scores_that_differ_by_little(monkeypatch, dtype, hd, shape, parts, sign):
    # Scores 2^20 - d, exact in 24 bits, d from 0 to 3 and the same for some 180 keys: parts have maxima that differ by 1 to 3.
    c, _ = plain.tree_case(random.Random(hd), [9, 6], [700, 1500], 4, 2, hd, 16, dtype, DEV)
    c["scale"] = float(sign)
    c["qkv"].zero_()
    c["qkv"].view(15, 8, hd)[:, :4, 0] = sign * 1024.0
    c["qkv"].view(15, 8, hd)[:, :4, 1] = sign * 1.0
    pages = c["block_table"].cpu()
    c["k_cache"].zero_()
    for b, kv in enumerate(c["kv_len"].tolist()):
        for j in range(kv):
            c["k_cache"][int(pages[b, j // 16]), :, j % 16, 0] = 1024.0
            c["k_cache"][int(pages[b, j // 16]), :, j % 16, 1] = -float((3, 1, 0, 2)[j // 181 % 4])
            c["v_cache"][int(pages[b, j // 16]), :, :, j % 16] = (-1.0) ** (j // 181)       # (a weight that is off is off in the result)
    want, spread = expected(c)
    within(run_shape(monkeypatch, c, shape, parts), want, exact_scores_tolerance(c, spread, want))


@in_parts
@every_shape
def test_scores_beyond_32_bits_once_scaled(monkeypatch, dtype, hd, shape, parts):
    # Products of 2^126 and 0, a scale of 8: the keys that have the greatest share the weight.
    c, _ = plain.tree_case(random.Random(hd + 1), [5, 7], [700, 1100], 4, 2, hd, 16, dtype, DEV)
    c["scale"] = 8.0
    c["qkv"].zero_()
    c["qkv"].view(12, 8, hd)[:, :4, 0] = 2.0 ** 63
    g = torch.Generator().manual_seed(hd)
    c["k_cache"].zero_()
    c["k_cache"][..., 0] = (torch.randint(0, 2, c["k_cache"].shape[:3], generator=g) * 2.0 ** 63).to(dtype).to(DEV)
    want, spread = expected(c)
    within(run_shape(monkeypatch, c, shape, parts), want, exact_scores_tolerance(c, spread, want))


@in_parts
@every_shape
def test_missing_pages_behind_the_last_masked_round_of_a_window(monkeypatch, dtype, hd, shape, parts):
    # The rows' windows begin at keys 1,001 to 1,008, in the last round before key 1,024, where the next 64 groups of 16 keys begin; some of those are in no page.
    c, _ = plain.tree_case(random.Random(hd + 2), [8, 8], [3000, 2100], 4, 2, hd, 16, dtype, DEV, window=2000, parents=[list(range(-1, 7))] * 2)
    c["positions"][8:] += 900                                # (the second request's begin there as well)
    c["v_cache"] += 3.0                                      # (values of one sign: weights for keys that are not there show)
    c["block_table"][:, [70, 95]] = -1
    clean = dict(c, block_table=c["block_table"].clone())
    c["block_table"][0, 100] = c["k_cache"].shape[0] + 3     # a page that the cache does not have is none either
    clean["block_table"][0, 100] = -1
    want, spread = expected(clean)
    got = run_shape(monkeypatch, c, shape, parts)
    within(got, want, plain.tree_tolerance(clean, spread, want))


@pytest.mark.parametrize("far", [-1, -3, -(2 ** 31), 2 ** 31 - 5, 2 ** 31 - 1])
@pytest.mark.parametrize("hd,dtype", [(64, BF16), (20, BF16), (64, F32), (22, F32)])
def test_rows_of_a_request_that_begins_nowhere_stay(hd, dtype, far):
    # (starts ascend)
    c, _ = plain.tree_case(random.Random(31), [6, 9], [40, 90], 4, 2, hd, 16, dtype, DEV)
    call = lambda out: kernels.backend().tree_attention(c["qkv"], out, c["k_cache"], c["v_cache"], c["block_table"], c["q_start"], c["q_len"], c["kv_len"],
                                                        c["visible"], 4, 2, hd, 16, c["scale"], 9, 99) or out
    whole = call(torch.full((15, 4 * hd), math.nan, dtype=dtype, device=DEV))
    assert bool(whole.isfinite().all())
    c["q_start"][0 if far < 0 else 1] = far
    got = call(torch.full((15, 4 * hd), math.nan, dtype=dtype, device=DEV))
    there, nobody = (slice(6, 15), slice(0, 6)) if far < 0 else (slice(0, 6), slice(6, 15))
    assert torch.equal(got[there], whole[there]) and bool(got[nobody].isnan().all())


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("scale", [22 ** -0.5, -0.3, 8.0])
def test_large_scores_of_heads_that_the_matrix_cores_do_not_take(scale, dtype):
    # Products of 2^20 - d, exact in 24 bits; and of 2^126 and 0, whose scaled scores are beyond 32 bits at the greatest scale.
    c, _ = plain.tree_case(random.Random(41), [9, 6], [700, 1500], 4, 2, 22, 16, dtype, DEV)
    c["scale"] = scale
    c["qkv"].zero_()
    sign = 1.0 if scale > 0 else -1.0
    c["qkv"].view(15, 8, 22)[:, :4, 0] = sign * 1024.0
    c["qkv"].view(15, 8, 22)[:, :4, 1] = sign * 1.0
    pages = c["block_table"].cpu()
    c["k_cache"].zero_()
    for b, kv in enumerate(c["kv_len"].tolist()):
        for j in range(kv):
            c["k_cache"][int(pages[b, j // 16]), :, j % 16, 0] = 1024.0
            c["k_cache"][int(pages[b, j // 16]), :, j % 16, 1] = -float((3, 1, 0, 2)[j // 181 % 4])
            c["v_cache"][int(pages[b, j // 16]), :, :, j % 16] = (-1.0) ** (j // 181)
    for far in (False, True):
        if far:
            c["qkv"].view(15, 8, 22)[:, :4, 0] = sign * 2.0 ** 63
            c["qkv"].view(15, 8, 22)[:, :4, 1] = 0.0
            c["k_cache"][..., 0] = (c["k_cache"][..., 1] == 0).to(dtype) * 2.0 ** 63
        want, spread = expected(c)
        out = torch.empty((15, 88), dtype=dtype, device=DEV)
        kernels.backend().tree_attention(c["qkv"], out, c["k_cache"], c["v_cache"], c["block_table"], c["q_start"], c["q_len"], c["kv_len"], c["visible"], 4, 2,
                                         22, 16, scale, 9, 1506)
        within(out, want, exact_scores_tolerance(c, spread, want))


@pytest.mark.parametrize("window", [-1, 1 << 31, (1 << 32) + 5])
def test_windows_that_32_bits_do_not_hold_are_refused(window):
    c, _ = plain.tree_case(random.Random(42), [4], [20], 4, 2, 64, 16, BF16, DEV, window=9)
    c["window"] = window
    with pytest.raises(ValueError):
        run_shape(pytest.MonkeyPatch(), c, 14, 1)


def check(monkeypatch, c, shape, parts, oracle=None):
    """Against 64 bits; rows of no request stay.  Twice, to the same bits."""
    want, spread = expected(oracle or c)
    got = run_shape(monkeypatch, c, shape, parts)
    nobody = want.isnan()
    assert bool(got.cpu()[nobody].isnan().all())
    tol = plain.tree_tolerance(c, spread, want)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol)[~nobody].all()), float((err / tol)[~nobody].max())
    again = run_shape(monkeypatch, c, shape, parts)
    assert torch.equal(again.nan_to_num(9.0), got.nan_to_num(9.0))
    return got


@in_parts
@every_shape
def test_uneven_trees(monkeypatch, dtype, hd, shape, parts):
    # from one row to more than a workgroup has, behind none to many rounds of keys, empty requests among them; seven query heads to a kv head, so that rows do not fill blocks
    c, _ = plain.tree_case(random.Random(51), [1, 0, 64, 13, 40, 2], [0, 50, 1100, 333, 64, 17], 14, 2, hd, 16, dtype, DEV, extra_rows=3)
    check(monkeypatch, c, shape, parts)


@in_parts
@pytest.mark.parametrize("less", [16, 8], ids=["16_less", "half"])
@every_shape
def test_heads_that_do_not_fill_the_instance(monkeypatch, dtype, hd, shape, parts, less):
    # (that of 64 takes 8 to 64 features, that of 128 up to 128 and so on)
    mine = hd - 16 if less == 16 else hd // 2 + 8
    c, _ = plain.tree_case(random.Random(52), [9, 33], [70, 700], 4, 2, mine, 32, dtype, DEV)
    check(monkeypatch, c, shape, parts)


@in_parts
@pytest.mark.parametrize("window", [1, 40, 600])
@every_shape
def test_windows(monkeypatch, dtype, hd, shape, parts, window):
    c, _ = plain.tree_case(random.Random(53), [20, 64, 1], [1333, 150, 40], 4, 2, hd, 16, dtype, DEV, window=window)
    c["block_table"][0, : max(0, 1333 - window) // 16] = -1  # (what lies behind all windows was given back)
    check(monkeypatch, c, shape, parts)


@in_parts
@every_shape
def test_any_set_of_nodes_and_rows_that_see_nothing(monkeypatch, dtype, hd, shape, parts):
    c, _ = plain.tree_case(random.Random(54), [64, 40], [300, 0], 4, 2, hd, 16, dtype, DEV)
    rng = random.Random(55)
    c["visible"][:64] = torch.tensor([rng.getrandbits(64) - (1 << 63) for _ in range(64)], dtype=torch.int64, device=DEV)
    c["visible"][64:] = torch.tensor([0 if i % 3 == 0 else 1 << (i % 40) for i in range(40)], device=DEV)
    c["visible"][65] = -1 << 40                              # only nodes that the request does not have
    got = check(monkeypatch, c, shape, parts)
    assert not bool(got[64].any()) and not bool(got[65].any())


@in_parts
@every_shape
def test_missing_pages(monkeypatch, dtype, hd, shape, parts):
    c, _ = plain.tree_case(random.Random(56), [12, 7], [1500, 200], 4, 2, hd, 16, dtype, DEV)
    c["v_cache"] += 3.0
    c["block_table"][:, 3] = -1
    c["block_table"][0, [60, 61, 80]] = -1
    oracle = dict(c, block_table=c["block_table"].clone())
    c["block_table"][0, 33], oracle["block_table"][0, 33] = c["k_cache"].shape[0], -1
    check(monkeypatch, c, shape, parts, oracle)


@in_parts
@pytest.mark.parametrize("number", [math.inf, -math.inf, math.nan])
@every_shape
def test_numbers_in_unseen_nodes(monkeypatch, dtype, hd, shape, parts, number):
    # node 3 of 12 holds no finite numbers: rows that do not see it are as if it held others; rows that do are as finite as the formula's
    c, _ = plain.tree_case(random.Random(57), [12, 5], [445, 20], 4, 2, hd, 16, dtype, DEV)
    place = 445 + 3
    page = int(c["block_table"][0, place // 16])
    c["v_cache"][page, :, : hd // 2, place % 16] = number
    c["k_cache"][page, 1, place % 16, 0] = number
    sees = torch.tensor([b >> 3 & 1 for b in c["visible"].tolist()[:12]] + [0] * 5, dtype=torch.bool)
    assert 0 < int(sees.sum()) < 12
    clean = dict(c, v_cache=c["v_cache"].clone(), k_cache=c["k_cache"].clone())
    clean["v_cache"][page, :, :, place % 16] = 0.5
    clean["k_cache"][page, :, place % 16] = 0.5
    got = run_shape(monkeypatch, c, shape, parts).cpu().double()
    want, spread = expected(clean)
    tol = plain.tree_tolerance(clean, spread, want)
    assert bool(((got - want).abs() <= tol)[~sees].all())
    assert torch.equal(got[sees].isfinite(), expected(c)[0][sees].isfinite())


@in_parts
@every_shape
def test_infinities_before_the_tree(monkeypatch, dtype, hd, shape, parts):
    c, _ = plain.tree_case(random.Random(58), [9], [700], 2, 1, hd, 16, dtype, DEV)
    c["v_cache"][int(c["block_table"][0, 20]), 0, 3, 5] = math.inf
    got = run_shape(monkeypatch, c, shape, parts).cpu().float().view(9, 2, hd)
    assert bool((got[:, :, 3] == math.inf).all())
    assert bool(got[:, :, :3].isfinite().all()) and bool(got[:, :, 4:].isfinite().all())


@in_parts
@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
@every_shape
def test_any_scale(monkeypatch, dtype, hd, shape, parts, scale):
    c, _ = plain.tree_case(random.Random(59), [9, 4], [570, 3], 4, 2, hd, 16, dtype, DEV, spread=0.5)
    c["scale"] = scale
    check(monkeypatch, c, shape, parts)


@pytest.mark.parametrize("parts", [2, 7, 64])
@every_shape
def test_a_long_context_in_any_number_of_parts(monkeypatch, dtype, hd, shape, parts):
    c, _ = plain.tree_case(random.Random(60), [24, 3], [4000, 900], 4, 2, hd, 16, dtype, DEV)
    check(monkeypatch, c, shape, parts)


def test_the_rule_chooses_every_shape():
    # (what the tests above ask for by name is what some sizes get)
    k = kernels.backend()
    chosen = set()
    for dt, size in ((1, 64), (1, 128), (1, 256), (0, 64), (0, 128), (0, 256)):
        for b in (1, 2, 8, 64):
            for n in (1, 8, 16, 32, 64):
                for group in (1, 7, 14):
                    for kv in (64, 512, 4096, 32768):
                        chosen.add((dt, size, k._tree_shape(b, b * n, 2, group, size, dt, n, kv)[0]))
    assert chosen == {(int(d is BF16), h, s) for d, h, s in SHAPES}
