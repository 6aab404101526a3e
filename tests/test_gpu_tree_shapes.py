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
