"""The operators for drafted tokens in plain 64-bit arithmetic, row by row, on the CPU: what the tests compare the kernels with."""
from __future__ import annotations

import math

import torch

F64 = torch.float64


def tree_attention(qkv, k_cache, v_cache, block_table, q_start, q_len, kv_len, visible, nq, nkv, hd, page_size, scale, window=0, positions=None):
    """(out, spread) float64 [T, nq * hd]: the attention of every row, and sum_j p_j |v_j|, which an error relative to the weights
    or the values is a share of.  Rows of no request are NaN.  A key in no page (table entry -1) is not seen."""
    t = qkv.shape[0]
    out = torch.full((t, nq * hd), math.nan, dtype=F64)
    spread = torch.zeros((t, nq * hd), dtype=F64)
    q = qkv.cpu()[:, : nq * hd].to(F64).view(t, nq, hd)
    keys, values, table = k_cache.cpu(), v_cache.cpu(), block_table.cpu()
    starts, lens, kvs, bits = q_start.tolist(), q_len.tolist(), kv_len.tolist(), visible.tolist()
    places = positions.tolist() if positions is not None else None
    for b, (s, n, kv) in enumerate(zip(starts, lens, kvs)):
        j = torch.arange(kv)
        page = table[b, j // page_size].long() if kv else torch.zeros(0, dtype=torch.long)
        k = keys[page.clamp(min=0), :, j % page_size, :].to(F64)            # [kv, nkv, hd]
        v = values[page.clamp(min=0), :, :, j % page_size].to(F64)
        for i in range(n):
            before = kv - n
            lo = max(0, places[s + i] - window + 1) if window else 0
            sees = [(x >= lo if x < before else (x - before < 64 and bits[s + i] >> (x - before) & 1)) and page[x] >= 0 for x in range(kv)]
            at = torch.tensor([x for x in range(kv) if sees[x]], dtype=torch.long)
            for h in range(nq):
                cols = slice(h * hd, (h + 1) * hd)
                if not len(at):
                    out[s + i, cols] = 0
                    continue
                p = torch.softmax(k[at, h // (nq // nkv)] @ q[s + i, h] * scale, 0)
                vv = v[at, h // (nq // nkv)]
                out[s + i, cols] = p @ vv
                spread[s + i, cols] = p @ vv.abs()
    return out, spread


def sample_row(x, temperature, top_k, top_p, uniform, min_p=0.0):
    """One row's token: the cuts by comparison of 64-bit weights, the draw in index order."""
    x = [float(v) for v in x]
    top = max(x)
    if not temperature > 0:
        return x.index(top)
    w = [math.exp((v - top) / temperature) for v in x]
    order = sorted(w, reverse=True)
    kept = [True] * len(w)
    if 0 < top_k < len(w):
        kept = [v >= order[top_k - 1] for v in w]
    if 0 < top_p < 1:
        need = top_p * math.fsum(v for v, keep in zip(w, kept) if keep)
        run, line = 0.0, 0.0
        for v in order:                                  # the weight with which the mass is reached
            line = v
            run += v
            if run >= need:
                break
        kept = [keep and v >= line for v, keep in zip(w, kept)]
    if min_p > 0:
        kept = [keep and v >= min(min_p, 1.0) for v, keep in zip(w, kept)]
    mass, run = math.fsum(v for v, keep in zip(w, kept) if keep), 0.0
    last = x.index(top)
    for i, (v, keep) in enumerate(zip(w, kept)):
        if keep:
            run += v
            last = i
            if run > uniform * mass:
                return i
    return last


def accept_drafts(tokens, parents, sampled, q_start, q_len):
    """(path, count, accepted) as lists."""
    tok, par, sam = tokens.tolist(), parents.tolist(), sampled.tolist()
    paths, counts, out = [], [], []
    for s, n in zip(q_start.tolist(), q_len.tolist()):
        path = [0] if n else []
        while path:
            nxt = [i for i in range(path[-1] + 1, n) if par[s + i] == path[-1] and tok[s + i] == sam[s + path[-1]]]
            if not nxt:
                break
            path.append(nxt[0])
        paths.append(path + [-1] * (64 - len(path)))
        counts.append(len(path))
        out.append([sam[s + i] for i in path] + [-1] * (64 - len(path)))
    return paths, counts, out


def keep_drafts(k_cache, v_cache, block_table, start, path, count):
    """New caches, from copies: every entry is read from the old ones."""
    k, v = k_cache.clone(), v_cache.clone()
    ps, table = k_cache.shape[-2], block_table.tolist()
    lead = (slice(None),) if k_cache.dim() == 5 else ()
    for b, (s, p, c) in enumerate(zip(start.tolist(), path.tolist(), count.tolist())):
        for i in range(c):
            a, z = s + p[i], s + i
            k[(*lead, table[b][z // ps], slice(None), z % ps)] = k_cache[(*lead, table[b][a // ps], slice(None), a % ps)]
            v[(*lead, table[b][z // ps], slice(None), slice(None), z % ps)] = v_cache[(*lead, table[b][a // ps], slice(None), slice(None), a % ps)]
    return k, v


def random_tree(rng, n, branch=5):
    """Parents of a tree of n nodes."""
    return [-1] + [rng.randrange(max(0, i - branch), i) for i in range(1, n)]


def tree_case(rng, lens, befores, nq, nkv, hd, page, dtype, device="cpu", window=0, parents=None, spread=1.0, extra_rows=0):
    """Operands of tree_attention for requests of those many nodes behind those many tokens, pages in random order, every number of the caches that no
    request has a NaN."""
    from easy_gpt.cpp_amd.kernels import draft_masks

    g = torch.Generator().manual_seed(rng.randrange(1 << 30))
    need = [max(1, -(-(n + b) // page)) for n, b in zip(lens, befores)]
    pages = sum(need) + 2
    ids = list(range(pages))
    rng.shuffle(ids)
    table, at = [], 0
    for k in need:
        table.append(ids[at : at + k] + [-1] * (max(need) - k))
        at += k
    t = sum(lens) + extra_rows
    qkv = (torch.randn((t, (nq + 2 * nkv) * hd), generator=g) * spread).to(dtype)
    k = torch.full((pages, nkv, page, hd), math.nan, dtype=dtype)
    v = torch.full((pages, nkv, hd, page), math.nan, dtype=dtype)
    visible, positions, parents_all = [], [], []
    for r, (n, b) in enumerate(zip(lens, befores)):
        for j in range(n + b):
            k[table[r][j // page], :, j % page] = torch.randn((nkv, hd), generator=g).to(dtype)
            v[table[r][j // page], :, :, j % page] = torch.randn((nkv, hd), generator=g).to(dtype)
        tree = random_tree(rng, n) if parents is None and n else (parents or [[]] * len(lens))[r]
        depth, mask = draft_masks(tree, window)
        visible += mask
        positions += [b + d for d in depth]
        parents_all.append(tree)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
    starts = [sum(lens[:r]) for r in range(len(lens))]
    return dict(qkv=qkv.to(device), k_cache=k.to(device), v_cache=v.to(device), block_table=i32(table), q_start=i32(starts), q_len=i32(lens),
                kv_len=i32([n + b for n, b in zip(lens, befores)]),
                visible=torch.tensor(visible + [0] * extra_rows, dtype=torch.int64, device=device), nq=nq, nkv=nkv, hd=hd, page_size=page,
                scale=hd ** -0.5, window=window, positions=i32(positions + [0] * extra_rows) if window else None), parents_all


def tree_tolerance(case, spread, out):
    """How far a kernel may be from 64 bits, element by element.  The scores' products are exact in float32's 24 bits (bfloat16) or rounded to
    them, their sums of hd terms off by at most hd 2^-24 of the terms' magnitude, which moves a weight by as much, relatively, and so does its exponential (2^-21, its
    argument's rounding included); sums over the L weights add L 2^-24; the weights of bfloat16 are rounded to 2^-8 before their product with the
    values, and the result to half a step of its type."""
    q = case["qkv"][:, : case["nq"] * case["hd"]].cpu().to(F64)
    keys = case["k_cache"].cpu().to(F64).nan_to_num(0, 0, 0)
    size = float(q.abs().view(-1, case["hd"]).sum(-1).max() * keys.abs().max()) * abs(case["scale"])      # of sum |q k| scale
    length = int(case["kv_len"].max())
    share = 2 * (case["hd"] + 4) * 2.0 ** -24 * size + 2.0 ** -20 + 2 * length * 2.0 ** -24
    if case["qkv"].dtype == torch.bfloat16:
        share += 2.0 ** -8
    return share * spread + torch.finfo(case["qkv"].dtype).eps / 2 * out.abs() * (1 + share) + 1e-30
