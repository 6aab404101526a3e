"""Drafted tokens, what needs no GPU: the bits of a tree, and what the library's entry points refuse before they touch a device."""
import random
import subprocess
import sys

import pytest

from easy_gpt.cpp_amd.csrc import build
from easy_gpt.cpp_amd.kernels import draft_masks


def test_a_node_sees_its_ancestors_and_itself():
    depth, mask = draft_masks([-1, 0, 0, 1, 3, 2])
    assert depth == [0, 1, 1, 2, 3, 2]
    assert mask == [0b1, 0b11, 0b101, 0b1011, 0b11011, 0b100101]


def test_a_window_counts_steps_up_the_tree():
    depth, mask = draft_masks([-1, 0, 1, 2, 1], window=2)
    assert depth == [0, 1, 2, 3, 2] and mask == [0b1, 0b11, 0b110, 0b1100, 0b10010]


def test_the_64th_node_is_the_sign_bit():
    depth, mask = draft_masks(list(range(-1, 63)))
    assert depth[63] == 63 and mask[63] == -1 and mask[62] == (1 << 63) - 1
    assert draft_masks([]) == ([], [])


@pytest.mark.parametrize("parents", [[0], [-1, -1], [-1, 1], [-1, 0, 3], [-1, 0, 2], list(range(-1, 64))], ids=str)
def test_what_is_no_tree_is_refused(parents):
    with pytest.raises(ValueError):
        draft_masks(parents)


def test_masks_of_random_trees():
    rng = random.Random(1)
    for _ in range(50):
        parents = [-1] + [rng.randrange(i) for i in range(1, rng.randint(1, 64))]
        depth, mask = draft_masks(parents)
        for i in range(len(parents)):
            seen, at = set(), i
            while at >= 0:
                seen.add(at)
                at = parents[at]
            assert {m for m in range(64) if mask[i] >> m & 1} == seen and depth[i] == len(seen) - 1


BAD, UNSUPPORTED = 1, 2
ENTRIES = """
import ctypes
lib = ctypes.CDLL({path!r})
p, f, none = ctypes.c_void_p(4096), ctypes.c_float, ctypes.c_void_p(None)
def tree(out=p, width=1, pages=1, pos=p, seqs=1, tokens=1, nq=2, nkv=1, hd=64, ps=16, window=0, dtype=1):
    return lib.egpt_tree_attention_generic(p, out, p, p, p, width, pages, p, p, p, p, pos, seqs, tokens, nq, nkv, hd, ps, f(1), window, dtype, none)
print(tree(out=none), tree(width=0), tree(pages=-1), tree(pos=none, window=5), tree(seqs=0), tree(tokens=-1), tree(nq=3, nkv=2), tree(hd=0), tree(ps=0),
      tree(window=-1), tree(dtype=2), tree(hd=257), tree(nq=70000, nkv=1), tree(tokens=0))
def accept(q=p, seqs=1, tokens=1, tok=p):
    return lib.egpt_accept_drafts(tok, p, p, q, p, seqs, tokens, p, p, p, none)
print(accept(q=none), accept(seqs=-1), accept(tokens=-1), accept(tok=none), accept(seqs=0))
def keep(k=p, width=1, pw=4, seqs=1, slabs=1, pages=1, ps=16, nkv=1, dk=8, dv=8, dtype=1):
    return lib.egpt_keep_drafts(k, p, p, width, p, p, pw, p, seqs, slabs, pages, ps, nkv, dk, dv, dtype, none)
print(keep(k=none), keep(width=0), keep(pw=0), keep(seqs=-1), keep(slabs=-1), keep(pages=-1), keep(ps=0), keep(nkv=0), keep(dk=0), keep(dv=0), keep(dtype=2),
      keep(slabs=70000), keep(seqs=0), keep(slabs=0))
"""


def test_entry_points_refuse_before_they_touch_a_device():
    p = subprocess.run([sys.executable, "-c", ENTRIES.format(path=build.ensure_built())], capture_output=True, text=True, timeout=110)
    assert p.returncode == 0, (p.returncode, p.stderr[-500:])
    tree, accept, keep = ([int(v) for v in line.split()] for line in p.stdout.splitlines())
    assert tree == [BAD] * 11 + [UNSUPPORTED] * 2 + [0]
    assert accept == [BAD] * 4 + [0]
    assert keep == [BAD] * 11 + [UNSUPPORTED, 0, 0]
