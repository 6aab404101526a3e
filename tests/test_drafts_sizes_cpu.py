"""Sizes of the operators for drafted tokens that 32 bits do not hold are refused before anything is launched, in a process of its own: a crash ends that one."""
import subprocess
import sys

from easy_gpt.cpp_amd.csrc import build

OK, UNSUPPORTED = 0, 2
CALLS = """
import ctypes
lib = ctypes.CDLL({path!r})
p, none, f = ctypes.c_void_p(4096), ctypes.c_void_p(None), ctypes.c_float
def tree(width, page, tokens=1):
    return lib.egpt_tree_attention_generic(p, p, p, p, p, width, 1, p, p, p, p, p, 1, tokens, 2, 1, 64, page, f(1), 0, 1, none)
print(tree(1 << 27, 16), tree((1 << 26) + 1, 16), tree(3, 1 << 30), tree(1 << 26, 16, 0))
"""


def test_tables_whose_tokens_cannot_be_counted_on_from_in_32_bits_are_refused():
    p = subprocess.run([sys.executable, "-c", CALLS.format(path=build.ensure_built())], capture_output=True, text=True, timeout=110)
    assert p.returncode == 0, (p.returncode, p.stderr[-500:])
    assert [int(v) for v in p.stdout.split()] == [UNSUPPORTED] * 3 + [OK]
