"""The loads of attention for trees stay in the group of keys that they are for: their addresses, computed by the kernel's own header, on the host."""
import os
import subprocess

from easy_gpt.cpp_amd.csrc import build

HERE = os.path.dirname(os.path.abspath(__file__))


def test_loads_read_what_they_are_for_and_nothing_else(tmp_path):
    program = tmp_path / "tree_loads_check"
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Wextra", "-I", build.HERE, os.path.join(HERE, "tree_loads_check.cpp"), "-o", str(program)], check=True,
                   timeout=110)
    p = subprocess.run([str(program)], capture_output=True, text=True, timeout=110)
    assert p.returncode == 0, p.stdout
    assert p.stdout.endswith(" places\n")
