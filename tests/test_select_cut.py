"""Lists of keys from a cut (csrc/select_cut.h, compiled by tests/select_cut.cpp): the largest keys, lower ones first among
equals, and never more than the list has room for, also where the blocks that are always taken fill it."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def test_lists_of_small_and_random_rows(tmp_path):
    exe = str(tmp_path / "select_cut")
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(HERE, "..", "x100-gemm_amd", "csrc"),
                           os.path.join(HERE, "select_cut.cpp"), "-o", exe])
    p = subprocess.run([exe], capture_output=True, text=True, timeout=100)
    assert p.returncode == 0, p.stderr
    # rows of n keys of 10 kinds; n_first + n_last = f in f ways, f <= n_sel <= n
    small = sum(10 ** n * sum(f * (n - f + 1) for f in range(1, n + 1)) for n in range(1, 6))
    assert int(p.stdout) == small + 200000
