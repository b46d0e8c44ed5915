"""Rows of a paged batch whose q_start holds anything (csrc/paged_rows.h, compiled by tests/paged_rows.cpp): the
search and the walk over value blocks end, and reach no row or position that is not their sequence's."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def test_every_small_q_start_and_long_broken_ones(tmp_path):
    exe = str(tmp_path / "paged_rows")
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(HERE, "..", "x100-gemm_amd", "csrc"),
                           os.path.join(HERE, "paged_rows.cpp"), "-o", exe])
    p = subprocess.run([exe], capture_output=True, text=True, timeout=100)
    assert p.returncode == 0, p.stderr
    small = sum((n + 3) ** (s + 1) for n in (4, 9) for s in range(1, 5))
    assert int(p.stdout) == small + 6000 + 4
