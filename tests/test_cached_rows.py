"""How the CTAs of a verification agree on a row's statistics, on the CPU: a C++
program (tests/cpp/row_stats_check.cpp) runs the kernel's own join through the
tree that its lanes form.  Every CTA of a cluster decides for itself which
drafts stand, so lanes that differ in a bit could end a call in two minds."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("cpp") / "row_stats_check")
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-mfma", "-ffp-contract=fast", "-I", os.path.join(CUDA, "include"),
                    "-I", os.path.join(ROOT, "glassboxai-transformer_b200", "csrc"),
                    os.path.join(ROOT, "tests", "cpp", "row_stats_check.cpp"), "-o", exe], check=True)
    return exe


@pytest.mark.parametrize("seed", [1, 2])
def test_every_lane_ends_with_the_same_row(check, seed):
    p = subprocess.run([check, "20000", str(seed)], capture_output=True, text=True, timeout=120)
    assert p.returncode == 0, p.stdout + p.stderr
    split, by_two_products = map(int, p.stdout.split())
    assert split == 0 and by_two_products > 2000
