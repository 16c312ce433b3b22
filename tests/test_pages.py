"""The host bookkeeping of the paged cache (gbx::PageTable), in a C++ program
(tests/cpp/pages_check.cpp) that keeps every token and compares after each of
many random steps.  No GPU."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "glassboxai-transformer_b200")


@pytest.fixture(scope="module")
def pages_check(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("cpp") / "pages_check")
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-I", os.path.join(ROOT, "include"),
                    os.path.join(ROOT, "tests", "cpp", "pages_check.cpp"), "-o", exe, "-L", PKG, "-lgbx_model", "-lgbx",
                    f"-Wl,-rpath,{PKG}"], check=True)
    return exe


@pytest.mark.parametrize("pages,size,steps,seed", [(40, 16, 3000, 1), (7, 16, 3000, 2), (300, 16, 1500, 3), (64, 32, 1500, 4),
                                                   (1, 128, 400, 5), (25, 64, 2000, 6)])
def test_random_steps(pages_check, pages, size, steps, seed):
    p = subprocess.run([pages_check, str(pages), str(size), str(steps), str(seed)], capture_output=True, text=True, timeout=300)
    assert p.returncode == 0 and p.stdout.split() == ["ok", str(steps)], p.stdout + p.stderr
