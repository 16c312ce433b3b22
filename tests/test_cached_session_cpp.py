"""gbx::Session from a C++ program (tests/cpp/session_check.cpp): what cannot be
said through the C ABI."""
import os
import subprocess

import pytest

from gguf_writer import GGML_F32, write_tiny_gpt2

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "glassboxai-transformer_b200")


@pytest.fixture(scope="module")
def session_check(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("cpp") / "session_check")
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-I", os.path.join(ROOT, "include"),
                    os.path.join(ROOT, "tests", "cpp", "session_check.cpp"), "-o", exe, "-L", PKG, "-lgbx_model", "-lgbx",
                    f"-Wl,-rpath,{PKG}"], check=True)
    return exe


def run(*args):
    p = subprocess.run(args, capture_output=True, text=True, timeout=300)
    assert p.returncode == 0 and p.stdout.split() == ["ok"], f"{p.returncode} {p.stdout}{p.stderr}"


def test_page_sizes_that_cannot_be(session_check):
    run(session_check, "sizes")

@pytest.mark.gpu
def test_a_model_is_loaded_once(session_check, cuda, tmp_path):
    path = str(tmp_path / "m.gguf")
    write_tiny_gpt2(path, GGML_F32, d=128, heads=2, ff=256, layers=2, ctx=64, vocab=700, seed=1)
    run(session_check, "reload", path)
