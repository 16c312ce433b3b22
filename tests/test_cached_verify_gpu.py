"""gbx_verify_tokens where the CTAs of a sequence's cluster could disagree:
draws on the border of an acceptance, whose two sides differ by the last bits of
fp32 row sums.  Either side is right there; half of one and half of the other
is not."""
import os
import subprocess

import numpy as np
import pytest

import kv_oracle
from test_kv_cache_gpu import dev, i32

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "glassboxai-transformer_b200")


def softmax(x, T):
    x = x.astype(np.float64) / T
    e = np.exp(x - x.max(-1, keepdims=True))
    return e / e.sum(-1, keepdims=True)


def next_of(p, q, rejected, u):
    """The first token whose running sum passes the draw, in 64 bits, and how near another one is (relative to the sum)."""
    r = np.maximum(p - q, 0) if rejected else p
    c = np.cumsum(r)
    want = u * c[-1]
    j = int(np.flatnonzero(c > want)[0])
    return j, min(c[j] - want, want - (c[j - 1] if j else -1)) / c[-1]


# clusters of 16 CTAs (few sequences) and of 8
@pytest.mark.parametrize("B,n,V,T,with_draft", [(3, 3, 4099, 1.0, True), (60, 2, 2003, 0.8, True), (9, 1, 50257, 1.0, True),
                                                (60, 3, 1500, 1.3, False)])
def test_draws_on_the_border_of_an_acceptance(gbx, cuda, B, n, V, T, with_draft):
    import torch
    rng = np.random.default_rng(B + n)
    base = rng.standard_normal((B, n + 1, V)) * 2
    logits = (base + 0.4 * rng.standard_normal(base.shape)).astype(np.float32)
    draft = (base[:, :n] + 0.4 * rng.standard_normal((B, n, V))).astype(np.float32)
    p, q = softmax(logits, T), softmax(draft, T)
    ids = np.empty((B, n), np.int64)
    for b in range(B):
        for i in range(n):
            if with_draft:      # likely tokens that the draft thinks likelier than the target does: p / q < 1
                ids[b, i] = np.argmax(np.where(p[b, i] < 0.98 * q[b, i], q[b, i], 0))
            else:
                ids[b, i] = np.argmax(p[b, i])
    if not with_draft:
        q = np.zeros_like(q)
        np.put_along_axis(q, ids[..., None], 1.0, 2)
    border = np.take_along_axis(p[:, :n], ids[..., None], 2)[..., 0] / np.take_along_axis(q, ids[..., None], 2)[..., 0]
    assert border.max() < 1
    lg, dl, idd = dev(logits), dev(draft) if with_draft else None, i32(ids)
    sides = set()
    for call in range(120):
        # within 3e-7 of the border, where fp32 sums decide
        u = np.concatenate([border * (1 + rng.uniform(-3e-7, 3e-7, border.shape)), rng.random((B, 1))], 1)
        out = torch.full((B, n + 1), -9, dtype=torch.int32, device="cuda")
        acc = torch.full((B,), -9, dtype=torch.int32, device="cuda")
        gbx.verify_tokens(lg, idd, out, acc, B=B, n_draft=n, vocab=V, temperature=T, uniforms=dev(u), draft_logits=dl)
        out, acc = out.cpu().numpy(), acc.cpu().numpy()
        assert acc.min() >= 0 and acc.max() <= n
        sides.update(acc.tolist())
        for b in range(B):
            a = int(acc[b])
            assert np.array_equal(out[b, :a], ids[b, :a]) and np.all(out[b, a + 1:] == -1), (call, b, out[b], a)
            want, margin = next_of(p[b, a], q[b, a] if a < n else 0.0, a < n, u[b, n])
            # the running sums are in 64 bits, of some 1e5 terms at most: 1e-11 covers them
            assert out[b, a] == want or margin < 1e-11, (call, b, out[b], a, want)
    assert {0, 1} <= sides      # both sides of a border were taken


@pytest.mark.parametrize("B", [5, 60])
def test_the_same_call_gives_the_same_tokens(gbx, cuda, B):
    import torch
    rng = np.random.default_rng(11)
    n, V = 4, 9001
    logits = (rng.standard_normal((B, n + 1, V)) * 2).astype(np.float32)
    draft = (logits[:, :n] + 0.3 * rng.standard_normal((B, n, V))).astype(np.float32)
    ids, u = draft.argmax(-1), rng.random((B, n + 1))
    want, wacc = kv_oracle.verify(logits, draft, ids, np.full(B, n), 1.0, u)
    args = dev(logits), i32(ids), dev(draft), dev(u)
    for _ in range(20):
        out = torch.full((B, n + 1), -9, dtype=torch.int32, device="cuda")
        acc = torch.full((B,), -9, dtype=torch.int32, device="cuda")
        gbx.verify_tokens(args[0], args[1], out, acc, B=B, n_draft=n, vocab=V, temperature=1.0, uniforms=args[3], draft_logits=args[2])
        assert np.array_equal(acc.cpu().numpy(), wacc) and np.array_equal(out.cpu().numpy(), want)


def test_calls_of_different_sizes_from_two_threads(gbx, cuda, tmp_path):
    """A call with many drafts and one with few, each on a thread of its own (tests/cpp/verify_threads.cpp): neither takes
    the shared memory that the other's launch needs."""
    exe = str(tmp_path / "verify_threads")
    home = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-I", os.path.join(ROOT, "include"), "-I", os.path.join(home, "include"),
                    os.path.join(ROOT, "tests", "cpp", "verify_threads.cpp"), "-o", exe, "-L", PKG, "-lgbx", "-L", os.path.join(home, "lib64"),
                    "-lcudart", "-lpthread", f"-Wl,-rpath,{PKG}:{home}/lib64"], check=True)
    p = subprocess.run([exe, "20000"], capture_output=True, text=True, timeout=300)
    assert p.returncode == 0 and p.stdout.split() == ["ok"], p.stdout + p.stderr


@pytest.mark.parametrize("T", [0.3, 1.0, 1.7])
def test_every_plain_sample_is_the_inversion_of_its_row(gbx, cuda, T):
    """Rows without drafts: the token of every draw, but for draws within 1e-11 of a border of the running sum."""
    import torch
    rng = np.random.default_rng(int(10 * T))
    B, V = 300, 5001
    logits = (rng.standard_normal((B, 1, V)) * 3).astype(np.float32)
    p, u = softmax(logits, T), rng.random((B, 1))
    out = torch.full((B, 1), -9, dtype=torch.int32, device="cuda")
    acc = torch.full((B,), -9, dtype=torch.int32, device="cuda")
    gbx.verify_tokens(dev(logits), None, out, acc, B=B, n_draft=0, vocab=V, temperature=T, uniforms=dev(u))
    got = out.cpu().numpy()[:, 0]
    assert not acc.cpu().numpy().any()
    for b in range(B):
        want, margin = next_of(p[b, 0], 0.0, False, u[b, 0])
        assert got[b] == want or margin < 1e-11, (b, got[b], want, margin)
