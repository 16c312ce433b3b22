"""The cached attention over pages whose value scales lie far apart.  A row's
result rests on the pages it sees, by the weight it gives them: a page with large
values that the row does not see, or hardly weighs, costs the others no bits."""
import numpy as np
import pytest

import kv_oracle
from test_kv_cache_gpu import Setup, run_attn

pytestmark = pytest.mark.gpu


def bound(s, kv_len, n_new, q, scale):
    """The output in 64 bits, and a bound on a kernel whose weights are fixed point relative to the largest product of
    weight and value scale that the row has among the four 16-token groups of a 64-token step: each of a step's
    weights is off by at most half of 2^-23 of that (and of the 2^-17 that keeps the largest below the top), which
    counts |code| times.  The rest is kv_oracle.attend's."""
    c, P = s.ref, s.P
    B, S, H, hd = q.shape
    G = H // s.heads
    out, tol = np.zeros((B, S, H, hd)), np.zeros((B, S, H, hd))
    for b in range(B):
        n, L = int(n_new[b]), int(kv_len[b])
        pages = np.array([int(s.table[b][t // P]) for t in range(L)])
        slot = np.arange(L) % P
        for i in range(n):
            t = np.arange(L - n + i + 1)
            for h in range(H):
                kc, vc = (c.codes[w][pages[t], h // G, slot[t]].astype(np.float64) for w in (0, 1))
                ks, vs = (c.scale[w][pages[t], h // G].astype(np.float64) for w in (0, 1))
                k, v, qq = kc * ks[:, None], vc * vs[:, None], q[b, i, h].astype(np.float64)
                x, A = k @ qq / scale, np.abs(k) @ np.abs(qq) / scale
                w = np.exp(x - x.max())
                w /= w.sum()
                out[b, i, h] = w @ v
                x2, A2, B2 = np.abs(x) * 1.4427, A * 1.4427, np.abs(k).sum(1) * np.abs(qq).max() / scale * 1.4427
                # (of tokens that no weight in fp32 reaches, nothing counts)
                near = w > 2.0 ** -120
                d = (B2 * 2.0 ** -23 + A2 * 2.0 ** -20 + 6 * 2.0 ** -24 * (x2 + x2.max() + 23))[near].max() * 0.6932 + 2.0 ** -22
                unit = np.zeros(L // 64 + 1)
                np.maximum.at(unit, t // 64, w * vs)
                fixed = np.zeros((L // 64 + 1, hd))
                np.add.at(fixed, t // 64, np.abs(vc))
                tol[b, i, h] = (2 * d + 2.0 ** -21 + (40 + L / 4) * 2.0 ** -23) * (w @ np.abs(v)) + \
                    (unit[:, None] * fixed).sum(0) * 2.0 ** -24 * (1 + 2.0 ** -16)
    return out, tol


def check(s, q, kv_len, n_new, scale):
    want, tol = bound(s, kv_len, n_new, q, scale)
    for ws in ("auto", None):
        got, _ = run_attn(s, q, kv_len, n_new, scale, workspace=ws)
        assert np.isfinite(got).all()
        err = np.abs(got.astype(np.float64) - want)
        assert np.all(err <= tol + 1e-38), f"{np.max(err / np.maximum(tol, 1e-38)):.3g} of the bound"
    assert int(s.err.item()) == 0


SHAPES = [(1, 64, 1), (5, 64, 1), (3, 64, 4), (40, 64, 1), (40, 32, 2), (40, 128, 1), (2, 128, 1), (12, 16, 1)]   # rows, width, queries a head


@pytest.mark.parametrize("S,hd,G", SHAPES)
@pytest.mark.parametrize("ratio", [1e3, 1e5, 1e8, 1e20])
def test_a_page_that_the_rows_do_not_see(gbx, cuda, S, hd, G, ratio):
    """Pages of 16 whose values grow by `ratio` from one to the next in the rows' own part: a row sees the smaller
    ones only."""
    heads, L = 2, 64 + 37 + S
    s = Setup(gbx, 16, heads, hd, 1, L, seed=S + hd)
    grow = np.maximum(np.arange(s.m) - (L - S) // 16, 0)
    for j, p in enumerate(s.table[0]):
        s.ref.scale[1][p] *= np.float32(min(ratio ** grow[j], 1e30) * 1e-8)
    s.upload()
    q = s.rng.standard_normal((1, S, heads * G, hd)).astype(np.float32)
    check(s, q, [L], [S], np.sqrt(hd) * 4)


@pytest.mark.parametrize("S,hd,G", SHAPES)
@pytest.mark.parametrize("ratio", [1e3, 1e5, 1e8])
def test_a_page_that_the_rows_hardly_weigh(gbx, cuda, S, hd, G, ratio):
    """Every fourth page has values `ratio` times larger, whose keys no row attends to: weights of ratio^-2 and below."""
    heads, L = 2, 300 + S
    s = Setup(gbx, 16, heads, hd, 1, L, seed=S * hd)
    big = s.table[0][1::4]
    s.ref.scale[1][big] *= np.float32(ratio)
    s.ref.scale[0][:] = np.float32(1 / 60)
    for w in range(16):       # column 0 of a key says whether it is wanted
        s.ref.codes[0][:, :, w, 0] = 100
        s.ref.codes[0][big, :, w, 0] = -100
    s.upload()
    q = s.rng.standard_normal((1, S, heads * G, hd)).astype(np.float32) * 0.05
    q[..., 0] = 60 / 200 * 2.1 * np.log(ratio) + 3
    check(s, q, [L], [S], 1.0)


@pytest.mark.parametrize("S", [1, 5, 40])
def test_pages_of_zero_and_of_tiny_values(gbx, cuda, S):
    """Scales of 0 beside others, and all of a row's values at 1e-30."""
    heads, hd, L = 2, 64, 130 + S
    for tiny in (0.0, 1e-30):
        s = Setup(gbx, 16, heads, hd, 1, L, seed=S)
        s.ref.scale[1][s.table[0][::2 if tiny == 0.0 else 1]] = np.float32(tiny)
        s.upload()
        q = s.rng.standard_normal((1, S, heads, hd)).astype(np.float32)
        check(s, q, [L], [S], 8.0)


@pytest.mark.parametrize("S,hd,G", SHAPES)
@pytest.mark.parametrize("P", [16, 64])
def test_large_values(gbx, cuda, S, hd, G, P):
    """Values up to 1e35: their sums in fixed point, 2^36 units and more, stay finite too."""
    heads, L = 2, 200 + S
    s = Setup(gbx, P, heads, hd, 1, L, seed=S * hd + 1)
    s.ref.scale[1][:] = np.float32(1e35 / 127) * s.rng.uniform(0.3, 1, s.ref.scale[1].shape).astype(np.float32)
    s.ref.codes[1][:] = 127 - np.abs(s.ref.codes[1]) // 2
    s.upload()
    q = s.rng.standard_normal((1, S, heads * G, hd)).astype(np.float32) * 0.1
    check(s, q, [L], [S], np.sqrt(hd))
