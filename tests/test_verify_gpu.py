"""gbx_verify_tokens against the 64-bit oracle (kv_oracle.verify).  The draws
are random: one within ~1e-6 of an acceptance's border or 1e-13 of a
cumulative one could go either way, which none of these seeds does."""
import numpy as np
import pytest

import kv_oracle
from test_kv_cache_gpu import dev, i32

pytestmark = pytest.mark.gpu


def run(gbx, logits, draft, ids, lens, T, u, off=0, err=None):
    import torch
    B, n1, V = logits.shape
    lg = torch.empty(logits.size + off, device="cuda")
    lg[off:] = dev(logits.astype(np.float32)).view(-1)
    dl = None
    if draft is not None:
        dl = torch.empty(draft.size + off, device="cuda")
        dl[off:] = dev(draft.astype(np.float32)).view(-1)
    out = torch.full((B, n1), -9, dtype=torch.int32, device="cuda")
    acc = torch.full((B,), -9, dtype=torch.int32, device="cuda")
    gbx.verify_tokens(lg[off:], i32(ids), out, acc, B=B, n_draft=n1 - 1, vocab=V, temperature=T,
                      uniforms=None if u is None else dev(u), draft_logits=None if dl is None else dl[off:],
                      draft_len=None if lens is None else i32(lens), err_flag=err)
    torch.cuda.synchronize()
    return out.cpu().numpy(), acc.cpu().numpy()


def inputs(rng, B, n, V, T, noise=0.5):
    base = rng.standard_normal((B, n + 1, V)) * 2
    logits = (base + noise * rng.standard_normal(base.shape)).astype(np.float32)
    draft = (base[:, :n] + noise * rng.standard_normal((B, n, V))).astype(np.float32)
    gumbel = -np.log(-np.log(rng.random((B, n, V)) * 0.999999 + 1e-9))
    ids = (draft / max(T, 0.05) + gumbel * (T > 0.01)).argmax(-1)
    return logits, draft, ids, rng.random((B, n + 1))


@pytest.mark.parametrize("B,n,V", [(1, 4, 50257), (7, 3, 1000), (40, 1, 257), (5, 8, 129), (3, 0, 5001), (9, 2, 1), (2, 40, 300),
                                   (4, 5, 4096)])
@pytest.mark.parametrize("T", [0.0, 0.7, 1.0])
def test_verification_matches_the_oracle(gbx, cuda, B, n, V, T):
    import torch
    rng = np.random.default_rng(B * 100 + n)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    for case, with_draft in enumerate((True, False, True)):
        logits, draft, ids, u = inputs(rng, B, n, V, T)
        lens = rng.integers(0, n + 1, B) if case else np.full(B, n)
        want, wacc = kv_oracle.verify(logits, draft if with_draft else None, ids, lens, T, u)
        got, acc = run(gbx, logits, draft if with_draft else None, ids, lens, T, u, off=case, err=err)
        assert np.array_equal(acc, wacc) and np.array_equal(got, want)
    assert int(err.item()) == 0


@pytest.mark.parametrize("B,n,V,T", [(20, 2, 50257, 0.8), (40, 1, 50257, 1.0), (2, 2, 70001, 0.9), (45, 2, 140001, 0.0), (38, 1, 9000, 1.2),
                                        (20, 1, 140001, 0.9)])
def test_large_vocabularies(gbx, cuda, B, n, V, T):
    """Clusters of 16 and 8 CTAs; exponentials kept in shared memory, and too many to be kept."""
    rng = np.random.default_rng(V + B)
    logits, draft, ids, u = inputs(rng, B, n, V, T)
    lens = rng.integers(0, n + 1, B)
    for d in (draft, None):
        want, wacc = kv_oracle.verify(logits, d, ids, lens, T, u)
        got, acc = run(gbx, logits, d, ids, lens, T, u)
        assert np.array_equal(acc, wacc) and np.array_equal(got, want)


def test_greedy_takes_the_first_of_equal_maxima_and_needs_no_draws(gbx, cuda):
    V = 50257
    logits = np.zeros((2, 3, V), np.float32)
    logits[0, 0, [40000, 7, 900]] = 3.0
    logits[0, 1, [V - 1, V - 2]] = 1.0
    logits[1, :, 5] = -np.inf
    ids = np.array([[7, V - 2], [0, 1]])
    out, acc = run(gbx, logits, None, ids, None, 0.0, None)
    assert acc.tolist() == [2, 1] and out.tolist() == [[7, V - 2, 0], [0, 0, -1]]


def test_verification_at_its_borders(gbx, cuda):
    """u = 0 and u next to 1; p = q; tokens of probability 0 are never picked nor, drafted, accepted."""
    V, T = 40, 1.0
    rng = np.random.default_rng(3)
    row = rng.standard_normal((1, 1, V)).astype(np.float32)
    logits = np.repeat(np.repeat(row, 2, 1), 6, 0)
    draft = np.repeat(row, 6, 0)
    logits[:, :, [0, 1, V - 1]] = -np.inf
    draft[:, :, [0, 1, V - 1]] = -np.inf
    ids = np.full((6, 1), 4)
    ids[3], ids[4] = 0, V - 1                      # drafted although the target never says them
    draft[3, 0, 0] = 2.0
    draft[4, 0, V - 1] = 30.0
    u = np.array([[0.0, 0.0], [0.5, 0.0], [1 - 2.0 ** -53, 1 - 2.0 ** -53], [0.0, 0.0], [0.0, 1 - 2.0 ** -53], [0.3, 0.3]])
    want, wacc = kv_oracle.verify(logits, draft, ids, np.ones(6, int), T, u)
    out, acc = run(gbx, logits, draft, ids, None, T, u)
    assert np.array_equal(acc, wacc) and np.array_equal(out, want)
    assert acc[3] == 0 and acc[4] == 0 and not np.isin(out[:, 0][acc == 0], [0, 1, V - 1]).any()
    # a rejection although p = q at that row (u = 1 is out of range, but must still end in a token of some probability)
    out, acc = run(gbx, logits[:1], draft[:1], ids[:1], None, T, np.array([[1.0, 0.25]]))
    assert acc[0] == 0 and 2 <= out[0, 0] < V - 1
    out, acc = run(gbx, logits[:1], None, ids[:1], None, T, np.array([[1.0, 1.0]]))
    assert acc[0] == 0 and out[0, 0] == V - 2


@pytest.mark.parametrize("T", [0.0, 0.8])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_rows_that_give_no_distribution_end_their_sequence(gbx, cuda, T, value):
    import torch
    rng = np.random.default_rng(5)
    B, n, V = 4, 3, 700
    logits, draft, ids, u = inputs(rng, B, n, V, T, noise=0.0)     # p = q: every draft is accepted
    if T <= 0.01:
        ids = logits[:, :n].argmax(-1)
    bad = slice(None) if value == -np.inf else 333
    logits[0, 0, bad] = value
    logits[1, 2, bad] = value
    logits[2, n, bad] = value
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    want, wacc = kv_oracle.verify(logits, draft, ids, np.full(B, n), T, u * 0.99)
    out, acc = run(gbx, logits, draft, ids, None, T, u * 0.99, err=err)
    assert np.array_equal(acc, wacc) and np.array_equal(out, want)
    assert acc.tolist() == [0, 2, 3, 3] and out[0, 0] == out[1, 2] == out[2, 3] == -1 and out[3, 3] >= 0
    assert int(err.item()) == gbx.VERIFY_BAD_ROW


def test_bad_ids_and_lengths_are_flagged(gbx, cuda):
    import torch
    rng = np.random.default_rng(6)
    for T in (0.0, 1.0):
        for draft_given in (True, False):
            logits, draft, ids, u = inputs(rng, 4, 2, 300, T, noise=0.0)
            ids = logits[:, :2].argmax(-1) if T == 0.0 else ids
            ids[0, 1], ids[1, 0] = 300, -1
            lens = np.array([2, 2, 3, -1])
            err = torch.zeros(1, dtype=torch.int32, device="cuda")
            u = u * 0.5
            want, wacc = kv_oracle.verify(logits, draft if draft_given else None, ids, lens, T, u)
            out, acc = run(gbx, logits, draft if draft_given else None, ids, lens, T, u, err=err)
            assert np.array_equal(acc, wacc) and np.array_equal(out, want)
            assert out[2, 0] == out[3, 0] == -1 and acc[2] == acc[3] == 0
            assert int(err.item()) == gbx.VERIFY_BAD_ID | gbx.VERIFY_BAD_ROW


def test_a_row_without_drafts_is_a_plain_sample(gbx, cuda):
    """n_draft = 0: inversion of the running sum, as gbx_select_tokens samples but for its convention at the border."""
    import torch
    rng = np.random.default_rng(7)
    B, V = 64, 50257
    logits = (rng.standard_normal((B, 1, V)) * 2).astype(np.float32)
    u = rng.random((B, 1))
    want, _ = kv_oracle.verify(logits, None, np.zeros((B, 0), int), np.zeros(B, int), 0.9, u)
    out, acc = run(gbx, logits, None, np.zeros((B, 0)), None, 0.9, u)
    assert np.array_equal(out, want) and not acc.any()
    sel = torch.empty(B, dtype=torch.int32, device="cuda")
    gbx.select_tokens(dev(logits[:, 0]), sel, rows=B, vocab=V, temperature=0.9, uniforms=dev(u[:, 0].copy()))
    assert (sel.cpu().numpy() == out[:, 0]).mean() > 0.9


@pytest.mark.parametrize("B,V,T", [(3, 50257, 0.7), (40, 50257, 1.0), (5, 700, 1.3), (3, 140001, 0.5), (4, 5000, 0.05), (3, 900, 1e30)])
def test_masks_of_the_lowest_float_and_large_logits(gbx, cuda, B, V, T):
    """Most of the vocabulary masked by the lowest float, a row of nothing else (uniform), and logits far from 0."""
    import torch
    rng = np.random.default_rng(V)
    n, low = 3, np.finfo(np.float32).min
    logits, draft, ids, u = inputs(rng, B, n, V, T)
    masked = rng.random((B, 1, V)) < 0.97
    masked[:, :, 5] = False
    logits[np.broadcast_to(masked, logits.shape)] = low
    draft[np.broadcast_to(masked, draft.shape)] = low
    ids = (draft + 0.5 * rng.standard_normal(draft.shape)).argmax(-1)
    logits[0, 1] = low
    draft[0, 1] = low
    logits[1] = np.where(masked[1], low, np.float32(1000) + logits[1])
    draft[1] = np.where(masked[1], low, np.float32(1000) + draft[1])
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    for d in (draft, None):
        want, wacc = kv_oracle.verify(logits, d, ids, np.full(B, n), T, u)
        got, acc = run(gbx, logits, d, ids, None, T, u, err=err)
        assert np.array_equal(acc, wacc) and np.array_equal(got, want)
    assert int(err.item()) == 0
