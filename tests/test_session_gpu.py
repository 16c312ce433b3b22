"""Cached generation end to end (gbx::Session through its C ABI): steps against
a plain GPT-2 in 64 bits whose keys and values go through the oracle's 8-bit
cache, and the session's own laws (forks, truncation, compaction, exhaustion,
speculative steps).

Tolerance of a step's logits.  The session's arithmetic is the forward's
(tests/test_model_gpu.py: 1e-5 + 1e-3 of the logit), and the cache adds one
thing: a key or value whose fp32 rounding (some 1e-6 of it) carries it over a
border between codes is off by a whole step, 1/127 of its page's largest.  That
happens to about one value in 1e5, so to none or one of a test's some 2e4; in
one of 64 columns of one of n >= 20 keys it moves a score by at most |q| step /
8 and a logit by under 1e-3 of the largest one.  So: 2e-3 of the largest."""
import importlib

import numpy as np
import pytest

import kv_oracle
from gguf_writer import GGML_F32, tiny_gpt2_tensors, write_tiny_gpt2

pytestmark = pytest.mark.gpu

DIMS = dict(d=128, heads=2, ff=256, layers=2, ctx=256, vocab=700)


@pytest.fixture(scope="module")
def gm():
    return importlib.import_module("glassboxai-transformer_b200.model")


@pytest.fixture(scope="module")
def model(gm, cuda, tmp_path_factory):
    path = str(tmp_path_factory.mktemp("session") / "tiny.gguf")
    write_tiny_gpt2(path, GGML_F32, seed=17, **DIMS)
    m = gm.Model(path)
    yield m
    m.close()


def boosted(gm, tmp_path, seed, **dims):
    """A tiny model and its tensors."""
    path = str(tmp_path / "m.gguf")
    kw = dict(DIMS, **dims)
    write_tiny_gpt2(path, GGML_F32, seed=seed, **kw)
    return gm.Model(path), tiny_gpt2_tensors(seed=seed, **kw), kw


class Plain:
    """GPT-2 in 64 bits over the oracle's cache; one sequence, its pages in order."""

    def __init__(self, t, kw, P, pages=16):
        self.t = {k: v.astype(np.float64) for k, v in t.items()}
        self.kw, self.hd = kw, kw["d"] // kw["heads"]
        self.caches = [kv_oracle.Cache(pages, kw["heads"], P, self.hd) for _ in range(kw["layers"])]
        self.table, self.n = np.arange(pages)[None], 0

    def _ln(self, x, name):
        m = x.mean(-1, keepdims=True)
        v = ((x - m) ** 2).mean(-1, keepdims=True)
        return (x - m) / np.sqrt(v + 1e-5) * self.t[name + ".weight"] + self.t[name + ".bias"]

    def step(self, ids):
        """Logits of every new token."""
        t, H, hd, d = self.t, self.kw["heads"], self.hd, self.kw["d"]
        S, fresh = len(ids), self.n == 0
        self.n += S
        x = t["token_embd.weight"][ids] + t["position_embd.weight"][self.n - S:self.n]
        for l, c in enumerate(self.caches):
            p = f"blk.{l}."
            qkv = self._ln(x, p + "attn_norm") @ t[p + "attn_qkv.weight"].T + t[p + "attn_qkv.bias"]
            q, k, v = (qkv[:, i * d:(i + 1) * d].reshape(1, S, H, hd) for i in range(3))
            c.append(self.table, [self.n], [S], k.astype(np.float32), v.astype(np.float32))
            if fresh and hd == 64:     # a prompt attends over its own keys and values as they are
                a = np.zeros((S, H, hd))
                for h in range(H):
                    s = np.where(np.tril(np.ones((S, S), bool)), q[0, :, h] @ k[0, :, h].T / np.sqrt(hd), -np.inf)
                    w = np.exp(s - s.max(-1, keepdims=True))
                    a[:, h] = (w / w.sum(-1, keepdims=True)) @ v[0, :, h]
            else:
                a, _ = kv_oracle.attend(c, self.table, [self.n], [S], q, np.sqrt(hd))
            x = x + a.reshape(S, d) @ t[p + "attn_output.weight"].T + t[p + "attn_output.bias"]
            u = self._ln(x, p + "ffn_norm") @ t[p + "ffn_up.weight"].T + t[p + "ffn_up.bias"]
            u = u * 0.5 * (1 + np.tanh(0.7978845608 * (u + 0.044715 * u ** 3)))
            x = x + u @ t[p + "ffn_down.weight"].T + t[p + "ffn_down.bias"]
        return self._ln(x, "output_norm") @ t["token_embd.weight"].T


def close(got, want):
    err, big = np.abs(got - want).max(), np.abs(want).max()
    assert err <= 2e-3 * big, f"{err:.3g} off, of {big:.3g}"


@pytest.mark.parametrize("d,heads,P", [(128, 2, 16), (128, 2, 64), (96, 2, 32), (64, 4, 16), (256, 2, 128)])
def test_steps_match_the_plain_model(gm, cuda, tmp_path, d, heads, P):
    """A prompt, single tokens, a chunk and single tokens again."""
    model, tensors, kw = boosted(gm, tmp_path, seed=d + heads, d=d, heads=heads)
    s = gm.Session(model, pages=40, page_size=P)
    rng = np.random.default_rng(d)
    seq, plain = s.new(), Plain(tensors, kw, P)
    for n in (21, 1, 1, 7, 1, 40, 1):
        ids = rng.integers(0, kw["vocab"], n)
        want = plain.step(ids)
        if n % 2:
            got = s.forward([seq], [ids], all_rows=True)
            close(got, want)
        else:
            close(s.forward([seq], [ids])[0], want[-1])
    assert s.length(seq) == 72
    s.close()
    model.close()
    gbx = importlib.import_module("glassboxai-transformer_b200")
    for call in (s.new, lambda: s.forward([0], [[1]]), s.compact, lambda: s.length(0)):
        with pytest.raises(gbx.GbxError, match="closed"):
            call()


def test_a_prompt_is_the_forward(gm, model):
    """Sequences that start together: bit for bit the forward of the same batch."""
    s = gm.Session(model, pages=20)
    ids = np.random.default_rng(0).integers(0, 700, (3, 50)).astype(np.int32)
    got = s.forward([s.new() for _ in range(3)], ids)
    assert np.array_equal(got.view(np.uint32), model.forward(ids.ravel(), batch=3).view(np.uint32))
    assert s.free_pages() == 17


def test_a_batch_is_its_sequences(gm, model):
    """Sequences of different lengths and counts together, and one by one in a second session."""
    rng = np.random.default_rng(1)
    a, b = gm.Session(model, 30, 16), gm.Session(model, 30, 16)
    sa, sb = [a.new() for _ in range(3)], [b.new() for _ in range(3)]
    prompts = [rng.integers(0, 700, n) for n in (5, 33, 16)]
    for i in range(3):
        a.forward([sa[i]], [prompts[i]])
        b.forward([sb[i]], [prompts[i]])
    for counts in ((1, 1, 1), (3, 1, 6), (2, 17, 1), (1, 1, 1)):
        toks = [rng.integers(0, 700, n) for n in counts]
        got = a.forward(sa, toks, all_rows=True)
        one = np.concatenate([b.forward([sb[i]], [toks[i]], all_rows=True) for i in range(3)])
        assert np.abs(got - one).max() <= 2e-3 * np.abs(one).max()
    last = a.forward(sa[::-1], [[7], [8, 9], [10]])
    ref = np.stack([b.forward([sb[2]], [[7]])[0], b.forward([sb[1]], [[8, 9]])[0], b.forward([sb[0]], [[10]])[0]])
    assert np.abs(last - ref).max() <= 2e-3 * np.abs(ref).max()
    assert [a.length(x) for x in sa] == [b.length(x) for x in sb]


def test_forks_truncation_and_compaction(gm, model):
    """Forks write to pages of their own; a truncated sequence continues; compaction changes nothing that is read."""
    rng = np.random.default_rng(2)
    prompt = rng.integers(0, 700, 40)
    a, b = gm.Session(model, 24, 16), gm.Session(model, 24, 16)
    base = a.new()
    a.forward([base], [prompt])
    free = a.free_pages()
    forks = [a.fork(base) for _ in range(3)]
    assert a.free_pages() == free
    toks = rng.integers(0, 700, (4, 12))
    everyone = [base] + forks
    alone = []
    for i in range(4):          # the same sequences, unshared, in a second session
        x = b.new()
        b.forward([x], [prompt])
        alone.append(x)
    for j in range(12):
        got = a.forward(everyone, toks[:, j:j + 1])
        want = b.forward(alone, toks[:, j:j + 1])
        assert np.array_equal(got.view(np.uint32), want.view(np.uint32)), j
    # holes in the pool, then compaction: the next steps are those of the session that did not compact
    for s, seqs in ((a, everyone), (b, alone)):
        s.release(seqs[1])
        s.truncate(seqs[2], 20)
    moved = a.compact()
    assert moved > 0 and a.compact() == 0
    for j in range(6):
        got = a.forward([everyone[i] for i in (0, 2, 3)], toks[[0, 2, 3], j:j + 1])
        want = b.forward([alone[i] for i in (0, 2, 3)], toks[[0, 2, 3], j:j + 1])
        assert np.array_equal(got.view(np.uint32), want.view(np.uint32)), j
    assert a.length(everyone[2]) == 26 and a.length(everyone[1]) == -1
    fresh = a.new()             # the released number, started anew
    assert fresh == everyone[1]
    assert np.array_equal(a.forward([fresh], [prompt])[0].view(np.uint32), model.forward(prompt).view(np.uint32))


def test_refusals_leave_the_sequences_as_they_were(gm, model, cuda):
    rng = np.random.default_rng(3)
    gbx = importlib.import_module("glassboxai-transformer_b200")
    s, twin = gm.Session(model, 5, 16), gm.Session(model, 5, 16)
    x, y = s.new(), s.new()
    tx = twin.new()
    p = rng.integers(0, 700, 30)
    s.forward([x], [p])
    twin.forward([tx], [p])
    bad = [lambda: s.forward([x], [rng.integers(0, 700, 60)]),          # 6 pages of 5
           lambda: s.forward([x, x], [[1], [2]]), lambda: s.forward([x, 99], [[1], [2]]), lambda: s.forward([x], [[]]),
           lambda: s.forward([x], [[700]]), lambda: s.forward([x, y], [[1], [-1]]), lambda: s.truncate(x, 31), lambda: s.fork(7),
           lambda: s.release(7), lambda: s.truncate(-1, 0), lambda: s.next_tokens([x], [[1]], temperature=0.5),
           lambda: s.verify([x], [[1, 2]], temperature=0.5), lambda: s.verify([x], [[1, 2]], draft_len=[2]),
           lambda: s.verify([x, x], [[1, 2], [3, 4]]), lambda: s.next_tokens([x], [[1]], temperature=float("nan"))]
    for call in bad:
        with pytest.raises(gbx.GbxError):
            call()
        assert s.length(x) == 30 and s.length(y) == 0 and s.free_pages() == 3
    for size, pages in ((24, 4), (0, 4), (16, 0), (16, -1)):
        with pytest.raises(gbx.GbxError):
            gm.Session(model, pages, size)
    got, want = s.forward([x], [[5]]), twin.forward([tx], [[5]])
    assert np.array_equal(got.view(np.uint32), want.view(np.uint32))
    long = gm.Session(model, 40, 16)
    z = long.new()
    long.forward([z], [rng.integers(0, 700, 256)])     # every position row there is
    with pytest.raises(gbx.GbxError, match="position"):
        long.forward([z], [[1]])
    # a forward that times out on the device: refused, then repeated with the same result as its twin
    prev = gbx.set_first_wait_limit(0)
    try:
        with pytest.raises(gbx.GbxError, match="timed out"):
            s.forward([x], [[6]])
    finally:
        gbx.set_first_wait_limit(prev)
    assert s.length(x) == 31
    assert np.isfinite(s.forward([x], [[6]])).all()


def test_next_tokens_select_as_the_reference_does(gm, model, orc):
    rng = np.random.default_rng(4)
    s, t = gm.Session(model, 20, 32), gm.Session(model, 20, 32)
    prompts = [rng.integers(0, 700, n) for n in (9, 40)]
    a, b = [s.new(), s.new()], [t.new(), t.new()]
    for T, u in ((0.0, None), (0.8, [0.2, 0.95]), (1.5, [0.5, 0.01])):
        got = s.next_tokens(a, prompts, T, u)
        logits = t.forward(b, prompts)
        want, _, _ = orc.select_tokens(logits, T, u if u else [0.0, 0.0])
        assert np.array_equal(got, want)
        prompts = [[int(g)] for g in got]


@pytest.mark.parametrize("T", [0.0, 0.9])
@pytest.mark.parametrize("with_logits", [False, True])
def test_speculative_steps(gm, model, T, with_logits):
    """Drafts, ragged, against the oracle on the logits of a twin session; what stays cached is the
    pending token and the accepted drafts."""
    rng = np.random.default_rng(5)
    V, k = 700, 4
    s, t = gm.Session(model, 60, 16), gm.Session(model, 60, 16)
    a, b = [s.new() for _ in range(3)], [t.new() for _ in range(3)]
    prompts = [rng.integers(0, V, n) for n in (14, 31, 50)]
    s.forward(a, prompts)
    t.forward(b, prompts)
    pending = np.array([1, 2, 3])
    accepted_any = 0
    for step in range(5):
        lens = rng.integers(0, k + 1, 3)
        lens[step % 3] = k
        before = [s.length(x) for x in a]
        # the drafts: mostly what the target would say greedily, found by stepping the twin and stepping it back
        drafts = np.zeros((3, k), np.int64)
        for i in range(3):
            tok = int(pending[i])
            for j in range(k):
                tok = int(t.forward([b[i]], [[tok]])[0].argmax()) if rng.random() < 0.8 else int(rng.integers(0, V))
                drafts[i, j] = tok
                if t.length(b[i]) == before[i] + j:      # a random draft: keep the twin in step
                    t.forward([b[i]], [[int(pending[i]) if j == 0 else int(drafts[i, j - 1])]])
            t.truncate(b[i], before[i])
        ids = np.concatenate([pending[:, None], drafts], 1)
        u = rng.random((3, k + 1))
        dl = (rng.standard_normal((3, k, V)) * 0.3).astype(np.float32) if with_logits else None
        rows = [ids[i, :lens[i] + 1] for i in range(3)]
        out, acc = s.verify(a, ids, T, None if T == 0 else u, dl, lens)
        assert [s.length(x) for x in a] == [n + 1 + int(c) for n, c in zip(before, acc)]
        assert np.all(acc <= lens)
        for i in range(3):
            assert np.array_equal(out[i, :acc[i]], drafts[i, :acc[i]]) and 0 <= out[i, acc[i]] < V and np.all(out[i, acc[i] + 1:] == -1)
        accepted_any += int(acc.sum())
        logits = t.forward(b, rows, all_rows=True)
        full = np.zeros((3, k + 1, V), np.float32)
        at = 0
        for i in range(3):
            full[i, :lens[i] + 1] = logits[at:at + lens[i] + 1]
            at += lens[i] + 1
            t.truncate(b[i], before[i] + 1 + int(acc[i]))
        # (the twin's own scores: the greedy search above may have grown a page's scale, so a draw or an
        # argmax next to a border may differ; there is none among these)
        n = lens.max()
        uu = np.concatenate([u[:, :n], u[:, k:]], 1)
        want, wacc = kv_oracle.verify(full[:, :n + 1], None if dl is None else dl[:, :n], ids[:, 1:n + 1], lens, T, uu)
        assert np.array_equal(acc, wacc) and np.array_equal(out[:, :n + 1], want)
        pending = np.array([out[i, acc[i]] for i in range(3)])
    if T == 0:
        assert accepted_any > 0


def test_two_sessions_of_one_model_take_turns(gm, model):
    """They share the model's buffers, not their caches."""
    rng = np.random.default_rng(6)
    a, b, alone = (gm.Session(model, 20, 16) for _ in range(3))
    p, q = rng.integers(0, 700, 20), rng.integers(0, 700, 35)
    x, y, z = a.new(), b.new(), alone.new()
    a.forward([x], [p])
    b.forward([y], [q])
    alone.forward([z], [p])
    for tok in rng.integers(0, 700, 5):
        got, _, want = a.forward([x], [[tok]]), b.forward([y], [[tok]]), alone.forward([z], [[tok]])
        assert np.array_equal(got.view(np.uint32), want.view(np.uint32))


def test_a_verification_that_fails_after_its_forward_is_undone(gm, model, cuda):
    gbx = importlib.import_module("glassboxai-transformer_b200")
    s = gm.Session(model, 6, 16)
    x = s.new()
    s.forward([x], [[1, 2, 3]])
    y = s.fork(x)                       # shares the page that the step writes to
    free = s.free_pages()
    for t in (float("inf"), 1e300):
        with pytest.raises(gbx.GbxError, match="temperature"):
            s.verify([x], [[4, 5, 6]], temperature=t, u=np.full((1, 3), 0.5))
        assert s.length(x) == s.length(y) == 3 and s.free_pages() == free
    out, acc = s.verify([x], [[4, 5, 6]])
    assert s.length(x) == 4 + acc[0] and s.length(y) == 3
