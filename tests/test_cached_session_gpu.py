"""What a step of a Session leaves behind when it fails after its keys and values
were appended: nothing.  Each case is compared bit for bit with a twin session
that never took the step, on pages that no fork shares unless said."""
import importlib

import numpy as np
import pytest

from gguf_writer import GGML_F32, gpt2_kv, raw_of, tiny_gpt2_tensors, write_gguf, write_tiny_gpt2

pytestmark = pytest.mark.gpu

DIMS = dict(d=128, heads=2, ff=256, layers=2, ctx=256, vocab=700)
gbx = importlib.import_module("glassboxai-transformer_b200")


@pytest.fixture(scope="module")
def gm():
    return importlib.import_module("glassboxai-transformer_b200.model")


@pytest.fixture(scope="module")
def model(gm, cuda, tmp_path_factory):
    path = str(tmp_path_factory.mktemp("session") / "tiny.gguf")
    write_tiny_gpt2(path, GGML_F32, seed=23, **DIMS)
    m = gm.Model(path)
    yield m
    m.close()


def model_with(gm, path, change, **dims):
    """A tiny model whose tensors went through change(tensors)."""
    kw = dict(DIMS, **dims)
    t = tiny_gpt2_tensors(seed=29, **kw)
    change(t)
    write_gguf(str(path), gpt2_kv(d=kw["d"], layers=kw["layers"], heads=kw["heads"], ff=kw["ff"], ctx=kw["ctx"]),
               [(name, list(a.shape), GGML_F32, raw_of(a, GGML_F32)) for name, a in t.items()])
    return gm.Model(str(path))


def same(a, b):
    assert np.isfinite(a).all() and np.array_equal(a.view(np.uint32), b.view(np.uint32)), np.abs(a - b).max()


def pair(gm, model, prompts, P=64, pages=12):
    """Two sessions with the same prompts; their sequences' numbers are the same."""
    s, t = gm.Session(model, pages, P), gm.Session(model, pages, P)
    for p in prompts:
        x = s.new()
        assert t.new() == x
        s.forward([x], [p])
        t.forward([x], [p])
    return s, t, list(range(len(prompts)))


def follow(s, t, seqs, rng, n=4):
    """The next steps of both are the same bits."""
    for _ in range(n):
        toks = rng.integers(0, 700, (len(seqs), 1))
        same(s.forward(seqs, toks), t.forward(seqs, toks))


@pytest.mark.parametrize("P", [16, 64, 128])
def test_a_step_that_times_out(gm, model, P):
    rng = np.random.default_rng(P)
    s, t, seqs = pair(gm, model, [rng.integers(0, 700, n) for n in (30, 16, 5)], P, 24)
    for call in (lambda: s.forward(seqs, rng.integers(0, 700, (3, 1))), lambda: s.forward(seqs[:1], [rng.integers(0, 700, 40)]),
                 lambda: s.next_tokens(seqs, rng.integers(0, 700, (3, 2))), lambda: s.verify(seqs, rng.integers(0, 700, (3, 4)))):
        prev = gbx.set_first_wait_limit(0)
        try:
            with pytest.raises(gbx.GbxError, match="timed out"):
                call()
        finally:
            gbx.set_first_wait_limit(prev)
        assert [s.length(x) for x in seqs] == [t.length(x) for x in seqs] and s.free_pages() == t.free_pages()
        follow(s, t, seqs, rng, 2)


@pytest.mark.parametrize("P", [16, 64])
def test_a_verification_whose_rows_are_nan(gm, tmp_path, P):
    """The position row of token 40 is NaN: so are its keys and values in every layer, and its logits."""
    def change(t):
        t["position_embd.weight"][40] = np.nan
    model = model_with(gm, tmp_path / "nan.gguf", change)
    rng = np.random.default_rng(P)
    s, t, seqs = pair(gm, model, [rng.integers(0, 700, n) for n in (37, 9)], P)
    drafts = rng.integers(0, 700, (2, 5))
    # tokens the target says itself, so that the row of token 40 is reached
    greedy = t.fork(0)
    tok = int(drafts[0, 0])
    for j in range(1, 4):
        tok = int(t.forward([greedy], [[tok]])[0].argmax())
        drafts[0, j] = tok
    t.release(greedy)
    for _ in range(2):
        with pytest.raises(gbx.GbxError, match="no distribution"):
            s.verify(seqs, drafts)
        assert [s.length(i) for i in seqs] == [37, 9]
    follow(s, t, seqs, rng, 3)      # tokens 37, 38 and 39 of the first


def test_a_verification_that_is_refused_after_its_forward(gm, model):
    """Keys and values of three tokens each were appended, to a page of its own and to one that two sequences share."""
    rng = np.random.default_rng(8)
    for _ in range(5):
        s, t, seqs = pair(gm, model, [rng.integers(0, 700, n) for n in (3, 20)])
        seqs.append(s.fork(0))
        assert t.fork(0) == seqs[2]
        with pytest.raises(gbx.GbxError, match="temperature"):
            s.verify(seqs, rng.integers(0, 700, (3, 3)), temperature=1e300, u=np.full((3, 3), 0.5))
        assert [s.length(x) for x in seqs] == [3, 20, 3] and s.free_pages() == t.free_pages()
        follow(s, t, seqs, rng)


def drafts_of(t, seqs, pending, k, right, rng):
    """[n, k] drafts: the first right[i] as the target says them itself (found on a fork), the others random."""
    out = rng.integers(0, 700, (len(seqs), k))
    for i, x in enumerate(seqs):
        f, tok = t.fork(x), int(pending[i])
        for j in range(right[i]):
            tok = int(t.forward([f], [[tok]])[0].argmax())
            out[i, j] = tok
        t.release(f)
    return out


@pytest.mark.parametrize("P", [16, 32, 64])
@pytest.mark.parametrize("with_len", [False, True])
def test_rejected_drafts_leave_nothing(gm, tmp_path, P, with_len):
    """Of one layer, whose keys and values depend on nothing but their token and place: after a verification the cache is
    what appending the pending token and the accepted drafts alone would have left, bit for bit.  Rejected drafts
    stand in the kept tokens' page, in one they share with a fork, and over the border to pages of their own."""
    model = model_with(gm, tmp_path / "one.gguf", lambda t: None, layers=1)
    rng = np.random.default_rng(P + with_len)
    s, t, seqs = pair(gm, model, [rng.integers(0, 700, n) for n in (3, 13, 30, 16)], P, 60)
    seqs.append(s.fork(1))
    assert t.fork(1) == seqs[4]
    k, counts = 4, set()
    for step in range(8):
        pending = rng.integers(0, 700, len(seqs))
        drafts = drafts_of(t, seqs, pending, k, rng.integers(0, k + 1, len(seqs)), rng)
        lens = rng.integers(0, k + 1, len(seqs)) if with_len else np.full(len(seqs), k)
        out, acc = s.verify(seqs, np.concatenate([pending[:, None], drafts], 1), draft_len=lens)
        counts.update((lens - acc).tolist())
        kept = [np.concatenate([pending[i:i + 1], drafts[i, :acc[i]]]) for i in range(len(seqs))]
        t.forward(seqs, kept)
        assert [s.length(x) for x in seqs] == [t.length(x) for x in seqs] and s.free_pages() == t.free_pages()
        follow(s, t, seqs, rng, 1)
    assert 0 in counts and len(counts) > 1      # with and without rejected drafts


def test_a_large_rejected_draft_does_not_coarsen_the_kept_tokens(gm, tmp_path):
    """A token whose keys and values are many times the others', drafted and rejected time and again: the page's scales
    stay those of the kept tokens, whose logits are a twin's that never saw it."""
    def change(t):
        t["blk.0.attn_norm.bias"][:] = 0
        t["token_embd.weight"][699] = 0
        t["token_embd.weight"][699, 5] = 50.0       # after the LayerNorm nearly all of the row is in one column
        t["blk.0.attn_qkv.weight"][128:, 5] *= 10
        t["output_norm.bias"][5] = -100             # its own logit (the tables are tied) far below the others
    model = model_with(gm, tmp_path / "big.gguf", change, layers=1)
    rng = np.random.default_rng(3)
    s, t, seqs = pair(gm, model, [rng.integers(0, 699, 10)], 64)
    for _ in range(6):
        pending = int(rng.integers(0, 699))
        out, acc = s.verify(seqs, [[pending, 699, 699]], temperature=0.5, u=np.full((1, 3), 1 - 2.0 ** -53))
        assert acc[0] == 0
        t.forward(seqs, [[pending]])
        toks = rng.integers(0, 699, (1, 1))
        same(s.forward(seqs, toks), t.forward(seqs, toks))


def test_a_prompt_does_not_depend_on_its_batch_mates(gm, model):
    """Prompts of different lengths, and beside sequences that go on: each has the logits of the forward of it alone
    (tests/test_model_gpu.py's bound for the model's arithmetic, 1e-5 + 1e-3 of the logit; the batches take other
    contraction shapes), not those of its keys and values in 8 bits."""
    rng = np.random.default_rng(12)
    s, t = gm.Session(model, 60, 16), gm.Session(model, 60, 16)
    prompts = [rng.integers(0, 700, n) for n in (50, 7, 33, 1, 64)]
    alone = [model.forward(p).ravel() for p in prompts]

    def as_alone(got, i):
        assert np.all(np.abs(got - alone[i]) <= 1e-5 + 1e-3 * np.abs(alone[i])), np.abs(got - alone[i]).max()

    seqs = [s.new() for _ in prompts]
    for i, row in enumerate(s.forward(seqs, prompts)):
        as_alone(row, i)
    # 1, 3 and 4 start while 0 and 2 go on with several tokens; the ones that go on take the steps they take alone
    mixed, single = [t.new() for _ in prompts], gm.Session(model, 60, 16)
    lone = [single.new() for _ in prompts]
    for sess, ids in ((t, mixed), (single, lone)):
        for i in (0, 2):
            sess.forward([ids[i]], [prompts[i]])
    more = {0: rng.integers(0, 700, 3), 2: rng.integers(0, 700, 9)}
    got = t.forward(mixed, [more.get(i, prompts[i]) for i in range(5)])
    for i in range(5):
        if i in more:
            want = single.forward([lone[i]], [more[i]])[0]
            # the 8-bit cache may round one value another way under another contraction shape
            assert np.abs(got[i] - want).max() <= 2e-3 * np.abs(want).max()
        else:
            as_alone(got[i], i)
    assert [t.length(x) for x in mixed] == [53, 7, 42, 1, 64]


@pytest.mark.parametrize("P,seed", [(16, 1), (32, 2), (64, 3)])
def test_random_steps_with_failures_between(gm, tmp_path, P, seed):
    """Prompts, tokens, chunks, verifications, forks, truncations, releases and compactions of a one-layer model, with
    failing steps in between, against a session that takes only what stood: the same bits at every step."""
    model = model_with(gm, tmp_path / "one.gguf", lambda t: None, layers=1)
    rng = np.random.default_rng(seed)
    s, t, live = gm.Session(model, 90, P), gm.Session(model, 90, P), []

    def fail():
        seqs = [x for x in live if s.length(x) < 240 and rng.random() < 0.7] or live[:1]
        kind = rng.integers(0, 3)
        if kind == 0:
            prev = gbx.set_first_wait_limit(0)
            try:
                with pytest.raises(gbx.GbxError, match="timed out"):
                    s.forward(seqs, [rng.integers(0, 700, rng.integers(1, 6)) for _ in seqs])
            finally:
                gbx.set_first_wait_limit(prev)
        elif kind == 1:
            with pytest.raises(gbx.GbxError, match="temperature"):
                s.verify(seqs, rng.integers(0, 700, (len(seqs), 4)), temperature=1e300, u=np.full((len(seqs), 4), 0.5))
        else:
            with pytest.raises(gbx.GbxError):
                s.forward(seqs + [seqs[0]], [[1]] * (len(seqs) + 1))

    for step in range(70):
        if live and step % 3 == 1:
            fail()
        kind = rng.integers(0, 9)
        ready = [x for x in live if s.length(x) < 235]
        if not ready or (kind == 0 and len(live) < 6):
            x = s.new()
            assert t.new() == x
            live.append(x)
            p = rng.integers(0, 700, rng.integers(1, 40))
            same(s.forward([x], [p]), t.forward([x], [p]))
        elif kind == 1 and len(live) < 6:
            x = int(rng.choice(live))
            live.append(s.fork(x))
            assert t.fork(x) == live[-1]
        elif kind == 2 and len(live) > 2:
            x = live.pop(int(rng.integers(0, len(live))))
            s.release(x)
            t.release(x)
        elif kind == 3:
            x = int(rng.choice(live))
            n = int(rng.integers(0, s.length(x) + 1))
            s.truncate(x, n)
            t.truncate(x, n)
        elif kind == 4:
            s.compact()
        elif kind in (5, 6):
            pending = rng.integers(0, 700, len(ready))
            drafts = drafts_of(t, ready, pending, 3, rng.integers(0, 4, len(ready)), rng)
            out, acc = s.verify(ready, np.concatenate([pending[:, None], drafts], 1))
            t.forward(ready, [np.concatenate([pending[i:i + 1], drafts[i, :acc[i]]]) for i in range(len(ready))])
        else:
            toks = [rng.integers(0, 700, 1 if kind == 7 else rng.integers(1, 5)) for _ in ready]
            same(s.forward(ready, toks), t.forward(ready, toks))
        assert [s.length(x) for x in live] == [t.length(x) for x in live] and s.free_pages() == t.free_pages()
    for x in live:
        if s.length(x) < 250:
            follow(s, t, [x], rng, 1)
