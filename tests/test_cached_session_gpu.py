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
