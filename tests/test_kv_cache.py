"""CPU checks of the cached-generation entry points: their refusals, which are
made before any CUDA call, and the oracle against its own definition."""
import numpy as np
import pytest

import kv_oracle


class _Cache:
    """A KVCache stand-in over made-up addresses: nothing is launched."""

    def __init__(self, gbx, **kw):
        import ctypes
        v = dict(k=1 << 20, v=2 << 20, k_scale=3 << 20, v_scale=4 << 20, pages=8, layers=2, page=16, heads=2, hd=64)
        v.update(kw)
        self.device, self._dev, self.heads = None, -1, v["heads"]
        self._c = gbx._KVCacheStruct(v["k"], v["v"], v["k_scale"], v["v_scale"], v["pages"], v["layers"], v["page"], v["heads"], v["hd"])
        self._ref = ctypes.byref(self._c)


APPEND = dict(k=16, v=16, table=16, kv_len=16, B=1, S=1, ld=128, max_pages=4)
ATTN = dict(q=1 << 30, out=1 << 31, table=16, kv_len=16, B=1, S=1, H=2, ld=128, ld_out=128, scale=8.0, max_pages=4)


def _refused(gbx, call, status, text):
    with pytest.raises(gbx.GbxError) as e:
        call()
    assert e.value.status == status and text in str(e.value), str(e.value)


def _append(gbx, cache, layer=0, **kw):
    a = dict(APPEND, **kw)
    gbx.kv_append(cache, layer, a.pop("k"), a.pop("v"), a.pop("table"), a.pop("kv_len"), stream=0, **a)


def _attn(gbx, cache, layer=0, **kw):
    a = dict(ATTN, **kw)
    gbx.attn_cached(cache, layer, a.pop("q"), a.pop("out"), a.pop("table"), a.pop("kv_len"), stream=0, **a)


@pytest.mark.parametrize("kw,text", [
    (dict(page=8), "tokens per page"), (dict(page=48), "tokens per page"), (dict(page=256), "tokens per page"),
    (dict(hd=8), "head width"), (dict(hd=72), "head width"), (dict(hd=144), "head width"), (dict(hd=0), "head width"),
    (dict(k=None), "null array"), (dict(v_scale=None), "null array"), (dict(pages=0), "pages"), (dict(layers=0), "layers"),
    (dict(heads=0), "heads"), (dict(k=(1 << 20) + 8), "alignment"), (dict(k_scale=(3 << 20) + 2), "alignment")])
def test_bad_caches_are_refused(gbx, kw, text):
    c = _Cache(gbx, **kw)
    _refused(gbx, lambda: _append(gbx, c), 1, text)
    _refused(gbx, lambda: gbx.kv_read(c, 0, 16, 16, 16, 16, B=1, S=1, ld=128, max_pages=4, stream=0), 1, text)
    _refused(gbx, lambda: gbx.kv_copy_pages(c, 16, 16, n=1, stream=0), 1, text)
    if kw.get("heads") != 0:
        _refused(gbx, lambda: _attn(gbx, c), 1, text)
        _refused(gbx, lambda: gbx.attn_cached_workspace(c, B=1, S=1, H=2, max_pages=4), 1, text)


def test_bad_calls_are_refused(gbx):
    c = _Cache(gbx)
    _refused(gbx, lambda: _append(gbx, c, layer=2), 1, "layer")
    _refused(gbx, lambda: _append(gbx, c, layer=-1), 1, "layer")
    _refused(gbx, lambda: _append(gbx, c, B=-1), 1, "B=-1")
    _refused(gbx, lambda: _append(gbx, c, ld=127), 1, "ld=127")
    _refused(gbx, lambda: _append(gbx, c, k=None), 1, "null")
    _refused(gbx, lambda: _append(gbx, c, table=None, max_pages=4), 1, "table")
    _refused(gbx, lambda: _append(gbx, c, max_pages=0), 1, "table")
    _refused(gbx, lambda: _append(gbx, c, kv_len=None), 1, "kv_len")
    _refused(gbx, lambda: _append(gbx, c, max_pages=1 << 27), 3, "pages of")
    _refused(gbx, lambda: _append(gbx, c, B=1 << 20, S=1 << 20), 3, "B=")
    _refused(gbx, lambda: _attn(gbx, c, H=3), 1, "query heads")
    _refused(gbx, lambda: _attn(gbx, c, H=0), 1, "query heads")
    for scale in (0.0, -1.0, float("inf"), float("nan"), 1e-40):
        _refused(gbx, lambda: _attn(gbx, c, scale=scale), 1, "scale")
    _refused(gbx, lambda: _attn(gbx, c, H=8192, S=1 << 20, ld=1 << 20, ld_out=1 << 20, q=1 << 45, out=1 << 46), 3, "query heads a key head")
    _refused(gbx, lambda: gbx.attn_cached_workspace(c, B=1, S=1 << 20, H=8192, max_pages=4), 3, "query heads a key head")
    _refused(gbx, lambda: _attn(gbx, c, ld=127), 1, "ld=127")
    _refused(gbx, lambda: _attn(gbx, c, ld_out=64), 1, "ld_out=64")
    _refused(gbx, lambda: _attn(gbx, c, out=1 << 30), 1, "overlaps")
    _refused(gbx, lambda: _attn(gbx, c, out_lo=(1 << 31) + 4), 1, "overlaps")
    _refused(gbx, lambda: _attn(gbx, c, q_lo=(1 << 31) - 4), 1, "overlaps")
    _refused(gbx, lambda: _attn(gbx, c, workspace=16, workspace_floats=-1), 1, "workspace")
    _refused(gbx, lambda: gbx.kv_copy_pages(c, 16, 16, n=-1, stream=0), 1, "n=-1")
    _refused(gbx, lambda: gbx.kv_copy_pages(c, None, 16, n=1, stream=0), 1, "null")
    ver = dict(B=1, n_draft=2, vocab=10, stream=0)
    _refused(gbx, lambda: gbx.verify_tokens(None, 16, 16, 16, **ver), 1, "null")
    _refused(gbx, lambda: gbx.verify_tokens(16, None, 16, 16, **ver), 1, "null")
    _refused(gbx, lambda: gbx.verify_tokens(16, 16, 16, 16, temperature=0.5, **ver), 1, "uniforms")
    _refused(gbx, lambda: gbx.verify_tokens(16, 16, 16, 16, temperature=float("nan"), **ver), 1, "temperature")
    _refused(gbx, lambda: gbx.verify_tokens(16, 16, 16, 16, temperature=float("inf"), **ver), 1, "temperature")
    _refused(gbx, lambda: gbx.verify_tokens(16, 16, 16, 16, **dict(ver, vocab=0)), 1, "vocab")
    _refused(gbx, lambda: gbx.verify_tokens(16, 16, 16, 16, **dict(ver, n_draft=-1)), 1, "n_draft")
    _refused(gbx, lambda: gbx.verify_tokens(16, 16, 16, 16, **dict(ver, n_draft=257)), 3, "n_draft")


def test_empty_calls_do_nothing(gbx):
    c = _Cache(gbx)
    _append(gbx, c, B=0, table=None, kv_len=None)
    _append(gbx, c, S=0, table=None, kv_len=None, k=None, v=None)
    _attn(gbx, c, B=0)
    gbx.kv_read(c, 0, 16, 16, None, None, B=1, S=1, ld=0, max_pages=4, stream=0)
    gbx.kv_copy_pages(c, None, None, n=0, stream=0)
    gbx.verify_tokens(None, None, None, None, B=0, n_draft=1, vocab=5, stream=0)
    assert gbx.attn_cached_workspace(c, B=0, S=1, H=2, max_pages=4) == 0


def test_wrong_tensors_are_refused(gbx):
    import torch
    k = torch.zeros((1, 2, 2, 16, 64), dtype=torch.int8)
    v = torch.zeros((1, 2, 2, 1, 64, 16), dtype=torch.int8)
    s = torch.zeros((1, 2, 2))
    cache = gbx.KVCache(k=k, v=v, k_scale=s, v_scale=s.clone())
    assert (cache.pages, cache.heads, cache.page, cache.hd) == (2, 2, 16, 64)
    t32 = torch.zeros((1, 2), dtype=torch.int32)
    for bad in (dict(v=v[:, :1]), dict(k_scale=s.double()), dict(v=v.float()), dict(k_scale=s[:, :1])):
        with pytest.raises(ValueError):
            gbx.KVCache(**dict(dict(k=k, v=v, k_scale=s, v_scale=s), **bad))
    with pytest.raises(ValueError):
        gbx.KVCache(layers=1, pages=1, heads=1, page=24, hd=64, device="cpu")
    with pytest.raises(ValueError, match="int32"):
        gbx.kv_append(cache, 0, k, k, torch.zeros((1, 2), dtype=torch.int64), 16, B=1, S=1, ld=128)
    with pytest.raises(ValueError, match="float32"):
        gbx.kv_append(cache, 0, s.double(), s, t32, 16, B=1, S=1, ld=128)
    with pytest.raises(ValueError, match="float64"):
        gbx.verify_tokens(1 << 20, None, 16, 16, B=1, n_draft=0, vocab=4, temperature=1.0, uniforms=s)
    for call in (lambda: gbx.kv_append(cache, 0, s, s, t32, t32, B=1, S=1, ld=128),
                 lambda: gbx.kv_copy_pages(cache, t32, t32, n=2),
                 lambda: gbx.verify_tokens(s, None, t32, t32, B=1, n_draft=0, vocab=2)):
        with pytest.raises(ValueError, match="not on a GPU"):
            call()
    with pytest.raises(ValueError, match="int32"):
        gbx.kv_copy_pages(cache, torch.zeros(4, dtype=torch.int32)[::2], 16, n=2)


def test_oracle_values_are_within_half_a_step():
    """Tokens appended one by one: each growth of a scale adds at most half a step of the new scale."""
    rng = np.random.default_rng(0)
    c = kv_oracle.Cache(4, 2, 16, 16)
    x = rng.standard_normal((1, 40, 2, 16)).astype(np.float32) * np.exp(rng.standard_normal((1, 40, 1, 1))).astype(np.float32)
    table = np.array([[2, 0, 3]])
    bound = np.zeros((40, 2))
    for t in range(40):
        first = t // 16 * 16
        before = c.scale[0][table[0][t // 16]].copy()
        c.append(table, [t + 1], [1], x[:, t:t + 1], x[:, t:t + 1])
        now = c.scale[0][table[0][t // 16]]
        if t > first:
            bound[first:t] += np.where(now != before, now / 2, 0)
        bound[t] = now / 2
    got = np.stack([c.values(0, table, 0, t) for t in range(40)])
    assert np.all(np.abs(got - x[0]) <= bound[..., None] * (1 + 2.0 ** -20))
    whole = kv_oracle.Cache(4, 2, 16, 16)
    whole.append(table, [40], [40], x, x)
    step = np.stack([whole.scale[0][table[0][t // 16]] for t in range(40)])
    got = np.stack([whole.values(0, table, 0, t) for t in range(40)])
    assert np.all(np.abs(got - x[0]) <= step[..., None] / 2 * (1 + 2.0 ** -20))


def test_oracle_verification_keeps_the_target_distribution():
    """First tokens of many verifications are distributed as the target's row, whatever drafted them."""
    rng = np.random.default_rng(1)
    V, N, T = 6, 40000, 0.9
    p_log, q_log = rng.standard_normal((1, 2, V)), rng.standard_normal((1, 1, V))
    p = np.exp(p_log[0, 0] / T) / np.exp(p_log[0, 0] / T).sum()
    q = np.exp(q_log[0, 0] / T) / np.exp(q_log[0, 0] / T).sum()
    ids = rng.choice(V, (N, 1), p=q)
    out, acc = kv_oracle.verify(np.repeat(p_log, N, 0), np.repeat(q_log, N, 0), ids, np.ones(N, int), T, rng.random((N, 2)))
    got = np.bincount(out[:, 0], minlength=V) / N
    # five standard deviations of a count
    assert np.all(np.abs(got - p) < 5 * np.sqrt(p * (1 - p) / N))
    assert abs(acc.mean() - np.minimum(p, q).sum()) < 5 * np.sqrt(0.25 / N)


@pytest.mark.parametrize("hd", range(16, 129, 16))
def test_the_attention_reads_stay_in_their_slot(hd):
    """The cached attention's shared-memory addresses, as attn_cached.cu forms them: every 16-byte read of a slot's
    keys (lane (n, c), pair g, chunk ch) and values (lane, column block j) lies inside the slot."""
    pitch = 16 * hd + 32
    chunks = 2 if hd > 64 else 1
    for n in range(8):
        for c in range(4):
            for g in range(8):
                for ch in range(chunks):
                    at = (n >> 1) * pitch + (n & 1) * hd + 2 * g * hd + min(64 * ch + 16 * c, hd - 16)
                    assert at % 16 == 0 and at + 16 <= (n >> 1) * pitch + 16 * hd
            for j in range(hd // 8):
                at = c * pitch + n * 16 + 8 * j * 16
                assert at % 16 == 0 and at + 16 <= c * pitch + 16 * hd


def test_temperatures_without_an_fp32_reciprocal_are_refused(gbx):
    for t in (1e38, 1e300):
        _refused(gbx, lambda: gbx.verify_tokens(16, 16, 16, 16, temperature=t, B=1, n_draft=1, vocab=4, uniforms=16), 1, "temperature")
