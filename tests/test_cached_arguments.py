"""What the bindings of the cache refuse before a launch: tensors on another device
than the call's, tensors that end too early, and strides that the kernels do not
read.  On the CPU the tensors say they are on GPU 0 and the library records its calls;
on the GPU host tensors stand beside a cache."""
import ctypes

import pytest


class On0:
    """A host tensor that says it is on GPU 0."""

    def __init__(self, t):
        self.t = t

    def get_device(self):
        return 0

    def __getattr__(self, name):
        return getattr(self.t, name)


class Calls:
    """In the library's place."""

    def __init__(self):
        self.made = []

    def __getattr__(self, name):
        return lambda *a: self.made.append(name) or 0


B, S, HEADS, HD, P, M, V, N = 3, 4, 2, 64, 16, 5, 50, 2
D = HEADS * HD


def arguments(make):
    """Each call's function, fixed arguments, and tensors that just suffice."""
    import torch
    f, i = (lambda *s: make(torch.zeros(s))), (lambda *s: make(torch.zeros(s, dtype=torch.int32)))  # noqa: E731
    index = dict(table=i(B, M), kv_len=i(B), err_flag=i(1))
    rows = dict(k=f(B * S, D), v=f(B * S, D), k_lo=f(B * S, D), v_lo=f(B * S, D))
    shape = dict(B=B, S=S, ld=D)
    return {
        "kv_append": (dict(shape), dict(index, **rows)),
        "kv_read": (dict(shape), dict(index, k_out=f(B * S, D), v_out=f(B * S, D))),
        "attn_cached": (dict(shape, H=HEADS, ld_out=D, scale=8.0, workspace_floats=9),
                        dict(index, q=f(B * S, D), out=f(B * S, D), q_lo=f(B * S, D), out_lo=f(B * S, D), workspace=f(9))),
        "kv_copy_pages": (dict(n=6), dict(src=i(6), dst=i(6), err_flag=i(1))),
        "verify_tokens": (dict(B=B, n_draft=N, vocab=V, temperature=1.0),
                          dict(logits=f(B, N + 1, V), draft_logits=f(B, N, V), draft_ids=i(B, N), draft_len=i(B), out_ids=i(B, N + 1),
                               n_accepted=i(B), uniforms=make(torch.zeros((B, N + 1), dtype=torch.float64)), err_flag=i(1))),
    }


CALLS = ["kv_append", "kv_read", "attn_cached", "kv_copy_pages", "verify_tokens"]


@pytest.fixture
def at0(gbx, monkeypatch):
    """(the recording library, call(name, fixed, tensors))"""
    lib = Calls()
    gbx._Torch.load()
    monkeypatch.setattr(gbx, "_lib", lib)
    monkeypatch.setattr(gbx._Torch, "device", staticmethod(lambda: 0))
    monkeypatch.setattr(gbx._Torch, "stream", staticmethod(lambda dev: 0))
    monkeypatch.setattr(gbx, "_device_of", lambda t: 0)
    c = gbx._KVCacheStruct(1 << 20, 2 << 20, 3 << 20, 4 << 20, 8, 1, P, HEADS, HD)

    class Cache:
        _dev, heads, hd, _ref = 0, HEADS, HD, ctypes.byref(c)

    def call(name, fixed, tensors):
        lead = () if name == "verify_tokens" else (Cache,) if name == "kv_copy_pages" else (Cache, 0)
        return getattr(gbx, name)(*lead, **fixed, **tensors)
    return lib, call


@pytest.mark.parametrize("name", CALLS)
def test_tensors_elsewhere_or_too_short_are_refused(at0, name):
    lib, call = at0
    fixed, tensors = arguments(On0)[name]
    call(name, fixed, tensors)                                  # just enough
    call(name, fixed, {k: 1 << 20 if k != "table" else t for k, t in tensors.items()})   # addresses are taken as they are
    assert lib.made == ["gbx_" + name] * 2
    for k, t in tensors.items():
        with pytest.raises(ValueError, match=f"^{k} is on cpu, the call runs on cuda:0"):
            call(name, fixed, dict(tensors, **{k: t.t}))
        with pytest.raises(ValueError, match=f"^{k} ends after|^table ends"):
            call(name, fixed, dict(tensors, **{k: On0(t.t.reshape(-1)[:-1].clone())}))
    assert len(lib.made) == 2


@pytest.mark.parametrize("name", ["kv_append", "kv_read", "attn_cached"])
def test_rows_of_a_wider_array_pass(at0, name):
    """Column blocks of a QKV output, whose last row ends with the array; with counts, rows behind the last need not be there."""
    import torch
    lib, call = at0
    fixed, tensors = arguments(On0)[name]
    wide = torch.zeros((B * S, 3 * D))
    first = "q" if name == "attn_cached" else "v" if name == "kv_append" else "k_out"
    lo = {"k_lo": None, "v_lo": None} if name == "kv_append" else {"q_lo": None} if name == "attn_cached" else {}
    other = {"k": On0(wide[:, D:])} if name == "kv_append" else {"v_out": On0(wide[:, D:])} if name == "kv_read" else {}
    call(name, dict(fixed, ld=3 * D), dict(tensors, **{first: On0(wide[:, 2 * D:])}, **other, **lo))
    with pytest.raises(ValueError, match=f"^{first} ends after"):
        call(name, dict(fixed, ld=3 * D), dict(tensors, **{first: On0(wide.view(-1)[2 * D + 1:])}, **other, **lo))
    with pytest.raises(ValueError, match=f"^{first} must be contiguous in its last"):
        call(name, fixed, dict(tensors, **{first: On0(torch.zeros((D, B * S)).t())}))
    counts = {"n" if name == "kv_read" else "n_new": On0(torch.zeros(B, dtype=torch.int32))}
    call(name, fixed, dict(tensors, **counts, **{first: On0(tensors[first].t[:-2])}))
    assert len(lib.made) == 2


def test_logits_with_strides_are_refused(at0):
    import torch
    lib, call = at0
    fixed, tensors = arguments(On0)["verify_tokens"]
    for k in ("logits", "draft_logits", "uniforms"):
        t = tensors[k].t
        cut = torch.zeros(t.shape[:-1] + (2 * t.shape[-1],), dtype=t.dtype)[..., :t.shape[-1]]
        with pytest.raises(ValueError, match=f"^{k} must be contiguous"):
            call("verify_tokens", fixed, dict(tensors, **{k: On0(cut)}))
    assert not lib.made


@pytest.mark.gpu
@pytest.mark.parametrize("name", CALLS)
def test_host_tensors_beside_a_cache_are_refused(gbx, cuda, name):
    cache = gbx.KVCache(layers=1, pages=B * M, heads=HEADS, page=P, hd=HD)
    fixed, tensors = arguments(lambda t: t.cuda())[name]
    lead = () if name == "verify_tokens" else (cache,) if name == "kv_copy_pages" else (cache, 0)
    for k, t in tensors.items():
        with pytest.raises(ValueError, match=f"^{k} is on cpu|the tensors are not on a GPU"):
            getattr(gbx, name)(*lead, **fixed, **dict(tensors, **{k: t.cpu()}))
