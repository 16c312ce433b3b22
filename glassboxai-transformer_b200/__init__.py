"""Python binding of the B200 hot-path C ABI (``include/gbx.h``, ``libgbx.so``).

The product is the C ABI; this module is a thin ctypes layer over it for the
test suite, the benchmark and Python callers.  Pointers are passed straight
through: arguments may be torch tensors (``data_ptr()``), raw integer device
addresses, or ``None`` for nullable pointers.  Every call raises ``GbxError``
on a non-zero status with the library's own message.

There is no fallback: importing this module fails loudly if ``libgbx.so``
has not been built (``make -C glassboxai-transformer_b200``).

Import it by path, e.g. ``importlib.import_module("glassboxai-transformer_b200")``.
"""
from __future__ import annotations

import ctypes
import os

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libgbx.so")
HEADER = os.path.join(os.path.dirname(HERE), "include", "gbx.h")

DT_F32, DT_F16, DT_BF16 = 0, 1, 30
EMBED_BAD_ID, EMBED_BAD_POS, EMBED_TIMEOUT = 1, 2, 4
KV_BAD_PAGE, KV_BAD_LEN, KV_BAD_PAIR, VERIFY_BAD_ID, VERIFY_BAD_ROW = 8, 16, 32, 64, 128

STATUS = {0: "GBX_OK", 1: "GBX_EINVAL", 2: "GBX_EDTYPE", 3: "GBX_ERANGE", 4: "GBX_ECUDA",
          5: "GBX_EIO", 6: "GBX_ENOTFOUND", 7: "GBX_ENOMEM"}


class GbxError(RuntimeError):
    def __init__(self, status: int, msg: str):
        super().__init__(f"{STATUS.get(status, status)}: {msg}")
        self.status = status


_vp = ctypes.c_void_p
_i64 = ctypes.c_int64
_int = ctypes.c_int
_f = ctypes.c_float

# name -> argtypes (restype int unless listed in _RESTYPES)
SIGNATURES = {
    "gbx_version": [],
    "gbx_status_string": [_int],
    "gbx_last_error": [],
    "gbx_set_pdl": [_int],
    "gbx_set_first_wait_limit": [ctypes.c_uint64],
    "gbx_dequant": [_vp, _int, _vp, _i64, _vp],
    "gbx_embed": [_vp, _vp, _int, _vp, _int, _vp, _vp, _i64, _int, _int, _int, _int, _int, _vp, _vp],
    "gbx_embed_layernorm": [_vp, _vp, _int, _vp, _int, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _int, _int, _int, _int,
                            _int, _f, _vp, _vp],
    "gbx_layernorm": [_vp, _vp, _vp, _vp, _i64, _int, _f, _vp],
    "gbx_layernorm_pair": [_vp, _vp, _vp, _vp, _vp, _i64, _int, _f, _vp],
    "gbx_residual_layernorm": [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _int, _f, _vp],
    "gbx_final_layernorm": [_vp, _vp, _vp, _vp, _vp, _i64, _int, _int, _f, _vp],
    "gbx_bias_gelu": [_vp, _vp, _vp, _i64, _int, _vp],
    "gbx_softmax_rows": [_vp, _vp, _i64, _int, _vp],
    "gbx_attn_softmax_rows": [_vp, _vp, _i64, _int, _int, _int, _f, _int, _vp],
    "gbx_attn_softmax_rows_pair": [_vp, _vp, _vp, _i64, _int, _int, _int, _f, _int, _vp],
    "gbx_attn_scores": [_vp, _vp, _vp, _vp, _i64, _vp, _int, _int, _int, _int, _int, _vp, _vp],
    "gbx_transpose_heads": [_vp, _i64, _vp, _int, _int, _int, _int, _vp],
    "gbx_attn_values": [_vp, _vp, _vp, _vp, _vp, _vp, _i64, _int, _int, _int, _int, _int, _vp, _vp],
    "gbx_attn_fused": [_vp, _vp, _vp, _vp, _i64, _vp, _vp, _vp, _vp, _i64, _int, _int, _int, _int, _f, _int, _vp, _vp],
    "gbx_logits": [_vp, _i64, _vp, _int, _vp, _int, _int, _vp],
    "gbx_select_tokens": [_vp, _i64, _int, ctypes.c_double, _vp, _vp, _vp, _vp, _vp],
    "gbx_split_tf32": [_vp, _vp, _vp, _i64, _vp],
    "gbx_linear_set_tiles": [_int, _int, _vp, _vp],
    "gbx_linear": [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _int, _int, _int, _vp, _vp],
    "gbx_linear_splitk": [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _int, _int, _int, _int, _vp, _i64, _vp, _vp],
    "gbx_linear_splitk_noalloc": [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _int, _int, _int, _int, _vp, _vp],
    "gbx_kv_append": [_vp, _int, _vp, _int, _vp, _vp, _int, _int, _vp, _vp, _vp, _vp, _i64, _vp, _vp],
    "gbx_kv_read": [_vp, _int, _vp, _int, _vp, _vp, _int, _int, _vp, _vp, _i64, _vp, _vp],
    "gbx_kv_copy_pages": [_vp, _vp, _vp, _int, _vp, _vp],
    "gbx_attn_cached": [_vp, _int, _vp, _vp, _i64, _vp, _int, _vp, _vp, _int, _int, _int, _f, _vp, _vp, _i64, _vp, _i64,
                        _vp, _vp],
    "gbx_attn_cached_workspace": [_vp, _int, _int, _int, _int],
    "gbx_verify_tokens": [_vp, _vp, _vp, _vp, _i64, _int, _int, ctypes.c_double, _vp, _vp, _vp, _vp, _vp],
}
_RESTYPES = {"gbx_status_string": ctypes.c_char_p, "gbx_last_error": ctypes.c_char_p,
             "gbx_set_first_wait_limit": ctypes.c_uint64, "gbx_attn_cached_workspace": _i64}

_lib = None


def lib():
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError(f"libgbx.so is not built ({LIB_PATH}); run make -C glassboxai-transformer_b200")
        L = ctypes.CDLL(LIB_PATH)
        for name, args in SIGNATURES.items():
            fn = getattr(L, name)
            fn.argtypes = args
            fn.restype = _RESTYPES.get(name, _int)
        _lib = L
    return _lib


lib()   # fail at import time when the library is missing


def _p(x):
    """Device address of a tensor / int / None."""
    if x is None:
        return None
    if isinstance(x, int):
        return x
    return x.data_ptr()


def _stream(stream):
    if stream is None:
        try:
            import torch
            if torch.cuda.is_available():
                return torch.cuda.current_stream().cuda_stream
        except ImportError:
            pass
        return None
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


def _check(rc: int):
    if rc != 0:
        raise GbxError(rc, lib().gbx_last_error().decode(errors="replace"))


def version() -> int:
    return lib().gbx_version()


def set_pdl(enable: bool) -> bool:
    """Programmatic dependent launch for the row kernels (process-wide);
    returns the previous setting."""
    return bool(lib().gbx_set_pdl(1 if enable else 0))


DEFAULT_WAIT_NS = 1_000_000_000


def set_first_wait_limit(ns: int) -> int:
    """Limit of the first consumer wait of the staged embedding and the
    tensor-core contractions (0: give up at once; for timeout tests).
    Returns the previous limit."""
    return int(lib().gbx_set_first_wait_limit(int(ns)))


def dequant(src, dtype: int, dst, n: int, stream=None):
    _check(lib().gbx_dequant(_p(src), dtype, _p(dst), n, _stream(stream)))


def embed(ids, wte, wte_dtype, wpe, wpe_dtype, out, *, n_tok, d, vocab, n_ctx, seq=None, pos_off=0,
          pos_ids=None, err_flag=None, stream=None):
    seq = n_tok if seq is None else seq
    _check(lib().gbx_embed(_p(ids), _p(wte), wte_dtype, _p(wpe), wpe_dtype, _p(pos_ids), _p(out), n_tok,
                           seq, pos_off, d, vocab, n_ctx, _p(err_flag), _stream(stream)))


def embed_layernorm(ids, wte, wte_dtype, wpe, wpe_dtype, h_out, y, gamma, beta, *, n_tok, d, vocab, n_ctx, seq=None,
                    pos_off=0, pos_ids=None, y_lo=None, eps=1e-5, err_flag=None, stream=None):
    """embed (into h_out, may be None) and the LayerNorm of its rows (into y;
    with y_lo, as a tf32 pair) in one pass."""
    seq = n_tok if seq is None else seq
    _check(lib().gbx_embed_layernorm(_p(ids), _p(wte), wte_dtype, _p(wpe), wpe_dtype, _p(pos_ids), _p(h_out), _p(y),
                                     _p(y_lo), _p(gamma), _p(beta), n_tok, seq, pos_off, d, vocab, n_ctx, eps,
                                     _p(err_flag), _stream(stream)))


def layernorm(x, y, gamma, beta, *, rows, d, eps=1e-5, stream=None):
    _check(lib().gbx_layernorm(_p(x), _p(y), _p(gamma), _p(beta), rows, d, eps, _stream(stream)))


def layernorm_pair(x, y_hi, y_lo, gamma, beta, *, rows, d, eps=1e-5, stream=None):
    """LayerNorm with the output as a tf32 pair (the x operand of linear)."""
    _check(lib().gbx_layernorm_pair(_p(x), _p(y_hi), _p(y_lo), _p(gamma), _p(beta), rows, d, eps, _stream(stream)))


def residual_layernorm(x, r, h_out, y, gamma, beta, *, rows, d, eps=1e-5, xbias=None, stream=None):
    _check(lib().gbx_residual_layernorm(_p(x), _p(r), _p(xbias), _p(h_out), _p(y), _p(gamma), _p(beta),
                                        rows, d, eps, _stream(stream)))


def final_layernorm(x, r, y, gamma, beta, *, n_seq, seq, d, eps=1e-5, stream=None):
    """y[b] = LayerNorm(r[t] + x[t]) for t = b*seq + seq - 1, the last row of
    each of n_seq sequences (x may be None)."""
    _check(lib().gbx_final_layernorm(_p(x), _p(r), _p(y), _p(gamma), _p(beta), n_seq, seq, d, eps, _stream(stream)))


def bias_gelu(x, out, bias, *, rows, F, stream=None):
    _check(lib().gbx_bias_gelu(_p(x), _p(out), _p(bias), rows, F, _stream(stream)))


def softmax_rows(x, out, *, rows, L, stream=None):
    _check(lib().gbx_softmax_rows(_p(x), _p(out), rows, L, _stream(stream)))


def attn_softmax_rows(scores, probs, *, rows, L, S, scale, q_off=0, causal=True, stream=None):
    _check(lib().gbx_attn_softmax_rows(_p(scores), _p(probs), rows, L, S, q_off, scale, 1 if causal else 0,
                                       _stream(stream)))


def logits(h, wte, wte_dtype, out, *, rows, vocab, d, stream=None):
    _check(lib().gbx_logits(_p(h), rows, _p(wte), wte_dtype, _p(out), vocab, d, _stream(stream)))


def select_tokens(logits, out_ids, *, rows, vocab, temperature=0.0, uniforms=None, out_best=None,
                  out_best_logit=None, stream=None):
    _check(lib().gbx_select_tokens(_p(logits), rows, vocab, float(temperature), _p(uniforms), _p(out_ids),
                                   _p(out_best), _p(out_best_logit), _stream(stream)))


ACT_NONE, ACT_GELU = 0, 1
LINEAR_TIMEOUT = 4


def split_tf32(x, hi, lo, *, n, stream=None):
    """hi = tf32(x), lo = tf32(x - hi): the operand pair gbx_linear reads."""
    _check(lib().gbx_split_tf32(_p(x), _p(hi), _p(lo), n, _stream(stream)))


def linear_set_tiles(k_block: int, pair_mode: int):
    """Tile form of the tensor-core contractions (process-wide): k_block 16 or
    32, pair_mode -1 auto / 0 never / 1 always CTA pairs.  Returns the
    previous (k_block, pair_mode)."""
    pk, pp = ctypes.c_int(0), ctypes.c_int(0)
    _check(lib().gbx_linear_set_tiles(k_block, pair_mode, ctypes.byref(pk), ctypes.byref(pp)))
    return pk.value, pp.value


def linear(x_hi, x_lo, w_hi, w_lo, y, *, M, N, K, bias=None, resid=None, y_lo=None, act=ACT_NONE, err_flag=None,
           stream=None):
    """y = act(x . w^T + bias) + resid on the tensor cores (tf32 pairs, see gbx.h)."""
    _check(lib().gbx_linear(_p(x_hi), _p(x_lo), _p(w_hi), _p(w_lo), _p(bias), _p(resid), _p(y), _p(y_lo), M, N, K,
                            act, _p(err_flag), _stream(stream)))


def attn_softmax_rows_pair(scores, probs_hi, probs_lo, *, rows, L, S, scale, q_off=0, causal=True, stream=None):
    """attn_softmax_rows with the probabilities as a tf32 pair (attn_values' P operand)."""
    _check(lib().gbx_attn_softmax_rows_pair(_p(scores), _p(probs_hi), _p(probs_lo), rows, L, S, q_off, scale,
                                            1 if causal else 0, _stream(stream)))


def attn_scores(q_hi, q_lo, k_hi, k_lo, dots, *, ld, B, S, H, hd, causal=True, err_flag=None, stream=None):
    """dots[(b*H+h)*S*S + p*S + s] = q[b, p, head h] . k[b, s, head h] on the tensor cores."""
    _check(lib().gbx_attn_scores(_p(q_hi), _p(q_lo), _p(k_hi), _p(k_lo), ld, _p(dots), B, S, H, hd,
                                 1 if causal else 0, _p(err_flag), _stream(stream)))


def transpose_heads(v, vt, *, ld, B, S, H, hd, stream=None):
    """vt[((b*H+h)*hd + i)*S + s] = v[(b*S + s)*ld + h*hd + i]."""
    _check(lib().gbx_transpose_heads(_p(v), ld, _p(vt), B, S, H, hd, _stream(stream)))


def attn_values(p_hi, p_lo, vt_hi, vt_lo, out, *, ld_out, B, S, H, hd, out_lo=None, causal=True, err_flag=None,
                stream=None):
    """out[(b*S+p)*ld_out + h*hd + i] = sum_s P[b, h, p, s] vt[b, h, i, s] on the tensor cores."""
    _check(lib().gbx_attn_values(_p(p_hi), _p(p_lo), _p(vt_hi), _p(vt_lo), _p(out), _p(out_lo), ld_out, B, S, H, hd,
                                 1 if causal else 0, _p(err_flag), _stream(stream)))


def linear_splitk(x_hi, x_lo, w_hi, w_lo, y, *, M, N, K, ksplit, workspace, workspace_floats=None, bias=None,
                  resid=None, y_lo=None, act=ACT_NONE, err_flag=None, stream=None):
    """linear with K in ksplit slices, partial sums in `workspace` (>= ksplit*M*N floats)."""
    if workspace_floats is None:
        workspace_floats = workspace.numel() if hasattr(workspace, "numel") else 0
    _check(lib().gbx_linear_splitk(_p(x_hi), _p(x_lo), _p(w_hi), _p(w_lo), _p(bias), _p(resid), _p(y), _p(y_lo), M,
                                   N, K, act, ksplit, _p(workspace), workspace_floats, _p(err_flag), _stream(stream)))


NOALLOC_SCRATCH_FLOATS = 1 << 22


def linear_splitk_noalloc(x_hi, x_lo, w_hi, w_lo, y, *, M, N, K, ksplit, bias=None, resid=None, y_lo=None,
                          act=ACT_NONE, err_flag=None, stream=None):
    """linear_splitk with the partial sums in the library's own scratch array
    (ksplit*M*N <= NOALLOC_SCRATCH_FLOATS); allocates nothing."""
    _check(lib().gbx_linear_splitk_noalloc(_p(x_hi), _p(x_lo), _p(w_hi), _p(w_lo), _p(bias), _p(resid), _p(y),
                                           _p(y_lo), M, N, K, act, ksplit, _p(err_flag), _stream(stream)))


def attn_fused(q_hi, q_lo, k_hi, k_lo, v_hi, v_lo, out, *, ld, ld_out, B, S, H, hd, scale, out_lo=None, causal=True,
               err_flag=None, stream=None):
    """Self-attention of every head in one fused launch (tf32 pairs in; see gbx.h)."""
    _check(lib().gbx_attn_fused(_p(q_hi), _p(q_lo), _p(k_hi), _p(k_lo), ld, _p(v_hi), _p(v_lo), _p(out), _p(out_lo),
                                ld_out, B, S, H, hd, scale, 1 if causal else 0, _p(err_flag), _stream(stream)))


class _KVCacheStruct(ctypes.Structure):
    """gbx_kv_cache of gbx.h."""
    _fields_ = [("k", _vp), ("v", _vp), ("k_scale", _vp), ("v_scale", _vp), ("pages", _i64), ("layers", ctypes.c_int32),
                ("page", ctypes.c_int32), ("heads", ctypes.c_int32), ("hd", ctypes.c_int32)]


class _Torch:
    """The few things of torch that a cache call needs, looked up once."""
    int32 = float32 = float64 = device = stream = None

    @classmethod
    def load(cls):
        import torch
        cls.int32, cls.float32, cls.float64 = torch.int32, torch.float32, torch.float64
        cls.device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else lambda: -1
        cls.stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _device_of(t):
    """CUDA device index of a tensor; -1 for an address, -2 for a host tensor."""
    if _Torch.int32 is None:
        _Torch.load()
    d = getattr(t, "device", None)
    if d is None or d.type != "cuda":
        return -1 if d is None else -2
    return _Torch.device() if d.index is None else d.index


def _elsewhere(dev):
    """Whether `dev` is a GPU other than the current one."""
    return dev >= 0 and dev != _Torch.device()


def _stream_on(dev, stream):
    """Handle of the stream to launch on: `stream`, or the device's current torch stream."""
    if dev == -2:
        raise ValueError("the tensors are not on a GPU")
    if stream is None:
        return _Torch.stream(dev) if dev >= 0 else _stream(None)
    return stream if isinstance(stream, int) else stream.cuda_stream


def _there(dev, fn, *args, **kw):
    """fn(...) with GPU `dev` current: a kernel runs where its tensors are."""
    import torch
    with torch.cuda.device(dev):
        return fn(*args, **kw)


class KVCache:
    """Paged 8-bit key/value cache (gbx_kv_cache): ``KVCache(layers=, pages=,
    heads=, page=, hd=)`` allocates its four tensors on `device`;
    ``KVCache(k=, v=, k_scale=, v_scale=)`` wraps tensors of the layout gbx.h
    gives.  The tensors stay reachable as ``.k .v .k_scale .v_scale``."""

    def __init__(self, *, layers=None, pages=None, heads=None, page=None, hd=None, k=None, v=None, k_scale=None,
                 v_scale=None, device="cuda"):
        import torch
        if k is None:
            if page not in (16, 32, 64, 128):
                raise ValueError(f"KVCache: {page} tokens per page (16, 32, 64 or 128)")
            k = torch.empty((layers, pages, heads, page, hd), dtype=torch.int8, device=device)
            v = torch.empty((layers, pages, heads, page // 16, hd, 16), dtype=torch.int8, device=device)
            k_scale = torch.empty((layers, pages, heads), dtype=torch.float32, device=device)
            v_scale = torch.empty((layers, pages, heads), dtype=torch.float32, device=device)
        layers, pages, heads, page, hd = k.shape
        want = {"k": (k, torch.int8, (layers, pages, heads, page, hd)),
                "v": (v, torch.int8, (layers, pages, heads, page // 16, hd, 16)),
                "k_scale": (k_scale, torch.float32, (layers, pages, heads)),
                "v_scale": (v_scale, torch.float32, (layers, pages, heads))}
        for name, (t, dtype, shape) in want.items():
            if t.dtype != dtype or tuple(t.shape) != shape or not t.is_contiguous() or t.device != k.device:
                raise ValueError(f"KVCache: {name} must be a contiguous {dtype} tensor {shape} on {k.device}")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.layers, self.pages, self.heads, self.page, self.hd = layers, pages, heads, page, hd
        self.device = k.device
        self._dev = _device_of(k)
        self._c = _KVCacheStruct(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), pages, layers, page,
                                 heads, hd)
        self._ref = ctypes.byref(self._c)


def _misplaced(name, t, dev, n):
    """Refuses a tensor on another device than the call's, or one that ends before the n-th entry from its start (that
    of its storage counts: it may be a view): the kernel would read an address that is not there."""
    if t.get_device() != dev:
        raise ValueError(f"{name} is on {t.device}, the call runs on cuda:{dev}")
    if t.untyped_storage().nbytes() // t.element_size() - t.storage_offset() < n:
        raise ValueError(f"{name} ends after {t.numel()} entries of {n}")


def _index(name, t, dev=-1, n=0):
    """Address of an index array of n entries: a contiguous int32 tensor (looked at where the call runs on GPU `dev` >=
    0), an address or None."""
    if t is None or t.__class__ is int:
        return t
    if t.dtype is not _Torch.int32 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor")
    if dev >= 0 and (t.numel() < n or t.get_device() != dev):
        _misplaced(name, t, dev, n)
    return t.data_ptr()


def _flag(t, dev):
    """Address of the status word: a tensor of at least its four bytes, an address or None."""
    if t is None or t.__class__ is int:
        return t
    if dev >= 0 and (t.get_device() != dev or t.numel() * t.element_size() < 4):
        _misplaced("err_flag", t, dev, -(-4 // t.element_size()))
    return t.data_ptr()


def _floats(name, t, dev, n, dtype=None, strided=False):
    """Address of an fp32 (or `dtype`) tensor with n entries of storage from its start, an address or None.  strided: it
    may be a view of rows that lie further apart."""
    if t is None or t.__class__ is int:
        return t
    if t.dtype is not (dtype or _Torch.float32):
        raise ValueError(f"{name} must be a {dtype or _Torch.float32} tensor")
    if dev >= 0:
        if t.is_contiguous():
            if t.numel() < n or t.get_device() != dev:
                _misplaced(name, t, dev, n)
        elif strided and (t.stride()[-1] == 1 or t.shape[-1] <= 1):
            if t.get_device() != dev or t.untyped_storage().nbytes() < 4 * (t.storage_offset() + n):
                _misplaced(name, t, dev, n)
        else:
            raise ValueError(f"{name} must be contiguous" + (" in its last dimension" if strided else ""))
    return t.data_ptr()


def kv_append(cache, layer, k, v, table, kv_len, *, B, S, ld, max_pages=None, n_new=None, k_lo=None, v_lo=None,
              err_flag=None, stream=None):
    """Appends row (b, i), i < n_new[b], of k and v (row stride ld) as token
    kv_len[b] - n_new[b] + i of sequence b.  max_pages: the table's row length
    (its last dimension when it is a tensor)."""
    dev = cache._dev
    if dev >= 0 and dev != _Torch.device():
        return _there(dev, kv_append, cache, layer, k, v, table, kv_len, B=B, S=S, ld=ld, max_pages=max_pages, n_new=n_new,
                      k_lo=k_lo, v_lo=v_lo, err_flag=err_flag, stream=stream)
    if max_pages is None:
        max_pages = table.shape[-1]
    at = dev if B > 0 and S > 0 else -1
    n = (B * S - 1) * ld + cache.heads * cache.hd if at >= 0 and n_new is None else 0   # with counts, rows behind a sequence's own need not be there
    rc = _lib.gbx_kv_append(
        cache._ref, layer, _index("table", table, at, B * max_pages), max_pages, _index("kv_len", kv_len, at, B),
        _index("n_new", n_new, at, B), B, S, _floats("k", k, at, n, None, True), _floats("k_lo", k_lo, at, n, None, True),
        _floats("v", v, at, n, None, True), _floats("v_lo", v_lo, at, n, None, True), ld, _flag(err_flag, at),
        _stream_on(dev, stream))
    if rc:
        _check(rc)


def kv_read(cache, layer, table, kv_len, k_out, v_out, *, B, S, ld, max_pages=None, n=None, err_flag=None, stream=None):
    """The fp32 values of each sequence's last n[b] tokens (the mirror of kv_append)."""
    dev = cache._dev
    if dev >= 0 and dev != _Torch.device():
        return _there(dev, kv_read, cache, layer, table, kv_len, k_out, v_out, B=B, S=S, ld=ld, max_pages=max_pages, n=n,
                      err_flag=err_flag, stream=stream)
    if max_pages is None:
        max_pages = table.shape[-1]
    at = dev if B > 0 and S > 0 else -1
    need = (B * S - 1) * ld + cache.heads * cache.hd if at >= 0 and n is None else 0
    rc = _lib.gbx_kv_read(
        cache._ref, layer, _index("table", table, at, B * max_pages), max_pages, _index("kv_len", kv_len, at, B), _index("n", n, at, B),
        B, S, _floats("k_out", k_out, at, need, None, True), _floats("v_out", v_out, at, need, None, True), ld,
        _flag(err_flag, at), _stream_on(dev, stream))
    if rc:
        _check(rc)


def kv_copy_pages(cache, src, dst, *, n, err_flag=None, stream=None):
    """Page dst[i] becomes page src[i], i < n, in every layer."""
    dev = cache._dev
    if dev >= 0 and dev != _Torch.device():
        return _there(dev, kv_copy_pages, cache, src, dst, n=n, err_flag=err_flag, stream=stream)
    rc = _lib.gbx_kv_copy_pages(cache._ref, _index("src", src, dev, n), _index("dst", dst, dev, n), n, _flag(err_flag, dev),
                                _stream_on(dev, stream))
    if rc:
        _check(rc)


def attn_cached_workspace(cache, *, B, S, H, max_pages) -> int:
    """Floats of workspace attn_cached can use for these sizes (0: none)."""
    if _elsewhere(cache._dev):
        return _there(cache._dev, attn_cached_workspace, cache, B=B, S=S, H=H, max_pages=max_pages)
    n = _lib.gbx_attn_cached_workspace(cache._ref, B, S, H, max_pages)
    if n < 0:
        _check(-n)
    return n


def attn_cached(cache, layer, q, out, table, kv_len, *, B, S, H, ld, ld_out, scale, max_pages=None, n_new=None, q_lo=None,
                out_lo=None, workspace=None, workspace_floats=None, err_flag=None, stream=None):
    """Attention of S rows per sequence over the cached tokens (see gbx.h)."""
    dev = cache._dev
    if dev >= 0 and dev != _Torch.device():
        return _there(dev, attn_cached, cache, layer, q, out, table, kv_len, B=B, S=S, H=H, ld=ld, ld_out=ld_out, scale=scale,
                      max_pages=max_pages, n_new=n_new, q_lo=q_lo, out_lo=out_lo, workspace=workspace,
                      workspace_floats=workspace_floats, err_flag=err_flag, stream=stream)
    if workspace_floats is None:
        workspace_floats = workspace.numel() if hasattr(workspace, "numel") else 0
    if max_pages is None:
        max_pages = table.shape[-1]
    at = dev if B > 0 and S > 0 else -1
    rows, width = (B * S - 1, H * cache.hd) if at >= 0 and n_new is None else (0, 0)
    n, n_out = rows * ld + width, rows * ld_out + width
    rc = _lib.gbx_attn_cached(
        cache._ref, layer, _floats("q", q, at, n, None, True), _floats("q_lo", q_lo, at, n, None, True), ld,
        _index("table", table, at, B * max_pages), max_pages, _index("kv_len", kv_len, at, B), _index("n_new", n_new, at, B), B, S, H,
        scale, _floats("out", out, at, n_out, None, True), _floats("out_lo", out_lo, at, n_out, None, True), ld_out,
        _floats("workspace", workspace, at, workspace_floats), workspace_floats, _flag(err_flag, at),
        _stream_on(dev, stream))
    if rc:
        _check(rc)


def verify_tokens(logits, draft_ids, out_ids, n_accepted, *, B, n_draft, vocab, temperature=0.0, uniforms=None,
                  draft_logits=None, draft_len=None, err_flag=None, stream=None):
    """Accepts drafted tokens against the target's logits and picks the next token (see gbx.h)."""
    dev = _device_of(logits)
    if dev >= 0 and dev != _Torch.device():
        return _there(dev, verify_tokens, logits, draft_ids, out_ids, n_accepted, B=B, n_draft=n_draft, vocab=vocab,
                      temperature=temperature, uniforms=uniforms, draft_logits=draft_logits, draft_len=draft_len,
                      err_flag=err_flag, stream=stream)
    at = dev if B > 0 and n_draft >= 0 else -1
    rows = B * (n_draft + 1)
    rc = _lib.gbx_verify_tokens(
        _floats("logits", logits, at, rows * vocab), _floats("draft_logits", draft_logits, at, B * n_draft * vocab),
        _index("draft_ids", draft_ids, at, B * n_draft), _index("draft_len", draft_len, at, B), B, n_draft, vocab, temperature,
        _floats("uniforms", uniforms, at, rows, _Torch.float64), _index("out_ids", out_ids, at, rows), _index("n_accepted", n_accepted, at, B),
        _flag(err_flag, at), _stream_on(dev, stream))
    if rc:
        _check(rc)
