"""Python binding of the model C ABI (``include/gbx_model.h``,
``libgbx_model.so``): the GGUFLoader and TransformerModel of
``include/gbx_model.hpp``.

``GGUF`` mirrors the reference's GGUFLoader (transformer.cu:480-740):
``get_tensor`` is getTensor (host fp32 values, the reference's decode),
``has_tensor`` is hasTensor, ``config`` the getters, ``tensor_gpu`` is
getTensorGPU and ``tensor_gpu_raw`` gives the tensor's GGUF bytes on the
device.  ``Model`` mirrors TransformerModel (transformer.cu:744-1051):
``forward(ids)`` returns the last token's logits; ``forward(ids, batch=B)``
runs B equal-length sequences and returns [B, vocab].  ``Session`` (no
counterpart in the reference) generates over a paged 8-bit key/value cache.

There is no fallback: importing fails loudly when the library is missing.
"""
from __future__ import annotations

import ctypes
import importlib
import os

import numpy as np

_gbx = importlib.import_module(__package__)
LIB_PATH = os.path.join(_gbx.HERE, "libgbx_model.so")
HEADER = os.path.join(os.path.dirname(_gbx.HERE), "include", "gbx_model.h")

_vp = ctypes.c_void_p
_i64 = ctypes.c_int64
_int = ctypes.c_int
_cp = ctypes.c_char_p

SIGNATURES = {
    "gbx_gguf_open": ([_cp], _vp),
    "gbx_gguf_close": ([_vp], None),
    "gbx_gguf_get_tensor": ([_vp, _cp, _vp, _i64], _i64),
    "gbx_gguf_has_tensor": ([_vp, _cp], _int),
    "gbx_gguf_config": ([_vp, _vp], _int),
    "gbx_gguf_tensor_gpu": ([_vp, _cp], _vp),
    "gbx_gguf_tensor_gpu_raw": ([_vp, _cp, _vp, _vp], _vp),
    "gbx_model_open": ([_cp], _vp),
    "gbx_model_close": ([_vp], None),
    "gbx_model_config": ([_vp, _vp], _int),
    "gbx_model_forward": ([_vp, _vp, _i64, _int, _vp], _int),
    "gbx_model_forward_hidden": ([_vp, _vp, _i64, _int, _vp, _i64], _int),
    "gbx_model_set_fused_attention": ([_vp, _int], _int),
    "gbx_model_next_token": ([_vp, _vp, _i64, ctypes.c_double, ctypes.c_double, _vp, _vp, _vp], _int),
    "gbx_session_open": ([_vp, _i64, _int], _vp),
    "gbx_session_close": ([_vp], None),
    "gbx_session_new": ([_vp], _int),
    "gbx_session_fork": ([_vp, _int], _int),
    "gbx_session_truncate": ([_vp, _int, _i64], _int),
    "gbx_session_release": ([_vp, _int], _int),
    "gbx_session_compact": ([_vp], _i64),
    "gbx_session_length": ([_vp, _int], _i64),
    "gbx_session_free_pages": ([_vp], _i64),
    "gbx_session_forward": ([_vp, _vp, _int, _vp, _i64, _vp, _int, _vp], _int),
    "gbx_session_next_tokens": ([_vp, _vp, _int, _vp, _i64, _vp, ctypes.c_double, _vp, _vp], _int),
    "gbx_session_verify": ([_vp, _vp, _int, _vp, _int, _vp, _vp, ctypes.c_double, _vp, _vp, _vp], _int),
    "gbx_sharded_open": ([_cp, _vp, _int], _vp),
    "gbx_sharded_close": ([_vp], None),
    "gbx_sharded_forward": ([_vp, _vp, _i64, _int, _vp], _int),
}

_lib = None


def lib():
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError(f"libgbx_model.so is not built ({LIB_PATH}); run make -C glassboxai-transformer_b200")
        _gbx.lib()   # the kernel library first (libgbx_model.so links it)
        L = ctypes.CDLL(LIB_PATH)
        for name, (args, res) in SIGNATURES.items():
            fn = getattr(L, name)
            fn.argtypes = args
            fn.restype = res
        _lib = L
    return _lib


lib()


def _err(status=None):
    msg = _gbx.lib().gbx_last_error().decode(errors="replace")
    return _gbx.GbxError(status if status is not None else 5, msg)


def _np_ptr(a):
    return a.ctypes.data_as(_vp)


class GGUF:
    """GGUFLoader over a GGUF file (host-side parse; no GPU needed except for
    the tensor_gpu* calls)."""

    def __init__(self, path: str):
        self.h = lib().gbx_gguf_open(path.encode())
        if not self.h:
            raise _err()

    def close(self):
        if self.h:
            lib().gbx_gguf_close(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def has_tensor(self, name: str) -> bool:
        return bool(lib().gbx_gguf_has_tensor(self.h, name.encode()))

    def get_tensor(self, name: str, cap: int) -> np.ndarray:
        out = np.empty(max(cap, 1), dtype=np.float32)
        n = lib().gbx_gguf_get_tensor(self.h, name.encode(), _np_ptr(out), cap)
        if n < 0:
            raise _err()
        return out[:n].copy()

    def config(self) -> dict:
        out = np.zeros(6, dtype=np.int32)
        if lib().gbx_gguf_config(self.h, _np_ptr(out)) != 0:
            raise _err()
        return dict(zip(("embed_dim", "num_layers", "num_heads", "ffn_dim", "vocab_size", "max_seq_len"),
                        out.tolist()))

    def tensor_gpu(self, name: str) -> int:
        p = lib().gbx_gguf_tensor_gpu(self.h, name.encode())
        if not p:
            raise _err(6)
        return p

    def tensor_gpu_raw(self, name: str):
        dt = ctypes.c_int(0)
        n = ctypes.c_int64(0)
        p = lib().gbx_gguf_tensor_gpu_raw(self.h, name.encode(), ctypes.byref(dt), ctypes.byref(n))
        if not p:
            raise _err(6)
        return p, dt.value, n.value


class Model:
    """TransformerModel on the current CUDA device."""

    def __init__(self, path: str):
        self.h = lib().gbx_model_open(path.encode())
        if not self.h:
            raise _err()
        out = np.zeros(6, dtype=np.int32)
        lib().gbx_model_config(self.h, _np_ptr(out))
        self.config = dict(zip(("embed_dim", "num_layers", "num_heads", "ffn_dim", "vocab", "n_ctx"),
                               out.tolist()))

    def close(self):
        if self.h:
            lib().gbx_model_close(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def forward(self, ids, batch: int = 1) -> np.ndarray:
        ids = np.ascontiguousarray(ids, dtype=np.int32).ravel()
        out = np.empty((batch, self.config["vocab"]), dtype=np.float32)
        rc = lib().gbx_model_forward(self.h, _np_ptr(ids), ids.size, batch, _np_ptr(out))
        if rc != 0:
            raise _err(rc)
        return out[0] if batch == 1 else out

    def forward_hidden(self, ids, batch: int = 1) -> np.ndarray:
        """The residual stream after the embedding and after each layer:
        [layers + 1, tokens, embed_dim]."""
        ids = np.ascontiguousarray(ids, dtype=np.int32).ravel()
        out = np.empty((self.config["num_layers"] + 1, ids.size, self.config["embed_dim"]), dtype=np.float32)
        rc = lib().gbx_model_forward_hidden(self.h, _np_ptr(ids), ids.size, batch, _np_ptr(out), out.size)
        if rc != 0:
            raise _err(rc)
        return out

    def set_fused_attention(self, on: bool) -> bool:
        """Fused attention (default) or the per-head products; returns the previous setting."""
        rc = lib().gbx_model_set_fused_attention(self.h, 1 if on else 0)
        if rc < 0 or rc > 1:
            raise _err(rc)
        return bool(rc)

    def next_token(self, ids, temperature=0.0, u=0.0):
        """(selected, best, best_logit) of one generate step with draw u."""
        ids = np.ascontiguousarray(ids, dtype=np.int32).ravel()
        sel, best, bl = ctypes.c_int32(0), ctypes.c_int32(0), ctypes.c_float(0)
        rc = lib().gbx_model_next_token(self.h, _np_ptr(ids), ids.size, float(temperature), float(u),
                                        ctypes.byref(sel), ctypes.byref(best), ctypes.byref(bl))
        if rc != 0:
            raise _err(rc)
        return sel.value, best.value, bl.value


class ShardedModel:
    """ShardedModel: a TransformerModel replica per listed device, one host
    thread per device, batches split into whole-sequence shards and the
    logits gathered on the host."""

    def __init__(self, path: str, devices, vocab: int):
        dev = np.ascontiguousarray(devices, dtype=np.int32)
        self.vocab = vocab
        self.h = lib().gbx_sharded_open(path.encode(), _np_ptr(dev), dev.size)
        if not self.h:
            raise _err()

    def close(self):
        if self.h:
            lib().gbx_sharded_close(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def forward(self, ids, batch: int) -> np.ndarray:
        ids = np.ascontiguousarray(ids, dtype=np.int32).ravel()
        out = np.empty((batch, self.vocab), dtype=np.float32)
        rc = lib().gbx_sharded_forward(self.h, _np_ptr(ids), ids.size, batch, _np_ptr(out))
        if rc != 0:
            raise _err(rc)
        return out


class Session:
    """Cached generation over a Model (gbx::Session): sequences in a paged 8-bit
    key/value cache of `pages` pages of `page_size` tokens; a step costs its
    new tokens only."""

    def __init__(self, model: Model, pages: int, page_size: int = 64):
        self.model = model   # outlives the session
        self.vocab = model.config["vocab"]
        self.h = lib().gbx_session_open(model.h, pages, page_size)
        if not self.h:
            raise _err()

    def close(self):
        if self.h:
            lib().gbx_session_close(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _open(self):
        if not self.h or not self.model.h:
            raise _gbx.GbxError(1, "the session or its model is closed")
        return self.h

    def new(self) -> int:
        """An empty sequence."""
        seq = lib().gbx_session_new(self._open())
        if seq < 0:
            raise _err(1)
        return seq

    def fork(self, seq: int) -> int:
        """A sequence that continues from where `seq` stands (its pages are shared until written to)."""
        new = lib().gbx_session_fork(self._open(), seq)
        if new < 0:
            raise _err(1)
        return new

    def truncate(self, seq: int, length: int):
        rc = lib().gbx_session_truncate(self._open(), seq, length)
        if rc:
            raise _err(rc)

    def release(self, seq: int):
        rc = lib().gbx_session_release(self._open(), seq)
        if rc:
            raise _err(rc)

    def compact(self) -> int:
        """Moves the pages in use to the lowest places; how many moved."""
        n = lib().gbx_session_compact(self._open())
        if n < 0:
            raise _err(4)
        return n

    def length(self, seq: int) -> int:
        return lib().gbx_session_length(self._open(), seq)

    def free_pages(self) -> int:
        return lib().gbx_session_free_pages(self._open())

    @staticmethod
    def _rows(seqs, tokens):
        """seqs, ids (one sequence after another) and counts as int32 arrays."""
        seqs = np.ascontiguousarray(seqs, dtype=np.int32).ravel()
        rows = [np.ascontiguousarray(t, dtype=np.int32).ravel() for t in tokens]
        if len(rows) != seqs.size:
            raise ValueError(f"{len(rows)} token lists for {seqs.size} sequences")
        counts = np.array([r.size for r in rows], dtype=np.int32)
        return seqs, np.ascontiguousarray(np.concatenate(rows)) if rows else np.zeros(0, np.int32), counts

    def forward(self, seqs, tokens, all_rows: bool = False) -> np.ndarray:
        """Appends tokens[i] (ids) to sequence seqs[i]; logits [n, vocab] of each
        sequence's last token, or of every token in order."""
        seqs, ids, counts = self._rows(seqs, tokens)
        out = np.empty((ids.size if all_rows else seqs.size, self.vocab), dtype=np.float32)
        rc = lib().gbx_session_forward(self._open(), _np_ptr(seqs), seqs.size, _np_ptr(ids), ids.size, _np_ptr(counts),
                                       1 if all_rows else 0, _np_ptr(out))
        if rc != 0:
            raise _err(rc)
        return out

    def next_tokens(self, seqs, tokens, temperature=0.0, u=None) -> np.ndarray:
        """forward, and each sequence's next token (the reference's rule; u: a draw in [0, 1) each)."""
        seqs, ids, counts = self._rows(seqs, tokens)
        out = np.empty(seqs.size, dtype=np.int32)
        u = None if u is None else np.ascontiguousarray(u, dtype=np.float64).ravel()
        if u is not None and u.size != seqs.size:
            raise ValueError("a draw for each sequence")
        rc = lib().gbx_session_next_tokens(self._open(), _np_ptr(seqs), seqs.size, _np_ptr(ids), ids.size, _np_ptr(counts),
                                           float(temperature), None if u is None else _np_ptr(u), _np_ptr(out))
        if rc != 0:
            raise _err(rc)
        return out

    def verify(self, seqs, tokens, temperature=0.0, u=None, draft_logits=None, draft_len=None):
        """One speculative step.  tokens [n, k + 1]: each sequence's pending token
        and k drafts; returns (ids [n, k + 1]: the accepted drafts, the next
        token, -1s; accepted [n])."""
        seqs = np.ascontiguousarray(seqs, dtype=np.int32).ravel()
        tokens = np.ascontiguousarray(tokens, dtype=np.int32)
        if tokens.ndim != 2 or tokens.shape[0] != seqs.size or tokens.shape[1] < 1:
            raise ValueError("tokens must be [sequences, drafts + 1]")
        k = tokens.shape[1] - 1
        u = None if u is None else np.ascontiguousarray(u, dtype=np.float64)
        if u is not None and u.shape != tokens.shape:
            raise ValueError("u must have the shape of tokens")
        if draft_logits is not None:
            draft_logits = np.ascontiguousarray(draft_logits, dtype=np.float32)
            if draft_logits.shape != (seqs.size, k, self.vocab):
                raise ValueError("draft_logits must be [sequences, drafts, vocab]")
        if draft_len is not None:
            draft_len = np.ascontiguousarray(draft_len, dtype=np.int32).ravel()
            if draft_len.size != seqs.size:
                raise ValueError("a draft count for each sequence")
        out = np.empty(tokens.shape, dtype=np.int32)
        acc = np.empty(seqs.size, dtype=np.int32)
        rc = lib().gbx_session_verify(self._open(), _np_ptr(seqs), seqs.size, _np_ptr(tokens), k,
                                      None if draft_len is None else _np_ptr(draft_len),
                                      None if draft_logits is None else _np_ptr(draft_logits), float(temperature),
                                      None if u is None else _np_ptr(u), _np_ptr(out), _np_ptr(acc))
        if rc != 0:
            raise _err(rc)
        return out, acc
