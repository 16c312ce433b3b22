"""The paged 8-bit cache, its attention and draft verification in 64 bits, as
plain loops over numpy arrays: what gbx_kv_append, gbx_kv_read,
gbx_kv_copy_pages, gbx_attn_cached and gbx_verify_tokens are checked against."""
import numpy as np


class Cache:
    """One layer: codes [pages, heads, P, hd] of keys and values, scales [pages, heads]."""

    def __init__(self, pages, heads, P, hd, rng=None):
        self.P, self.heads, self.hd, self.pages = P, heads, hd, pages
        shape = (pages, heads, P, hd)
        if rng is None:
            self.codes = [np.zeros(shape, np.int8) for _ in range(2)]
            self.scale = [np.zeros((pages, heads), np.float32) for _ in range(2)]
        else:
            self.codes = [rng.integers(-127, 128, shape).astype(np.int8) for _ in range(2)]
            self.scale = [((0.5 + rng.random((pages, heads))) / 60).astype(np.float32) for _ in range(2)]

    def copy(self):
        c = Cache(1, 1, self.P, self.hd)
        c.pages, c.heads = self.pages, self.heads
        c.codes = [x.copy() for x in self.codes]
        c.scale = [x.copy() for x in self.scale]
        return c

    # device layouts
    def k_dev(self):
        return self.codes[0][None]

    def v_dev(self):
        p, h, P, hd = self.codes[1].shape
        return np.ascontiguousarray(self.codes[1].reshape(p, h, P // 16, 16, hd).transpose(0, 1, 2, 4, 3))[None]

    def append(self, table, kv_len, n_new, k, v, skip=()):
        """k, v: [B, S, heads, hd] fp32; sequences in `skip` are left out."""
        for b in range(len(kv_len)):
            if b in skip:
                continue
            first = int(kv_len[b]) - int(n_new[b])
            i = 0
            while i < n_new[b]:
                t = first + i
                page, slot = int(table[b][t // self.P]), t % self.P
                n = min(self.P - slot, int(n_new[b]) - i)
                if 0 <= page < self.pages:
                    for w, x in enumerate((k, v)):
                        for h in range(self.heads):
                            self._block(w, page, h, slot, x[b, i:i + n, h])
                i += n

    def _block(self, w, page, h, slot, x):
        codes, scale = self.codes[w], self.scale[w]
        with np.errstate(all="ignore"):
            if not np.all(np.isfinite(x)):
                s = np.float32(np.nan)
            else:
                a = np.abs(x).max()
                s = np.float32(np.float64(a) / 127) if a >= 2.0 ** -100 else np.float32(0)
            if slot:
                old = scale[page, h]
                s = np.float32(np.nan) if np.isnan(old) or np.isnan(s) else max(old, s)
                if not s == old:
                    was = codes[page, h, :slot].astype(np.float64)
                    codes[page, h, :slot] = np.rint(was * np.float64(old) / np.float64(s)) if s > 0 else 0
            scale[page, h] = s
            codes[page, h, slot:slot + len(x)] = np.rint(x.astype(np.float64) / np.float64(s)) if s > 0 else 0

    def values(self, w, table, b, t):
        """[heads, hd] fp32 of token t of sequence b, or None on a page outside the pool."""
        page = int(table[b][t // self.P])
        if not 0 <= page < self.pages:
            return None
        return self.codes[w][page, :, t % self.P].astype(np.float32) * self.scale[w][page][:, None]


def attend(cache, table, kv_len, n_new, q, scale, skip=()):
    """out [B, S, H, hd] in fp64, NaN-filled where no row is computed, and the
    bound on an fp32-grade kernel's error at each entry.

    A query enters as 24-bit fixed point: every entry is off by at most qmax 2^-23
    (half a unit of qmax / 8355704, and the rounding of the product that scales
    it), so with B_t = qmax sum_i |k_ti| / scale and A_t = sum_i |q_i k_ti| /
    scale the score x_t (in units of log 2) is off by B 2^-23, plus the fp32
    joining of three exact sums and its scaling by three factors (8 roundings
    of at most 2^-24 of A, doubled), plus the rounding of x - max + 23; the
    weight's exponential adds 2^-22.  A weight is fixed point too, off by half
    of 2^-23 of its 64-token step's largest (in terms of the step's largest
    value), and the running sums add (L/4 + 40) 2^-23 of sum w |v|.  An error
    of d in every score moves the output by at most 2 d sum w |v|."""
    B, S, H, hd = q.shape
    G = H // cache.heads
    out = np.full((B, S, H, hd), np.nan)
    tol = np.zeros((B, S, H, hd))
    for b in range(B):
        if b in skip:
            continue
        n, L = int(n_new[b]), int(kv_len[b])
        got = [t for t in range(L) if cache.values(0, table, b, t) is not None]
        if got:
            K = np.stack([cache.codes[0][int(table[b][t // cache.P]), :, t % cache.P].astype(np.float64) *
                          cache.scale[0][int(table[b][t // cache.P])].astype(np.float64)[:, None] for t in got])
            V = np.stack([cache.codes[1][int(table[b][t // cache.P]), :, t % cache.P].astype(np.float64) *
                          cache.scale[1][int(table[b][t // cache.P])].astype(np.float64)[:, None] for t in got])
        pos = np.array(got)
        for i in range(n):
            see = pos <= L - n + i if got else np.zeros(0, bool)
            for h in range(H):
                if not see.any():
                    out[b, i, h] = 0.0
                    continue
                k, v = K[see, h // G], V[see, h // G]
                qq = q[b, i, h].astype(np.float64)
                with np.errstate(all="ignore"):
                    x = k @ qq / scale
                    A = np.abs(k) @ np.abs(qq) / scale
                    w = np.exp(x - x.max())
                    w /= w.sum()
                    out[b, i, h] = w @ v
                    x2, A2 = np.abs(x) * 1.4427, A * 1.4427
                    B2 = np.abs(k).sum(1) * np.abs(qq).max() / scale * 1.4427
                    d = (B2 * 2.0 ** -23 + A2 * 2.0 ** -20 + 6 * 2.0 ** -24 * (x2 + x2.max() + 23)).max() * 0.6932 + 2.0 ** -22
                    step = pos[see] // 64
                    top = np.zeros(step.max() + 1)
                    np.maximum.at(top, step, w)
                    fixed = top[step].sum() * np.abs(v).max() * 2.0 ** -24
                    tol[b, i, h] = (2 * d + 2.0 ** -21 + (40 + L / 4) * 2.0 ** -23) * (w @ np.abs(v)) + fixed
    return out, tol


def verify(logits, draft_logits, ids, lens, T, u):
    """(out_ids, accepted) as gbx_verify_tokens defines them, in fp64.
    logits [B, n + 1, V], draft_logits [B, n, V] or None."""
    B, n1, V = logits.shape
    n = n1 - 1
    out, acc = np.full((B, n1), -1, np.int64), np.zeros(B, np.int64)

    def dist(row):
        row = row.astype(np.float64)
        if np.isnan(row).any() or row.max() in (np.inf, -np.inf):
            return None
        e = np.exp((row - row.max()) / T) if T > 0.01 else row
        return e / e.sum() if T > 0.01 else e

    for b in range(B):
        if not 0 <= lens[b] <= n:
            continue
        i, nxt, q = 0, None, None
        while i < lens[b]:
            p = dist(logits[b, i])
            d = int(ids[b, i])
            if p is None:
                break
            if T <= 0.01:
                if int(np.argmax(p)) != d:
                    break
            else:
                if draft_logits is None:
                    q = np.zeros(V)
                    if 0 <= d < V:
                        q[d] = 1.0
                else:
                    q = dist(draft_logits[b, i])
                    if q is None:
                        break
                if not 0 <= d < V or not u[b, i] * q[d] < p[d]:
                    break
            i += 1
        acc[b] = i
        out[b, :i] = ids[b, :i]
        p = dist(logits[b, i])
        if p is None or (i < lens[b] and T > 0.01 and draft_logits is not None and dist(draft_logits[b, i]) is None):
            continue
        if T <= 0.01:
            nxt = int(np.argmax(p))
        else:
            r = np.maximum(p - q, 0) if i < lens[b] else p
            if not r.sum() > 0:
                r = p
            c = np.cumsum(r)
            over = np.flatnonzero(c > u[b, n] * c[-1])
            nxt = int(over[0]) if over.size else int(np.flatnonzero(r > 0)[-1])
        out[b, i] = nxt
    return out, acc
