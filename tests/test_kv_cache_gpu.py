"""The paged 8-bit cache on the GPU: appending, reading back, attending and
copying pages against the 64-bit oracle (kv_oracle.py).  Codes and scales are
compared bit for bit; attention within the oracle's derived bound."""
import numpy as np
import pytest

import kv_oracle

pytestmark = pytest.mark.gpu


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def i32(a):
    return dev(np.asarray(a, np.int32))


class Setup:
    """A cache with B sequences of random tables over it, on both sides."""

    def __init__(self, gbx, P, heads, hd, B, tokens, seed, layers=1, layer=0, spare=3):
        import torch
        self.gbx, self.P, self.heads, self.hd, self.B, self.layer = gbx, P, heads, hd, B, layer
        self.rng = np.random.default_rng(seed)
        self.m = -(-tokens // P)
        pages = B * self.m + spare
        self.ref = kv_oracle.Cache(pages, heads, P, hd, self.rng)
        self.table = self.rng.permutation(pages)[:B * self.m].reshape(B, self.m)
        self.cache = gbx.KVCache(layers=layers, pages=pages, heads=heads, page=P, hd=hd)
        for t in (self.cache.k, self.cache.v):
            t.fill_(77)
        for t in (self.cache.k_scale, self.cache.v_scale):
            t.fill_(float("nan"))      # other layers: never to be read
        self.upload()
        self.err = torch.zeros(1, dtype=torch.int32, device="cuda")

    def upload(self):
        l = self.layer
        self.cache.k[l], self.cache.v[l] = dev(self.ref.k_dev())[0], dev(self.ref.v_dev())[0]
        self.cache.k_scale[l], self.cache.v_scale[l] = dev(self.ref.scale[0]), dev(self.ref.scale[1])

    def check(self, what=""):
        import torch
        torch.cuda.synchronize()
        l = self.layer
        for w, (codes, scale) in enumerate(((self.cache.k, self.cache.k_scale), (self.cache.v, self.cache.v_scale))):
            want = (self.ref.k_dev, self.ref.v_dev)[w]()[0]
            got = codes[l].cpu().numpy()
            assert np.array_equal(got, want), f"{what}: {'KV'[w]} codes differ at {np.argwhere(got != want)[:5].tolist()}"
            gs = scale[l].cpu().numpy()
            assert np.array_equal(gs, self.ref.scale[w], equal_nan=True), f"{what}: {'KV'[w]} scales"

    def append(self, kv_len, n_new, k, v, S, skip=(), **kw):
        """k, v: [B, S, heads, hd]."""
        d = self.heads * self.hd
        self.ref.append(self.table, kv_len, n_new, k, v, skip)
        self.gbx.kv_append(self.cache, self.layer, dev(k.reshape(-1, d)), dev(v.reshape(-1, d)), i32(self.table), i32(kv_len),
                           B=self.B, S=S, ld=d, n_new=i32(n_new), err_flag=self.err, **kw)


def tokens(rng, *shape):
    """Keys or values whose size varies over the tokens."""
    x = rng.standard_normal(shape) * np.exp(rng.standard_normal(shape[:-1]))[..., None]
    return x.astype(np.float32)


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("P,heads,hd,B,S", [
    (16, 2, 64, 3, 1), (16, 3, 16, 2, 7), (32, 1, 128, 2, 33), (64, 2, 80, 2, 150), (128, 2, 32, 2, 300), (16, 25, 64, 1, 40),
    (32, 2, 48, 5, 3), (128, 1, 112, 1, 129), (64, 12, 64, 2, 64)])
def test_append_matches_the_oracle(gbx, cuda, P, heads, hd, B, S):
    s = Setup(gbx, P, heads, hd, B, S + 2 * P + 5, seed=S * hd, layers=2, layer=1)
    rng = s.rng
    n_new = rng.integers(0, S + 1, B)
    n_new[0] = S
    before = rng.integers(0, 2 * P, B)
    s.append(before + n_new, n_new, tokens(rng, B, S, heads, hd), tokens(rng, B, S, heads, hd), S)
    s.check()
    assert int(s.err.item()) == 0
    # full prompts from the first slot
    s.append([S] * B, [S] * B, tokens(rng, B, S, heads, hd), tokens(rng, B, S, heads, hd), S)
    s.check("prompt")


@pytest.mark.parametrize("P,hd", [(16, 64), (64, 96)])
def test_append_token_by_token_and_roll_back(gbx, cuda, P, hd):
    """Scales grow as larger tokens come; rejected tokens are overwritten."""
    s = Setup(gbx, P, 2, hd, 2, 3 * P, seed=5)
    length = np.array([0, P - 2])
    for step in range(P + 6):
        n = np.array([step % 3, 1])
        length = length + n
        s.append(length, n, tokens(s.rng, 2, 3, 2, hd), tokens(s.rng, 2, 3, 2, hd), 3)
        s.check(f"step {step}")
        if step % 4 == 3:
            length = length - np.minimum(length, [2, 1])


def test_append_of_a_pair_with_strides_and_without_alignment(gbx, cuda):
    import torch
    P, heads, hd, B, S = 16, 3, 64, 2, 5
    for off, ld in ((0, 3 * heads * hd + 4), (1, 3 * heads * hd + 5), (2, 3 * heads * hd)):
        s = Setup(gbx, P, heads, hd, B, 40, seed=off)
        d = heads * hd
        hi = torch.randn(B * S * ld + 8, device="cuda")
        lo = torch.randn(B * S * ld + 8, device="cuda") * 2.0 ** -12
        n_new, kv_len = [5, 2], [19, 2]
        full = (hi + lo)[off:off + B * S * ld].view(B, S, ld).cpu().numpy()
        k, v = full[..., :d].reshape(B, S, heads, hd), full[..., d:2 * d].reshape(B, S, heads, hd)
        s.ref.append(s.table, kv_len, n_new, k, v)
        gbx.kv_append(s.cache, 0, hi[off:], hi[off + d:], i32(s.table), i32(kv_len), B=B, S=S, ld=ld, n_new=i32(n_new),
                      k_lo=lo[off:], v_lo=lo[off + d:])
        s.check(f"offset {off}")


def test_append_special_values(gbx, cuda):
    """Zero, tiny, huge and non-finite blocks; a scale of 0 or NaN that meets new tokens; ties."""
    P, heads, hd, B = 16, 1, 16, 9
    s = Setup(gbx, P, heads, hd, B, P, seed=3)
    x = np.zeros((B, 2, heads, hd), np.float32)
    x[1] = 2.0 ** -101
    x[2] = np.float32(2.0 ** -100)
    x[3, 0] = 3e38
    x[4, 1, 0, 3] = np.nan
    x[5, 0, 0, 0] = -np.inf
    x[6] = -1.0
    x[7, 0, 0] = 127.0
    x[7, 1, 0] = np.arange(16) + 0.5      # ties at a scale of 1
    x[8] = np.float32(1e-45)
    y = tokens(s.rng, B, 2, heads, hd)
    s.append([2] * B, [2] * B, x, y, 2)
    s.check("start")
    assert np.isnan(s.ref.scale[0][s.table[4, 0], 0]) and s.ref.scale[0][s.table[1, 0], 0] == 0
    assert s.ref.codes[0][s.table[7, 0], 0, 1].tolist() == [0, 2, 2, 4, 4, 6, 6, 8, 8, 10, 10, 12, 12, 14, 14, 16]
    s.append([4] * B, [2] * B, y, x, 2)
    s.check("next tokens")
    s.append([2] * B, [2] * B, y, y, 2)   # started anew: the NaN is gone
    s.check("anew")
    assert np.isfinite(s.ref.scale[0][s.table[:, 0]]).all()


def test_append_flags_bad_pages_and_lengths(gbx, cuda):
    P, heads, hd, B, S = 16, 2, 32, 6, 4
    s = Setup(gbx, P, heads, hd, B, 3 * P, seed=9)
    kv_len, n_new = np.array([18, 4, 4, 49, 3, 10]), np.array([4, 5, -1, 4, 4, 4])
    x = tokens(s.rng, B, S, heads, hd)
    s.table[0, 1] = s.ref.pages            # tokens 16, 17 of sequence 0 are lost, 14 and 15 are not
    s.append(kv_len, n_new, x, x, S, skip=(1, 2, 3, 4))
    s.check()
    assert int(s.err.item()) == gbx.KV_BAD_PAGE | gbx.KV_BAD_LEN
    s.err.zero_()
    s.table[0, 1] = -1
    s.append([18, 0, 0, 0, 0, 0], [4, 0, 0, 0, 0, 0], x, x, S)
    s.check()
    assert int(s.err.item()) == gbx.KV_BAD_PAGE


# ------------------------------------------------------------------ read
@pytest.mark.parametrize("P,hd,off", [(16, 64, 0), (32, 80, 0), (128, 16, 1)])
def test_read_returns_the_values_and_leaves_the_rest(gbx, cuda, P, hd, off):
    import torch
    heads, B, S = 3, 4, 21
    s = Setup(gbx, P, heads, hd, B, 60, seed=P)
    s.table[3, 0] = s.ref.pages + 7
    kv_len, n = np.array([60, 21, 0, 8]), np.array([21, 5, 0, 8])
    ld = heads * hd + (5 if off else 4)
    ko = torch.full((B * S * ld + 4,), 7.0, device="cuda")
    vo = torch.full((B * S * ld + 4,), 7.0, device="cuda")
    gbx.kv_read(s.cache, 0, i32(s.table), i32(kv_len), ko[off:], vo[off:], B=B, S=S, ld=ld, n=i32(n), err_flag=s.err)
    for w, got in enumerate((ko, vo)):
        want = np.full(B * S * ld + 4, 7.0, np.float32)
        rows = want[off:off + B * S * ld].reshape(B, S, ld)
        for b in range(B):
            for i in range(n[b]):
                x = s.ref.values(w, s.table, b, int(kv_len[b] - n[b] + i))
                if x is not None:
                    rows[b, i, :heads * hd] = x.ravel()
        assert np.array_equal(got.cpu().numpy(), want)
    assert int(s.err.item()) == gbx.KV_BAD_PAGE
    alone = torch.full_like(vo, 7.0)
    gbx.kv_read(s.cache, 0, i32(s.table), i32(kv_len), None, alone[off:], B=B, S=S, ld=ld, n=i32(n))
    assert torch.equal(alone, vo)


# ------------------------------------------------------------------ attention
def run_attn(s, q, kv_len, n_new, scale, pair=False, workspace="auto", fill=None, ld_extra=0, off=0):
    """(out, out_lo) as numpy [B, S, H, hd] from q [B, S, H, hd]."""
    import torch
    gbx = s.gbx
    B, S, H, hd = q.shape
    ld = H * hd + ld_extra
    buf = np.zeros((B * S, ld), np.float32)
    buf[:, :H * hd] = q.reshape(B * S, -1)
    qd = torch.zeros(buf.size + off, device="cuda")
    qd[off:] = dev(buf).view(-1)
    qh, ql = qd, None
    if pair:
        qh, ql = torch.empty_like(qd), torch.empty_like(qd)
        gbx.split_tf32(qd, qh, ql, n=qd.numel())
    out = torch.full((B * S * ld + off,), float("nan") if fill is None else fill, device="cuda")
    lo = torch.full_like(out, 5.0) if pair else None
    ws = None
    if workspace == "auto":
        n = gbx.attn_cached_workspace(s.cache, B=B, S=S, H=H, max_pages=s.table.shape[1])
        ws = torch.full((max(n, 1),), float("nan"), device="cuda")
    gbx.attn_cached(s.cache, s.layer, qh[off:], out[off:], i32(s.table), i32(kv_len), B=B, S=S, H=H, ld=ld, ld_out=ld, scale=scale,
                    n_new=i32(n_new), q_lo=ql[off:] if pair else None, out_lo=lo[off:] if pair else None, workspace=ws, err_flag=s.err)
    torch.cuda.synchronize()
    cut = lambda t: t[off:].cpu().numpy().reshape(B * S, ld)[:, :H * hd].reshape(q.shape)  # noqa: E731
    if ld_extra:
        rest = out[off:].view(B * S, ld)[:, H * hd:]
        assert bool(torch.isnan(rest).all()) if fill is None else bool((rest == fill).all())
    return cut(out), cut(lo) if pair else None


def assert_attn(got, want, tol, live):
    assert np.isfinite(got[live]).all()
    err = np.abs(got[live].astype(np.float64) - want[live])
    worst = np.max(err / np.maximum(tol[live], 1e-30)) if err.size else 0
    assert np.all(err <= tol[live] + 1e-30), f"worst error {worst:.3g} of its bound"


ATTN = [  # P, heads, G, hd, S, lengths before the call's rows
    (16, 2, 1, 64, 1, [0, 1, 15, 16, 63, 64, 65, 500]),
    (16, 12, 1, 64, 1, [1022]),
    (64, 3, 1, 64, 1, [127, 700, 0]),
    (32, 1, 4, 128, 1, [333, 31]),
    (128, 2, 8, 64, 1, [260, 100]),
    (16, 2, 1, 64, 5, [0, 12, 60, 123]),
    (16, 1, 3, 80, 4, [77, 5]),
    (32, 2, 2, 96, 9, [40, 0]),
    (64, 2, 1, 16, 3, [200, 1]),
    (16, 1, 5, 112, 1, [90]),
    (64, 1, 1, 64, 70, [130, 0, 3]),
    (32, 1, 2, 48, 37, [64]),
    (128, 1, 16, 128, 2, [300]),
    (16, 1, 1, 64, 1, [5000]),
    (128, 1, 2, 128, 1, [9000, 17]),
]


@pytest.mark.parametrize("P,heads,G,hd,S,before", ATTN)
@pytest.mark.parametrize("pair", [False, True])
def test_attention_matches_the_oracle(gbx, cuda, P, heads, G, hd, S, before, pair):
    B, H = len(before), heads * G
    s = Setup(gbx, P, heads, hd, B, max(before) + S, seed=sum(before) + hd + S)
    q = (s.rng.standard_normal((B, S, H, hd)) * 2).astype(np.float32)
    n_new = np.full(B, S)
    kv_len = np.array(before) + n_new
    scale = float(np.sqrt(hd))
    want, tol = kv_oracle.attend(s.ref, s.table, kv_len, n_new, q, scale)
    out, lo = run_attn(s, q, kv_len, n_new, scale, pair=pair, ld_extra=4)
    if pair:
        tol = tol + np.abs(want) * 2.0 ** -20       # a tf32 pair carries 21 bits; q's own pair is in the queries' halves
        tol = tol + pair_slack(s, q, want)
        out = out.astype(np.float64) + lo
    assert_attn(out, want, tol, np.ones(B * S * H * hd, bool).reshape(q.shape))
    assert int(s.err.item()) == 0
    without, _ = run_attn(s, q, kv_len, n_new, scale, workspace=None)
    assert_attn(without, want, tol, np.ones(q.shape, bool))


def pair_slack(s, q, want):
    """q split into a tf32 pair loses up to 2^-22 of each entry: as a score error, A 2^-22 log2(e) and its weight."""
    big = max(np.abs(s.ref.scale[0]).max() * 127, 1e-30)
    A = np.abs(q.astype(np.float64)).sum(-1, keepdims=True) * big / np.sqrt(q.shape[-1])
    vmax = np.abs(s.ref.scale[1]).max() * 127
    return 2 * A * 2.0 ** -22 * vmax * np.ones_like(want)


@pytest.mark.parametrize("hd", range(16, 129, 16))
@pytest.mark.parametrize("rows", [1, 12, 50])
def test_attention_of_every_head_width_uses_its_whole_ring(gbx, cuda, hd, rows):
    """Caches long enough that every warp goes through all its slots several times."""
    s = Setup(gbx, 16, 2, hd, 1, 4200, seed=hd)
    q = s.rng.standard_normal((1, rows, 2, hd)).astype(np.float32)
    kv_len, n_new = np.array([4200]), np.array([rows])
    pick = [0, rows - 1]
    want, tol = kv_oracle.attend(s.ref, s.table, [4200 - rows + 1], [1], q[:, :1], 8.0)
    want1, tol1 = kv_oracle.attend(s.ref, s.table, kv_len, [1], q[:, rows - 1:], 8.0)
    for ws in ("auto", None):
        out, _ = run_attn(s, q, kv_len, n_new, 8.0, workspace=ws)
        assert np.isfinite(out).all()
        assert_attn(out[:, pick], np.concatenate([want, want1], 1), np.concatenate([tol, tol1], 1), np.ones((1, 2, 2, hd), bool))
    assert int(s.err.item()) == 0


@pytest.mark.parametrize("S,G,P", [(1, 1, 16), (5, 1, 32), (4, 3, 64), (40, 1, 16)])
def test_attention_ragged_rows(gbx, cuda, S, G, P):
    """Rows past a sequence's own are left as they were; sequences without rows or tokens too."""
    heads, hd, B = 2, 64, 6
    s = Setup(gbx, P, heads, hd, B, 200, seed=S)
    n_new = np.array([S, 0, min(S, 2), S, 0, 1])
    kv_len = np.array([S, 50, 101, 190, 0, 1])
    q = s.rng.standard_normal((B, S, heads * G, hd)).astype(np.float32)
    q[np.arange(S)[None] >= n_new[:, None]] = np.nan
    want, tol = kv_oracle.attend(s.ref, s.table, kv_len, n_new, q, 8.0)
    out, _ = run_attn(s, q, kv_len, n_new, 8.0, fill=3.0, ld_extra=8)
    live = np.broadcast_to((np.arange(S)[None] < n_new[:, None])[..., None, None], q.shape)
    assert np.all(out[~live] == 3.0)
    assert_attn(out, want, tol, live)
    assert int(s.err.item()) == 0


@pytest.mark.parametrize("ld_extra,off", [(0, 0), (1, 0), (4, 1), (2, 3)])
def test_attention_strides_and_alignment(gbx, cuda, ld_extra, off):
    s = Setup(gbx, 16, 2, 64, 2, 90, seed=off)
    q = s.rng.standard_normal((2, 2, 4, 64)).astype(np.float32)
    kv_len, n_new = np.array([90, 33]), np.array([2, 2])
    want, tol = kv_oracle.attend(s.ref, s.table, kv_len, n_new, q, 8.0)
    for pair in (False, True):
        out, lo = run_attn(s, q, kv_len, n_new, 8.0, pair=pair, ld_extra=ld_extra, off=off)
        extra = np.abs(want) * 2.0 ** -20 + pair_slack(s, q, want) if pair else 0
        assert_attn(out if not pair else out.astype(np.float64) + lo, want, tol + extra, np.ones(q.shape, bool))


def test_attention_sees_nothing_beyond_the_length(gbx, cuda):
    """NaN scales and table entries out of range behind the last token's page; stale codes behind the last token."""
    P, heads, hd = 16, 2, 64
    s = Setup(gbx, P, heads, hd, 3, 160, seed=1)
    kv_len, n_new = np.array([70, 64, 1]), np.array([3, 1, 1])
    for b in range(3):
        first_free = -(-int(kv_len[b]) // P)
        for j in range(first_free, s.m):
            for w in range(2):
                s.ref.scale[w][s.table[b, j]] = np.nan
        s.table[b, min(first_free + 1, s.m - 1):] = 1 << 30
    s.upload()
    q = s.rng.standard_normal((3, 3, heads, hd)).astype(np.float32)
    want, tol = kv_oracle.attend(s.ref, s.table, kv_len, n_new, q, 8.0)
    out, _ = run_attn(s, q, kv_len, n_new, 8.0)
    live = np.broadcast_to((np.arange(3)[None] < n_new[:, None])[..., None, None], q.shape)
    assert_attn(out, want, tol, live)
    assert int(s.err.item()) == 0


@pytest.mark.parametrize("which", ["k", "v"])
def test_a_poisoned_page_reaches_only_the_rows_that_see_it(gbx, cuda, which):
    P, heads, hd, S = 16, 2, 64, 6
    s = Setup(gbx, P, heads, hd, 2, 64, seed=2)
    kv_len, n_new = np.array([35, 35]), np.array([S, S])   # rows are tokens 29 .. 34; the third page starts at 32
    page, h = int(s.table[0, 2]), 1
    s.ref.scale[0 if which == "k" else 1][page, h] = np.nan
    s.upload()
    q = s.rng.standard_normal((2, S, heads, hd)).astype(np.float32)
    want, tol = kv_oracle.attend(s.ref, s.table, kv_len, n_new, q, 8.0)
    out, _ = run_attn(s, q, kv_len, n_new, 8.0)
    bad = np.zeros(q.shape, bool)
    bad[0, 3:, h] = True
    assert np.isnan(out[bad]).all() and np.isnan(want[bad]).all()
    assert_attn(out, want, tol, ~bad)


def test_attention_special_queries(gbx, cuda):
    """Zero, huge, tiny and NaN rows next to ordinary ones of the same tile."""
    s = Setup(gbx, 16, 1, 64, 1, 100, seed=4)
    q = s.rng.standard_normal((1, 8, 1, 64)).astype(np.float32)
    q[0, 1] = 0.0
    q[0, 2] *= 1e-30
    q[0, 3] *= 300.0
    q[0, 4, 0, 5] = np.nan
    q[0, 5] *= 1e-42                      # subnormal entries
    kv_len, n_new = np.array([100]), np.array([8])
    want, tol = kv_oracle.attend(s.ref, s.table, kv_len, n_new, q, 8.0)
    out, _ = run_attn(s, q, kv_len, n_new, 8.0)
    live = np.ones(q.shape, bool)
    live[0, 4] = False
    assert np.isnan(out[0, 4]).all()
    assert_attn(out, want, tol, live)


def test_attention_flags_bad_pages_and_lengths(gbx, cuda):
    P, heads, hd, B, S = 16, 2, 64, 6, 2
    s = Setup(gbx, P, heads, hd, B, 90, seed=6)
    s.table[0, 1] = s.ref.pages            # 16 of its 40 tokens are not to be had
    s.table[1, :] = -3                     # none is: zeros
    kv_len, n_new = np.array([40, 20, 30, 97, 2, 50]), np.array([2, 2, 3, 1, -1, 2])
    q = s.rng.standard_normal((B, S, heads, hd)).astype(np.float32)
    want, tol = kv_oracle.attend(s.ref, s.table, kv_len, n_new, q, 8.0, skip=(2, 3, 4))
    out, _ = run_attn(s, q, kv_len, n_new, 8.0, fill=9.0)
    live = np.zeros(q.shape, bool)
    live[[0, 1, 5]] = True
    assert np.all(out[~live] == 9.0) and np.all(out[1] == 0.0)
    assert_attn(out, want, tol, live)
    assert int(s.err.item()) == gbx.KV_BAD_PAGE | gbx.KV_BAD_LEN


def test_attention_far_into_the_pool(gbx, cuda):
    """Pages whose codes lie past 2^31 bytes."""
    import torch
    P, heads, hd = 128, 8, 128             # 131,072 bytes a page
    pages = (1 << 31) // (P * heads * hd) + 40
    cache = gbx.KVCache(layers=1, pages=pages, heads=heads, page=P, hd=hd)
    s = Setup(gbx, P, heads, hd, 1, 300, seed=8)
    far = np.array([[pages - 1, pages - 30, 1]])
    for j in range(3):
        p = int(s.table[0, j])
        for a, b in ((cache.k, s.cache.k), (cache.v, s.cache.v), (cache.k_scale, s.cache.k_scale), (cache.v_scale, s.cache.v_scale)):
            a[0, int(far[0, j])] = b[0, p]
    q = s.rng.standard_normal((1, 2, heads, hd)).astype(np.float32)
    kv_len, n_new = np.array([300]), np.array([2])
    want, tol = kv_oracle.attend(s.ref, s.table, kv_len, n_new, q, 11.0)
    near = s.cache
    s.cache, s.table = cache, far
    out, _ = run_attn(s, q, kv_len, n_new, 11.0)
    assert_attn(out, want, tol, np.ones(q.shape, bool))
    x = dev(tokens(s.rng, 2, heads * hd))
    for c, t in ((cache, far), (near, None)):
        t = far if t is not None else near_table(s, near)
        gbx.kv_append(c, 0, x, x, i32(t), i32([301]), B=1, S=2, ld=heads * hd, n_new=i32([1]))
    got = [torch.empty((1, heads * hd), device="cuda") for _ in range(4)]
    gbx.kv_read(cache, 0, i32(far), i32([301]), got[0], got[1], B=1, S=1, ld=heads * hd)
    gbx.kv_read(near, 0, i32(near_table(s, near)), i32([301]), got[2], got[3], B=1, S=1, ld=heads * hd)
    assert torch.equal(got[0], got[2]) and torch.equal(got[1], got[3])
    gbx.kv_copy_pages(cache, i32([pages - 1]), i32([pages - 2]), n=1)
    assert torch.equal(cache.k[0, pages - 1], cache.k[0, pages - 2]) and torch.equal(cache.v[0, pages - 1], cache.v[0, pages - 2])


def near_table(s, near):
    rng = np.random.default_rng(8)         # Setup's own table of that seed
    m = s.m
    kv_oracle.Cache(m + 3, s.heads, s.P, s.hd, rng)
    return rng.permutation(m + 3)[:m].reshape(1, m)


@pytest.mark.parametrize("P,heads,G,hd,S,before", [(16, 1, 1, 64, 20, [5000]), (64, 1, 8, 128, 3, [3000]), (32, 1, 1, 96, 66, [2500]),
                                                   (128, 1, 2, 16, 40, [1500, 0])])
def test_attention_of_many_rows_cut_into_pieces(gbx, cuda, P, heads, G, hd, S, before):
    """More rows than 16 over caches long enough for several clusters, which meet in the workspace."""
    B, H = len(before), heads * G
    s = Setup(gbx, P, heads, hd, B, max(before) + S, seed=S)
    q = (s.rng.standard_normal((B, S, H, hd)) * 2).astype(np.float32)
    n_new = np.full(B, S)
    kv_len = np.array(before) + n_new
    assert gbx.attn_cached_workspace(s.cache, B=B, S=S, H=H, max_pages=s.m) > 0
    want, tol = kv_oracle.attend(s.ref, s.table, kv_len, n_new, q, 9.0)
    for ws in ("auto", None):
        out, _ = run_attn(s, q, kv_len, n_new, 9.0, workspace=ws)
        assert_attn(out, want, tol, np.ones(q.shape, bool))
    assert int(s.err.item()) == 0


@pytest.mark.parametrize("S,tokens_", [(1, 300), (1, 40000), (30, 300)])
def test_attention_reports_a_timeout(gbx, cuda, S, tokens_):
    """The first wait for a copy gives up at once: NaN rows and the status, and the next call is as ever."""
    s = Setup(gbx, 16, 1, 64, 1, tokens_, seed=S)
    q = s.rng.standard_normal((1, S, 1, 64)).astype(np.float32)
    clean, _ = run_attn(s, q, [tokens_], [S], 8.0)
    prev = gbx.set_first_wait_limit(0)
    try:
        out, _ = run_attn(s, q, [tokens_], [S], 8.0, fill=1.0)
    finally:
        gbx.set_first_wait_limit(prev)
    assert np.isnan(out).all() and int(s.err.item()) == gbx.LINEAR_TIMEOUT
    s.err.zero_()
    again, _ = run_attn(s, q, [tokens_], [S], 8.0)
    assert np.array_equal(clean, again) and int(s.err.item()) == 0


def test_calls_on_two_streams(gbx, cuda):
    """Two caches, each with its own workspace, on two streams at once."""
    import torch
    sets = [Setup(gbx, 16, 2, 64, 2, 3000, seed=i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    qs = [s.rng.standard_normal((2, 1, 2, 64)).astype(np.float32) for s in sets]
    want = [run_attn(s, q, [3000, 1700], [1, 1], 8.0)[0] for s, q in zip(sets, qs)]
    args = []
    for s, q in zip(sets, qs):
        n = gbx.attn_cached_workspace(s.cache, B=2, S=1, H=2, max_pages=s.m)
        args.append((dev(q.reshape(2, -1)), torch.empty(2, 128, device="cuda"), i32(s.table), i32([3000, 1700]), i32([1, 1]),
                     torch.empty(max(n, 1), device="cuda")))
    torch.cuda.synchronize()
    for _ in range(20):
        for s, st, (q, out, table, kv_len, n_new, ws) in zip(sets, streams, args):
            gbx.attn_cached(s.cache, 0, q, out, table, kv_len, B=2, S=1, H=2, ld=128, ld_out=128, scale=8.0, n_new=n_new, workspace=ws,
                            stream=st)
    torch.cuda.synchronize()
    for w, a in zip(want, args):
        assert np.array_equal(w.reshape(2, 128), a[1].cpu().numpy())


# ------------------------------------------------------------------ page copies
@pytest.mark.parametrize("P,heads,hd,layers,n", [(16, 12, 64, 3, 5), (128, 1, 16, 1, 1), (32, 25, 64, 2, 40), (64, 3, 112, 4, 9)])
def test_copy_pages(gbx, cuda, P, heads, hd, layers, n):
    import torch
    g = torch.Generator(device="cuda").manual_seed(n)
    pages = 2 * n + 4
    c = gbx.KVCache(layers=layers, pages=pages, heads=heads, page=P, hd=hd)
    for t in (c.k, c.v):
        t.copy_(torch.randint(-127, 128, t.shape, generator=g, device="cuda"))
    for t in (c.k_scale, c.v_scale):
        t.copy_(torch.rand(t.shape, generator=g, device="cuda"))
    ids = torch.randperm(pages, generator=g, device="cuda").int()
    src, dst = ids[:n].contiguous(), ids[n:2 * n].contiguous()
    want = [t.clone() for t in (c.k, c.v, c.k_scale, c.v_scale)]
    for t in want:
        t[:, dst.long()] = t[:, src.long()]
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    gbx.kv_copy_pages(c, src, dst, n=n, err_flag=err)
    for a, b in zip((c.k, c.v, c.k_scale, c.v_scale), want):
        assert torch.equal(a, b)
    assert int(err.item()) == 0


@pytest.mark.parametrize("pairs,done,bits", [
    ([(1, 2), (1, 3)], [0, 1], 0),                     # one source twice
    ([(1, 2), (3, 2)], [0], 32),                       # one target twice: the first stands
    ([(1, 2), (2, 3)], [1], 32),                       # a chain: the target that is read is left alone
    ([(1, 2), (2, 1)], [], 32),                        # a swap
    ([(4, 4), (1, 2)], [1], 0),                        # a page onto itself
    ([(1, 9), (0, 5)], [1], 8), ([(-1, 3), (0, 5)], [1], 8),
    ([(1, 2), (3, 2), (2, 5), (0, 1)], [2], 32)])
def test_copy_pages_that_clash_are_left_out(gbx, cuda, pairs, done, bits):
    import torch
    c = gbx.KVCache(layers=2, pages=9, heads=3, page=16, hd=32)
    for t in (c.k, c.v):
        t.copy_(torch.randint(-127, 128, t.shape, device="cuda"))
    for t in (c.k_scale, c.v_scale):
        t.copy_(torch.rand(t.shape, device="cuda"))
    want = [t.clone() for t in (c.k, c.v, c.k_scale, c.v_scale)]
    for i in done:
        for t in want:
            t[:, pairs[i][1]] = t[:, pairs[i][0]]
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    gbx.kv_copy_pages(c, i32([p[0] for p in pairs]), i32([p[1] for p in pairs]), n=len(pairs), err_flag=err)
    for a, b in zip((c.k, c.v, c.k_scale, c.v_scale), want):
        assert torch.equal(a, b)
    assert int(err.item()) == bits


# ------------------------------------------------------------------ together
def _chain(gbx, s, kv_len, n_new, k, v, q, out, logits, st, B, S):
    """One decode step of a layer with drafts: append, attend, verify."""
    d = s.heads * s.hd
    gbx.kv_append(s.cache, 0, k, v, st["table"], kv_len, B=B, S=S, ld=d, n_new=n_new)
    gbx.attn_cached(s.cache, 0, q, out, st["table"], kv_len, B=B, S=S, H=s.heads, ld=d, ld_out=d, scale=8.0, n_new=n_new,
                    workspace=st["ws"])
    gbx.verify_tokens(logits, st["ids"], st["out_ids"], st["acc"], B=B, n_draft=S - 1, vocab=st["V"], temperature=0.9,
                      uniforms=st["u"])


@pytest.mark.parametrize("pdl", [False, True])
def test_a_captured_step_replays_on_new_inputs(gbx, cuda, pdl):
    """append -> attention -> verification in one CUDA graph on a side stream, replayed with other tokens and lengths,
    equals the same calls made one by one on a second cache."""
    import torch
    B, S, heads, hd, P, V = 3, 4, 2, 64, 16, 1000
    d = heads * hd
    old = gbx.set_pdl(pdl)
    try:
        a, b = Setup(gbx, P, heads, hd, B, 200, seed=11), Setup(gbx, P, heads, hd, B, 200, seed=11)
        g = torch.Generator(device="cuda").manual_seed(1)
        new = lambda *sh: torch.randn(*sh, generator=g, device="cuda")  # noqa: E731
        steps = [(new(B * S, d), new(B * S, d), new(B * S, d), new(B, S, V)) for _ in range(4)]
        lens = [np.array([4 + 5 * i, 60 + 4 * i, 100 + i]) for i in range(4)]
        state = lambda: dict(table=i32(a.table), ws=torch.empty(1 << 20, device="cuda"), ids=i32(np.full((B, S - 1), 7)),  # noqa: E731
                             out_ids=i32(np.zeros((B, S))), acc=i32(np.zeros(B)), V=V,
                             u=torch.full((B, S), 0.4, dtype=torch.float64, device="cuda"))
        n_new, st_a, st_b = i32([4, 2, 1]), state(), state()
        k, v, q, lg = (torch.empty_like(t) for t in steps[0])
        out, kv_len = torch.zeros(B * S, d, device="cuda"), i32([0, 0, 0])
        side = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        kv_len.copy_(i32(lens[0]))
        for dst, src in zip((k, v, q, lg), steps[0]):
            dst.copy_(src)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            _chain(gbx, a, kv_len, n_new, k, v, q, out, lg, st_a, B, S)
        for (kk, vv, qq, ll), ln in zip(steps, lens):
            for dst, src in zip((k, v, q, lg, kv_len), (kk, vv, qq, ll, i32(ln))):
                dst.copy_(src)
            graph.replay()
            ref = torch.zeros(B * S, d, device="cuda")
            _chain(gbx, b, i32(ln), n_new, kk, vv, qq, ref, ll, st_b, B, S)
            torch.cuda.synchronize()
            for x, y in ((a.cache.k, b.cache.k), (a.cache.v, b.cache.v), (st_a["out_ids"], st_b["out_ids"]), (st_a["acc"], st_b["acc"])):
                assert torch.equal(x, y)
            rows = torch.zeros(B, S, 1, dtype=torch.bool, device="cuda")
            for i, n in enumerate((4, 2, 1)):
                rows[i, :n] = True
            rows = rows.expand(B, S, d).reshape(B * S, d)
            assert torch.equal(out[rows], ref[rows])
    finally:
        gbx.set_pdl(old)


@pytest.mark.parametrize("tokens_,cut", [(6000, False), (40000, True)])
def test_the_same_call_gives_the_same_bits(gbx, cuda, tokens_, cut):
    """One cluster, and several that meet in a workspace: no atomics, no order that changes."""
    s = Setup(gbx, 16, 1, 64, 1, tokens_, seed=12)
    q = s.rng.standard_normal((1, 1, 1, 64)).astype(np.float32)
    assert not cut or s.gbx.attn_cached_workspace(s.cache, B=1, S=1, H=1, max_pages=s.m) > 0
    first, _ = run_attn(s, q, [tokens_], [1], 8.0)
    for _ in range(5):
        again, _ = run_attn(s, q, [tokens_], [1], 8.0)
        assert np.array_equal(first, again)


@pytest.mark.parametrize("hd,S", [(64, 1), (64, 4), (32, 20), (128, 20)])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_far_from_zero(gbx, cuda, hd, S, sign):
    """Rows whose one best key is ahead by more than any rounding, at scores of 10^2 to 10^15 in size, above and
    below 0: they return that key's value, to 2^-19 of it (the weight's fixed point half of 2^-23 over a ratio of value
    scales of at least 1/3; fewer than 20 fp32 roundings and two approximations of 2^-22)."""
    heads, L = 2, 300
    s = Setup(gbx, 16, heads, hd, 1, L, seed=hd + S)
    rng = np.random.default_rng(17)
    best = rng.integers(0, L - S, (S, heads))
    big = 10.0 ** rng.uniform(2, 15, (S, heads))
    s.ref.scale[0][:] = np.float32(1 / 60)
    q = np.zeros((1, S, heads, hd), np.float32)
    want = np.zeros(q.shape)
    for h in range(heads):
        for i in range(S):
            # key columns i mod hd, one to a row: its best token is ahead (or least behind) by half
            c = i % hd
            for t in range(L):
                s.ref.codes[0][s.table[0, t // 16], h, t % 16, c] = 60 if sign > 0 else 120
            t = int(best[i, h])
            s.ref.codes[0][s.table[0, t // 16], h, t % 16, c] = 120 if sign > 0 else 60
            q[0, i, h, c] = sign * big[i, h]
            want[0, i, h] = s.ref.codes[1][s.table[0, t // 16], h, t % 16].astype(np.float64) * s.ref.scale[1][s.table[0, t // 16], h]
    s.upload()
    out, _ = run_attn(s, q, [L], [S], 1.0)[:2]
    err = np.abs(out.astype(np.float64) - want)
    assert np.all(err <= np.abs(want) * 2.0 ** -19 + 1e-30), f"{np.argwhere(err > np.abs(want) * 2.0 ** -19)[:5].tolist()}"


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("steps", [2, 3, 5, 6, 7, 9])
def test_rows_shared_by_any_number_of_blocks(gbx, cuda, hd, steps):
    """Prompts whose 64-token steps leave a row block to 2 .. 8 CTAs, with a last step that is not full."""
    L, S, B = 64 * steps - 17, 70, 2
    s = Setup(gbx, 64, 2, hd, B, 64 * steps, seed=steps)
    q = np.random.default_rng(steps).standard_normal((B, S, 4, hd)).astype(np.float32)
    kv_len, n_new = [L, L - 40], [S, 33]
    want, tol = kv_oracle.attend(s.ref, s.table, kv_len, n_new, q, 9.0)
    live = ~np.isnan(want)
    for ws in ("auto", None):
        out, _ = run_attn(s, q, kv_len, n_new, 9.0, workspace=ws)
        assert_attn(out, want, tol, live)
        assert np.isnan(out[~live]).all()
    assert int(s.err.item()) == 0
