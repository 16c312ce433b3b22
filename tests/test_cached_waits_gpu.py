"""The cached attention under first-wait limits about as long as the wait
itself, so that some lanes of a warp see their copies land just as others give
up: a warp goes one way or the other as a whole.  Each row then comes out either
with the bits of the undisturbed call, or as NaN with the status set."""
import numpy as np
import pytest

from test_kv_cache_gpu import Setup, dev, i32

pytestmark = pytest.mark.gpu


# one CTA, a cluster, several clusters that meet in the workspace; the rows kernel alone, in clusters and cut
@pytest.mark.parametrize("B,heads,G,hd,S,length", [(40, 12, 1, 64, 1, 200), (2, 4, 1, 64, 3, 1500), (1, 1, 2, 128, 1, 30000),
                                                   (30, 8, 1, 64, 70, 150), (1, 4, 2, 32, 40, 1500), (1, 1, 1, 96, 40, 9000)])
def test_limits_near_the_wait_itself(gbx, cuda, B, heads, G, hd, S, length):
    import torch
    s = Setup(gbx, 16, heads, hd, B, length, seed=S + B)
    H = heads * G
    d = H * hd
    q, table = dev(s.rng.standard_normal((B * S, d)).astype(np.float32)), i32(s.table)
    kv_len = i32([length - b % 7 for b in range(B)])
    ws = torch.empty(max(1, gbx.attn_cached_workspace(s.cache, B=B, S=S, H=H, max_pages=s.m)), device="cuda")
    cold = torch.empty(1 << 26, device="cuda")     # larger than L2

    def call(out):
        gbx.attn_cached(s.cache, 0, q, out, table, kv_len, B=B, S=S, H=H, ld=d, ld_out=d, scale=8.0, workspace=ws, err_flag=s.err)

    want = torch.full_like(q, 7.0)
    call(want)
    torch.cuda.synchronize()
    assert int(s.err.item()) == 0 and bool(torch.isfinite(want).all())
    got = torch.full_like(q, 7.0)
    prev = gbx.set_first_wait_limit(0)
    try:
        for limit in (1, 300, 700, 1000, 1300, 1600, 2000, 2500, 3000, 4000):
            gbx.set_first_wait_limit(limit)
            for flush in (True, True, True, False):
                if flush:
                    cold.fill_(1.0)
                s.err.zero_()
                call(got)
                err = int(s.err.item())
                assert err in (0, gbx.LINEAR_TIMEOUT)
                lost = torch.isnan(got.view(B * S * H, hd))
                assert bool((lost.all(1) == lost.any(1)).all())                  # a row as a whole
                assert err or not bool(lost.any())
                same = got.view(torch.int32) == want.view(torch.int32)
                assert bool((same.view(B * S * H, hd) | lost).all())
    finally:
        gbx.set_first_wait_limit(prev)
    s.err.zero_()
    call(got)
    assert torch.equal(got, want) and int(s.err.item()) == 0
