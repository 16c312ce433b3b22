"""The recoding of a page's earlier tokens when its scale grows: every code under
ratios that end in ties and next to them, bit for bit with the oracle."""
import numpy as np
import pytest

from test_kv_cache_gpu import Setup

pytestmark = pytest.mark.gpu


# rows kernel (few new rows) and page kernel
@pytest.mark.parametrize("P,hd,S", [(16, 16, 1), (32, 64, 3), (64, 80, 1), (128, 128, 2), (128, 64, 200), (64, 48, 70), (16, 112, 40)])
def test_recoded_codes(gbx, cuda, P, hd, S):
    B, heads = 8, 2
    first = np.array([1, 5, P // 2, P - 1, P // 2 + 1, 3, P - 2, 7])
    s = Setup(gbx, P, heads, hd, B, P + S + 1, seed=P + hd)
    for grow in ([2, 4, 6, 8, 10, 12, 254, 1000], [3, 5, 7, 1.5, 1.25, 127, 129, 1 + 2.0 ** -20], s.rng.uniform(1, 9, B).tolist()):
        grow = np.array(grow)
        # earlier tokens: codes at a scale of 1 / 64, every value of them
        n0 = int(first.max())
        x = s.rng.integers(-127, 128, (B, n0, heads, hd)).astype(np.float32) / 64
        x[:, 0, :, 0], x[:, 0, :, 1] = 127 / 64, -127 / 64
        s.append(first, first, x, -x, n0)
        s.check("before")
        y = np.zeros((B, S, heads, hd), np.float32)
        y[...] = (127 / 64 * grow[:, None, None, None] * s.rng.uniform(-1, 1, y.shape)).astype(np.float32)
        y[:, 0, :, 3] = (127 / 64 * grow[:, None]).astype(np.float32)     # a scale of grow / 64, exactly for the first eight
        n = np.where(np.arange(B) % 2, S, 1)
        s.append(first + n, n, y, -y, S)
        s.check(f"after {grow}")
    assert int(s.err.item()) == 0
