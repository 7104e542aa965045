"""Rotation at positions whose number, or whose angle, has more bits than f32 holds."""
import numpy as np
import pytest

from paged_batches import EPS
from test_paged_gpu import _append, _far, _frequencies

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("length", [131075, 300001, 4194301, 16777219, 100000007, 2 ** 31 - 256])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_the_rotation_of_far_positions(ctx, length, kind):
    """Bound: the angle (of up to 2^31, in 64 bits here as there) is off by 2^-21 at most, its functions by 2^-22, the sum by 2^-23 of it; one rounding to the type."""
    heads, kvh, dim, rot = 2, 1, 64, 64                              # (the three rows are on one page)
    b = _far(length % 97, [(3, length)], heads, kvh, dim, 256, kind)
    proj = np.random.default_rng(length % 89).normal(0, 2, (b.rows, (heads + 2 * kvh) * dim)).astype(np.float32)
    freq = _frequencies(rot, 1e4)
    q, k, _ = _append(ctx, b, proj, "f32", rot, freq)
    x = proj.reshape(b.rows, -1, dim).astype(np.float64)
    for i in range(3):
        p = length - 3 + i
        a = p * (freq[0].astype(np.float64) + freq[1].astype(np.float64))
        lo, hi = x[i, :heads + kvh, :32], x[i, :heads + kvh, 32:]
        want = np.concatenate([lo * np.cos(a) - hi * np.sin(a), lo * np.sin(a) + hi * np.cos(a)], 1)
        off = EPS[kind] / 2 * np.abs(want) + 2.0 ** -20 * np.tile(np.abs(lo) + np.abs(hi), 2) + 2.0 ** -25
        assert (np.abs(q[i] - want[:heads]) <= off[:heads]).all(), (p, np.abs(q[i] - want[:heads]).max())
        assert (np.abs(k[b.table[0, p // 256], :, p % 256] - want[heads:]) <= off[heads:]).all(), p
