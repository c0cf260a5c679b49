"""Cross attention over long keys, whose walk is shared out and joined again: every share's part of the result by itself.

Element d of the keys' and values' width is zero outside the d-th of as many windows of the sequence, so that column d of out is made of one window
alone: a share that is lost or carries a wrong weight shows in full, not as one of hundreds that average out.  Bounds are those of
test_gpu_model_attention.py, (2 r + (Lk + 16) u) of a column: at most 0.5 % of it in single precision, where a share is a third of a window or more."""
import numpy as np
import pytest

from test_gpu_model_attention import Oracle, compare, inputs, unit, within  # noqa: F401

pytestmark = pytest.mark.gpu


def windows(Lk, D):
    return (np.arange(Lk) * D // Lk)[:, None] == np.arange(D)[None, :]


# B, H, Hk, Lq, Lk, D: up to 32 rows of a key head (256 shares of at most 5 tiles), more rows, several heads
@pytest.mark.parametrize("dt", [np.float32, np.float64])
@pytest.mark.parametrize("shape", [(1, 3, 1, 1, 40000, 100), (1, 1, 1, 17, 40000, 64), (1, 1, 1, 40, 40000, 32), (2, 2, 1, 33, 9001, 64), (1, 2, 2, 1, 8190, 63), (1, 1, 1, 70, 30000, 128)])
def test_share_by_share(G, rng, dt, shape):
    B, H, Hk, Lq, Lk, D = shape
    q, k, v, do = inputs(rng, dt, B, H, Hk, Lq, Lk, D, D)
    on = windows(Lk, D)
    mask = np.ones((B, Lk), bool)
    mask[0, ::7] = False
    mask[-1, Lk // 3:Lk // 3 + 700] = False
    compare(G, q, np.where(on, k, 0).astype(dt), np.where(on, 1 + np.abs(v), 0).astype(dt), do, mask)
