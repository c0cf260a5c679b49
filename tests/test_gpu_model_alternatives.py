"""The best alternatives of TokenLogProbs where wavefronts hand elements from lane to lane, a few lanes at a time and in several turns."""
import numpy as np
import pytest

from deepnet_amd.tensor import Tensor

pytestmark = pytest.mark.gpu
TYPES = [np.float32, np.float64]


def best(x, K):
    """Indices of the K largest of each row in descending order, equal ones by ascending index; NaN counts as missing."""
    x = np.where(np.isnan(x), -np.inf, x)
    out = np.empty((len(x), K), np.int64)
    for row, least, to in zip(x, np.partition(x, -K, axis=1)[:, -K], out):
        at = np.flatnonzero(row >= least)
        to[:] = at[np.argsort(-row[at], kind="stable")[:K]]
    return out


def alternatives(G, X, K):
    tv, ti = G.zeros(X.Shape[:-1] + [K], X.DataType), G.zeros(X.Shape[:-1] + [K], np.int64)
    Tensor.FillTokenLogProbs(X, topLogProbs=tv, topTokens=ti)
    return G.toNumpy(ti)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("lanes", [1, 2, 3, 4, 5, 7, 8, 9, 20])
@pytest.mark.parametrize("rows,vocab", [(2, 40000), (600, 20011)])
def test_a_few_lanes_better_in_every_step(G, rng, dt, lanes, rows, vocab):
    """A row is walked in steps of 4096 elements or fewer; each holds a few elements above everything before, other lanes' from step to step, and
    some lanes' twice with one element that the list has taken already."""
    x = rng.standard_normal((rows, vocab)).astype(dt)
    x[:, :64] += 5
    for j in range(512, vocab - 512, 512):
        at = j + rng.permutation(512)[:lanes]
        x[:, at] = (10 + j / 512 + rng.random((rows, lanes))).astype(dt)
        x[:, at ^ 1] = x[:, at] - dt(0.001)          # the neighbour in the same lane comes close behind
    want, X = best(x, 50), G.ofNumpy(x)
    for K in (1, 8, 50):
        np.testing.assert_array_equal(alternatives(G, X, K), want[:, :K])
    down = G.ofNumpy(np.ascontiguousarray(x[:520, :9000].T)).T     # the vocabulary along a strided axis
    np.testing.assert_array_equal(alternatives(G, down, 8), best(x[:520, :9000], 8))


@pytest.mark.parametrize("dt, nan", [(np.float32, 0x7FC00000), (np.float32, 0x7FA00001), (np.float32, 0xFF800001),
                                     (np.float64, 0x7FF8000000000000), (np.float64, 0x7FF4000000000001), (np.float64, 0xFFF0000000000001)])
@pytest.mark.parametrize("rows,vocab", [(4, 30000), (600, 9001)])
def test_no_kind_of_nan_hides_the_numbers_beside_it(G, rng, dt, nan, rows, vocab):
    """Quiet and signaling NaNs right behind and far behind the best element, in its lane: the alternatives are those of the numbers."""
    x = rng.standard_normal((rows, vocab)).astype(dt)
    bits = x.view(np.uint32 if dt == np.float32 else np.uint64)
    at = rng.integers(vocab - 3000, vocab - 2000, rows)
    for r in range(rows):
        x[r, at[r]] = 50
        bits[r, at[r] + 1:at[r] + 4] = nan
        bits[r, at[r] + 1024] = nan
    tok = np.zeros(rows, np.int64)
    lp, lse, ent, tv, ti = (G.toNumpy(t) for t in Tensor.tokenLogProbs(G.ofNumpy(x), G.ofNumpy(tok), 5))
    np.testing.assert_array_equal(ti, best(x, 5))
    for t in (lp, lse, ent, tv):
        assert np.isnan(t).all()
