"""Token embedding and its gradient against plain sums in 64 bits.

Bounds (u: half a step of the type, 2^-24 or 2^-53).  The lookup is one product: its bits are NumPy's.  The gradient sums m addends in
double precision (each addition off by at most 2^-53 of a partial sum, itself at most sum|x|), multiplies once and rounds once to
the type: |got - exact| <= u |exact| + (m + 2) 2^-53 scale sum|x|; the reference's own double sum is allowed the same again."""
import ctypes as C

import numpy as np
import pytest

from deepnet_amd import abi, native
from deepnet_amd.tensor import Tensor
from deepnet_amd import layout as L

pytestmark = pytest.mark.gpu
TYPES = [np.float32, np.float64]


def zipf(rng, n, vocab):
    return np.clip(np.exp(rng.random(n) * np.log(vocab + 1)).astype(np.int64) - 1, 0, vocab - 1)


def check_grad(got, tokens, g, vocab, scale, base=None):
    dt = got.dtype
    u = np.finfo(dt).eps / 2
    g = g.reshape(-1, g.shape[-1]).astype(np.float64)
    ref, mag, cnt = np.zeros((vocab, g.shape[1])), np.zeros((vocab, g.shape[1])), np.bincount(tokens.ravel(), minlength=vocab)
    np.add.at(ref, tokens.ravel(), g)
    np.add.at(mag, tokens.ravel(), np.abs(g))
    s = float(dt.type(scale))
    exact = ref * s + (0 if base is None else base.astype(np.float64))
    bound = u * np.abs(exact) + 2 * (cnt[:, None] + 3) * 2.0 ** -53 * (abs(s) * mag + (0 if base is None else np.abs(base))) + np.finfo(dt).smallest_subnormal
    err = np.abs(got.astype(np.float64) - exact)
    assert (err <= bound).all(), f"worst {np.max(err / np.maximum(bound, 1e-300))} of the bound"
    if base is None:
        assert not got[cnt == 0].any()
    else:
        np.testing.assert_array_equal(got[cnt == 0], base[cnt == 0])


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n,vocab,width", [(1, 1, 1), (1, 7, 4), (3, 5, 3), (16, 1000, 1024), (257, 100, 130), (5000, 333, 65), (4, 10, 5000), (70000, 50, 8)])
def test_lookup(G, rng, dt, n, vocab, width):
    table = rng.standard_normal((vocab, width)).astype(dt)
    tok = rng.integers(0, vocab, n)
    for scale in (None, 1.0, -3.7):
        got = G.toNumpy(Tensor.embedding(G.ofNumpy(table), G.ofNumpy(tok), scale))
        np.testing.assert_array_equal(got, table[tok] * dt(1 if scale is None else scale))


@pytest.mark.parametrize("dt", TYPES)
def test_lookup_layouts(G, rng, dt):
    table = rng.standard_normal((40, 70)).astype(dt)
    tok = rng.integers(0, 40, (6, 5))
    T, K = G.ofNumpy(table), G.ofNumpy(tok)
    # a transposed table, rows of a wider table at an odd start, tokens in reversed and transposed order, broadcast tokens, a strided target
    np.testing.assert_array_equal(G.toNumpy(Tensor.embedding(G.ofNumpy(np.ascontiguousarray(table.T)).T, K)), table[tok])
    np.testing.assert_array_equal(G.toNumpy(Tensor.embedding(T[:, 1:68], K, 2.0)), table[:, 1:68][tok] * dt(2))
    np.testing.assert_array_equal(G.toNumpy(Tensor.embedding(T.reverseAxis(0), K.T.reverseAxis(1))), table[::-1][tok.T[:, ::-1]])
    np.testing.assert_array_equal(G.toNumpy(Tensor.embedding(T, G.ofNumpy(tok[:1]).broadcastTo([4, 5]))), table[np.broadcast_to(tok[:1], (4, 5))])
    out = G.filled([5, 6, 80], dt(-1), dt)
    view = out.permuteAxes([1, 0, 2])[:, :, 3:73]
    view.FillEmbedding(T, K)
    want = np.full((5, 6, 80), -1, dt)
    want.transpose(1, 0, 2)[:, :, 3:73] = table[tok]
    np.testing.assert_array_equal(G.toNumpy(out), want)
    # a single token (rank 0), no tokens, an empty table that nothing names
    np.testing.assert_array_equal(G.toNumpy(Tensor.embedding(T, G.scalar(7, np.int64))), table[7])
    assert Tensor.embedding(T, G.zeros([0, 3], np.int64)).Shape == [0, 3, 70]
    assert Tensor.embedding(G.zeros([0, 4], dt), G.zeros([0], np.int64)).Shape == [0, 4]


@pytest.mark.parametrize("bad", [-1, 40, 2 ** 40, -2 ** 63])
def test_tokens_outside_the_table(G, rng, bad):
    table = rng.standard_normal((40, 12)).astype(np.float32)
    tok = rng.integers(0, 40, 300)
    tok[[5, 299]] = bad
    T, K = G.ofNumpy(table), G.ofNumpy(tok)
    out = G.filled([300, 12], np.float32(9), np.float32)
    with pytest.raises(IndexError):
        out.FillEmbedding(T, K)
    ok = (tok >= 0) & (tok < 40)
    want = np.full((300, 12), 9, np.float32)
    want[ok] = table[tok[ok]]
    np.testing.assert_array_equal(G.toNumpy(out), want)
    g = rng.standard_normal((300, 12)).astype(np.float32)
    g[~ok] = np.nan                                   # what such a row holds is not used
    d = G.filled([40, 12], np.float32(9), np.float32)
    with pytest.raises(IndexError):
        d.FillEmbeddingGrad(K, G.ofNumpy(g))
    check_grad(G.toNumpy(d), tok[ok], g[ok], 40, 1.0)
    out.FillEmbedding(T, G.ofNumpy(np.where(ok, tok, 0)))   # the flag was cleared with the report


# one token, one workgroup's sort, its border, one pass and several through memory, pieces that end inside and between runs
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n,vocab,width", [(1, 1, 1), (1, 9, 5), (2, 3, 1), (7, 3, 4), (64, 500, 33), (1000, 1, 6), (1025, 40, 130), (8191, 5000, 9), (8192, 511, 8),
                                           (8193, 512, 7), (8193, 1, 3), (20000, 100000, 16), (50001, 70, 20), (40000, 300000, 2), (300, 20, 1500)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_gradient(G, rng, dt, n, vocab, width, accumulate):
    tok = zipf(rng, n, vocab)
    g = rng.standard_normal((n, width)).astype(dt)
    base = rng.standard_normal((vocab, width)).astype(dt)
    d = G.ofNumpy(base)
    d.FillEmbeddingGrad(G.ofNumpy(tok), G.ofNumpy(g), 1.7, accumulate)
    first = G.toNumpy(d)
    check_grad(first, tok, g, vocab, 1.7, base if accumulate else None)
    d = G.ofNumpy(base)
    d.FillEmbeddingGrad(G.ofNumpy(tok), G.ofNumpy(g), 1.7, accumulate)
    np.testing.assert_array_equal(G.toNumpy(d), first)   # the same bits again


@pytest.mark.parametrize("dt", TYPES)
def test_gradient_of_one_token_that_fills_many_pieces(G, rng, dt):
    tok = np.full(30000, 2)
    tok[::1000] = 1
    g = (rng.standard_normal((30000, 131)) * 1e3).astype(dt)
    check_grad(G.toNumpy(Tensor.embeddingGrad(G.ofNumpy(tok), G.ofNumpy(g), 4)), tok, g, 4, 1.0)


@pytest.mark.parametrize("dt", TYPES)
def test_gradient_layouts(G, rng, dt):
    tok = rng.integers(0, 30, (8, 50))
    g = rng.standard_normal((8, 50, 21)).astype(dt)
    K, D = G.ofNumpy(tok), G.ofNumpy(g)
    check_grad(G.toNumpy(Tensor.embeddingGrad(K, D, 30)), tok, g, 30, 1.0)
    check_grad(G.toNumpy(Tensor.embeddingGrad(K.T, D.permuteAxes([1, 0, 2]), 30)), tok.T, g.transpose(1, 0, 2), 30, 1.0)
    check_grad(G.toNumpy(Tensor.embeddingGrad(K, D[:, :, 1:18], 30)), tok, g[:, :, 1:18], 30, 1.0)
    check_grad(G.toNumpy(Tensor.embeddingGrad(K, D.reverseAxis(2), 30)), tok, g[:, :, ::-1], 30, 1.0)
    # a gradient that is the same for every token (broadcast), and one upstream value per row
    one = np.ascontiguousarray(np.broadcast_to(g[:1, :1], g.shape))
    check_grad(G.toNumpy(Tensor.embeddingGrad(K, G.ofNumpy(g[:1, :1]).broadcastTo([8, 50, 21]), 30)), tok, one, 30, 1.0)
    # a strided target: a transposed matrix inside a larger one; what lies around it stays
    out = G.filled([25, 40], dt(5), dt)
    view = out[2:23, 4:34].T
    view.FillEmbeddingGrad(K, D)
    got = G.toNumpy(out)
    check_grad(np.ascontiguousarray(got[2:23, 4:34].T), tok, g, 30, 1.0)
    got[2:23, 4:34] = 5
    assert (got == 5).all()
    # no tokens: zeros, or nothing
    d = G.filled([3, 4], dt(5), dt)
    d.FillEmbeddingGrad(G.zeros([0], np.int64), G.zeros([0, 4], dt), accumulate=True)
    assert (G.toNumpy(d) == 5).all()
    d.FillEmbeddingGrad(G.zeros([0], np.int64), G.zeros([0, 4], dt))
    assert not G.toNumpy(d).any()


def test_scratch_memory_of_the_caller(G, rng):
    for n, vocab, width in ((500, 40, 12), (9000, 4000, 5)):
        tok, g = rng.integers(0, vocab, n), rng.standard_normal((n, width)).astype(np.float32)
        need = G.scratchBytes("embedding_grad", n, vocab, width)
        d = G.zeros([vocab, width], np.float32)
        guard = G.filled([need + 64], np.uint8(0xA5), np.uint8)
        d.FillEmbeddingGrad(G.ofNumpy(tok), G.ofNumpy(g), scratch=guard[:need])
        check_grad(G.toNumpy(d), tok, g, vocab, 1.0)
        assert (G.toNumpy(guard)[need:] == 0xA5).all()
        with pytest.raises(ValueError):
            d.FillEmbeddingGrad(G.ofNumpy(tok), G.ofNumpy(g), scratch=guard[:need - 1])


def test_rows_beyond_two_to_the_32_elements(G):
    width, vocab = 1024, (1 << 22) + 5                # 17 GB of floats
    table = Tensor.new([vocab, width], G.Dev, np.float32)
    tok = np.array([0, vocab - 1, 1 << 21, vocab - 2])
    rows = np.arange(4 * width, dtype=np.float32).reshape(4, width)
    for i, t in enumerate(tok):
        table[int(t)] = G.ofNumpy(rows[i])
    np.testing.assert_array_equal(G.toNumpy(Tensor.embedding(table, G.ofNumpy(tok), 2.0)), rows * 2)
    table.FillEmbeddingGrad(G.ofNumpy(tok), G.ofNumpy(rows))
    for i, t in enumerate(tok):
        np.testing.assert_array_equal(G.toNumpy(table[int(t)]), rows[i])
    assert not G.toNumpy(table[vocab - 4]).any() and not G.toNumpy(table[(1 << 22) - 1]).any()
    assert float(table.sum()) == float(G.ofNumpy(rows).sum())


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n,vocab,width", [(512, 3000, 20), (513, 3000, 20), (257, 70000, 1), (500, 1200, 1030), (512, 1, 300), (300, 5000, 64), (1024, 700, 30)])
def test_gradient_of_few_tokens(G, rng, dt, n, vocab, width):
    """Around the number up to which one launch does it all: many blocks of rows to clear, one token named by every position, rows in several
    pieces, read and written along another axis too."""
    tok = zipf(rng, n, vocab) if vocab > 1 else np.zeros(n, np.int64)
    g = rng.standard_normal((n, width)).astype(dt)
    d = G.filled([vocab, width], dt(np.nan), dt)
    d.FillEmbeddingGrad(G.ofNumpy(tok), G.ofNumpy(g))
    check_grad(G.toNumpy(d), tok, g, vocab, 1.0)
    d = G.filled([width, vocab], dt(np.nan), dt)
    d.T.FillEmbeddingGrad(G.ofNumpy(tok), G.ofNumpy(np.ascontiguousarray(g.T)).T, 0.3)
    check_grad(np.ascontiguousarray(G.toNumpy(d).T), tok, g, vocab, 0.3)
