"""Log probabilities of tokens, entropy, top alternatives and their gradient against the formulas in 64 bits.

Bounds for a row with maximum m, d_j = x_j - m and weights p_j (E[.] the mean under p), u half a step of the type.  A term e^d carries
the rounding of d (u |d|), of d log2(e) and of its constant (2 u |d|) and of the exponential (2 u): relative 3 u |d| + 2 u.  Terms of one
sign are added up in groups five roundings deep (5 u; the terms that are exactly 1 are counted, without a rounding), the groups in
double precision, at most n additions: n 2^-53.  The sums are rescaled, by a factor off by 2 u, at most once for each 4096 logits.
Hence with c = 7 + 2 ceil(n / 4096) and s1 = u (3 E|d| + c) + n 2^-53
  lse, log_prob:  s1, and the last rounding u |result|;
  entropy = log s - a / s:  s1 for log s; the terms e^d d carry 2 u more, so a / s is off by u (3 E d^2 + (c + 2) E|d|) + n 2^-53 E|d| + s1 E|d|.
The oracle's own arithmetic is double precision: it is allowed the double-precision bound besides (the 4 below covers it for doubles)."""
import numpy as np
import pytest

from deepnet_amd.tensor import Tensor

pytestmark = pytest.mark.gpu
TYPES = [np.float32, np.float64]


def reference(x, tok, top):
    x = x.astype(np.float64)
    n = x.shape[-1]
    m = x.max(-1, keepdims=True)
    z = x - m
    e = np.exp(z)
    s = e.sum(-1)
    p = e / s[..., None]
    zf = np.where(np.isfinite(z), z, 0)
    lse = m[..., 0] + np.log(s)
    ent = np.log(s) - (p * zf).sum(-1)
    lp = np.take_along_axis(x, tok[..., None], -1)[..., 0] - m[..., 0] - np.log(s)
    order = np.argsort(-x, axis=-1, kind="stable")[..., :top]
    tv = np.take_along_axis(x, order, -1) - m - np.log(s)[..., None]
    e1, e2 = (p * np.abs(zf)).sum(-1), (p * zf * zf).sum(-1)
    return lp, lse, ent, tv, order, e1, e2, n


def within(got, ref, bound, what):
    got = got.astype(np.float64)
    inf = np.isinf(ref)
    np.testing.assert_array_equal(got[inf], ref[inf])
    err = np.abs(got[~inf] - ref[~inf])
    b = np.broadcast_to(bound, ref.shape)[~inf]
    assert (err <= b).all(), f"{what}: worst {np.max(err / b)} of the bound"


def check(x, tok, top, res):
    dt = x.dtype
    u = np.finfo(dt).eps / 2 * (4 if dt == np.float64 else 1)
    lp, lse, ent, tv, order, e1, e2, n = reference(x, tok, top)
    c = 7 + 2 * -(-n // 4096)
    s1 = u * (3 * e1 + c) + n * 2.0 ** -53
    within(res[1], lse, s1 + u * np.abs(lse), "lse")
    within(res[0], lp, s1 + u * np.abs(np.where(np.isinf(lp), 0, lp)), "log_probs")
    within(res[2], ent, s1 + u * (3 * e2 + (c + 2) * e1) + n * 2.0 ** -53 * e1 + s1 * e1 + u * np.abs(ent), "entropy")
    if top:
        np.testing.assert_array_equal(res[4], order)
        within(res[3], tv, s1[..., None] + u * np.abs(np.where(np.isinf(tv), 0, tv)), "top_log_probs")


def run(G, x, tok, top):
    return [G.toNumpy(t) for t in Tensor.tokenLogProbs(G.ofNumpy(x), G.ofNumpy(tok), top)]


# one logit; fewer than a vector, a wavefront, a workgroup; odd sizes around the workgroup's step; rows shared by workgroups, and not
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 2, 2), (5, 63, 0), (2, 64, 64), (7, 65, 20), (4, 1023, 5), (3, 4096, 1), (3, 4097, 7), (2, 8191, 64),
                                            (1, 128000, 20), (2, 100003, 50), (300, 5000, 3), (600, 2051, 0), (600, 2051, 9), (1, 3000, 0)])
@pytest.mark.parametrize("spread", [1.0, 20.0])
def test_against_the_formulas(G, rng, dt, rows, vocab, top, spread):
    x = (rng.standard_normal((rows, vocab)) * spread).astype(dt)
    tok = rng.integers(0, vocab, rows)
    check(x, tok, top, run(G, x, tok, top))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 70000), (700, 1500)])
def test_ties_go_to_the_lowest_index(G, rng, dt, rows, vocab):
    x = rng.integers(-3, 4, (rows, vocab)).astype(dt)
    tok = rng.integers(0, vocab, rows)
    check(x, tok, 64, run(G, x, tok, 64))
    x[:] = 0.25
    check(x, tok, 30, run(G, x, tok, 30))
    x = np.sort(rng.standard_normal((rows, vocab)).astype(dt), axis=-1)     # ascending: every element is the best so far
    check(x, tok, 17, run(G, x, tok, 17))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("vocab", [300, 20000])
def test_logits_that_cannot_be_chosen(G, rng, dt, vocab):
    x = rng.standard_normal((6, vocab)).astype(dt)
    tok = rng.integers(0, vocab, 6)
    x[0, vocab // 2:] = -np.inf
    x[1, :] = -np.inf
    x[1, 77] = -3                                    # one choice: probability 1, entropy 0
    x[2, 1:] = np.finfo(dt).min                      # the type's lowest value
    x[3, 5:] = -np.inf                               # fewer choices than alternatives asked for
    tok[0], tok[1], tok[2] = vocab - 1, 77, 0
    res = run(G, x, tok, 8)
    check(x, tok, 8, res)
    assert res[0][1] == 0 and res[2][1] == 0 and res[0][0] == -np.inf
    # a row that leaves nothing
    x[4] = -np.inf
    res = run(G, x, tok, 8)
    assert res[0][4] == -np.inf and res[1][4] == -np.inf and res[2][4] == 0
    assert (res[3][4] == -np.inf).all() and (res[4][4] == np.arange(8)).all()
    # NaN, +inf: NaN in the row's results and nowhere else; a NaN is no alternative
    x[4] = 1
    x[4, 3] = np.nan
    x[5, 2] = np.inf
    res = run(G, x, tok, 8)
    for r in (4, 5):
        assert np.isnan(res[0][r]) and np.isnan(res[1][r]) and np.isnan(res[2][r]) and np.isnan(res[3][r]).all()
    assert (res[4][4] == [0, 1, 2, 4, 5, 6, 7, 8]).all() and res[4][5][0] == 2
    check(x[:4], tok[:4], 8, [t[:4] for t in res])
    y = np.full((1, 3), np.nan, dt)
    y[0, 1] = 2
    assert (run(G, y, np.array([1]), 3)[4] == [[1, -2 ** 63 + 4, -2 ** 63 + 4]]).all()


@pytest.mark.parametrize("dt", TYPES)
def test_entropy_of_a_dominant_logit(G, rng, dt):
    """s = 1 + tiny: the entropy is made of the tiny rest, to the precision of its terms and of the double-precision sum s, of whose up
    to n additions each rounds by at most 2^-53 s, s < 2 here (log s passes that on unchanged: its slope is 1 / s)."""
    x = rng.standard_normal((4, 5000)).astype(dt)
    x[:, 11] = [25, 30, 33, 36]
    tok = np.full(4, 11)
    res = run(G, x, tok, 2)
    check(x, tok, 2, res)
    ent = reference(x, tok, 2)[2]
    # terms of weight p carry a relative error of at most u (3 |d| + 13), |d| <= 42, below 140 u: the same for their sum
    assert np.abs(res[2] - ent).max() <= (np.finfo(dt).eps / 2 * 140 * np.abs(ent)).max() + 5000 * 2.0 ** -52


@pytest.mark.parametrize("dt", TYPES)
def test_layouts_and_optional_results(G, rng, dt):
    x = rng.standard_normal((5, 7, 301)).astype(dt)
    tok = rng.integers(0, 301, (5, 7))
    X, K = G.ofNumpy(x), G.ofNumpy(tok)
    down = lambda r: [G.toNumpy(t) for t in r]
    check(x, tok, 4, down(Tensor.tokenLogProbs(X, K, 4)))
    check(x.transpose(1, 0, 2), tok.T, 4, down(Tensor.tokenLogProbs(X.permuteAxes([1, 0, 2]), K.T, 4)))
    check(x[:, :, 1:300], tok % 299, 4, down(Tensor.tokenLogProbs(X[:, :, 1:300], G.ofNumpy(tok % 299), 4)))
    check(x[:, :, ::-1], tok, 4, down(Tensor.tokenLogProbs(X.reverseAxis(2), K, 4)))
    tok5 = rng.integers(0, 5, (301, 7))
    check(x.transpose(2, 1, 0), tok5, 2, down(Tensor.tokenLogProbs(X.permuteAxes([2, 1, 0]), G.ofNumpy(tok5), 2)))
    check(np.broadcast_to(x[:1], x.shape), tok, 3, down(Tensor.tokenLogProbs(G.ofNumpy(x[:1]).broadcastTo([5, 7, 301]), K, 3)))
    # rank 1: one row; strided targets; each result alone
    check(x[0, 0], tok[0, 0], 3, down(Tensor.tokenLogProbs(X[0, 0], K[0, 0], 3)))
    wide = G.filled([5, 7, 9], dt(-5), dt)
    idx = G.filled([7, 5, 4], -1, np.int64)
    Tensor.FillTokenLogProbs(X, K, wide[:, :, 0], wide[:, :, 1], wide[:, :, 2], wide[:, :, 4:8], idx.permuteAxes([1, 0, 2]))
    w = G.toNumpy(wide)
    check(x, tok, 4, [w[..., 0], w[..., 1], w[..., 2], w[..., 4:8], G.toNumpy(idx).transpose(1, 0, 2)])
    assert (w[..., 3] == -5).all() and (w[..., 8] == -5).all()
    alone = G.zeros([5, 7], dt)
    Tensor.FillTokenLogProbs(X, lse=alone)
    np.testing.assert_array_equal(G.toNumpy(alone), w[..., 1])
    Tensor.FillTokenLogProbs(X, entropy=alone)
    np.testing.assert_array_equal(G.toNumpy(alone), w[..., 2])
    Tensor.FillTokenLogProbs(X, K, alone)
    np.testing.assert_array_equal(G.toNumpy(alone), w[..., 0])
    assert [t.Shape for t in Tensor.tokenLogProbs(G.zeros([0, 9], dt), G.zeros([0], np.int64), 2)] == [[0], [0], [0], [0, 2], [0, 2]]


def test_tokens_outside_the_vocabulary(G, rng):
    x = rng.standard_normal((6, 50)).astype(np.float32)
    tok = np.array([0, 49, 50, -1, 2 ** 40, 7])
    out = [G.filled([6], np.float32(9), np.float32) for _ in range(2)]
    with pytest.raises(IndexError):
        Tensor.FillTokenLogProbs(G.ofNumpy(x), G.ofNumpy(tok), out[0], out[1])
    lp, lse = G.toNumpy(out[0]), G.toNumpy(out[1])
    good = np.array([True, True, False, False, False, True])
    assert (lp[~good] == 9).all()
    check(x[good], tok[good], 0, [lp[good], lse[good], reference(x[good], tok[good], 0)[2].astype(np.float32)])
    d = G.filled([6, 50], np.float32(9), np.float32)
    with pytest.raises(IndexError):
        d.FillTokenLogProbsGrad(G.ofNumpy(x), G.ofNumpy(tok), out[1], out[1])
    d = G.toNumpy(d)
    assert (d[~good] == 9).all() and not (d[good] == 9).any()


# ---- gradient ------------------------------------------------------------------------------------------------------------------------
def grad_reference(x, tok, lse, ent, g, h):
    """The formula on the given lse and entropy, and the bound: e^lp carries the rounding of lp and of its exponent (3 u |lp| + 2 u), the
    factors after it at most 6 roundings; the target column one more addition of g."""
    u = np.finfo(x.dtype).eps / 2 * (4 if x.dtype == np.float64 else 1)
    x, lse, ent, g, h = (a.astype(np.float64) for a in (x, lse[..., None], ent[..., None], g[..., None], h[..., None]))
    with np.errstate(invalid="ignore"):
        lp = np.where(lse == -np.inf, -np.inf, x - lse)
    p = np.exp(lp)
    lf = np.where(p > 0, lp, 0)                      # an element of probability 0 adds nothing, whatever its logarithm
    d = -p * (g + h * (lf + ent))
    onehot = np.zeros(x.shape)
    np.put_along_axis(onehot, tok[..., None], 1, -1)
    dead = lse == -np.inf
    mag = p * (np.abs(g) + np.abs(h) * (np.abs(lf) + np.abs(ent)))
    full = np.where(dead, 0, d + g * onehot)
    tiny = 2.0 ** -126 if u > 2 ** -30 else 0.0      # the exponential flushes denormal results
    bound = mag * u * (3 * np.abs(lf) + 8) + u * (np.abs(full) + np.abs(g) * onehot) + tiny * (1 + np.abs(g) + np.abs(h) * (np.abs(lf) + np.abs(ent)))
    return full, bound


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (4, 1000), (5, 1023), (3, 4096), (2, 8195), (300, 777), (1, 100001)])
@pytest.mark.parametrize("entropy", [False, True])
def test_gradient(G, rng, dt, rows, vocab, entropy):
    x = (rng.standard_normal((rows, vocab)) * 3).astype(dt)
    if vocab > 10:
        x[0, -3:] = -np.inf
        x[rows - 1, : vocab // 2] = np.finfo(dt).min
    if rows > 2:
        x[1] = -np.inf
    tok = rng.integers(0, vocab, rows)
    g, h = rng.standard_normal(rows).astype(dt), rng.standard_normal(rows).astype(dt)
    X, K = G.ofNumpy(x), G.ofNumpy(tok)
    _, lse, ent = Tensor.tokenLogProbs(X, K)
    args = (X, K, lse, G.ofNumpy(g)) + ((ent, G.ofNumpy(h)) if entropy else ())
    ref, bound = grad_reference(x, tok, G.toNumpy(lse), G.toNumpy(ent), g, h if entropy else np.zeros_like(h))
    d = Tensor.tokenLogProbsGrad(*args)
    got = G.toNumpy(d).astype(np.float64)
    err = np.abs(got - ref)
    assert (err <= bound).all(), f"worst {np.max(err / np.maximum(bound, 1e-300))} of the bound"
    X.FillTokenLogProbsGrad(*args)                   # in place
    np.testing.assert_array_equal(G.toNumpy(X), G.toNumpy(d))


def test_gradient_layouts(G, rng):
    x = rng.standard_normal((4, 6, 130))
    tok = rng.integers(0, 128, (4, 6))
    g = rng.standard_normal((4, 1))
    X, K = G.ofNumpy(x), G.ofNumpy(tok)
    for view, xv in ((lambda t: t[:, :, 1:129], x[:, :, 1:129]), (lambda t: t[:, :, 1:129].reverseAxis(2), x[:, :, 1:129][..., ::-1]),
                     (lambda t: t[:, :, 1:129].reverseAxis(0), x[::-1, :, 1:129])):
        V = view(X)
        _, lse, ent = Tensor.tokenLogProbs(V, K)
        gb = G.ofNumpy(g).broadcastTo([4, 6])
        out = G.filled([6, 130, 4], 3.0, np.float64)
        target = out[:, 1:129, :].permuteAxes([1, 2, 0])
        target.FillTokenLogProbsGrad(V, K, lse, gb, ent, gb)
        gg = np.ascontiguousarray(np.broadcast_to(g, (4, 6)))
        ref, bound = grad_reference(np.ascontiguousarray(xv), tok, G.toNumpy(lse), G.toNumpy(ent), gg, gg)
        got = G.toNumpy(target)
        assert (np.abs(got - ref) <= bound).all()
        full = G.toNumpy(out)
        assert (full[:, 0] == 3).all() and (full[:, 129] == 3).all()


def test_gradient_against_differences(G, rng):
    x = rng.standard_normal((3, 17))
    tok = rng.integers(0, 17, 3)
    g, h = rng.standard_normal(3), rng.standard_normal(3)

    def value(y):
        lp, _, ent = (G.toNumpy(t) for t in Tensor.tokenLogProbs(G.ofNumpy(y), G.ofNumpy(tok)))
        return float((g * lp + h * ent).sum())

    X, K = G.ofNumpy(x), G.ofNumpy(tok)
    _, lse, ent = Tensor.tokenLogProbs(X, K)
    d = G.toNumpy(Tensor.tokenLogProbsGrad(X, K, lse, G.ofNumpy(g), ent, G.ofNumpy(h)))
    step = 1e-5                                      # central differences: step^2 |f'''| / 6 + 2^-52 |f| / step, with room: 1e-8
    for r in range(3):
        for j in range(17):
            up, dn = x.copy(), x.copy()
            up[r, j] += step
            dn[r, j] -= step
            assert abs((value(up) - value(dn)) / (2 * step) - d[r, j]) < 1e-8


def test_scratch_memory_of_the_caller(G, rng):
    x = rng.standard_normal((3, 50000)).astype(np.float32)
    tok = rng.integers(0, 50000, 3)
    need = G.scratchBytes("token_log_probs", np.float32, 3, 50000, 6)
    assert need > 0 and G.scratchBytes("token_log_probs", np.float32, 4096, 50000, 6) == 0
    out = [G.zeros([3], np.float32) for _ in range(3)] + [G.zeros([3, 6], np.float32), G.zeros([3, 6], np.int64)]
    guard = G.filled([need + 64], np.uint8(0xA5), np.uint8)
    Tensor.FillTokenLogProbs(G.ofNumpy(x), G.ofNumpy(tok), *out, scratch=guard[:need])
    check(x, tok, 6, [G.toNumpy(t) for t in out])
    assert (G.toNumpy(guard)[need:] == 0xA5).all()
    with pytest.raises(ValueError):
        Tensor.FillTokenLogProbs(G.ofNumpy(x), G.ofNumpy(tok), *out, scratch=guard[:need - 1])


def test_logits_beyond_two_to_the_32_elements(G, rng):
    rows, vocab = 8200, 1 << 19                       # 17 GB of floats; the rows that are looked at lie at both ends
    big = Tensor.new([rows, vocab], G.Dev, np.float32)
    x = rng.standard_normal((2, vocab)).astype(np.float32)
    big[0:1], big[rows - 1:rows] = G.ofNumpy(x[:1]), G.ofNumpy(x[1:])
    pick = big.Relayout(type(big.Layout)((2, vocab), big.Layout.Offset, ((rows - 1) * vocab, 1)))
    tok = np.array([5, vocab - 1])
    check(x, tok, 5, [G.toNumpy(t) for t in Tensor.tokenLogProbs(pick, G.ofNumpy(tok), 5)])
