"""Cross attention in single precision at the ends of the type's range: gradients far below and above what they are made of.

Bounds as in test_gpu_model_attention.py (r, u), without its absolute allowances for probabilities near 2^-126: none is here.  A product of two
parts below 2^-126 may vanish (6 of them stand for one product): n 6 2^-126 for a sum of n.  dS is held with a factor 2^64: nothing
below 2^-126 is lost of it, and results round at the least denormal, 2^-149."""
import numpy as np
import pytest

from deepnet_amd import native
from deepnet_amd.tensor import Tensor

from test_gpu_model_attention import Oracle, inputs, unit, within

pytestmark = pytest.mark.gpu
F32 = np.float32


def grad_bounds(o, do, out, lse, least=0.0, part=6 * 2.0 ** -126):
    """d_q, d_k, d_v and their bounds, for an oracle whose scores leave every key a probability above 2^-60.  part: what may vanish of a
    product of d_out and v; least: the same of one of dS and of each of the three roundings that make dS."""
    do, out, lse, u = do.astype(np.float64), out.astype(np.float64), lse.astype(np.float64)[..., None], o.u
    T = lambda a: a.transpose(0, 1, 3, 2)
    p = np.exp(o.s - lse)
    assert p.min() > 2.0 ** -60
    dp, dpa = do @ T(o.v), np.abs(do) @ T(np.abs(o.v))
    delta, da = (do * out).sum(-1, keepdims=True), np.abs(do * out).sum(-1, keepdims=True)
    ds = p * (dp - delta) * o.scale
    n, rows = do.shape[-1], do.shape[2]
    rp = o.r[..., None] + 4 * u * np.abs(lse)
    e = np.abs(ds) * (rp + 8 * u) + abs(o.scale) * p * ((n + 2) * u * (dpa + da) + n * part) + 3 * least
    tiny = 2.0 ** -149
    return [(ds @ o.k, (e + (o.lk + 4) * u * np.abs(ds)) @ np.abs(o.k) + o.lk * least + tiny),
            (T(ds) @ o.q, T(e + (rows + 4) * u * np.abs(ds)) @ np.abs(o.q) + rows * least + tiny),
            (T(p) @ do, T(p * (rp + (rows + 4) * u)) @ np.abs(do) + rows * part)]


def check(G, q, k, v, do, scale):
    o = Oracle(q, k, v, None, float(F32(scale)), unit(F32))
    on, ln = o.out.astype(F32), o.lse.astype(F32)
    got = Tensor.crossAttentionGrad(*(G.ofNumpy(t) for t in (do, q, k, v, on, ln)), scale=scale)
    for g, (ref, bound), what in zip(got, grad_bounds(o, do, on, ln), ("d_q", "d_k", "d_v")):
        within(G.toNumpy(g), ref, bound, what)


# widths of the bf16 parts (32, 64, 96, 128), one that takes the float instructions, shares of both walks
WIDTHS = [(70, 90, 32), (160, 200, 64), (40, 75, 96), (130, 70, 128), (50, 90, 63), (100, 2000, 64), (2000, 100, 64)]


@pytest.mark.parametrize("Lq, Lk, D", WIDTHS)
def test_scores_gradients_far_below_upstream(G, rng, Lq, Lk, D):
    """d_out around 2^-80 and a scale of 2^-40: dS lies around 2^-128, where a float cut in three bf16 numbers keeps 6 bits."""
    q, k, v, do = inputs(rng, F32, 1, 2, 2, Lq, Lk, D, D)
    check(G, q, k, v, do * F32(2.0 ** -80), 2.0 ** -40)


@pytest.mark.parametrize("Lq, Lk, D", WIDTHS)
def test_scores_gradients_far_above_upstream(G, rng, Lq, Lk, D):
    """dS around 2^112, beyond what a factor 2^64 leaves room for: q and k are small, the scale is large."""
    q, k, v, do = inputs(rng, F32, 1, 2, 2, Lq, Lk, D, D)
    check(G, q * F32(2.0 ** -32), k * F32(2.0 ** -32), v, do * F32(2.0 ** 53), 2.0 ** 61)


@pytest.mark.parametrize("D", [32, 64, 128, 5])
def test_scores_gradients_at_the_top_of_the_range(G, D):
    """Two keys with opposite values and equal scores: dS = +-(a b), finite, but the next bf16 number above it is infinite."""
    q = np.zeros((1, 1, 40, D), F32)
    k, v, do = np.zeros((1, 1, 2, D), F32), np.zeros((1, 1, 2, D), F32), np.zeros((1, 1, 40, D), F32)
    k[0, 0, :, 0] = 2.0 ** -10, -2.0 ** -10
    a, b = F32(2.0 ** 63 * (2 - 2.0 ** -9)), F32(2.0 ** 63)              # a b / 2 x scale 4 = 2^127 (2 - 2^-9): above bf16's largest, 2^127 (2 - 2^-7)
    v[0, 0, :, 1], do[0, 0, :, 1] = (a, -a), b
    lse, out = np.full((1, 1, 40), np.log(2), F32), np.zeros((1, 1, 40, D), F32)
    dq, dk, dv = (G.toNumpy(t).astype(np.float64) for t in Tensor.crossAttentionGrad(*(G.ofNumpy(t) for t in (do, q, k, v, out, lse)), scale=4.0))
    # P is e^(-lse) with lse rounded (u log 2) and its conversion to another base and the exponential: 6 u in all; each further step 1 u
    want = np.zeros_like(dq)
    want[..., 0] = 2.0 ** 126 * (2 - 2.0 ** -9) * 2.0 ** -10 * 4
    assert (np.abs(dq - want) <= 12 * 2.0 ** -24 * want).all()
    assert not dk.any()                                                  # q is zero
    want = np.zeros_like(dv)
    want[..., 1] = 40 * 0.5 * float(b)
    assert (np.abs(dv - want) <= 50 * 2.0 ** -24 * want).all()


def test_an_infinity_upstream_reaches_its_own_row_only(G, rng):
    q, k, v, do = inputs(rng, F32, 1, 1, 1, 50, 60, 64, 64)
    do[0, 0, 7, 3] = np.inf
    Q, K, V, DO = (G.ofNumpy(t) for t in (q, k, v, do))
    out, lse = Tensor.crossAttention(Q, K, V)
    dq, dk, dv = (G.toNumpy(t) for t in Tensor.crossAttentionGrad(DO, Q, K, V, out, lse))
    bad = np.zeros(50, bool)
    bad[7] = True
    assert not np.isfinite(dq[0, 0, bad]).any() and np.isfinite(dq[0, 0, ~bad]).all()
    assert (dv[0, 0, :, 3] == np.inf).all() and np.isfinite(np.delete(dv[0, 0], 3, 1)).all()


@pytest.mark.parametrize("Lq, D", [(70, 64), (40, 128), (33, 32), (20, 64), (70, 62)])
@pytest.mark.parametrize("which", "q k v do".split())
def test_elements_of_which_bf16_parts_hold_half(G, rng, Lq, D, which):
    """One operand around 2^-122, where three bf16 parts keep 12 bits; the others and the scale bring the scores to about 1 and dS to where a float
    holds it.  The float instructions keep denormals: a sum of n products is besides off by n 2^-149, dS by three such roundings."""
    t = dict(zip(("q", "k", "v", "do"), inputs(rng, F32, 1, 2, 2, Lq, 12, D, D)))
    n = t[which].shape
    t[which] = (np.where(rng.random(n) < 0.5, -1, 1) * (1 + rng.random(n)) * 2.0 ** -122).astype(F32)
    scale = 4.0
    if which in "qk":
        other = "k" if which == "q" else "q"
        t[other], t["do"], scale = t[other] * F32(2.0 ** 60), t["do"] * F32(2.0 ** -56), 2.0 ** 58
    else:
        t["q"] *= F32(2.0 ** -20)
    q, k, v, do = (t[x] for x in ("q", "k", "v", "do"))
    o = Oracle(q, k, v, None, scale, unit(F32))
    out, lse = Tensor.crossAttention(*(G.ofNumpy(x) for x in (q, k, v)), scale=scale)
    within(G.toNumpy(out), o.out, (o.p * (2 * o.r + 28 * o.u)[..., None]) @ np.abs(o.v) + 12 * 2.0 ** -149, "out")
    within(G.toNumpy(lse), o.lse, o.lse_bound(), "lse")
    on, ln = o.out.astype(F32), o.lse.astype(F32)
    got = Tensor.crossAttentionGrad(*(G.ofNumpy(x) for x in (do, q, k, v, on, ln)), scale=scale)
    for g, (ref, bound), what in zip(got, grad_bounds(o, do, on, ln, 2.0 ** -149, 2.0 ** -149), ("d_q", "d_k", "d_v")):
        within(G.toNumpy(g), ref, bound, what)



@pytest.mark.parametrize("Lq, Lk, D", WIDTHS)
def test_the_float_instructions_by_option(G, rng, Lq, Lk, D):
    """attention_bf16x3 = 0: the same bounds, and for layouts that would take the parts other bits (sums rounded at other places)."""
    q, k, v, do = inputs(rng, F32, 1, 2, 2, Lq, Lk, D, D)
    scale = float(F32(1 / np.sqrt(D)))
    o = Oracle(q, k, v, None, scale, unit(F32))
    results = []
    for parts in (1, 0):
        with native.option("attention_bf16x3", parts):
            out, lse = (G.toNumpy(t) for t in Tensor.crossAttention(*(G.ofNumpy(t) for t in (q, k, v)), scale=scale))
            within(out, o.out, o.out_bound(), "out")
            within(lse, o.lse, o.lse_bound(), "lse")
            on, ln = o.out.astype(F32), o.lse.astype(F32)
            got = [G.toNumpy(t) for t in Tensor.crossAttentionGrad(*(G.ofNumpy(t) for t in (do, q, k, v, on, ln)), scale=scale)]
            for g, (ref, bound), what in zip(got, o.grad(do, on, ln), ("d_q", "d_k", "d_v")):
                within(g, ref, bound, what)
            results.append([out, *got])
    for a, b in zip(*results):
        assert np.array_equal(a, b) == (D % 4 != 0)
