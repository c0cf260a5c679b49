"""Cross attention and its gradient against the formulas in 64 bits.

Bounds, u half a step of the type, |.| sums of absolute products.  A score is a sum of Dk products (Dk + 1) u S_abs, its scaling and
the exponent's subtraction add 6 u (|S| + |m|), the exponential 2 u (4 u with its base's constant): every probability before
normalisation is off by at most r = max over the keys of (Dk + 4) u S_abs + 6 u (|S| + |m|) + 4 u, relatively.  Sums over Lk keys add
Lk u.  (Where the products of single precision are taken of bf16 parts they are exact but for 2 u of dropped ones; Dk - 1 additions and those
of the five smaller parts, 5 Dk 2^-8 u, make (Dk + 4) u, too.)  So
  out:  sum_j P_j |v_j| (2 r + (Lk + 16) u)          lse:  r + (Lk + 8) u + 4 u |lse|
Backward, with out and lse as given: P_j is off by r + 4 u |lse| relatively, dP by (Dv + 2) u (|d_out||v|) and delta by (Dv + 2) u
(|d_out||out|), dS by e = |dS| (r + 4 u |lse| + 8 u) + scale P (those two); the last product adds (n + 4) u of its absolute sum.
Single precision flushes: a probability, a product or a partial sum below t = 2^-126 counts as zero, so every probability is besides off
by t absolutely (which dS passes on times scale (|d_out||v| + |d_out||out|)), and every sum of n products by n t.
Double precision: the oracle's own rounding is of the same size, every bound is taken four times."""
import numpy as np
import pytest

from deepnet_amd.tensor import Tensor

pytestmark = pytest.mark.gpu
TYPES = [np.float32, np.float64]


def unit(dt):
    return np.finfo(dt).eps / 2 * (4 if dt == np.float64 else 1)


class Oracle:
    def __init__(self, q, k, v, mask, scale, u):
        q, k, v = (t.astype(np.float64) for t in (q, k, v))
        self.group = q.shape[1] // k.shape[1]
        b, lk = k.shape[0], k.shape[2]
        self.mask = np.ones((b, lk), bool) if mask is None else mask
        on = self.mask[:, None, :, None]
        self.q, self.k0, self.v0 = q, np.where(on, k, 0), np.where(on, v, 0)
        self.k, self.v = (np.repeat(t, self.group, 1) for t in (self.k0, self.v0))
        self.scale, self.u, self.dk, self.lk = scale, u, q.shape[3], lk
        kt = self.k.transpose(0, 1, 3, 2)
        s = q @ kt * scale
        sabs = np.abs(q) @ np.abs(kt) * abs(scale)
        keys = np.broadcast_to(self.mask[:, None, None, :], s.shape)
        self.s = np.where(keys, s, -np.inf)
        m = self.s.max(-1, keepdims=True, initial=-np.inf)
        mz = np.where(np.isfinite(m), m, 0)
        self.keys = keys
        e = np.where(keys, np.exp(self.s - mz), 0)
        tot = e.sum(-1, keepdims=True)
        self.p = e / np.where(tot == 0, 1, tot)
        self.out = self.p @ self.v
        with np.errstate(divide="ignore"):
            self.lse = (mz + np.log(tot))[..., 0]
        fin = np.where(keys, s, 0)
        self.r = np.where(keys, (self.dk + 4) * u * sabs + 6 * u * (np.abs(fin) + np.abs(mz)) + 4 * u, 0).max(-1, initial=0.0)

    def out_bound(self):
        t = 2.0 ** -126 if self.u > 2 ** -30 else 1e-300
        return (self.p * (2 * self.r + (self.lk + 16) * self.u)[..., None] + t) @ np.abs(self.v) + self.lk * t

    def lse_bound(self):
        return self.r + (self.lk + 8) * self.u + 4 * self.u * np.abs(np.where(np.isfinite(self.lse), self.lse, 0))

    def grad(self, do, out, lse):
        do, out, lse, u = do.astype(np.float64), out.astype(np.float64), lse.astype(np.float64), self.u
        lz = np.where(np.isfinite(lse), lse, 0)[..., None]
        p = np.where(self.keys & np.isfinite(lse)[..., None], np.exp(np.where(self.keys, self.s, 0) - lz), 0)
        vt = self.v.transpose(0, 1, 3, 2)
        dp, dpa = do @ vt, np.abs(do) @ np.abs(vt)
        delta, da = (do * out).sum(-1, keepdims=True), np.abs(do * out).sum(-1, keepdims=True)
        ds = p * (dp - delta) * self.scale
        n = do.shape[-1]
        rp = self.r[..., None] + 4 * u * np.abs(lz)
        t = 2.0 ** -126 if u > 2 ** -30 else 0.0
        e = np.abs(ds) * (rp + 8 * u) + abs(self.scale) * (p * (n + 2) * u + t) * (dpa + da)
        rows = do.shape[2] * self.group
        dq = ds @ self.k
        bq = (e + (self.lk + 4) * u * np.abs(ds)) @ np.abs(self.k) + (self.lk + n) * t
        T = lambda a: a.transpose(0, 1, 3, 2)
        fold = lambda a: a.reshape(a.shape[0], -1, self.group, *a.shape[2:]).sum(2)
        dk = fold(T(ds) @ self.q)
        bk = fold(T(e + (rows + 4) * u * np.abs(ds)) @ np.abs(self.q)) + (rows + n) * t
        dv = fold(T(p) @ do)
        bv = fold(T(p * (rp + (rows + 4) * u) + t) @ np.abs(do)) + rows * t
        return [(a, b + 1e-300) for a, b in ((dq, bq), (dk, bk), (dv, bv))]


def within(got, ref, bound, what):
    got = got.astype(np.float64)
    inf = np.isinf(ref)
    np.testing.assert_array_equal(got[inf], ref[inf])
    err = np.abs(got - np.where(inf, 0, ref))[~inf]
    b = np.broadcast_to(bound, ref.shape)[~inf]
    assert (err <= b).all(), f"{what}: worst {np.max(err / b)} of the bound"


def inputs(rng, dt, B, H, Hk, Lq, Lk, Dk, Dv, std=1.0):
    mk = lambda *s: (rng.standard_normal(s) * std).astype(dt)
    return mk(B, H, Lq, Dk), mk(B, Hk, Lk, Dk), mk(B, Hk, Lk, Dv), mk(B, H, Lq, Dv)


def compare(G, q, k, v, do, mask=None, scale=None, up=None, grads=True):
    """Forward and backward of `up`(array) -> tensor against the oracle."""
    dt = q.dtype.type
    up = up or G.ofNumpy
    sc = float(dt(1 / np.sqrt(q.shape[3]) if scale is None else scale))
    o = Oracle(q, k, v, mask, sc, unit(dt))
    Q, K, V, DO = (up(t) for t in (q, k, v, do))
    M = None if mask is None else G.ofNumpy(mask)
    out, lse = Tensor.crossAttention(Q, K, V, M, scale)
    within(G.toNumpy(out), o.out, o.out_bound(), "out")
    within(G.toNumpy(lse), o.lse, o.lse_bound(), "lse")
    if not grads:
        return
    on, ln = o.out.astype(dt), o.lse.astype(dt)
    got = Tensor.crossAttentionGrad(DO, Q, K, V, up(on), G.ofNumpy(ln), M, scale)
    for g, (ref, bound), what in zip(got, o.grad(do, on, ln), ("d_q", "d_k", "d_v")):
        within(G.toNumpy(g), ref, bound, what)


# B, H, Hk, Lq, Lk, Dk, Dv: single positions, sizes around a tile, a wavefront's and a workgroup's rows, shared heads, widths around the
# instantiated ones, one query over many keys (split), many queries over one key
SHAPES = [(1, 1, 1, 1, 1, 1, 1), (1, 1, 1, 1, 5, 3, 7), (2, 2, 2, 5, 31, 16, 16), (1, 2, 1, 16, 32, 32, 32), (1, 1, 1, 33, 33, 33, 17), (2, 4, 2, 31, 65, 48, 48),
          (1, 3, 3, 130, 97, 64, 64), (1, 6, 2, 77, 130, 40, 40), (1, 2, 2, 129, 64, 96, 80), (2, 2, 1, 65, 161, 128, 128), (1, 1, 1, 40, 70, 100, 128),
          (3, 8, 2, 1, 1000, 64, 64), (1, 16, 16, 1, 3001, 128, 128), (1, 1, 1, 700, 1, 64, 64), (2, 8, 1, 3, 517, 20, 64), (1, 1, 1, 1500, 40, 65, 9)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_against_the_formulas(G, rng, dt, shape):
    compare(G, *inputs(rng, dt, *shape))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", [(3, 4, 2, 20, 75, 32, 32), (3, 2, 2, 1, 900, 64, 64), (4, 2, 1, 140, 200, 24, 40)])
def test_masked_keys(G, rng, dt, shape):
    B, Lk = shape[0], shape[4]
    q, k, v, do = inputs(rng, dt, *shape)
    mask = rng.random((B, Lk)) < 0.6
    mask[0] = np.arange(Lk) < Lk // 2                # padding behind the sequence
    mask[1] = False                                  # a sequence without keys
    mask[2, :] = False
    mask[2, Lk - 1] = True                           # one key, the last
    compare(G, q, k, v, do, mask)
    # what masked places hold is not used
    k2, v2 = k.copy(), v.copy()
    k2.transpose(0, 2, 1, 3)[~mask], v2.transpose(0, 2, 1, 3)[~mask] = np.nan, np.inf
    compare(G, q, k2, v2, do, mask)
    M = G.ofNumpy(mask)
    a = Tensor.crossAttention(*(G.ofNumpy(t) for t in (q, k, v)), M)
    b = Tensor.crossAttention(*(G.ofNumpy(t) for t in (q, k2, v2)), M)
    for x, y in zip(a, b):
        np.testing.assert_array_equal(G.toNumpy(x), G.toNumpy(y))
    assert not G.toNumpy(a[0])[1].any() and (G.toNumpy(a[1])[1] == -np.inf).all()
    g = Tensor.crossAttentionGrad(G.ofNumpy(do), G.ofNumpy(q), G.ofNumpy(k2), G.ofNumpy(v2), *a, M)
    assert not G.toNumpy(g[0])[1].any()
    for t in g[1:]:
        assert not G.toNumpy(t).transpose(0, 2, 1, 3)[~mask].any()
    # a mask that is the same for every sequence, as a broadcast view and reversed in memory
    same = G.ofNumpy(np.ascontiguousarray(mask[0][::-1])).reverseAxis(0).broadcastTo([B, Lk])
    o = Oracle(q, k, v, np.broadcast_to(mask[0], (B, Lk)), float(dt(1 / np.sqrt(q.shape[3]))), unit(dt))
    out, _ = Tensor.crossAttention(G.ofNumpy(q), G.ofNumpy(k), G.ofNumpy(v), same)
    within(G.toNumpy(out), o.out, o.out_bound(), "out")


@pytest.mark.parametrize("dt", TYPES)
def test_layouts(G, rng, dt):
    q, k, v, do = inputs(rng, dt, 2, 4, 2, 37, 70, 36, 36)
    blhd = lambda t: G.ofNumpy(np.ascontiguousarray(t.transpose(0, 2, 1, 3))).permuteAxes([0, 2, 1, 3])
    compare(G, q, k, v, do, up=blhd)
    odd = lambda t: G.ofNumpy(np.concatenate([np.full(t.shape[:3] + (1,), np.nan, dt), t, np.full(t.shape[:3] + (2,), np.nan, dt)], 3))[:, :, :, 1:1 + t.shape[3]]
    compare(G, q, k, v, do, up=odd)                  # rows at odd starts with odd pitches, NaN beside them
    down = lambda t: G.ofNumpy(np.ascontiguousarray(t.transpose(0, 1, 3, 2))).permuteAxes([0, 1, 3, 2])
    compare(G, q, k, v, do, up=down)                 # width not the contiguous axis
    rev = lambda t: G.ofNumpy(np.ascontiguousarray(t[:, :, ::-1, ::-1])).reverseAxis(2).reverseAxis(3)
    compare(G, q, k, v, do, up=rev)
    compare(G, q, k, v, do, scale=0.0)
    compare(G, q, k, v, do, scale=-0.3)
    # one encoder sequence for the whole batch (broadcast), strided targets with a frame that stays
    k1, v1 = np.broadcast_to(k[:1], k.shape), np.broadcast_to(v[:1], v.shape)
    sc = float(dt(1 / np.sqrt(36)))
    o = Oracle(q, k1, v1, None, sc, unit(dt))
    K, V = (G.ofNumpy(t[:1]).broadcastTo(list(t.shape)) for t in (k, v))
    frame = G.filled([2, 37, 4, 40], dt(7), dt)
    lse = G.filled([37, 4, 2], dt(7), dt)
    target, lview = frame[:, :, :, 2:38].permuteAxes([0, 2, 1, 3]), lse.permuteAxes([2, 1, 0])
    target.FillCrossAttention(G.ofNumpy(q), K, V, lse=lview)
    within(G.toNumpy(target), o.out, o.out_bound(), "out")
    within(G.toNumpy(lview), o.lse, o.lse_bound(), "lse")
    f = G.toNumpy(frame)
    assert (f[..., :2] == 7).all() and (f[..., 38:] == 7).all()
    on, ln = o.out.astype(dt), o.lse.astype(dt)
    Q, DO, O, LSE = G.ofNumpy(q), G.ofNumpy(do), G.ofNumpy(on), G.ofNumpy(ln)
    full = [G.toNumpy(t) for t in Tensor.crossAttentionGrad(DO, Q, K, V, O, LSE)]
    for g, (ref, bound), what in zip(full, o.grad(do, on, ln), ("d_q", "d_k", "d_v")):
        within(g, ref, bound, what)
    # each gradient alone, into strided targets
    frames = [G.filled([t.shape[0], t.shape[2], t.shape[1], 40], dt(7), dt) for t in (q, k, v)]
    views = [f[:, :, :, 1:37].permuteAxes([0, 2, 1, 3]) for f in frames]
    Tensor.FillCrossAttentionGrad(views[0], None, None, DO, Q, K, V, O, LSE)
    Tensor.FillCrossAttentionGrad(None, views[1], views[2], DO, Q, K, V, O, LSE)
    for a, b, f in zip(views, full, frames):
        np.testing.assert_array_equal(G.toNumpy(a), b)
        f = G.toNumpy(f)
        assert (f[..., 0] == 7).all() and (f[..., 37:] == 7).all()


@pytest.mark.parametrize("dt", TYPES)
def test_large_scores(G, rng, dt):
    """Scores of several hundred: the running maximum carries the softmax; a later tile raises it again and again."""
    q, k, v, do = inputs(rng, dt, 1, 2, 2, 40, 300, 64, 64, std=4.0)
    compare(G, q, k, v, do, scale=1.0)
    k *= np.linspace(0.01, 3, 300)[None, None, :, None].astype(dt)
    compare(G, q, k, v, do, scale=1.0)


@pytest.mark.parametrize("dt", TYPES)
def test_empty_extents(G, dt):
    z = lambda *s: G.zeros(list(s), dt)
    assert Tensor.crossAttention(z(0, 2, 3, 8), z(0, 2, 5, 8), z(0, 2, 5, 8))[0].Shape == [0, 2, 3, 8]
    assert Tensor.crossAttention(z(2, 2, 0, 8), z(2, 2, 5, 8), z(2, 2, 5, 8))[0].Shape == [2, 2, 0, 8]
    one = G.ones([2, 2, 3, 8], dt)
    out, lse = Tensor.crossAttention(one, z(2, 2, 0, 8), z(2, 2, 0, 8))      # no keys at all
    assert not G.toNumpy(out).any() and (G.toNumpy(lse) == -np.inf).all()
    dq, dk, dv = Tensor.crossAttentionGrad(one, one, z(2, 2, 0, 8), z(2, 2, 0, 8), out, lse)
    assert not G.toNumpy(dq).any()
    k = G.ones([2, 2, 5, 8], dt)                                              # no queries: the keys' gradients are zero
    dk, dv = G.filled([2, 2, 5, 8], dt(3), dt), G.filled([2, 2, 5, 8], dt(3), dt)
    Tensor.FillCrossAttentionGrad(None, dk, dv, z(2, 2, 0, 8), z(2, 2, 0, 8), k, k, z(2, 2, 0, 8), z(2, 2, 0))
    assert not G.toNumpy(dk).any() and not G.toNumpy(dv).any()


def test_gradient_against_differences(G, rng):
    q, k, v, do = inputs(rng, np.float64, 1, 2, 1, 3, 6, 5, 4)
    mask = np.array([[1, 1, 0, 1, 1, 1]], bool)
    M = G.ofNumpy(mask)

    def value(a, b, c):
        return float((do * G.toNumpy(Tensor.crossAttention(G.ofNumpy(a), G.ofNumpy(b), G.ofNumpy(c), M)[0])).sum())

    Q, K, V = (G.ofNumpy(t) for t in (q, k, v))
    out, lse = Tensor.crossAttention(Q, K, V, M)
    grads = [G.toNumpy(t) for t in Tensor.crossAttentionGrad(G.ofNumpy(do), Q, K, V, out, lse, M)]
    step = 1e-5                                       # central differences: step^2 |f'''| / 6 + 2^-52 |f| / step, with room: 1e-8
    for which in range(3):
        for at in np.ndindex(grads[which].shape):
            hi, lo = [t.copy() for t in (q, k, v)], [t.copy() for t in (q, k, v)]
            hi[which][at] += step
            lo[which][at] -= step
            assert abs((value(*hi) - value(*lo)) / (2 * step) - grads[which][at]) < 1e-8


@pytest.mark.parametrize("dt", TYPES)
def test_the_same_bits_again_and_scratch_of_the_caller(G, rng, dt):
    for shape in ((2, 4, 4, 1, 2000, 64, 64), (1, 4, 2, 200, 300, 64, 64)):
        q, k, v, do = inputs(rng, dt, *shape)
        B, H, Hk, Lq, Lk, Dk, Dv = shape
        Q, K, V, DO = (G.ofNumpy(t) for t in (q, k, v, do))
        out, lse = Tensor.crossAttention(Q, K, V)
        grads = Tensor.crossAttentionGrad(DO, Q, K, V, out, lse)
        need = G.scratchBytes("cross_attention", dt, B, H, Hk, Lq, Lk, Dv)
        guard = G.filled([need + 64], np.uint8(0xA5), np.uint8)
        o2, l2 = G.zeros(out.Shape, dt), G.zeros(lse.Shape, dt)
        o2.FillCrossAttention(Q, K, V, lse=l2, scratch=guard[:need])
        g2 = [G.zeros(t.Shape, dt) for t in grads]
        Tensor.FillCrossAttentionGrad(*g2, DO, Q, K, V, out, lse, scratch=guard[:need])
        for a, b in zip((out, lse, *grads), (o2, l2, *g2)):
            np.testing.assert_array_equal(G.toNumpy(a), G.toNumpy(b))
        assert (G.toNumpy(guard)[need:] == 0xA5).all()


def test_keys_beyond_two_to_the_32_elements(G, rng):
    """A cache of [key; head; batch-wide rows]: a key's row lies 2^25 elements after the one before it, the last beyond 2^32."""
    q, k, v, do = inputs(rng, np.float32, 1, 1, 1, 3, 140, 32, 32)
    pitch = 1 << 25
    cache = Tensor.new([140, pitch], G.Dev, np.float32)                       # 18.8 GB, two columns blocks of it in use
    cache[:, 64:96] = G.ofNumpy(k[0, 0])
    cache[:, 96:128] = G.ofNumpy(v[0, 0])
    mk = lambda off: cache.Relayout(type(cache.Layout)((1, 1, 140, 32), off, (0, 0, pitch, 1)))
    out, lse = Tensor.crossAttention(G.ofNumpy(q), mk(64), mk(96))
    o = Oracle(q, k, v, None, float(np.float32(1 / np.sqrt(32))), unit(np.float32))
    within(G.toNumpy(out), o.out, o.out_bound(), "out")
    grads = Tensor.crossAttentionGrad(G.ofNumpy(do), G.ofNumpy(q), mk(64), mk(96), out, lse)
    for g, (ref, bound), what in zip(grads, o.grad(do, G.toNumpy(out), G.toNumpy(lse)), ("d_q", "d_k", "d_v")):
        within(G.toNumpy(g), ref, bound, what)


@pytest.mark.parametrize("dt, shape", [(np.float32, (1, 16, 16, 379, 706, 96, 1)), (np.float32, (1, 8, 8, 557, 764, 128, 16)), (np.float32, (1, 8, 8, 120, 2000, 8, 96)),
                                       (np.float64, (1, 16, 16, 604, 390, 8, 96)), (np.float64, (1, 4, 4, 142, 1171, 128, 8)), (np.float64, (2, 2, 2, 1, 3000, 3, 100))])
def test_scratch_that_was_asked_for_suffices_for_unlike_widths(G, rng, dt, shape):
    B, H, Hk, Lq, Lk, Dk, Dv = shape
    q, k, v, do = inputs(rng, dt, *shape)
    Q, K, V, DO = (G.ofNumpy(t) for t in (q, k, v, do))
    scratch = G.zeros([G.scratchBytes("cross_attention", dt, B, H, Hk, Lq, Lk, max(Dk, Dv))], np.uint8)
    o = Oracle(q, k, v, None, float(dt(1 / np.sqrt(Dk))), unit(dt))
    out, lse = G.zeros([B, H, Lq, Dv], dt), G.zeros([B, H, Lq], dt)
    out.FillCrossAttention(Q, K, V, lse=lse, scratch=scratch)
    within(G.toNumpy(out), o.out, o.out_bound(), "out")
    grads = [G.zeros(list(t.shape), dt) for t in (q, k, v)]
    Tensor.FillCrossAttentionGrad(*grads, DO, Q, K, V, out, lse, scratch=scratch)
    for g, (ref, bound), what in zip(grads, o.grad(do, G.toNumpy(out), G.toNumpy(lse)), ("d_q", "d_k", "d_v")):
        within(G.toNumpy(g), ref, bound, what)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("Lq, D", [(1, 20), (1, 72), (70, 20), (70, 72), (1, 7)])
def test_a_key_that_scores_minus_infinity(G, rng, dt, Lq, D):
    """Such a key has probability 0, at widths that fill no instruction too: what is computed beyond the width must not meet it."""
    q, k, v, do = inputs(rng, dt, 1, 2, 2, Lq, 45, D, D)
    q = np.abs(q)                              # an infinity of the keys times any of these is that infinity
    k[:, :, 7, 0] = k[:, :, 40, 0] = -np.inf
    mask = np.ones((1, 45), bool)
    mask[0, [7, 40]] = False                   # the oracle leaves them out
    o = Oracle(q, k, v, mask, float(dt(1 / np.sqrt(D))), unit(dt))
    out, lse = Tensor.crossAttention(*(G.ofNumpy(t) for t in (q, k, v)))
    within(G.toNumpy(out), o.out, o.out_bound(), "out")
    within(G.toNumpy(lse), o.lse, o.lse_bound(), "lse")


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("bad", [np.inf, np.nan])
def test_masked_keys_have_no_gradient_whatever_is_upstream(G, rng, dt, bad):
    q, k, v, do = inputs(rng, dt, 2, 2, 1, 40, 90, 24, 24)
    mask = np.arange(90)[None, :] < np.array([[50], [71]])
    do[0, 1, 3, 5] = bad
    Q, K, V, DO, M = (G.ofNumpy(t) for t in (q, k, v, do, mask))
    out, lse = Tensor.crossAttention(Q, K, V, M)
    dq, dk, dv = (G.toNumpy(t) for t in Tensor.crossAttentionGrad(DO, Q, K, V, out, lse, M))
    for t in (dk, dv):
        assert (t[~np.broadcast_to(mask[:, None], t.shape[:3])] == 0).all()
        assert np.isfinite(t[1]).all()         # the other sequence is not touched by it
    assert np.isfinite(dq[1]).all() and np.isfinite(dq[0, 0]).all() and not np.isfinite(dq[0, 1, 3]).any()


@pytest.mark.parametrize("shape", [(1, 4, 2, 70, 150, 16, 24), (1, 2, 2, 40, 333, 64, 64), (1, 1, 1, 130, 90, 128, 128)])
def test_elements_that_have_no_bf16_parts(G, rng, shape):
    """Single precision: 2^127 and more, which rounds to an infinity in fewer bits; here in the values, with small upstream gradients."""
    q, k, v, do = inputs(rng, np.float32, *shape)
    v[0, 0, 5, 3] = 3e38
    v[0, -1, -1, 0] = -2e38
    compare(G, q, k, v, do * np.float32(1e-30))


@pytest.mark.parametrize("dt", TYPES)
def test_a_walk_longer_than_the_mask_words_kept_at_a_time(G, rng, dt):
    """More sequences than workgroups fit at once, so that each is one walk; they share the same keys and values (a broadcast view)."""
    B, Lq, Lk, D = 2100, 40, 8300, 4
    q, k, v, do = inputs(rng, dt, 1, 1, 1, Lq, Lk, D, D)
    mask = np.ones((B, Lk), bool)
    mask[:, 100:8200] = False
    mask[1, :] = False
    mask[1, 8290:] = True
    mask[2, :] = False
    mask[3, :] = True
    Q, K, V, DO = (G.ofNumpy(t).broadcastTo([B, 1, t.shape[2], D]) for t in (q, k, v, do))
    M = G.ofNumpy(mask)
    out, lse = Tensor.crossAttention(Q, K, V, M)
    dq = G.zeros([B, 1, Lq, D], dt)
    Tensor.FillCrossAttentionGrad(dq, None, None, DO, Q, K, V, out, lse, M)
    for b in (0, 1, 2, 3, B - 1):
        o = Oracle(q, k, v, mask[b:b + 1], float(dt(1 / np.sqrt(D))), unit(dt))
        go, gl, gq = (G.toNumpy(t[b:b + 1]) for t in (out, lse, dq))
        within(go, o.out, o.out_bound(), "out")
        within(gl, o.lse, o.lse_bound(), "lse")
        ref, bound = o.grad(do, go, gl)[0]
        within(gq, ref, bound, "d_q")


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("Lq, H, Hk", [(37, 6, 2), (64, 4, 1), (31, 5, 1)])
def test_tiles_that_cross_the_heads_of_a_group(G, rng, dt, Lq, H, Hk):
    """[B; L; H; D] tensors: a tile of 32 rows of a shared key head ends in the next query head, whose rows lie before those of the first one."""
    q, k, v, do = inputs(rng, dt, 2, H, Hk, Lq, 75, 16, 32)
    compare(G, q, k, v, do, up=lambda t: G.ofNumpy(np.ascontiguousarray(t.transpose(0, 2, 1, 3))).permuteAxes([0, 2, 1, 3]))


@pytest.mark.parametrize("dt", TYPES)
def test_rows_far_apart(G, rng, dt):
    """Rows of a tile more than 2^31 bytes apart: keys of every 2^25th element, many query rows."""
    q, k, v, do = inputs(rng, dt, 1, 1, 1, 50, 40, 32, 32)
    pitch = 1 << 25
    cache = Tensor.new([40, pitch], G.Dev, dt)
    cache[:, 64:96] = G.ofNumpy(k[0, 0])
    cache[:, 96:128] = G.ofNumpy(v[0, 0])
    mk = lambda off: cache.Relayout(type(cache.Layout)((1, 1, 40, 32), off, (0, 0, pitch, 1)))
    out, lse = Tensor.crossAttention(G.ofNumpy(q), mk(64), mk(96))
    o = Oracle(q, k, v, None, float(dt(1 / np.sqrt(32))), unit(dt))
    within(G.toNumpy(out), o.out, o.out_bound(), "out")
    grads = Tensor.crossAttentionGrad(G.ofNumpy(do), G.ofNumpy(q), mk(64), mk(96), out, lse)
    for g, (ref, bound), what in zip(grads, o.grad(do, G.toNumpy(out), G.toNumpy(lse)), ("d_q", "d_k", "d_v")):
        within(G.toNumpy(g), ref, bound, what)


def test_elements_whose_last_part_is_a_denormal(G, rng):
    """One key: out is its value.  Below 2^-109 the last of three bf16 parts has bits under 2^-133, the least bf16 has: off by half of it."""
    q, k, v, do = inputs(rng, np.float32, 1, 1, 1, 70, 1, 64, 64)
    v *= np.exp2(rng.integers(-120, -105, v.shape)).astype(np.float32)
    out, _ = Tensor.crossAttention(*(G.ofNumpy(t) for t in (q, k, v)))
    err = np.abs(G.toNumpy(out).astype(np.float64) - v[:, :, :1])
    assert (err <= 2.0 ** -134 + 2 * 2.0 ** -24 * np.abs(v[:, :, :1])).all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", [(1, 3, 1, 1, 40000, 16, 100), (1, 1, 1, 40, 20000, 32, 32), (2, 1, 1, 7, 9001, 5, 3)])
def test_long_sequences_in_many_shares(G, rng, dt, shape):
    """More than 64 shares; some of them without a key."""
    q, k, v, do = inputs(rng, dt, *shape)
    mask = np.ones((shape[0], shape[4]), bool)
    mask[0, 1000:7000] = False
    mask[-1, 8000:] = rng.random(shape[4] - 8000) < 0.7
    compare(G, q, k, v, do, mask, grads=False)
