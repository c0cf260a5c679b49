"""The language-model operators as a program uses them: one training step of a small decoder over encoder states, its gradients against
differences; the same calls captured into graphs and replayed; on streams of their own and from several host threads."""
import ctypes as C
import threading

import numpy as np
import pytest

from deepnet_amd import native
from deepnet_amd.tensor import Tensor

pytestmark = pytest.mark.gpu


class Step:
    """Tokens -> embedding -> attention to encoder states (+ the embedding) -> logits on the same table -> log probabilities, and back."""

    def __init__(self, G, rng, dt, B=2, L=5, H=2, D=8, V=23, S=9):
        self.G, self.dt, self.shape = G, dt, (B, L, H, D, V, S)
        self.table = rng.standard_normal((V, H * D)).astype(dt)
        self.enc = rng.standard_normal((B, S, 2 * D)).astype(dt)     # keys and values of one shared head, side by side
        self.tok, self.nxt = rng.integers(0, V, (B, L)), rng.integers(0, V, (B, L))
        self.mask = np.arange(S)[None, :] < rng.integers(2, S + 1, (B, 1))
        self.g, self.h = rng.standard_normal((B, L)).astype(dt), rng.standard_normal((B, L)).astype(dt)

    def heads(self, x, n):
        B, L, H, D, V, S = self.shape
        return x.reshape([B, x.Shape[1], n, D]).permuteAxes([0, 2, 1, 3])

    def forward(self, table, enc):
        B, L, H, D, V, S = self.shape
        G = self.G
        T, E, K, M = G.ofNumpy(table), G.ofNumpy(enc), G.ofNumpy(self.tok), G.ofNumpy(self.mask)
        x = Tensor.embedding(T, K, np.sqrt(H * D))
        q = self.heads(x, H)
        k, v = self.heads(E[:, :, :D], 1), self.heads(E[:, :, D:], 1)
        out, lse = Tensor.crossAttention(q, k, v, M)
        y = x + out.permuteAxes([0, 2, 1, 3]).reshape([B, L, H * D])
        logits = (y.reshape([B * L, H * D]) @ T.T).reshape([B, L, V])
        lp, row_lse, ent, tv, ti = Tensor.tokenLogProbs(logits, G.ofNumpy(self.nxt), 3)
        return T, E, K, M, x, q, k, v, out, lse, y, logits, lp, row_lse, ent, tv, ti

    def value(self, table, enc):
        r = self.forward(table, enc)
        return float((self.g * self.G.toNumpy(r[12]) + self.h * self.G.toNumpy(r[14])).sum())

    def gradients(self):
        B, L, H, D, V, S = self.shape
        G = self.G
        T, E, K, M, x, q, k, v, out, lse, y, logits, lp, row_lse, ent, tv, ti = self.forward(self.table, self.enc)
        d_logits = Tensor.tokenLogProbsGrad(logits, G.ofNumpy(self.nxt), row_lse, G.ofNumpy(self.g), ent, G.ofNumpy(self.h)).reshape([B * L, V])
        d_table = d_logits.T @ y.reshape([B * L, H * D])
        d_y = (d_logits @ T).reshape([B, L, H * D])
        dq, dk, dv = Tensor.crossAttentionGrad(self.heads(d_y, H), q, k, v, out, lse, M)
        d_x = d_y + dq.permuteAxes([0, 2, 1, 3]).reshape([B, L, H * D])
        d_table.FillEmbeddingGrad(K, d_x, np.sqrt(H * D), accumulate=True)
        d_enc = G.zeros(list(self.enc.shape), self.dt)
        d_enc[:, :, :D], d_enc[:, :, D:] = dk[:, 0], dv[:, 0]
        return G.toNumpy(d_table), G.toNumpy(d_enc)


def test_gradients_of_a_step_against_differences(G, rng):
    s = Step(G, rng, np.float64)
    got = s.gradients()
    step = 1e-6     # central differences: step^2 |f'''| / 6 ~ 1e-12 x thousands, rounding 2^-52 x 1e2 / step ~ 2e-8: bound 1e-6 x (1 + |d|)
    for which, base in enumerate((s.table, s.enc)):
        for at in [tuple(rng.integers(0, n) for n in base.shape) for _ in range(40)]:
            args = [[s.table.copy(), s.enc.copy()] for _ in range(2)]
            args[0][which][at] += step
            args[1][which][at] -= step
            d = (s.value(*args[0]) - s.value(*args[1])) / (2 * step)
            assert abs(d - got[which][at]) <= 1e-6 * (1 + abs(d)), (which, at, d, got[which][at])


def test_single_and_double_precision_agree(G, rng):
    """The step in single precision is a handful of sums of at most 32 products and one softmax: 1e-3 of each tensor's largest value is
    more than a thousand half steps (2^-24)."""
    s = Step(G, rng, np.float64)
    f = Step(G, rng, np.float32)
    for name in ("table", "enc", "g", "h"):
        x = getattr(s, name).astype(np.float32)
        setattr(f, name, x)
        setattr(s, name, x.astype(np.float64))
    f.tok, f.nxt, f.mask = s.tok, s.nxt, s.mask
    for a, b in zip(s.gradients(), f.gradients()):
        assert np.abs(a - b).max() <= 1e-3 * np.abs(a).max()


def _hip():
    hip = C.CDLL("libamdhip64.so")
    for f in ("hipStreamBeginCapture", "hipStreamEndCapture", "hipGraphInstantiate", "hipGraphLaunch", "hipGraphExecDestroy", "hipGraphDestroy"):
        getattr(hip, f).restype = C.c_int
    return hip


class Calls:
    """Every operator once, on tensors made beforehand; sizes that need scratch memory."""

    def __init__(self, G, rng, scratch=True):
        dt = np.float32
        n, vocab, width, V = 9000, 700, 36, 9000
        self.G = G
        up = lambda *s: G.ofNumpy(rng.standard_normal(s).astype(dt))
        self.table, self.d_rows, self.logits, self.q, self.k, self.v, self.do = up(vocab, width), up(n, width), up(3, V), up(2, 4, 1, 32), up(2, 2, 700, 32), up(2, 2, 700, 32), up(2, 4, 1, 32)
        self.tok, self.tok3 = G.ofNumpy(rng.integers(0, vocab, n)), G.ofNumpy(rng.integers(0, V, 3))
        self.g = up(3)
        z = lambda *s, t=dt: G.zeros(list(s), t)
        self.rows, self.d_table, self.lp, self.lse, self.ent, self.tv, self.ti = z(n, width), z(vocab, width), z(3), z(3), z(3), z(3, 5), z(3, 5, t=np.int64)
        self.d_logits, self.out, self.al, self.dq, self.dk, self.dv = z(3, V), z(2, 4, 1, 32), z(2, 4, 1), z(2, 4, 1, 32), z(2, 2, 700, 32), z(2, 2, 700, 32)
        self.inputs = [self.table, self.d_rows, self.logits, self.q, self.k, self.v, self.do]
        self.results = [self.rows, self.d_table, self.lp, self.lse, self.ent, self.tv, self.ti, self.d_logits, self.out, self.al, self.dq, self.dk, self.dv]
        sb = lambda *a: G.zeros([max(G.scratchBytes(*a), 16)], np.uint8) if scratch else None
        self.s1, self.s2, self.s3 = sb("embedding_grad", n, vocab, width), sb("token_log_probs", dt, 3, V, 5), sb("cross_attention", dt, 2, 4, 2, 1, 700, 32)

    def issue(self):
        self.rows.FillEmbedding(self.table, self.tok, 2.0)
        self.d_table.FillEmbeddingGrad(self.tok, self.d_rows, 2.0, scratch=self.s1)
        Tensor.FillTokenLogProbs(self.logits, self.tok3, self.lp, self.lse, self.ent, self.tv, self.ti, scratch=self.s2)
        self.d_logits.FillTokenLogProbsGrad(self.logits, self.tok3, self.lse, self.g, self.ent, self.g)
        self.out.FillCrossAttention(self.q, self.k, self.v, lse=self.al, scratch=self.s3)
        Tensor.FillCrossAttentionGrad(self.dq, self.dk, self.dv, self.do, self.q, self.k, self.v, self.out, self.al, scratch=self.s3)

    def snapshot(self):
        self.G.synchronize()
        return [self.G.toNumpy(t).copy() for t in self.results]

    def poison(self):
        for t in self.results:
            t.FillConst(t.DataType.type(-7))
        self.G.synchronize()

    def change(self):
        for t in self.inputs:
            t.FillMultiply(t, t.scalarLike(np.float32(-0.75)))
        self.G.synchronize()


class OnStream:
    def __init__(self, G):
        self.G, self.lib, self.s = G, native.load(), C.c_void_p()

    def __enter__(self):
        native.check(self.lib.dnh_stream_create(C.byref(self.s)))
        self.G.Cfg.Stream, self.G.Cfg.Stacktrace = self.s.value, False
        return self.s

    def __exit__(self, *exc):
        self.G.synchronize()
        self.G.Cfg.Stream, self.G.Cfg.Stacktrace = 0, True
        native.check(self.lib.dnh_stream_destroy(self.s))


def capture(hip, stream, issue):
    graph, gexec = C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 1) == 0      # thread-local mode
    try:
        issue()
    finally:
        rc = hip.hipStreamEndCapture(stream, C.byref(graph))
    assert rc == 0 and graph.value
    assert hip.hipGraphInstantiate(C.byref(gexec), graph, None, None, C.c_size_t(0)) == 0
    return graph, gexec


def test_two_graphs_replayed_with_eager_work_between(G, rng):
    """Both are captured on one stream that has run nothing before (nothing may be allocated meanwhile), each with scratch memory of its
    own, and replayed on two streams at once; every replay must give the eager calls' bits."""
    hip = _hip()
    with OnStream(G) as stream:
        sets = [Calls(G, rng), Calls(G, rng)]
        G.synchronize()
        graphs = [capture(hip, stream, c.issue) for c in sets]
        other = C.c_void_p()
        native.check(native.load().dnh_stream_create(C.byref(other)))
        try:
            for rep in range(4):
                for c in sets:
                    c.poison()
                assert hip.hipGraphLaunch(graphs[0][1], stream) == 0
                assert hip.hipGraphLaunch(graphs[1][1], other) == 0
                native.check(native.load().dnh_stream_sync(other))
                got = [c.snapshot() for c in sets]
                for c, g in zip(sets, got):
                    c.poison()
                    c.issue()
                    for a, b in zip(g, c.snapshot()):
                        np.testing.assert_array_equal(a, b)
                    c.change()
        finally:
            for graph, gexec in graphs:
                hip.hipGraphExecDestroy(gexec)
                hip.hipGraphDestroy(graph)
            native.check(native.load().dnh_stream_destroy(other))


def test_capture_without_scratch_memory_is_refused(G, rng):
    hip = _hip()
    with OnStream(G) as stream:
        c = Calls(G, rng, scratch=False)
        c.issue()                                        # eager: the stream's workspace
        G.synchronize()
        refused = []

        def issue():
            for f in (lambda: c.d_table.FillEmbeddingGrad(c.tok, c.d_rows),
                      lambda: Tensor.FillTokenLogProbs(c.logits, c.tok3, c.lp, topLogProbs=c.tv, topTokens=c.ti),
                      lambda: c.out.FillCrossAttention(c.q, c.k, c.v),
                      lambda: Tensor.FillCrossAttentionGrad(c.dq, None, None, c.do, c.q, c.k, c.v, c.out, c.al)):
                try:
                    f()
                except ValueError as e:
                    refused.append(str(e))
            c.rows.FillEmbedding(c.table, c.tok)         # needs none, and the capture goes on after the refusals

        graph, gexec = capture(hip, stream, issue)
        assert len(refused) == 4 and all("scratch" in r for r in refused)
        c.poison()
        assert hip.hipGraphLaunch(gexec, stream) == 0
        G.synchronize()
        np.testing.assert_array_equal(G.toNumpy(c.rows), G.toNumpy(c.table)[G.toNumpy(c.tok)])
        hip.hipGraphExecDestroy(gexec)
        hip.hipGraphDestroy(graph)


def test_host_threads_on_one_stream_and_on_streams_of_their_own(G, rng):
    sets = [Calls(G, rng, scratch=False) for _ in range(4)]
    want = []
    for c in sets:
        c.issue()
        want.append(c.snapshot())
        c.poison()
    errors = []

    def work(c, w, own):
        try:
            for _ in range(5):
                if own:
                    with OnStream(G):
                        c.issue()
                else:
                    c.issue()
                for a, b in zip(c.snapshot(), w):
                    np.testing.assert_array_equal(a, b)
        except BaseException as e:                       # noqa: BLE001 (reported by the main thread)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(c, w, i % 2 == 1)) for i, (c, w) in enumerate(zip(sets, want))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[0]
