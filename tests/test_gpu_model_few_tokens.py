"""The embedding's gradient of up to 512 tokens, captured into a graph without scratch memory."""
import numpy as np
import pytest

from test_gpu_model_embedding import check_grad
from test_gpu_model_run import OnStream, _hip, capture

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [np.float32, np.float64])
@pytest.mark.parametrize("accumulate", [False, True])
def test_captured_without_scratch_memory(G, rng, dt, accumulate):
    hip = _hip()
    with OnStream(G) as s:
        sets = []
        for n, vocab, width in ((1, 9, 5), (512, 700, 36), (500, 40, 130)):
            tok, g, base = rng.integers(0, vocab, n), rng.standard_normal((n, width)).astype(dt), rng.standard_normal((vocab, width)).astype(dt)
            sets.append((G.ofNumpy(tok), G.ofNumpy(g), G.ofNumpy(base), G.ofNumpy(base), tok, g, base))
        G.synchronize()

        def issue():
            for K, D, d, *_ in sets:
                d.FillEmbeddingGrad(K, D, 1.7, accumulate)

        graph, gexec = capture(hip, s, issue)
        for rep in range(3):
            for K, D, d, b, *_ in sets:
                d.CopyFrom(b)
            G.synchronize()
            assert hip.hipGraphLaunch(gexec, s) == 0
            G.synchronize()
            for K, D, d, b, tok, g, base in sets:
                got = G.toNumpy(d)
                check_grad(got, tok, g, len(base), 1.7, base if accumulate else None)
                d.CopyFrom(b)                                # the eager call gives the same bits
                d.FillEmbeddingGrad(K, D, 1.7, accumulate)
                np.testing.assert_array_equal(G.toNumpy(d), got)
        hip.hipGraphExecDestroy(gexec)
        hip.hipGraphDestroy(graph)
