"""Which stream learns of a token outside the table when the call was captured into a graph."""
import ctypes as C

import numpy as np
import pytest

from deepnet_amd import abi, native

from test_gpu_model_run import _hip, capture

pytestmark = pytest.mark.gpu


def stream():
    s = C.c_void_p()
    native.check(native.load().dnh_stream_create(C.byref(s)))
    return s


def error_of(s):
    code = C.c_int32()
    native.check(native.load().dnh_async_error(s, C.byref(code)))
    return code.value


def test_a_graph_does_not_report_to_a_stream_that_came_later(G, rng):
    hip, lib = _hip(), native.load()
    table = rng.standard_normal((10, 8)).astype(np.float32)
    T, K, bad, out = G.ofNumpy(table), G.ofNumpy(np.arange(5)), G.ofNumpy(np.array([3, 10, 4])), G.zeros([5, 8], np.float32)
    G.synchronize()
    d = lambda t: t.Backend._opt(t)

    def call(s, target, tokens):
        native.check(lib.dnh_embedding(d(target), d(T), d(tokens), None, s))

    a = stream()
    graph, gexec = capture(hip, a, lambda: call(a, out[0:3], bad))
    assert hip.hipGraphLaunch(gexec, a) == 0
    assert error_of(a) == abi.DNH_ERR_INDEX_OUT_OF_RANGE     # reported where it was captured, and cleared
    assert error_of(a) == abi.DNH_OK
    b = stream()
    assert hip.hipGraphLaunch(gexec, b) == 0
    native.check(lib.dnh_stream_sync(b))
    assert error_of(b) == abi.DNH_OK and error_of(a) == abi.DNH_ERR_INDEX_OUT_OF_RANGE
    native.check(lib.dnh_stream_destroy(a))
    later = [stream() for _ in range(3)]
    try:
        for s in later:                                      # each takes a word of its own
            call(s, out, K)
            assert error_of(s) == abi.DNH_OK
        for s in later:
            assert hip.hipGraphLaunch(gexec, s) == 0
            native.check(lib.dnh_stream_sync(s))
            assert [error_of(x) for x in later] == [abi.DNH_OK] * 3
        call(later[0], out[0:3], bad)                        # their own errors they do report
        assert error_of(later[0]) == abi.DNH_ERR_INDEX_OUT_OF_RANGE and error_of(later[1]) == abi.DNH_OK
    finally:
        hip.hipGraphExecDestroy(gexec)
        hip.hipGraphDestroy(graph)
        for s in [b, *later]:
            native.check(lib.dnh_stream_destroy(s))


def test_a_word_that_no_graph_has_is_cleared_for_the_next_stream(G):
    lib = native.load()
    T, bad, out = G.zeros([10, 8], np.float32), G.ofNumpy(np.array([3, 10, 4])), G.zeros([3, 8], np.float32)
    G.synchronize()
    a = stream()
    native.check(lib.dnh_embedding(*(t.Backend._opt(t) for t in (out, T, bad)), None, a))
    native.check(lib.dnh_stream_destroy(a))
    b = stream()
    native.check(lib.dnh_embedding(*(t.Backend._opt(t) for t in (out[0:1], T, bad[0:1])), None, b))
    assert error_of(b) == abi.DNH_OK
    native.check(lib.dnh_stream_destroy(b))
