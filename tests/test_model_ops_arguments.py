"""CPU: what the language-model operators refuse, and the scratch memory they ask for.  Every refusal comes before any device work, so
the descriptors here need no memory behind them."""
import ctypes as C

import numpy as np
import pytest

from deepnet_amd import abi, native

F32, F64, I64, I32, BOOL = np.float32, np.float64, np.int64, np.int32, np.bool_


def d(shape, dt=F32, stride=None, base=4096):
    if stride is None:
        stride, n = [], 1
        for s in reversed(shape):
            stride.insert(0, n)
            n *= max(s, 1)
    return abi.make_descriptor(base, dt, shape, stride, 0)


def call(name, *args):
    refs = [C.byref(a) if isinstance(a, abi.DnhTensor) else a for a in args]
    return getattr(native.load(), "dnh_" + name)(*refs, None)


def refused(name, *args, status=abi.DNH_ERR_INVALID_ARG, says=""):
    assert call(name, *args) == status, native.last_error()
    assert says in native.last_error(), native.last_error()


NOT = abi.DNH_ERR_NOT_SUPPORTED


def test_embedding():
    t, table, tok = d([5, 8]), d([10, 8]), d([5], I64)
    refused("embedding", None, table, tok, None, says="null")
    refused("embedding", t, None, tok, None, says="null")
    refused("embedding", t, table, None, None, says="null")
    refused("embedding", t, table, d([5], I32), None, says="int64")
    refused("embedding", d([5, 8], F64), table, tok, None, says="single")
    refused("embedding", d([5, 8], I32), d([10, 8], I32), tok, None, status=NOT)
    refused("embedding", d([5, 7]), table, tok, None, says="row length")
    refused("embedding", d([4, 8]), table, tok, None, says="shape")
    refused("embedding", d([5]), table, tok, None, says="shape")
    refused("embedding", t, d([10, 2, 4]), tok, None, says="matrix")
    refused("embedding", d([5, 8], stride=[0, 1]), table, tok, None, says="broadcast")
    refused("embedding", d([5, 8], base=0), table, tok, None, says="null base")
    big = 1 << 31
    refused("embedding", d([big, 1]), d([10, 1]), d([big], I64), None, status=NOT, says="rows")
    refused("embedding", t, d([big, 8]), tok, None, status=NOT, says="rows")
    refused("embedding", d([5, 1 << 24]), d([10, 1 << 24]), tok, None, status=NOT)
    refused("embedding_grad", table, tok, t, None, 2, None, 0, says="accumulate")
    refused("embedding_grad", d([10, 8], stride=[0, 1]), tok, t, None, 0, None, 0, says="broadcast")
    refused("embedding_grad", table, tok, d([6, 8]), None, 0, None, 0, says="shape")
    refused("embedding_grad", d([10, 1]), d([1 << 28], I64), d([1 << 28, 1]), None, 0, None, 0, status=NOT, says="tokens")


def test_token_log_probs():
    x, tok, row, top, idx = d([4, 50]), d([4], I64), d([4]), d([4, 3]), d([4, 3], I64)
    S = (None, 0)
    refused("token_log_probs", row, row, row, top, idx, None, tok, *S, says="null")
    refused("token_log_probs", None, None, None, None, None, x, None, *S, says="nothing")
    refused("token_log_probs", row, None, None, None, None, x, None, *S, says="together")
    refused("token_log_probs", None, row, None, None, None, x, tok, *S, says="together")
    refused("token_log_probs", None, row, None, top, None, x, None, *S, says="together")
    refused("token_log_probs", row, None, None, None, None, x, d([4], I32), *S, says="int64")
    refused("token_log_probs", row, None, None, None, None, x, d([5], I64), *S, says="shape")
    refused("token_log_probs", d([4], F64), None, None, None, None, x, tok, *S, says="single")
    refused("token_log_probs", None, d([4, 1]), None, None, None, x, None, *S, says="shape")
    refused("token_log_probs", None, None, d([4], stride=[0]), None, None, x, None, *S, says="broadcast")
    refused("token_log_probs", None, None, None, top, d([4, 3]), x, None, *S, says="int64")
    refused("token_log_probs", None, None, None, d([4, 2]), idx, x, None, *S, says="alternatives")
    refused("token_log_probs", None, None, None, d([4, 51]), d([4, 51], I64), x, None, *S, says="51 alternatives of 50")
    refused("token_log_probs", None, None, None, d([4, 65]), d([4, 65], I64), d([4, 500]), None, *S, status=NOT, says="64")
    refused("token_log_probs", None, d([4], I32), None, None, None, d([4, 50], I32), None, *S, status=NOT)
    refused("token_log_probs", None, row, None, None, None, d([4, 0]), None, *S, says="without logits")
    refused("token_log_probs", None, d([]), None, None, None, d([]), None, *S, says="last axis")
    refused("token_log_probs", None, d([1 << 24]), None, None, None, d([1 << 24, 2]), None, *S, status=NOT, says="rows")
    refused("token_log_probs", None, d([1]), None, None, None, d([1, 1 << 31]), None, *S, status=NOT)
    g = d([4, 50])
    refused("token_log_probs_grad", None, x, tok, row, None, row, None, says="null")
    refused("token_log_probs_grad", g, x, None, row, None, row, None, says="null")
    refused("token_log_probs_grad", g, x, tok, None, None, row, None, says="null")
    refused("token_log_probs_grad", g, x, tok, row, None, None, None, says="null")
    refused("token_log_probs_grad", g, x, tok, row, row, row, None, says="together")
    refused("token_log_probs_grad", d([4, 49]), x, tok, row, None, row, None, says="shape")
    refused("token_log_probs_grad", d([4, 50], stride=[50, 0]), x, tok, row, None, row, None, says="broadcast")
    refused("token_log_probs_grad", g, x, tok, d([3]), None, row, None, says="shape")
    refused("token_log_probs_grad", g, x, tok, row, None, d([4], F64), None, says="single")


def test_cross_attention():
    q, k, v, o, l = d([2, 4, 5, 8]), d([2, 2, 7, 8]), d([2, 2, 7, 6]), d([2, 4, 5, 6]), d([2, 4, 5])
    S = (None, None, 0)
    f = lambda *a, **kw: refused("cross_attention", *a, *S, **kw)
    f(None, l, q, k, v, None, says="null")
    f(o, l, None, k, v, None, says="null")
    f(o, l, q, k, d([2, 2, 7, 6], F64), None, says="single")
    f(d([2, 4, 5, 6], I32), None, d([2, 4, 5, 8], I32), d([2, 2, 7, 8], I32), d([2, 2, 7, 6], I32), None, status=NOT)
    f(o, l, d([4, 5, 8]), k, v, None, says="rank")
    f(o, l, d([3, 4, 5, 8]), k, v, None, says="batch")
    f(o, l, q, k, d([2, 2, 6, 6]), None, says="positions")
    f(o, l, q, d([2, 2, 7, 9]), v, None, says="width")
    f(o, l, d([2, 3, 5, 8]), k, v, None, says="share")
    f(o, l, q, d([2, 0, 7, 8]), d([2, 0, 7, 6]), None, says="share")
    f(d([2, 4, 5, 5]), l, q, k, v, None, says="out")
    f(d([2, 4, 5, 6], stride=[120, 30, 0, 1]), l, q, k, v, None, says="broadcast")
    f(o, d([2, 4, 6]), q, k, v, None, says="lse")
    f(o, l, q, k, v, d([2, 7]), says="mask")
    f(o, l, q, k, v, d([2, 8], BOOL), says="mask")
    f(d([2, 4, 5, 129]), l, q, k, d([2, 2, 7, 129]), None, status=NOT, says="128")
    f(d([2, 4, 5, 0]), l, q, k, d([2, 2, 7, 0]), None, says="width")
    f(d([1, 1, 1 << 31, 1]), None, d([1, 1, 1 << 31, 1]), d([1, 1, 1, 1]), d([1, 1, 1, 1]), None, status=NOT)
    f(d([1 << 12, 1 << 12, 1, 1]), None, d([1 << 12, 1 << 12, 1, 1]), d([1 << 12, 1 << 12, 1, 1]), d([1 << 12, 1 << 12, 1, 1]), None, status=NOT, says="tiles")
    g = lambda *a, **kw: refused("cross_attention_grad", *a, *S, **kw)
    g(q, k, v, None, q, k, v, o, l, None, says="null")
    g(None, None, None, o, q, k, v, o, l, None, says="nothing")
    g(q, k, None, o, q, k, v, o, l, None, says="together")
    g(d([2, 4, 5, 7]), k, v, o, q, k, v, o, l, None, says="d_q")
    g(q, d([2, 2, 7, 7]), v, o, q, k, v, o, l, None, says="d_k")
    g(q, k, d([2, 2, 7, 7]), o, q, k, v, o, l, None, says="d_v")
    g(q, k, v, o, q, k, v, o, None, None, says="null")
    g(q, k, v, d([2, 4, 5, 7]), q, k, v, o, l, None, says="d_out")


def test_scratch_queries():
    """They touch no device; sizes grow with the work, are zero where none is needed, and refuse what the operators refuse."""
    lib, n = native.load(), C.c_size_t()

    def ask(name, *args):
        native.check(getattr(lib, f"dnh_{name}_scratch_bytes")(*args, C.byref(n)))
        return n.value

    assert ask("embedding_grad", 0, 10, 10) == 0 and ask("embedding_grad", 100, 10, 0) == 0
    # two lists of 32-bit numbers and two partial rows of doubles for every piece of 8 tokens
    assert ask("embedding_grad", 1024, 100, 16) == 2 * 4096 + 128 * 2 * 16 * 8
    assert ask("embedding_grad", 1 << 20, 50000, 64) > ask("embedding_grad", 1 << 16, 50000, 64)
    assert ask("token_log_probs", abi.DNH_F32, 5000, 50000, 5) == 0 and ask("token_log_probs", abi.DNH_F32, 1, 1000, 5) == 0
    assert ask("token_log_probs", abi.DNH_F64, 1, 128000, 20) > 0
    assert ask("cross_attention", abi.DNH_F32, 0, 4, 2, 5, 7, 8) == 0
    assert ask("cross_attention", abi.DNH_F32, 1, 4, 4, 1, 4000, 64) > 4 * 64 * 4
    for name, bad in (("embedding_grad", (-1, 1, 1)), ("embedding_grad", (1 << 28, 1, 1)), ("embedding_grad", (1, 1 << 31, 1)),
                      ("token_log_probs", (abi.DNH_I32, 1, 1, 0)), ("token_log_probs", (abi.DNH_F32, 1, 1, 65)),
                      ("cross_attention", (abi.DNH_F32, 1, 3, 2, 1, 1, 8)), ("cross_attention", (abi.DNH_F32, 1, 2, 0, 1, 1, 8)),
                      ("cross_attention", (abi.DNH_F32, 1, 2, 2, 1, 1, 129))):
        assert getattr(lib, f"dnh_{name}_scratch_bytes")(*bad, C.byref(n)) == abi.DNH_ERR_INVALID_ARG
    assert lib.dnh_embedding_grad_scratch_bytes(1, 1, 1, None) == abi.DNH_ERR_INVALID_ARG


def test_not_available_on_the_host_device(H):
    from deepnet_amd.tensor import Tensor
    with pytest.raises(NotImplementedError):
        Tensor.embedding(H.ofNumpy(np.zeros((3, 2), F32)), H.ofNumpy(np.zeros(2, I64)))


def test_extents_of_attention():
    """Large work that fits the grids is taken (the query is answered), what does not fit is refused by the query and by the call alike."""
    lib, n = native.load(), C.c_size_t()
    assert lib.dnh_cross_attention_scratch_bytes(abi.DNH_F32, 64, 16, 16, 1 << 16, 1 << 16, 64, C.byref(n)) == abi.DNH_OK
    assert lib.dnh_cross_attention_scratch_bytes(abi.DNH_F32, 128, 64, 64, 1 << 16, 1 << 16, 64, C.byref(n)) == NOT
    assert lib.dnh_cross_attention_scratch_bytes(abi.DNH_F64, 1 << 40, 1 << 20, 1, 1 << 40, 1 << 40, 64, C.byref(n)) == NOT
    big = [128, 64, 1 << 16, 4]
    refused("cross_attention", d(big), None, d(big), d(big), d(big), None, None, None, 0, status=NOT, says="tiles")


def test_the_memory_of_a_shared_walk_stays_bounded():
    """Parts of at most 256 MB: work that fills the chip by itself is not cut into shares for the sake of its end."""
    lib, n = native.load(), C.c_size_t()
    for args in ((16, 16, 16, 8000, 1 << 20, 64), (1, 128, 128, 16000, 1 << 18, 128)):
        native.check(lib.dnh_cross_attention_scratch_bytes(abi.DNH_F32, *args, C.byref(n)))
        rows = args[0] * args[1] * args[3]
        assert n.value <= (1 << 28) + rows * 4 * 4
