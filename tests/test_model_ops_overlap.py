"""Targets of the language-model operators that share memory with a source or with each other are refused before any device work; views that
lie beside each other in one tensor are not (on the GPU, with real memory)."""
import numpy as np
import pytest

from deepnet_amd import abi
from deepnet_amd.tensor import Tensor

from test_model_ops_arguments import F32, F64, I64, refused

S = (None, None, 0)
PAGE = 1 << 30


def at(place, shape, dt=F32, stride=None, offset=0):
    """A view of the place-th of memory ranges that lie far apart."""
    if stride is None:
        stride, n = [], 1
        for s in reversed(shape):
            stride.insert(0, n)
            n *= max(s, 1)
    return abi.make_descriptor((place + 1) * PAGE, dt, shape, stride, offset)


def over(name, *args):
    refused(name, *args, says="overlaps")


def test_embedding():
    table, tok = at(0, [10, 8]), at(1, [5], I64)
    over("embedding", at(0, [5, 8]), table, tok, None)                       # the table's first rows
    over("embedding", at(0, [5, 8], offset=40), table, tok, None)            # its last ones
    over("embedding", at(0, [5, 8], offset=79), table, tok, None)
    over("embedding", at(0, [5, 8], offset=-39), table, tok, None)
    over("embedding", at(1, [5, 8]), table, tok, None)                       # other element sizes
    over("embedding", at(0, [5, 8], F64, offset=-1), at(0, [10, 8], F64), tok, None)
    over("embedding", at(0, [5, 8], stride=[16, 2]), table, tok, None)       # a corner
    over("embedding", at(0, [5, 8], stride=[-8, -1], offset=60), table, tok, None)
    over("embedding_grad", at(0, [10, 8]), tok, at(0, [5, 8], offset=8), None, 0, None, 0)
    over("embedding_grad", at(1, [10, 8]), tok, at(0, [5, 8]), None, 1, None, 0)


def test_token_log_probs():
    x, tok, row, top, idx = at(0, [4, 50]), at(1, [4], I64), at(2, [4]), at(3, [4, 3]), at(4, [4, 3], I64)
    over("token_log_probs", row, row, None, None, None, x, tok, None, 0)     # one target twice
    over("token_log_probs", row, at(0, [4], offset=7), None, None, None, x, tok, None, 0)
    over("token_log_probs", None, None, at(0, [4], stride=[50], offset=3), None, None, x, None, None, 0)    # a column of the logits
    over("token_log_probs", None, None, None, at(0, [4, 3], stride=[50, 1]), idx, x, None, None, 0)
    over("token_log_probs", row, None, None, top, at(1, [4, 3], I64), x, tok, None, 0)
    over("token_log_probs", None, row, None, top, at(3, [4, 3], I64), x, None, None, 0)
    # the gradient may take the logits' place, but no other view of them
    over("token_log_probs_grad", at(0, [4, 50], offset=50), x, tok, row, None, row, None)
    over("token_log_probs_grad", at(0, [4, 50], stride=[-50, 1], offset=150), x, tok, row, None, row, None)
    over("token_log_probs_grad", at(2, [4, 50]), x, tok, row, None, row, None)


def test_cross_attention():
    q, k, v, o, l = at(0, [2, 4, 5, 8]), at(1, [2, 2, 7, 8]), at(2, [2, 2, 7, 8]), at(3, [2, 4, 5, 8]), at(4, [2, 4, 5])
    over("cross_attention", q, l, q, k, v, None, *S)                         # in place
    over("cross_attention", at(2, [2, 4, 5, 8], offset=100), l, q, k, v, None, *S)
    over("cross_attention", o, at(3, [2, 4, 5]), q, k, v, None, *S)
    over("cross_attention", o, at(0, [2, 4, 5]), q, k, v, None, *S)
    over("cross_attention", at(0, [2, 4, 5, 8], stride=[160, 8, 32, 1]), l, q, k, v, None, *S)       # the same memory, other axes
    dq, dk, dv, do = at(5, [2, 4, 5, 8]), at(6, [2, 2, 7, 8]), at(7, [2, 2, 7, 8]), at(8, [2, 4, 5, 8])
    over("cross_attention_grad", dq, dk, dk, do, q, k, v, o, l, None, *S)
    over("cross_attention_grad", q, dk, dv, do, q, k, v, o, l, None, *S)
    over("cross_attention_grad", do, dk, dv, do, q, k, v, o, l, None, *S)
    over("cross_attention_grad", None, dk, v, do, q, k, v, o, l, None, *S)
    over("cross_attention_grad", at(4, [2, 4, 5, 8]), dk, dv, do, q, k, v, o, l, None, *S)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [np.float32, np.float64])
def test_views_beside_each_other_are_taken(G, rng, dt):
    """Everything an attention call has, and its gradient, as columns of two tensors; rows of logits between each other; ranges that meet, end to end."""
    B, L, H, D = 2, 9, 2, 8
    one = rng.standard_normal((B, L, 5, H, D)).astype(dt)
    one[:, :, 4] = 0
    X, Y = G.ofNumpy(one), G.zeros([B, L, 3, H, D], dt)
    view = lambda t, i: t[:, :, i].permuteAxes([0, 2, 1, 3])
    q, k, v, do, out = (view(X, i) for i in range(5))
    lse = G.zeros([B, H, L], dt)
    out.FillCrossAttention(q, k, v, lse=lse)
    apart = [G.ofNumpy(np.ascontiguousarray(one[:, :, i].transpose(0, 2, 1, 3))) for i in range(4)]
    o2, l2 = Tensor.crossAttention(*apart[:3])
    np.testing.assert_array_equal(G.toNumpy(out), G.toNumpy(o2))
    np.testing.assert_array_equal(G.toNumpy(lse), G.toNumpy(l2))
    Tensor.FillCrossAttentionGrad(view(Y, 0), view(Y, 1), view(Y, 2), do, q, k, v, out, lse)
    for i, g in enumerate(Tensor.crossAttentionGrad(apart[3], *apart[:3], o2, l2)):
        np.testing.assert_array_equal(G.toNumpy(view(Y, i)), G.toNumpy(g))
    # logits and their gradient row by row in turn, and in place
    pair = G.ofNumpy(rng.standard_normal((6, 2, 50)).astype(dt))
    tok, g = G.ofNumpy(rng.integers(0, 50, 6)), G.ofNumpy(rng.standard_normal(6).astype(dt))
    _, row_lse, _ = Tensor.tokenLogProbs(pair[:, 0], tok)
    want = G.toNumpy(Tensor.tokenLogProbsGrad(pair[:, 0], tok, row_lse, g))
    pair[:, 1].FillTokenLogProbsGrad(pair[:, 0], tok, row_lse, g)
    np.testing.assert_array_equal(G.toNumpy(pair[:, 1]), want)
    pair[:, 0].FillTokenLogProbsGrad(pair[:, 0], tok, row_lse, g)
    np.testing.assert_array_equal(G.toNumpy(pair[:, 0]), want)
    # a table and, right behind it, its rows
    block = G.ofNumpy(rng.standard_normal((20, 4)).astype(dt))
    block[10:16].FillEmbedding(block[:10], G.ofNumpy(np.arange(6)), 2.0)
    np.testing.assert_array_equal(G.toNumpy(block[10:16]), G.toNumpy(block[:6]) * dt(2))
