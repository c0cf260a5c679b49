"""Timed cases of the language-model operators: token embedding and its gradient, token log probabilities and their gradient,
cross attention and its gradient.

Every case is a dict of plain values.  `prepare` makes a case's inputs on the GPU, `run` makes one pass through the operator: with
`own` false in its plain form (elementary torch operations), with `own` true through the entry points of libtensor_hip.so on
descriptors that the program keeps, as it keeps its buffers.  `exact` computes the same outputs in 64 bits from the definition.
"""
import math

import numpy as np
import torch

own = False

_T = {"float32": torch.float32, "float64": torch.float64}
_BYTES = {"float32": 4, "float64": 8}


# ---- cases ------------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one decoding step of 16 sequences: their newest tokens enter the model
        dict(name="embed_decode_step", op="embed", dtype="float32", tokens=16, vocab=32000, width=1024),
        # a training batch of 64 Ki tokens
        dict(name="embed_batch", op="embed", dtype="float32", tokens=65536, vocab=50000, width=1024),
        # a short ragged batch of a model trained in double precision, with a width that is no power of two
        dict(name="embed_grad_odd_f64", op="embed_grad", dtype="float64", tokens=4095, vocab=10007, width=300),
        # the embedding's gradient of a training batch; token frequencies fall off like 1 / rank
        dict(name="embed_grad_batch", op="embed_grad", dtype="float32", tokens=32768, vocab=50000, width=1024),
        # one sampled token of one sequence, with the alternatives that a serving interface shows
        dict(name="logprobs_one_row", op="logprobs", dtype="float32", rows=1, vocab=128000, pad=0, top=20),
        # scoring the tokens of a batch; the vocabulary is padded to a round size with columns that cannot be chosen
        dict(name="logprobs_batch", op="logprobs", dtype="float32", rows=4096, vocab=50048, pad=41, top=5),
        # gradient of log probability and entropy, ragged sizes, double precision
        dict(name="logprobs_grad_odd_f64", op="logprobs_grad", dtype="float64", rows=333, vocab=32003, pad=0),
        # the loss gradient of a training batch
        dict(name="logprobs_grad_batch", op="logprobs_grad", dtype="float32", rows=4096, vocab=50048, pad=41),
        # one decoding step of 16 sequences over encoder states of up to 2000 positions, four query heads on each key head
        dict(name="attend_decode_step", op="attend", dtype="float32", batch=16, heads=16, kv_heads=4, queries=1, keys=2000, width=64, blhd=True),
        # a batch of target sentences over encoder states of up to 1500 positions
        dict(name="attend_batch", op="attend", dtype="float32", batch=8, heads=16, kv_heads=16, queries=512, keys=1500, width=64, blhd=True),
        # training step of a wide-headed decoder block
        dict(name="attend_grad_batch", op="attend_grad", dtype="float32", batch=4, heads=16, kv_heads=16, queries=512, keys=1024, width=128, blhd=True),
        # ragged small training step in double precision, shared key heads
        dict(name="attend_grad_odd_f64", op="attend_grad", dtype="float64", batch=2, heads=6, kv_heads=2, queries=77, keys=333, width=40, blhd=False),
    ]


def _spread(rng, lo, hi):
    """An integer of [lo, hi], uniform over its logarithm; every other one is made odd."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:
        n |= 1
    return max(lo, min(hi, n))


def draw(rng):
    op = rng.choice(["embed", "embed_grad", "logprobs", "logprobs_grad", "attend", "attend_grad"])
    dtype = rng.choice(["float32", "float32", "float64"])
    half = 2 if dtype == "float64" else 1
    if op in ("embed", "embed_grad"):
        width = _spread(rng, 16, 2048)
        vocab = _spread(rng, 500, min(130000, 25_000_000 // width // half))
        tokens = _spread(rng, 1, min(65536, 30_000_000 // width // half))
        return dict(op=op, dtype=dtype, tokens=tokens, vocab=vocab, width=width)
    if op in ("logprobs", "logprobs_grad"):
        vocab = _spread(rng, 500, 130000)
        rows = _spread(rng, 1, min(4096, 100_000_000 // vocab // half))
        pad = rng.choice([0, rng.randrange(1, 100)])
        case = dict(op=op, dtype=dtype, rows=rows, vocab=vocab, pad=pad)
        if op == "logprobs":
            case["top"] = rng.choice([0, 1, 5, 20, 50])
        return case
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4])
    width = rng.choice([16, 32, 40, 64, 64, 80, 96, 128, 128, rng.randrange(9, 128)])
    batch = rng.choice([1, 2, 3, 8])
    keys = _spread(rng, 1, 4000)
    queries = _spread(rng, 1, max(1, min(1024, 3_000_000_000 // (batch * heads * keys * width) // half ** 2)))
    return dict(op=op, dtype=dtype, batch=batch, heads=heads, kv_heads=kv_heads, queries=queries, keys=keys, width=width,
                blhd=rng.random() < 0.5)


def work(case):
    s = _BYTES[case["dtype"]]
    op = case["op"]
    if op == "embed":
        n, d = case["tokens"], case["width"]
        # a row that several tokens name is read once: the expected number of different tokens
        rank = np.arange(case["vocab"], dtype=np.float64)
        p = np.log((rank + 2) / (rank + 1)) / math.log(case["vocab"] + 1)
        rows = int(round(float((1 - np.exp(n * np.log1p(-p))).sum())))
        return {"bytes": 8 * n + (rows + n) * d * s, "flops": n * d}
    if op == "embed_grad":
        n, d = case["tokens"], case["width"]
        return {"bytes": 8 * n + (n + case["vocab"]) * d * s, "flops": n * d}
    if op == "logprobs":
        r, v = case["rows"], case["vocab"]
        return {"bytes": r * v * s + r * (8 + 3 * s) + r * case["top"] * (8 + s), "flops": 6 * r * v}
    if op == "logprobs_grad":
        r, v = case["rows"], case["vocab"]
        return {"bytes": 2 * r * v * s + r * (8 + 4 * s), "flops": 6 * r * v}
    b, h, g, lq, lk, d = (case[k] for k in ("batch", "heads", "kv_heads", "queries", "keys", "width"))
    lk_seen = 3 * lk / 4                 # sequences fill between half and all of the padded length
    q_bytes, kv_bytes, lse_bytes = b * h * lq * d * s, b * g * lk * d * s, b * h * lq * s
    if op == "attend":
        return {"bytes": int(2 * q_bytes + 2 * 0.75 * kv_bytes + lse_bytes + b * lk), "flops": int(4 * b * h * lq * lk_seen * d)}
    return {"bytes": int(4 * q_bytes + (2 * 0.75 + 2) * kv_bytes + lse_bytes + b * lk), "flops": int(10 * b * h * lq * lk_seen * d)}


# ---- inputs -----------------------------------------------------------------------------------------------------------------

def _tokens(n, vocab, gen):
    """Token numbers whose frequency falls off like 1 / rank, the frequent ones first."""
    u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
    return (torch.exp(u * math.log(vocab + 1)).long() - 1).clamp_(0, vocab - 1)


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt, op = _T[case["dtype"]], case["op"]

    def normal(*shape, std=1.0):
        x = torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)
        if dt == torch.float64:          # all 53 bits of the significand in use
            x = x.double() + 1e-8 * torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)
        return x.mul_(std)

    if op in ("embed", "embed_grad"):
        n, v, d = case["tokens"], case["vocab"], case["width"]
        tokens = _tokens(n, v, gen)
        if op == "embed":
            return dict(table=normal(v, d, std=d ** -0.5), tokens=tokens, scale=math.sqrt(d))
        return dict(d_out=normal(n, d, std=0.1), tokens=tokens, scale=math.sqrt(d))
    if op in ("logprobs", "logprobs_grad"):
        r, v, pad = case["rows"], case["vocab"], case["pad"]
        logits = normal(r, v, std=2.5)
        if pad:
            logits[:, v - pad:] = -math.inf
        st = dict(logits=logits, tokens=_tokens(r, v - pad, gen))
        if op == "logprobs_grad":
            st["d_log_probs"] = normal(r, std=1.0 / r)
            st["d_entropy"] = normal(r, std=0.01 / r)
            st["lse"], st["entropy"] = _plain_statistics(logits)
        return st
    b, h, g, lq, lk, d = (case[k] for k in ("batch", "heads", "kv_heads", "queries", "keys", "width"))

    def heads(n, l):                     # a projection's output: heads side by side in each position's row, or heads first
        return normal(b, l, n, d).permute(0, 2, 1, 3) if case["blhd"] else normal(b, n, l, d)

    st = dict(q=heads(h, lq), k=heads(g, lk), v=heads(g, lk), scale=d ** -0.5)
    lengths = torch.randint((lk + 1) // 2, lk + 1, (b, 1), generator=gen, device="cuda")
    st["key_mask"] = torch.arange(lk, device="cuda")[None, :] < lengths
    if op == "attend_grad":
        st["d_out"] = heads(h, lq)
        st["out"], st["lse"] = _plain_attend(st)
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = case
    if own:
        _prepare_own(case, st)
    return st


# ---- the plain form -----------------------------------------------------------------------------------------------------------

def _plain_statistics(x):
    """lse and entropy of each row; a column that cannot be chosen (-inf) adds nothing to either."""
    m = x.max(dim=-1, keepdim=True).values
    z = x - m
    e = torch.exp(z)
    total = e.sum(dim=-1)
    zsum = torch.where(e > 0, e * z, torch.zeros_like(e)).sum(dim=-1)
    log_total = torch.log(total)
    return m[..., 0] + log_total, log_total - zsum / total


def _plain_logprobs(st, top):
    x, tokens = st["logits"], st["tokens"]
    lse, entropy = _plain_statistics(x)
    log_probs = torch.take_along_dim(x, tokens[:, None], dim=1)[:, 0] - lse
    if not top:
        return log_probs, lse, entropy
    # the k largest, one after the other; among equal ones the lowest index
    left = x.clone()
    index = torch.arange(x.shape[1], device=x.device)
    values, indices = [], []
    for _ in range(top):
        m = left.max(dim=1, keepdim=True).values
        i = torch.where(left == m, index, x.shape[1]).min(dim=1, keepdim=True).values
        values.append(m)
        indices.append(i)
        left.scatter_(1, i, -math.inf)
    return log_probs, lse, entropy, torch.cat(values, 1) - lse[:, None], torch.cat(indices, 1)


def _plain_logprobs_grad(st):
    x, lse, entropy = st["logits"], st["lse"][:, None], st["entropy"][:, None]
    log_p = x - lse
    p = torch.exp(log_p)
    p_log_p = torch.where(p > 0, p * (log_p + entropy), torch.zeros_like(p))
    g, h = st["d_log_probs"][:, None], st["d_entropy"][:, None]
    d = -(g * p + h * p_log_p)
    d.scatter_add_(1, st["tokens"][:, None], g)
    return d


def _plain_probs(st):
    """q, k and v as [batch, key head, queries x shared heads or keys, width], and the scaled scores with masked keys at -inf."""
    q, k, v, mask = st["q"], st["k"], st["v"], st["key_mask"]
    b, h, lq, d = q.shape
    g, lk = k.shape[1], k.shape[2]
    q = q.reshape(b, g, h // g * lq, d)
    seen = mask[:, None, :, None]
    k = torch.where(seen, k, torch.zeros_like(k))
    v = torch.where(seen, v, torch.zeros_like(v))
    s = torch.matmul(q, k.transpose(2, 3)) * st["scale"]
    return q, k, v, torch.where(mask[:, None, None, :], s, torch.full_like(s, -math.inf))


def _plain_attend(st):
    q, k, v, s = _plain_probs(st)
    b, h, lq, d = st["q"].shape
    m = s.max(dim=-1, keepdim=True).values
    e = torch.exp(s - m)
    total = e.sum(dim=-1, keepdim=True)
    out = torch.matmul(e / total, v).reshape(b, h, lq, d)
    return out, (m + torch.log(total)).reshape(b, h, lq)


def _plain_attend_grad(st):
    q, k, v, s = _plain_probs(st)
    b, h, lq, d = st["q"].shape
    g = k.shape[1]
    rows = (b, g, h // g * lq)
    d_out, out = st["d_out"].reshape(*rows, d), st["out"].reshape(*rows, d)
    p = torch.exp(s - st["lse"].reshape(*rows, 1))
    d_v = torch.matmul(p.transpose(2, 3), d_out)
    delta = (d_out * out).sum(dim=-1, keepdim=True)
    d_s = p * (torch.matmul(d_out, v.transpose(2, 3)) - delta) * st["scale"]
    return torch.matmul(d_s, k).reshape(b, h, lq, d), torch.matmul(d_s.transpose(2, 3), q), d_v


def _run_plain(st):
    case = st["case"]
    op = case["op"]
    if op == "embed":
        return st["table"][st["tokens"]] * st["scale"]
    if op == "embed_grad":
        # sums of thousands of addends for the frequent tokens: held in 64 bits
        total = torch.zeros(case["vocab"], case["width"], device="cuda", dtype=torch.float64)
        total.index_add_(0, st["tokens"], st["d_out"].double())
        return (total * st["scale"]).to(st["d_out"].dtype)
    if op == "logprobs":
        return _plain_logprobs(st, case["top"])
    if op == "logprobs_grad":
        return _plain_logprobs_grad(st)
    if op == "attend":
        return _plain_attend(st)
    return _plain_attend_grad(st)


# ---- the library's entry points -------------------------------------------------------------------------------------------------

def _prepare_own(case, st):
    import ctypes

    from deepnet_amd import abi, native

    dt, op = _T[case["dtype"]], case["op"]
    scalar = ctypes.c_float if case["dtype"] == "float32" else ctypes.c_double

    def new(*shape, dtype=dt):
        return torch.empty(*shape, device="cuda", dtype=dtype)

    def desc(t):
        np_type = {torch.float32: np.float32, torch.float64: np.float64, torch.int64: np.int64, torch.bool: np.bool_}[t.dtype]
        d = abi.make_descriptor(t.data_ptr(), np_type, t.shape, t.stride(), 0)
        return d, ctypes.byref(d)

    if op == "embed":
        st["outputs"] = new(case["tokens"], case["width"])
        entry, args = "dnh_embedding", [st["outputs"], st["table"], st["tokens"], "scale"]
    elif op == "embed_grad":
        st["outputs"] = new(case["vocab"], case["width"])
        entry, args = "dnh_embedding_grad", [st["outputs"], st["tokens"], st["d_out"], "scale", 0, "scratch"]
    elif op == "logprobs":
        r, top = case["rows"], case["top"]
        o = [new(r), new(r), new(r)]
        if top:
            o += [new(r, top), new(r, top, dtype=torch.int64)]
        st["outputs"] = tuple(o)
        entry, args = "dnh_token_log_probs", o + [None] * (5 - len(o)) + [st["logits"], st["tokens"], "scratch"]
    elif op == "logprobs_grad":
        st["outputs"] = torch.empty_like(st["logits"])
        entry = "dnh_token_log_probs_grad"
        args = [st["outputs"], st["logits"], st["tokens"], st["lse"], st["entropy"], st["d_log_probs"], st["d_entropy"]]
    elif op == "attend":
        o = (new(*st["q"].shape), new(*st["q"].shape[:3]))
        st["outputs"] = o
        entry, args = "dnh_cross_attention", [*o, st["q"], st["k"], st["v"], st["key_mask"], "scale", "scratch"]
    else:
        o = (new(*st["q"].shape), new(*st["k"].shape), new(*st["v"].shape))
        st["outputs"] = o
        entry = "dnh_cross_attention_grad"
        args = [*o, st["d_out"], st["q"], st["k"], st["v"], st["out"], st["lse"], st["key_mask"], "scale", "scratch"]

    keep, call = [], []
    for a in args:
        if isinstance(a, torch.Tensor):
            d, ref = desc(a)
            keep.append(d)
            call.append(ref)
        elif a == "scale":
            value = scalar(st["scale"])
            keep.append(value)
            call.append(ctypes.addressof(value))
        elif a == "scratch":              # the stream's workspace, which the library keeps
            call += [None, 0]
        else:
            call.append(a)
    st["keep"], st["args"] = keep, call
    st["entry"], st["check"] = getattr(native.load(), entry), native.check


def _run_own(st):
    st["check"](st["entry"](*st["args"], torch.cuda.current_stream().cuda_stream))
    return st["outputs"]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------------------

def _single(x, case):
    """A scalar argument as the operator receives it: one element of the case's type."""
    return torch.tensor(x, dtype=_T[case["dtype"]]).double().item()


def exact(case, seed):
    st = _inputs(case, seed)
    op = case["op"]
    if op == "embed":
        return torch.index_select(st["table"], 0, st["tokens"]).double().mul_(_single(st["scale"], case))
    if op == "embed_grad":
        # tokens sorted; each token's rows added up by halving, neighbours of one token first
        tokens, order = torch.sort(st["tokens"], stable=True)
        rows = st["d_out"].double()[order]
        while True:
            first = torch.ones_like(tokens, dtype=torch.bool)
            first[1:] = tokens[1:] != tokens[:-1]
            place = torch.arange(len(tokens), device="cuda")
            start = torch.cummax(torch.where(first, place, 0), 0).values
            odd = (place - start) % 2 == 1          # every second row of a token joins the one before it
            if not bool(odd.any()):
                break
            at = torch.nonzero(odd)[:, 0]
            rows[at - 1] += rows[at]
            tokens, rows = tokens[~odd], rows[~odd]
        total = torch.zeros(case["vocab"], case["width"], device="cuda", dtype=torch.float64)
        total[tokens] = rows * _single(st["scale"], case)
        return total
    if op == "logprobs":
        x = st["logits"].double()
        lse = torch.logsumexp(x, dim=1)
        log_p = x - lse[:, None]
        entropy = torch.special.entr(torch.exp(log_p)).sum(dim=1)
        out = [log_p.gather(1, st["tokens"][:, None])[:, 0], lse, entropy]
        if case["top"]:
            del x
            tops = [torch.sort(part, dim=1, descending=True, stable=True).indices[:, :case["top"]] for part in _row_pieces(st["logits"])]
            index = torch.cat(tops)
            out += [log_p.gather(1, index), index]
        return tuple(out)
    if op == "logprobs_grad":
        x = st["logits"].double()
        log_p = x - torch.logsumexp(x, dim=1, keepdim=True)
        p = torch.exp(log_p)
        entr = torch.special.entr(p)
        entropy = entr.sum(dim=1, keepdim=True)
        g, h = st["d_log_probs"].double()[:, None], st["d_entropy"].double()[:, None]
        d = h * (entr - p * entropy) - g * p
        rows = torch.arange(case["rows"], device="cuda")
        d[rows, st["tokens"]] += g[:, 0]
        return d
    q, k, v = st["q"].double(), st["k"].double(), st["v"].double()
    b, h, lq, d = q.shape
    g, lk = k.shape[1], k.shape[2]
    scale = _single(st["scale"], case)
    outs, lses, d_qs = [], [], []
    d_ks, d_vs = [], []
    for bi in range(b):                  # the keys that the sequence has, and no others
        n = int(st["key_mask"][bi].sum())
        for gi in range(g):
            kk, vv = k[bi, gi, :n].contiguous(), v[bi, gi, :n].contiguous()
            dk, dv = torch.zeros(lk, d, device="cuda", dtype=torch.float64), torch.zeros(lk, d, device="cuda", dtype=torch.float64)
            for hi in range(gi * (h // g), (gi + 1) * (h // g)):
                qq = q[bi, hi].contiguous()
                log_w = qq @ kk.t() * scale
                lse = torch.logsumexp(log_w, dim=1)
                w = torch.softmax(log_w, dim=1)
                o = w @ vv
                if op == "attend":
                    outs.append(o)
                    lses.append(lse)
                    continue
                do = st["d_out"][bi, hi].double().contiguous()
                dw = do @ vv.t()
                dz = w * (dw - (dw * w).sum(dim=1, keepdim=True)) * scale
                d_qs.append(dz @ kk)
                dk[:n] += dz.t() @ qq
                dv[:n] += w.t() @ do
            d_ks.append(dk)
            d_vs.append(dv)
    if op == "attend":
        return torch.stack(outs).reshape(b, h, lq, d), torch.stack(lses).reshape(b, h, lq)
    return torch.stack(d_qs).reshape(b, h, lq, d), torch.stack(d_ks).reshape(b, g, lk, d), torch.stack(d_vs).reshape(b, g, lk, d)


def _row_pieces(x):
    """Pieces of a few hundred rows, so that a stable sort of each fits beside the rest."""
    return x.split(max(1, 30_000_000 // x.shape[1]))
