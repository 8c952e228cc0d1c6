"""The operators that read an encoder's states, as they are measured.

Four operators: cross attention to states of another length (training steps,
prompts, single tokens), writing key / value states to an 8-bit cache and
reading them back, attention of new tokens over that cache, and attention of
a batch over one shared prefix plus each sequence's own states.

``run`` computes them in elementary torch operations in 32 bits, or, where
``own`` is true, through this package's public entry points.
"""

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
_E4M3_MAX = 448.0


# ------------------------------------------------------------------ the cases
def _case(name, op, dtype, batch, heads, groups, queries, states, head_dim, *, ragged=False, empty=False, prefix=0,
          capacity=0):
    return {"name": name, "op": op, "dtype": dtype, "batch": batch, "heads": heads, "groups": groups,
            "queries": queries, "states": states, "head_dim": head_dim, "ragged": ragged, "empty": empty,
            "prefix": prefix, "capacity": capacity}


def listed():
    return [
        # A small decoder trained on the half6d3r encoder's 195 patch states and its CLS state, 3 heads of 64.
        _case("train-vit-states", "train", "bf16", 8, 3, 3, 64, 196, 64),
        # Image positions that read a short text: many queries, few states, padded texts, grouped heads.
        _case("train-wide-queries", "train", "f16", 4, 12, 4, 4096, 77, 64, ragged=True),
        # A long document's states under a long target, heads of 128: bound by the matrix products.
        _case("train-long", "train", "bf16", 4, 16, 16, 2048, 4096, 128),
        # A serving prompt over long padded states, four query heads to a key head, odd sizes.
        _case("prompt-grouped", "forward", "bf16", 2, 32, 8, 1023, 8191, 128, ragged=True),
        # One new token over one image's states: latency.
        _case("token-one-image", "forward", "bf16", 1, 3, 3, 1, 196, 64),
        # One new token for each of a serving batch over long padded states: bound by reading them.
        _case("token-batch", "forward", "bf16", 64, 32, 8, 1, 4096, 128, ragged=True),
        # One new state appended to each sequence's cache: latency.
        _case("cache-append", "cache", "bf16", 32, 8, 8, 0, 1, 128, capacity=2048),
        # A prompt's states written to the cache and read back.
        _case("cache-prompt", "cache", "f16", 16, 8, 8, 0, 4096, 128, capacity=4096),
        # A new token of two sequences over a short 8-bit cache: latency.
        _case("cached-token-small", "cached", "bf16", 2, 3, 3, 1, 777, 64, ragged=True, capacity=777),
        # A serving batch's new tokens over a long 8-bit cache.
        _case("cached-token-batch", "cached", "bf16", 64, 32, 8, 1, 8192, 128, ragged=True, capacity=8192),
        # Four questions about one image: the shared states are the encoder's 196.
        _case("prefix-one-image", "prefix", "bf16", 4, 3, 3, 1, 33, 64, ragged=True, prefix=196),
        # A serving batch that shares a long document, each with an answer of its own so far.
        _case("prefix-batch", "prefix", "bf16", 64, 32, 8, 1, 512, 128, ragged=True, prefix=16384),
    ]


def _cost(case):
    w = work(case)
    # a pass's cost in microseconds at about 1e15 flop/s and 6e12 byte/s
    return w["flops"] / 1e9 + w["bytes"] / 6e6


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["train", "train", "forward", "forward", "cache", "cached", "prefix"])
    limit = 0.9 * max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        groups = rng.choice([1, 2, 3, 4, 6, 8, 16])
        heads = groups * rng.choice([1, 1, 2, 3, 4, 8])
        batch = _log(rng, 1, 64)
        dtype = rng.choice(["bf16", "bf16", "f16"])
        head_dim = rng.choice([32, 64, 64, 80, 96, 128, 128])
        queries, prefix, capacity = 1, 0, 0
        ragged = rng.random() < 0.6
        empty = ragged and batch > 1 and rng.random() < 0.3
        if op == "train":
            # a softmax over one or two states has hardly a gradient: nothing to compare
            queries, states = _log(rng, 1, 4096), _log(rng, 16, 8192)
        elif op == "forward":
            if rng.random() < 0.5:
                queries, states = rng.choice([1, 1, 2, 3]), _log(rng, 1, 32768)
            else:
                queries, states = _log(rng, 4, 4096), _log(rng, 1, 16384)
        elif op == "cache":
            states = 1 if rng.random() < 0.4 else _log(rng, 2, 8192)
            heads, queries, ragged, empty = groups, 0, False, False
            capacity = states + _log(rng, 1, 4096)
        elif op == "cached":
            queries, states = rng.choice([1, 1, 1, 2, 4]), _log(rng, 1, 32768)
            capacity = states + rng.choice([0, 1, 64])
        else:
            states, prefix = _log(rng, 1, 4096), _log(rng, 1, 32768)
        case = _case("", op, dtype, batch, heads, groups, queries, states, head_dim, ragged=ragged, empty=empty,
                     prefix=prefix, capacity=capacity)
        scores = 4.0 * batch * heads * max(queries, 1) * (states + prefix)
        held = 2.0 * batch * groups * (states + capacity) * head_dim * 2
        if _cost(case) <= limit and scores <= 4e9 and held <= 8e9:
            del case["name"]
            return case


def work(case):
    """Each input read once, each output written once; padded states are not read."""
    b, h, g, m, n, d = (case[k] for k in ("batch", "heads", "groups", "queries", "states", "head_dim"))
    mean = 0.75 * n if case["ragged"] else float(n)  # mean length of the padded sequences
    total = mean * (b - 1 if case["empty"] else b)
    if case["op"] == "train":
        return {"bytes": 2 * (4.0 * b * h * m * d + 2 * g * d * (total + b * n)), "flops": 14.0 * h * m * d * total}
    if case["op"] == "forward":
        return {"bytes": 2 * (2.0 * b * h * m * d + 2 * g * d * total), "flops": 4.0 * h * m * d * total}
    if case["op"] == "cache":
        return {"bytes": 2.0 * b * g * n * (6 * d + 2), "flops": 4.0 * b * g * n * d}
    if case["op"] == "cached":
        return {"bytes": 4.0 * b * h * m * d + 2 * g * total * (d + 1), "flops": 4.0 * h * m * d * total}
    p = case["prefix"]
    return {"bytes": 2 * (2.0 * b * h * m * d + 2 * g * d * (p + total)), "flops": 4.0 * h * m * d * (p * b + total)}


# ------------------------------------------------------------------ the inputs
def prepare(case, seed):
    rng = torch.Generator(device="cuda").manual_seed(int(seed))
    b, h, g, m, n, d = (case[k] for k in ("batch", "heads", "groups", "queries", "states", "head_dim"))
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=rng, device="cuda", dtype=dtype) * scale

    state = {"op": case["op"], "scale": d ** -0.5, "lengths": None}
    if case["ragged"]:
        lengths = torch.randint((n + 1) // 2, n + 1, (b,), generator=rng, device="cuda", dtype=torch.int32)
        if case["empty"]:
            lengths[b // 2] = 0
        state["lengths"] = lengths
    if case["op"] == "cache":
        c = case["capacity"]
        state["k"], state["v"] = normal(b, g, n, d), normal(b, g, n, d, scale=0.5)
        state["start"] = torch.randint(0, c - n + 1, (b,), generator=rng, device="cuda", dtype=torch.int32)
        for name in ("keys", "values"):
            state[name] = torch.zeros(b, g, c, d, device="cuda", dtype=torch.float8_e4m3fn)
        for name in ("key_exponents", "value_exponents"):
            state[name] = torch.full((b, g, c), 127, device="cuda", dtype=torch.uint8)
        return state
    state["q"] = normal(b, h, m, d)
    if case["op"] == "cached":  # a cache as its rows are written: codes and one power of two for each row
        c = case["capacity"]
        for name, exps in (("keys", "key_exponents"), ("values", "value_exponents")):
            rows = torch.randn((b, g, c, d), generator=rng, device="cuda", dtype=dtype)
            rows *= torch.rand((b, g, c, 1), generator=rng, device="cuda", dtype=dtype) + 0.5
            codes, exponent = _quantise(rows)
            state[name], state[exps] = codes, exponent
        if state["lengths"] is None:
            state["lengths"] = torch.full((b,), n, device="cuda", dtype=torch.int32)
        return state
    state["k"], state["v"] = normal(b, g, n, d), normal(b, g, n, d)
    if case["op"] == "train":
        state["grad"] = normal(b, h, m, d)
    if case["op"] == "prefix":
        state["prefix_k"], state["prefix_v"] = normal(g, case["prefix"], d), normal(g, case["prefix"], d)
    return state


# ------------------------------------------------------------------ the plain forms
def _quantise(x):
    """e4m3 codes and exponent bytes of rows: the smallest power of two 2^e with amax <= 448 * 2^e."""
    x = x.float()
    mantissa, exponent = torch.frexp(x.abs().amax(-1, keepdim=True))
    e = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8).clamp(min=-126)
    e = torch.where(mantissa == 0, torch.zeros_like(e), e)
    codes = torch.ldexp(x, -e).to(torch.float8_e4m3fn)
    return codes, (e.squeeze(-1) + 127).to(torch.uint8)


def _dequantise(codes, exponents):
    return torch.ldexp(codes.float(), exponents.int().unsqueeze(-1) - 127)


def _grouped(x, groups):
    """(B, H, M, D) in 32 bits with the rows of a key head's query heads together: (B, G, H/G * M, D)."""
    b, h, m, d = x.shape
    return x.float().reshape(b, groups, h // groups * m, d)


def _visible(lengths, n, device):
    if lengths is None:
        return None
    return (torch.arange(n, device=device) < lengths.unsqueeze(1))[:, None, None, :]


def _softmax_parts(scores, visible):
    """exp(scores - rowmax) and its row sum; a row with nothing visible has zeros."""
    if visible is not None:
        scores = scores.masked_fill(~visible, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(scores - top)
    return p, p.sum(-1, keepdim=True)


def _states(x, visible):
    x = x.float()
    return x if visible is None else x.masked_fill(~visible.transpose(-1, -2), 0.0)


def _plain_attention(q, k, v, scale, lengths):
    """Probabilities and outputs, rows grouped."""
    visible = _visible(lengths, k.shape[2], q.device)
    k, v = _states(k, visible), _states(v, visible)
    rows = _grouped(q, k.shape[1])
    p, total = _softmax_parts(torch.matmul(rows, k.transpose(-1, -2)) * scale, visible)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    return rows, k, v, p, torch.matmul(p, v)


def _plain(s):
    op = s["op"]
    if op == "cache":
        got = []
        at = s["start"].long()[:, None] + torch.arange(s["k"].shape[2], device="cuda")  # (B, n) rows of the cache
        seq = torch.arange(at.shape[0], device="cuda")[:, None]
        for x, name, exps in ((s["k"], "keys", "key_exponents"), (s["v"], "values", "value_exponents")):
            codes, e = _quantise(x)
            s[name].view(torch.uint8).transpose(1, 2)[seq, at] = codes.view(torch.uint8).transpose(1, 2)
            s[exps].transpose(1, 2)[seq, at] = e.transpose(1, 2)
            codes = s[name].view(torch.uint8).transpose(1, 2)[seq, at].view(torch.float8_e4m3fn)
            read = _dequantise(codes, s[exps].transpose(1, 2)[seq, at])
            got.append(read.to(x.dtype).transpose(1, 2).contiguous())
        return got
    q, scale, lengths = s["q"], s["scale"], s["lengths"]
    if op == "cached":
        k = _dequantise(s["keys"], s["key_exponents"])
        v = _dequantise(s["values"], s["value_exponents"])
        return _plain_attention(q, k, v, scale, lengths)[-1].reshape(q.shape).to(q.dtype)
    if op == "forward":
        return _plain_attention(q, s["k"], s["v"], scale, lengths)[-1].reshape(q.shape).to(q.dtype)
    if op == "prefix":
        g, d = s["prefix_k"].shape[0], q.shape[-1]
        visible = _visible(lengths, s["k"].shape[2], q.device)
        k, v, rows = _states(s["k"], visible), _states(s["v"], visible), _grouped(q, g)
        b, _, r, _ = rows.shape
        own_scores = torch.matmul(rows, k.transpose(-1, -2)) * scale
        if visible is not None:
            own_scores = own_scores.masked_fill(~visible, -math.inf)
        pre = rows.transpose(0, 1).reshape(g, b * r, d)  # every sequence's rows against the one prefix
        pre_scores = torch.matmul(pre, s["prefix_k"].float().transpose(-1, -2)) * scale
        top = torch.maximum(pre_scores.amax(-1, keepdim=True).reshape(g, b, r, 1).transpose(0, 1),
                            own_scores.amax(-1, keepdim=True))
        own_p = torch.exp(own_scores - top)
        pre_p = torch.exp(pre_scores - top.transpose(0, 1).reshape(g, b * r, 1))
        total = own_p.sum(-1, keepdim=True) + pre_p.sum(-1, keepdim=True).reshape(g, b, r, 1).transpose(0, 1)
        out = torch.matmul(own_p, v)
        out = out + torch.matmul(pre_p, s["prefix_v"].float()).reshape(g, b, r, d).transpose(0, 1)
        return (out / total).reshape(q.shape).to(q.dtype)
    rows, k, v, p, out = _plain_attention(q, s["k"], s["v"], scale, lengths)
    grad = _grouped(s["grad"], k.shape[1])
    ds = torch.matmul(grad, v.transpose(-1, -2))
    ds = p * (ds - (grad * out).sum(-1, keepdim=True))
    dq = torch.matmul(ds, k) * scale
    dk = torch.matmul(ds.transpose(-1, -2), rows) * scale
    dv = torch.matmul(p.transpose(-1, -2), grad)
    return {"out": out.reshape(q.shape).to(q.dtype), "dq": dq.reshape(q.shape).to(q.dtype),
            "dk": dk.to(q.dtype), "dv": dv.to(q.dtype)}


# ------------------------------------------------------------------ the framework's operators
def _framework(s):
    from intp_preliminary_b200 import (StateCache, cached_cross_attention, cross_attention,
                                       shared_prefix_attention)

    op = s["op"]
    if op == "cache":
        cache = StateCache(s["keys"], s["key_exponents"], s["values"], s["value_exponents"])
        cache.write(s["k"], s["v"], start=s["start"])
        return list(cache.read(s["k"].shape[2], start=s["start"], dtype=s["k"].dtype))
    q, scale, lengths = s["q"], s["scale"], s["lengths"]
    if op == "cached":
        cache = StateCache(s["keys"], s["key_exponents"], s["values"], s["value_exponents"])
        return cached_cross_attention(q, cache, scale=scale, lengths=lengths)
    if op == "forward":
        return cross_attention(q, s["k"], s["v"], scale=scale, lengths=lengths)
    if op == "prefix":
        return shared_prefix_attention(q, s["prefix_k"], s["prefix_v"], s["k"], s["v"], scale=scale, lengths=lengths)
    q, k, v = (s[n].detach().requires_grad_() for n in ("q", "k", "v"))
    out = cross_attention(q, k, v, scale=scale, lengths=lengths)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), s["grad"])
    return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}


def run(state):
    return _framework(state) if own else _plain(state)


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "cache":
        # Nearest e4m3 value, ties to the even one, from the list of all its values.
        table = torch.arange(0, 127, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn).double()
        got = []
        for x in (s["k"], s["v"]):
            x = x.double()
            amax = x.abs().amax(-1, keepdim=True)
            e = torch.ceil(torch.log2(amax / _E4M3_MAX))
            e = torch.where(amax > _E4M3_MAX * torch.exp2(e), e + 1, e)
            e = torch.where(amax <= _E4M3_MAX * torch.exp2(e - 1), e - 1, e)
            unit = torch.exp2(torch.where(amax == 0, torch.zeros_like(e), e))
            y = (x.abs() / unit).contiguous()
            hi = torch.searchsorted(table, y).clamp(max=126)
            lo = (hi - 1).clamp(min=0)
            below, above = y - table[lo], table[hi] - y
            pick = torch.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)
            got.append(table[pick] * unit * torch.sign(x))
        return got
    q, scale = s["q"].double(), s["scale"]
    b, h, m, d = q.shape
    g = case["groups"]
    if case["op"] == "cached":
        k = s["keys"].double() * torch.exp2(s["key_exponents"].double() - 127).unsqueeze(-1)
        v = s["values"].double() * torch.exp2(s["value_exponents"].double() - 127).unsqueeze(-1)
    else:
        k, v = s["k"], s["v"]
    lengths = [k.shape[2]] * b if s["lengths"] is None else s["lengths"].tolist()
    train = case["op"] == "train"
    out = torch.zeros_like(q)
    dq, dk, dv = torch.zeros_like(q), None, None
    if train:
        dk, dv = torch.zeros(k.shape, device="cuda").double(), torch.zeros(k.shape, device="cuda").double()
    for i in range(b):
        for j in range(h):
            head = j // (h // g)
            kk, vv = k[i, head, : lengths[i]].double(), v[i, head, : lengths[i]].double()
            if case["op"] == "prefix":
                kk = torch.cat([s["prefix_k"][head].double(), kk])
                vv = torch.cat([s["prefix_v"][head].double(), vv])
            if kk.shape[0] == 0:
                continue
            p = torch.softmax(scale * (q[i, j] @ kk.T), dim=-1)
            out[i, j] = p @ vv
            if train:
                go = s["grad"][i, j].double()
                dp = go @ vv.T
                ds = p * (dp - (p * dp).sum(-1, keepdim=True))
                dq[i, j] = scale * (ds @ kk)
                dk[i, head, : lengths[i]] += scale * (ds.T @ q[i, j])
                dv[i, head, : lengths[i]] += p.T @ go
    return {"out": out, "dq": dq, "dk": dk, "dv": dv} if train else out
