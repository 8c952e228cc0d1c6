"""The operators of a decoder's own tokens, as they are measured.

Three operators: turning queries and keys by positions of several axes (a
patch's place on the hex lattice, a video's time, height and width), appending
a step's keys and values to a paged cache with that rotation on the way, and
attention of new tokens over the pages, the whole sequence or a sliding window
with a few first states that stay visible.

``run`` computes them in elementary torch operations in 32 bits (angles in 64),
or, where ``own`` is true, through this package's public entry points.
"""

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BASE = 10000.0


# ------------------------------------------------------------------ the cases
def _rotate(name, dtype, batch, heads, groups, rows, head_dim, sections, *, train=False, place="grid", far=0,
            interleaved=False):
    return {"name": name, "op": "rotate", "dtype": dtype, "batch": batch, "heads": heads, "groups": groups,
            "rows": rows, "head_dim": head_dim, "sections": sections, "train": train, "place": place, "far": far,
            "interleaved": interleaved}


def _append(name, dtype, batch, heads, groups, rows, head_dim, sections, *, held, page, ragged=False, place="row",
            interleaved=False):
    return {"name": name, "op": "append", "dtype": dtype, "batch": batch, "heads": heads, "groups": groups,
            "rows": rows, "head_dim": head_dim, "sections": sections, "held": held, "page": page, "ragged": ragged,
            "place": place, "interleaved": interleaved}


def _attend(name, dtype, batch, heads, groups, rows, states, head_dim, *, page, ragged=False, empty=False, window=0,
            sinks=0):
    return {"name": name, "op": "attend", "dtype": dtype, "batch": batch, "heads": heads, "groups": groups,
            "rows": rows, "states": states, "head_dim": head_dim, "page": page, "ragged": ragged, "empty": empty,
            "window": window, "sinks": sinks}


def listed():
    return [
        # One image's 195 patches and its CLS token, turned by their places on the lattice: latency.
        _rotate("rotate-one-image", "bf16", 1, 3, 3, 196, 64, "16,16", place="lattice"),
        # The same in a training step of 256 images: both directions of q and k.
        _rotate("rotate-train-images", "bf16", 256, 3, 3, 196, 64, "16,16", train=True, place="lattice"),
        # Frames of a long video in a training step, far from its beginning, grouped heads of 128.
        _rotate("rotate-train-video", "bf16", 2, 32, 8, 16384, 128, "16,24,24", train=True, far=100000),
        # 32-bit heads of 80 whose first 64 columns turn in neighbouring pairs, odd length.
        _rotate("rotate-partial-f32", "f32", 3, 12, 12, 1001, 80, "32", interleaved=True),
        # A serving batch's new token: q turned, k turned into its page, v beside it: latency.
        _append("append-token", "bf16", 32, 32, 8, 1, 128, "64", held=2000, page=16, ragged=True),
        # Prompts of images and text, padded to the longest, into fragmented pages.
        _append("append-prompt", "bf16", 16, 32, 8, 4096, 128, "16,24,24", held=0, page=64, ragged=True, place="grid"),
        # Further prompts behind what is held, odd sizes, pages that end inside any power of two.
        _append("append-odd", "f16", 3, 6, 2, 777, 96, "32", held=1001, page=24, ragged=True, interleaved=True),
        # One new token of two sequences over short caches: latency.
        _attend("attend-token-small", "bf16", 2, 3, 3, 1, 777, 64, page=16, ragged=True),
        # A serving batch's new tokens over long caches of unequal lengths: bound by reading them.
        _attend("attend-token-batch", "bf16", 64, 32, 8, 1, 8192, 128, page=16, ragged=True),
        # One reader of a very long document: the pages have to be split.
        _attend("attend-token-long", "bf16", 1, 32, 8, 1, 131071, 128, page=64),
        # Several guessed tokens a sequence, some of them padding, one sequence finished; odd sizes.
        _attend("attend-guesses", "f16", 17, 12, 4, 5, 4001, 80, page=24, ragged=True, empty=True),
        # A stream that keeps its last thousand states and its first four in sight.
        _attend("attend-window", "bf16", 48, 16, 4, 1, 16384, 64, page=16, ragged=True, window=1024, sinks=4),
    ]


def _cost(case):
    w = work(case)
    # a pass's cost in microseconds at about 1e15 flop/s and 6e12 byte/s
    return w["flops"] / 1e9 + w["bytes"] / 6e6


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _draw_sections(rng, head_dim):
    """Pairs of each axis, in whole groups of four: the whole head or its front half."""
    pairs = rng.choice([head_dim // 2, head_dim // 2, head_dim // 8 * 2]) // 4
    axes = min(rng.choice([1, 2, 3]), pairs)
    cuts = sorted(rng.sample(range(1, pairs), axes - 1))
    return ",".join(str(4 * (b - a)) for a, b in zip([0, *cuts], [*cuts, pairs]))


def draw(rng):
    op = rng.choice(["rotate", "rotate", "append", "append", "attend", "attend", "attend"])
    limit = 0.9 * max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        groups = rng.choice([1, 2, 3, 4, 6, 8])
        heads = groups * rng.choice([1, 1, 2, 3, 4, 8])
        batch = _log(rng, 1, 64)
        dtype = rng.choice(["bf16", "bf16", "f16"])
        head_dim = rng.choice([32, 64, 64, 72, 80, 96, 128, 128])
        page = rng.choice([8, 16, 16, 24, 32, 64, 128])
        ragged = rng.random() < 0.7
        if op == "rotate":
            case = _rotate("", rng.choice([dtype, dtype, "f32"]), batch, heads, groups, _log(rng, 1, 16384), head_dim,
                           _draw_sections(rng, head_dim), train=rng.random() < 0.5,
                           place=rng.choice(["grid", "grid", "lattice"]), far=rng.choice([0, 1000, 1000000]),
                           interleaved=rng.random() < 0.3)
        elif op == "append":
            rows = rng.choice([1, 1, 2, 5]) if rng.random() < 0.4 else _log(rng, 2, 8192)
            case = _append("", dtype, batch, heads, groups, rows, head_dim, _draw_sections(rng, head_dim),
                           held=rng.choice([0, _log(rng, 1, 8192)]), page=page, ragged=ragged,
                           place=rng.choice(["row", "grid"]), interleaved=rng.random() < 0.3)
        else:
            rows = rng.choice([1, 1, 1, 2, 3, 8])
            window = rng.choice([0, 0, _log(rng, 1, 4096)])
            case = _attend("", dtype, batch, heads, groups, rows, _log(rng, rows, 65536), head_dim, page=page,
                           ragged=ragged, empty=ragged and batch > 1 and rng.random() < 0.3, window=window,
                           sinks=rng.choice([0, 1, 4, 20]) if window else 0)
        held = 2.0 * batch * groups * head_dim * _capacity(case) * 4 if op != "rotate" else 0
        if _cost(case) <= limit and held <= 12e9:
            del case["name"]
            return case


def _capacity(case):
    """States that a sequence's row of the page table has room for."""
    most = case["held"] + case["rows"] if case["op"] == "append" else case["states"]
    return (most + case["page"] - 1) // case["page"] * case["page"]


def _seen(case):
    """States that a sequence's rows read, and scores of one head, at the mean length."""
    mean = 0.75 * case["states"] if case["ragged"] else float(case["states"])
    if not case["window"]:
        return mean, case["rows"] * mean
    row = min(mean, case["window"] + case["sinks"])
    return min(mean, row + case["rows"] - 1), case["rows"] * row


def work(case):
    """Each input read once, each output written once; padded rows and states are neither."""
    b, h, g, n, d = (case[k] for k in ("batch", "heads", "groups", "rows", "head_dim"))
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "attend":
        states, scores = _seen(case)
        live = b - 1 if case["empty"] else b
        return {"bytes": 2.0 * b * h * n * d * size + 2 * g * d * states * live * size,
                "flops": 4.0 * h * d * scores * live}
    pairs = sum(int(s) for s in case["sections"].split(","))
    if case["op"] == "rotate":
        passes = 2 if case["train"] else 1
        return {"bytes": passes * (2.0 * b * (h + g) * n * d * size), "flops": passes * 6.0 * b * (h + g) * n * pairs}
    rows = b * n * (0.75 if case["ragged"] and n > 1 else 1.0)
    return {"bytes": 2.0 * size * d * (b * n * h + 2 * g * rows), "flops": 6.0 * pairs * (b * n * h + g * rows)}


# ------------------------------------------------------------------ the inputs
def _frequencies(case):
    """Pair i of R / 2 turns by base^(-2 i / R) radians for each step along its axis."""
    sections = [int(s) for s in case["sections"].split(",")]
    pairs = sum(sections)
    return [_BASE ** (-i / pairs) for i in range(pairs)], [a for a, s in enumerate(sections) for _ in range(s)]


def _places(case, rng):
    """(B, n, axes): whole numbers along a grid, or points of the hex lattice with one at its origin."""
    b, n, axes = case["batch"], case["rows"], case["sections"].count(",") + 1
    i = torch.arange(n, device="cuda")
    if case["place"] == "lattice":
        row, column = i // 14, i % 14
        points = torch.stack((column * 0.5, row * 3 ** 0.5 + (column % 2) * (3 ** 0.5 / 2), i * 0.25), dim=-1)
        return points[:, :axes].float().roll(1, 0).expand(b, n, axes)
    steps = torch.stack((i // 196, i // 14 % 14, i % 14), dim=-1)[:, :axes] if axes > 1 else i[:, None]
    offset = torch.randint(0, case.get("far", 0) + 1, (b, 1, 1), generator=rng, device="cuda")
    return (offset + steps).to(torch.int32)


def _page_table(lengths, capacity, page, rng):
    """Each sequence's pages, dealt from a shuffled pool; -1 where a sequence has none."""
    width = capacity // page
    need = [(int(x) + page - 1) // page for x in lengths]
    pages = len(need) * width + 3  # a pool that is never used up
    pool = torch.randperm(pages, generator=rng, device="cuda").to(torch.int32)
    table = torch.full((len(need), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, c in enumerate(need):
        table[i, :c] = pool[at:at + c]
        at += c
    return table, pages


def prepare(case, seed):
    rng = torch.Generator(device="cuda").manual_seed(int(seed))
    b, h, g, n, d = (case[k] for k in ("batch", "heads", "groups", "rows", "head_dim"))
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=rng, device="cuda", dtype=dtype)

    def tokens(heads):
        # as a projection leaves them: (B, n, heads * D) seen as (B, heads, n, D)
        return normal(b, n, heads, d).transpose(1, 2)

    state = {"op": case["op"], "case": case, "q": tokens(h)}
    if case["op"] != "attend":
        state["frequencies"], state["axes"] = _frequencies(case)
        state["interleaved"] = case["interleaved"]
        state["positions"] = _places(case, rng) if case["place"] != "row" else None
        state["k"] = tokens(g)
        if own:
            from intp_preliminary_b200 import RotaryAxes

            state["rotary"] = RotaryAxes(state["frequencies"], state["axes"], interleaved=state["interleaved"],
                                         device="cuda")
    if case["op"] == "rotate":
        if case["train"]:
            state["grad_q"], state["grad_k"] = tokens(h), tokens(g)
        return state
    state["counts"] = None
    if case["op"] == "append":
        state["v"] = tokens(g)
        held, most = case["held"], case["held"] + n
        start = torch.full((b,), held, dtype=torch.int32, device="cuda")
        if case["ragged"]:
            start = torch.randint(held // 2, held + 1, (b,), generator=rng, device="cuda", dtype=torch.int32)
            if n > 1:
                state["counts"] = torch.randint((n + 1) // 2, n + 1, (b,), generator=rng, device="cuda",
                                                dtype=torch.int32)
        lengths = start + (n if state["counts"] is None else state["counts"])
    else:
        most = case["states"]
        lengths = torch.full((b,), most, dtype=torch.int32, device="cuda")
        if case["ragged"]:
            lengths = torch.randint(max((most + 1) // 2, n), most + 1, (b,), generator=rng, device="cuda",
                                    dtype=torch.int32)
        if case["ragged"] and n > 1:
            state["counts"] = torch.randint(1, n + 1, (b,), generator=rng, device="cuda", dtype=torch.int32)
        if case["empty"]:
            if state["counts"] is None:
                state["counts"] = torch.full((b,), n, dtype=torch.int32, device="cuda")
            state["counts"][b // 2] = 0
        start = lengths - (n if state["counts"] is None else state["counts"])
        state["window"], state["sinks"] = case["window"] or None, case["sinks"]
        state["scale"] = d ** -0.5
    state["start"] = start
    state["page_table"], pages = _page_table(lengths.tolist(), _capacity(case), case["page"], rng)
    state["keys"], state["values"] = normal(pages, g, case["page"], d), normal(pages, g, case["page"], d)
    if own:
        from intp_preliminary_b200 import PagedCache

        state["cache"] = PagedCache(state["keys"], state["values"])
    return state


# ------------------------------------------------------------------ the plain forms
def _turned(x, s, positions, sign=1.0):
    """x (B, heads, n, D) with its pairs turned by their angles, in 32 bits, rounded once."""
    frequency = torch.tensor(s["frequencies"], dtype=torch.float64, device=x.device)
    axis = torch.tensor(s["axes"], device=x.device)
    angle = positions.double()[:, None, :, axis] * frequency
    c, sn = torch.cos(angle).float(), (sign * torch.sin(angle)).float()
    pairs = frequency.shape[0]
    y = x.float().clone()
    if s["interleaved"]:
        one, two = y[..., 0:2 * pairs:2].clone(), y[..., 1:2 * pairs:2].clone()
        y[..., 0:2 * pairs:2] = one * c - two * sn
        y[..., 1:2 * pairs:2] = two * c + one * sn
    else:
        one, two = y[..., :pairs].clone(), y[..., pairs:2 * pairs].clone()
        y[..., :pairs] = one * c - two * sn
        y[..., pairs:2 * pairs] = two * c + one * sn
    return y.to(x.dtype)


def _row_positions(s):
    n, axes = s["q"].shape[2], max(s["axes"]) + 1
    at = s["start"].long()[:, None] + torch.arange(n, device="cuda")
    return at[:, :, None].expand(-1, -1, axes)


def _plain(s):
    q = s["q"]
    if s["op"] == "rotate":
        out = {name: _turned(s[name], s, s["positions"]) for name in ("q", "k")}
        if s["case"]["train"]:
            out["dq"] = _turned(s["grad_q"], s, s["positions"], -1.0)
            out["dk"] = _turned(s["grad_k"], s, s["positions"], -1.0)
        return out
    keys, values, table, start, counts = s["keys"], s["values"], s["page_table"].long(), s["start"].long(), s["counts"]
    page = keys.shape[2]
    b, _, n, d = q.shape
    at = start[:, None] + torch.arange(n, device="cuda")
    if s["op"] == "append":
        positions = s["positions"] if s["positions"] is not None else _row_positions(s)
        k = _turned(s["k"], s, positions)
        there = torch.arange(n, device="cuda") < (counts[:, None] if counts is not None else n)
        seq, row = there.expand(b, n).nonzero(as_tuple=True)
        to = at[seq, row]
        where = table[seq, to // page]
        keys[where, :, to % page] = k[seq, :, row]
        values[where, :, to % page] = s["v"][seq, :, row]
        return [_turned(q, s, positions), keys, values]
    g = keys.shape[1]
    dense = [x[table.clamp(min=0)].transpose(1, 2).reshape(b, g, -1, d).float() for x in (keys, values)]
    j = torch.arange(dense[0].shape[2], device="cuda")
    sees = j <= at[:, :, None]
    if s["window"] is not None:
        sees &= (j > at[:, :, None] - s["window"]) | (j < s["sinks"])
    if counts is not None:
        sees &= (torch.arange(n, device="cuda") < counts[:, None])[:, :, None]
    out = torch.zeros(q.shape, dtype=torch.float32, device="cuda")
    for i in range(g):  # a key head's query heads together
        rows = q[:, i * (q.shape[1] // g):(i + 1) * (q.shape[1] // g)].float()
        scores = torch.matmul(rows, dense[0][:, i:i + 1].transpose(-1, -2)) * s["scale"]
        scores = scores.masked_fill(~sees[:, None], -math.inf)
        top = scores.amax(-1, keepdim=True)
        p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
        total = p.sum(-1, keepdim=True)
        part = torch.matmul(p, dense[1][:, i:i + 1]) / torch.where(total == 0, torch.ones_like(total), total)
        out[:, i * (q.shape[1] // g):(i + 1) * (q.shape[1] // g)] = part
    return out.to(q.dtype)


# ------------------------------------------------------------------ the framework's operators
def _framework(s):
    from intp_preliminary_b200 import paged_attention, rotate_positions

    q = s["q"]
    if s["op"] == "attend":
        return paged_attention(q, s["cache"], page_table=s["page_table"], start=s["start"], counts=s["counts"],
                               scale=s["scale"], window=s["window"], sinks=s["sinks"])
    if s["op"] == "append":
        turned = s["cache"].append(s["k"], s["v"], page_table=s["page_table"], start=s["start"], counts=s["counts"],
                                   rotary=s["rotary"], positions=s["positions"], q=q)
        return [turned, s["cache"].keys, s["cache"].values]
    if not s["case"]["train"]:
        out = rotate_positions(q, s["k"], rotary=s["rotary"], positions=s["positions"])
        return {"q": out[0], "k": out[1]}
    leaves = [x.detach().requires_grad_() for x in (q, s["k"])]
    out = rotate_positions(*leaves, rotary=s["rotary"], positions=s["positions"])
    dq, dk = torch.autograd.grad(out, leaves, (s["grad_q"], s["grad_k"]))
    return {"q": out[0].detach(), "k": out[1].detach(), "dq": dq, "dk": dk}


def run(state):
    return _framework(state) if own else _plain(state)


# ------------------------------------------------------------------ 64 bits
def _turned_64(x, s, positions, inverse=False):
    """As complex numbers times e^(i angle), one head at a time, in place of what x holds."""
    y = x.double()
    pairs = len(s["frequencies"])
    angle = torch.zeros(*positions.shape[:2], pairs, dtype=torch.float64, device="cuda")
    for i, (f, a) in enumerate(zip(s["frequencies"], s["axes"])):
        angle[:, :, i] = positions[:, :, a].double() * f
    turn = torch.polar(torch.ones_like(angle), -angle if inverse else angle)
    real = slice(0, 2 * pairs, 2) if s["interleaved"] else slice(0, pairs)
    imag = slice(1, 2 * pairs, 2) if s["interleaved"] else slice(pairs, 2 * pairs)
    for i in range(x.shape[1]):
        z = torch.complex(y[:, i, :, real].contiguous(), y[:, i, :, imag].contiguous()) * turn
        y[:, i, :, real], y[:, i, :, imag] = z.real, z.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotate":
        out = {name: _turned_64(s[name], s, s["positions"]) for name in ("q", "k")}
        if case["train"]:
            out.update({"d" + x: _turned_64(s["grad_" + x], s, s["positions"], True) for x in ("q", "k")})
        return out
    q, table, page = s["q"], s["page_table"].tolist(), case["page"]
    b, h, n, d = q.shape
    g = case["groups"]
    counts = [n] * b if s["counts"] is None else s["counts"].tolist()
    starts = s["start"].tolist()
    if case["op"] == "append":
        positions = s["positions"] if s["positions"] is not None else _row_positions(s)
        turned = [_turned_64(q, s, positions)]
        for new, held in ((_turned_64(s["k"], s, positions), s["keys"]), (s["v"].double(), s["values"])):
            held = held.double()
            for i in range(b):
                row = 0
                while row < counts[i]:  # a page's rows at once
                    at = starts[i] + row
                    some = min(page - at % page, counts[i] - row)
                    held[table[i][at // page], :, at % page:at % page + some] = new[i, :, row:row + some]
                    row += some
            turned.append(held)
        return turned
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for i in range(b):
        length = starts[i] + counts[i]
        own_pages = torch.tensor(table[i][:(length + page - 1) // page], dtype=torch.long, device="cuda")
        j = torch.arange(length, device="cuda")
        for x in range(g if counts[i] else 0):
            k = s["keys"][own_pages, x].reshape(-1, d)[:length].double()
            v = s["values"][own_pages, x].reshape(-1, d)[:length].double()
            for row in range(counts[i]):
                at = starts[i] + row
                sees = j <= at
                if case["window"]:
                    sees &= (j > at - case["window"]) | (j < case["sinks"])
                heads = slice(x * (h // g), (x + 1) * (h // g))
                scores = (q[i, heads, row].double() @ k[sees].T) * s["scale"]
                out[i, heads, row] = torch.softmax(scores, dim=-1) @ v[sees]
    return out
