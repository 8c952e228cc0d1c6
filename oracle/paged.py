"""float64 restatement of a decoder's own tokens: positions that turn pairs of columns, a paged
cache, attention of new tokens over it, and elementwise error bounds for the kernels.

Where a kernel may round, with u the unit roundoff of the output type (half its eps):
  turned values: the angle is a 64-bit product (2 roundings of 2^-53 of it, one more here); its
        part within an eighth of a turn, x, is rounded to 32 bits and multiplied by 2 pi (2.7 * 2^-24 of
        pi / 4 at most: 2.1 * 2^-24), sin x and cos x are sums of a power series whose first term left
        out is 2e-9 (0.1 * 2^-24) and whose last sum is rounded to half of 2^-24, the terms before it
        adding 0.7 * 2^-24 at most: below 4 * 2^-24 + 3 * 2^-53 |t| of |x1| + |x2|.  Two fp32
        products and a sum: 2 * 2^-24 more.  The result is rounded once: u |y| (f16: at most 2^-25
        below its normal range).
  attention: the bound of a kernel that multiplies each probability as two 16-bit numbers, as
        oracle.cross_attention's ``two_part`` derives it, but for the two parts: the first leaves less than
        (eps + 2^-22) of the probability, eps = 2 u, the second is that rounded: 2 u^2 (and 2^-22 u, within the
        sum's other terms).  A probability's unit is that of the row's reference, which is at most the largest.  In
        f16 the parts are multiples of 2^-31 of it and their sum off by 2^-32 at most, whatever the probability.
        The result is rounded once (f16: 2^-25 at least).
"""

from __future__ import annotations

import torch


def _u(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def turn(x, positions, frequencies, axes, *, interleaved=False, inverse=False):
    """``(y, bound)`` of x (B, heads, n, D) on the CPU; positions (B, n, axes) or (n, axes)."""
    dtype = x.dtype
    x = x.detach().cpu().double()
    positions = positions.detach().cpu().double().expand(x.shape[0], x.shape[2], -1)
    pairs = len(axes)
    y, size, angles = x.clone(), x.abs(), torch.zeros_like(x)
    for i, (f, a) in enumerate(zip(frequencies, axes)):
        one, two = (2 * i, 2 * i + 1) if interleaved else (i, pairs + i)
        t = (positions[:, None, :, a] * f) * (-1 if inverse else 1)
        c, s = torch.cos(t), torch.sin(t)
        y[..., one] = x[..., one] * c - x[..., two] * s
        y[..., two] = x[..., two] * c + x[..., one] * s
        size[..., one] = size[..., two] = x[..., one].abs() + x[..., two].abs()
        angles[..., one] = angles[..., two] = t.abs()
    bound = size * (6 * 2.0 ** -24 + 3 * 2.0 ** -53 * angles) + _u(dtype) * y.abs()
    bound[..., 2 * pairs:] = 0
    if dtype == torch.float16:
        bound[..., :2 * pairs] += 2.0 ** -25
    return y, bound


def place(page_table, page_size, pages, sequence, state):
    """(page, row) of a sequence's state, or None."""
    if state < 0 or state // page_size >= page_table.shape[1]:
        return None
    page = int(page_table[sequence, state // page_size])
    return (page, state % page_size) if 0 <= page < pages else None


def append(keys, values, k, v, *, page_table, start, counts=None):
    """Writes rows of k, v into (pages, G, S, D) tensors of any dtype, in place, on the CPU."""
    for b in range(k.shape[0]):
        for i in range(k.shape[2] if counts is None else min(max(int(counts[b]), 0), k.shape[2])):
            at = place(page_table, keys.shape[2], keys.shape[0], b, int(start[b]) + i)
            if at is not None:
                keys[at[0], :, at[1]] = k[b, :, i].to(keys.dtype)
                values[at[0], :, at[1]] = v[b, :, i].to(values.dtype)


def attend(q, keys, values, *, page_table, start, scale, counts=None, window=None, sinks=0):
    """``(out, bound)`` in float64 on the CPU."""
    dtype = q.dtype
    q, keys, values = (t.detach().cpu().double() for t in (q, keys, values))
    page_table = page_table.cpu()
    batch, heads, rows, dim = q.shape
    groups = keys.shape[1]
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    u = _u(dtype)
    for b in range(batch):
        for m in range(rows if counts is None else min(max(int(counts[b]), 0), rows)):
            at = int(start[b]) + m
            states = torch.arange(min(at + 1, page_table.shape[1] * keys.shape[2]) if at >= 0 else 0)
            if window is not None:
                states = states[(states > at - window) | (states < sinks)]
            pages = page_table[b, states // keys.shape[2]].long()
            there = (pages >= 0) & (pages < keys.shape[0])
            pages, slots = pages[there], (states % keys.shape[2])[there]
            if not len(pages):
                continue
            for h in range(heads):
                g = h // (heads // groups)
                kk, vv = keys[pages, g, slots], values[pages, g, slots]
                s = scale * (kk @ q[b, h, m])
                if not bool((s != -float("inf")).any()):
                    continue
                p = torch.softmax(s, -1)
                out[b, h, m] = p @ vv
                # a score of -inf is exact: its probability is zero
                size = torch.where(s == -float("inf"), torch.zeros_like(s), scale * (kk.abs() @ q[b, h, m].abs()))
                score = 2.0 ** -23 * ((dim + 8) * size + 4 * s[s != -float("inf")].abs().max())
                rel = 2 * u ** 2 + 2.0 ** -22 * (1 + 64 + len(pages) / 16)
                w = p * (score + rel)
                bound[b, h, m] = w @ vv.abs() + w.sum() * (p @ vv.abs()) + u * out[b, h, m].abs()
                if dtype == torch.float16:
                    bound[b, h, m] += 2.0 ** -25 + 2.0 ** -32 * p.max() * vv.abs().sum(0)
    return out, bound
