"""float64 restatement of cross attention to encoder states, its gradients, the
8-bit state cache's rounding, and elementwise error bounds for 16-bit kernels.

The bounds follow from where a kernel may round, with u the unit roundoff of a
16-bit type (half its eps) and fp32 sums:
  out:  each probability is rounded once (u), its exponential is within 1e-4 of
        itself (a 7.5e-5 polynomial, fp32 scores, two of them in a split), and the
        result is rounded once: (u_p + EXP) sum_j p_j |v_j| + u |out|.
  P, dS of the backward: the same EXP, plus the row sum's own (it is an fp32 log
        within 2e-4), one rounding each; delta carries the rounding of out.
f16 operands below 2^-14 lose bits: at most 2^-25 each.

``two_part`` bounds a kernel that multiplies each probability as two 16-bit numbers, so that
hardly more than the result's own rounding remains.  Relative to p_j |v_j|, with D products in
a score, n states and n / 16 matrix instructions in a sum:
  the two parts leave out u_p^2 (f16 also 2^-25 of the largest);
  ex2.approx 2^-22;  fp32 sums (n / 16 + 64) 2^-22, joins of warps and parts among them;
  a score's own error, absolute in its exponent: a sum of D fp32 products, 2^-23 (D + 8)
  scale sum |q k|, and four roundings of numbers of the largest score's size.
The row sum carries the same once more.
"""

from __future__ import annotations

import torch

EXP = 2.5e-4
LSE = 2e-4


def _u(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def _lengths(lengths, batch, n):
    return [n] * batch if lengths is None else [min(max(int(x), 0), n) for x in lengths]


def cross_attention(q, k, v, *, scale, lengths=None, prefix=None, out_dtype=None, p_dtype=None, key_weight=None,
                    two_part=False):
    """``(out, lse, bound)`` in float64 on the CPU; ``prefix`` = (k, v) of shape (G, P, D).

    ``key_weight`` (B, G, N): the size of a unit of each value row (8-bit states), for
    the loss of small f16 probabilities.  ``two_part``: see the module's text."""
    out_dtype = out_dtype or q.dtype
    p_dtype = p_dtype or q.dtype
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    batch, heads, queries, dim = q.shape
    groups, n = k.shape[1], k.shape[2]
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full((batch, heads, queries), -float("inf"), dtype=torch.float64)
    u_p, u_o = _u(p_dtype), _u(out_dtype)
    for b, length in enumerate(_lengths(lengths, batch, n)):
        for h in range(heads):
            g = h // (heads // groups)
            kk, vv = k[b, g, :length], v[b, g, :length]
            if prefix is not None:
                kk = torch.cat([prefix[0][g].detach().cpu().double(), kk])
                vv = torch.cat([prefix[1][g].detach().cpu().double(), vv])
            if kk.shape[0] == 0:
                continue
            s = scale * (q[b, h] @ kk.T)
            lse[b, h] = torch.logsumexp(s, -1)
            p = torch.exp(s - lse[b, h][:, None])
            out[b, h] = p @ vv
            if two_part:
                score = 2.0 ** -23 * ((dim + 8) * scale * (q[b, h].abs() @ kk.abs().T) + 4 * s.abs().amax(-1, keepdim=True))
                rel = u_p ** 2 + 2.0 ** -22 * (1 + 64 + kk.shape[0] / 16)
                mean = p @ vv.abs()
                bound[b, h] = (p * (score + rel)) @ vv.abs() + (p * (score + rel)).sum(-1, keepdim=True) * mean
                bound[b, h] += u_o * out[b, h].abs() + (2.0 ** -25 if out_dtype == torch.float16 else 0.0)
                if p_dtype == torch.float16:
                    bound[b, h] += 2.0 ** -25 * p.amax(-1, keepdim=True) * vv.abs().sum(0)
                continue
            bound[b, h] = (u_p + EXP) * (p @ vv.abs()) + u_o * out[b, h].abs()
            if p_dtype == torch.float16:
                if key_weight is None:
                    # the running reference is at most 2^8 below the row's maximum
                    bound[b, h] += 2.0 ** -25 * p.amax(-1, keepdim=True) * vv.abs().sum(0) * 2.0
                else:
                    w = key_weight[b, g, :length].detach().cpu().double()
                    bound[b, h] += 2.0 ** -25 * (p * w).amax(-1, keepdim=True) * (vv.abs() / w[:, None]).sum(0) * 2.0
            bound[b, h] += 1e-7
    return out, lse, bound


def cross_attention_gradients(q, k, v, grad, *, scale, lengths=None, scaled=False):
    """``((dq, dk, dv), (their bounds))`` in float64 on the CPU.

    ``scaled``: for a kernel that brings P and dS into f16's range by powers of two, so that a
    bound knows no absolute size but the result's own.  With r = |dO| max |v_j| + |delta| of a query
    row (lengths of vectors), at least |dS|, it holds 2^e dS with 2^14 <= 2^e r: what f16 loses below
    2^-14 is at most 2^-25 of that unit, 2^-39 r (dk: of the key's own |v_j| and the largest |dO| and
    |delta| of the rows that read it).  P is held as 2^12 P: 2^-37.  The result loses at most 2^-25 when it is rounded (f16's last step is 2^-24)."""
    dtype = q.dtype
    u = _u(dtype)
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    last = 1e-7
    if scaled:
        last = 2.0 ** -25 if dtype == torch.float16 else 0.0
    out, _, out_bound = cross_attention(q, k, v, scale=scale, lengths=lengths)
    q, k, v, grad = (t.detach().cpu().double() for t in (q, k, v, grad))
    batch, heads = q.shape[:2]
    groups, n = k.shape[1], k.shape[2]

    def delta_of(b, h):
        return (grad[b, h] * out[b, h]).sum(-1, keepdim=True).abs()

    d = [torch.zeros_like(t) for t in (q, k, v)]
    e = [torch.zeros_like(t) for t in (q, k, v)]
    rel = u + EXP + 2 * LSE
    for b, length in enumerate(_lengths(lengths, batch, n)):
        if length == 0:
            continue
        for h in range(heads):
            g = h // (heads // groups)
            kk, vv, go = k[b, g, :length], v[b, g, :length], grad[b, h]
            p = torch.softmax(scale * (q[b, h] @ kk.T), -1)
            dp = go @ vv.T
            ds = p * (dp - (p * dp).sum(-1, keepdim=True))
            delta_bound = (go.abs() * out_bound[b, h]).sum(-1, keepdim=True)
            ds_bound = rel * ds.abs() + p * (delta_bound + 1e-5 * (go.abs() @ vv.abs().T))
            ds_row, ds_all, p_tiny = tiny, tiny, tiny
            if scaled:
                ds_row = 2.0 ** -39 * (go.norm(dim=-1, keepdim=True) * vv.norm(dim=-1).max() + delta_of(b, h))
                of_group = range(g * (heads // groups), (g + 1) * (heads // groups))
                most = max(float(grad[b, x].norm(dim=-1).max()) for x in of_group)
                ds_all = 2.0 ** -39 * (most * vv.norm(dim=-1) + max(float(delta_of(b, x).max()) for x in of_group))
                p_tiny = 2.0 ** -37
            p_bound = rel * p + p_tiny
            d[0][b, h] = scale * (ds @ kk)
            d[1][b, g, :length] += scale * (ds.T @ q[b, h])
            d[2][b, g, :length] += p.T @ go
            e[0][b, h] = scale * ((ds_bound + ds_row) @ kk.abs())
            e[1][b, g, :length] += scale * ((ds_bound + ds_all).T @ q[b, h].abs())
            e[2][b, g, :length] += p_bound.T @ go.abs()
    return tuple(d), tuple(x + u * t.abs() + last for x, t in zip(e, d))


def e4m3_values() -> torch.Tensor:
    """The non-negative finite e4m3 values in order (index = code)."""
    values = []
    for code in range(127):
        exponent, mantissa = code >> 3, code & 7
        values.append((mantissa / 8) * 2.0 ** -6 if exponent == 0 else (1 + mantissa / 8) * 2.0 ** (exponent - 7))
    return torch.tensor(values, dtype=torch.float64)


def quantise_rows(x):
    """``(values, exponents)``: each row of x as e4m3 codes times a power of two, in float64."""
    x = x.detach().cpu().double()
    finite = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))
    amax = finite.amax(-1)
    exponents = torch.zeros_like(amax)
    flat, flat_e = amax.reshape(-1), exponents.reshape(-1)
    for i, a in enumerate(flat.tolist()):
        if a > 0:
            e = -126
            while a > 448 * 2.0 ** e:
                e += 1
            flat_e[i] = e
    unit = torch.exp2(exponents)[..., None]
    table = e4m3_values()
    y = (finite / unit).contiguous()
    hi = torch.searchsorted(table, y).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    below, above = y - table[lo], table[hi] - y
    code = torch.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)
    values = table[code] * unit * torch.sign(x)
    return torch.where(torch.isfinite(x), values, torch.full_like(x, float("nan"))), exponents.long()
