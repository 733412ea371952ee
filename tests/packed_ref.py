"""Packed causal attention in 64 bits, and how far the kernels may be from it.

A value is off by at most half a step of a rounding: u = eps / 2 of the 16-bit type, relative to it.  The forward rounds
each weight P once (its operand of P V) and o once, so with A = P |v|
    |o - o*| <= u A + u |o*|.
The backward rounds P (operand of dV), dS (operand of dQ and dK) and each gradient once; with an o as above delta =
rowsum(o dO) is off by at most e_i = sum_d |dO_id| u (A_id + |o_id|) (less where it takes o before its rounding), and dS by P e:
    |dV - dV*| <= u P^T |dO| + u |dV*|,
    |dQ - dQ*| <= sm (u |dS| + P e) |K| + u |dQ*|,   |dK - dK*| <= sm (u |dS| + P e)^T |Q| + u |dK*|.
32-bit arithmetic adds FP32 = 2^-16 of the sums of absolute values (weights: the exponent s c - m, of size up to 2^6 here,
is off by some 2^-24 of that and of the D products behind s; sums of up to 2^12 terms), terms of the second order in u are
below 2 % of the first.  fp16 weights below 2^-14 have steps of 2^-24, so half a step is 2^-25 of the row's reference weight
1 (the row's sum is at least 1): N 2^-25 max|v| more for N keys, the same for P and dS in the backward.
"""
import torch

FP32 = 2.0 ** -16


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def sees(nq, nk, causal, device):
    i, j = torch.arange(nq, device=device)[:, None], torch.arange(nk, device=device)[None, :]
    return j <= i + nk - nq if causal else torch.ones(nq, nk, dtype=torch.bool, device=device)


def one(q, k, v, grad, seen, sm, dtype):
    """One head of one sequence, all in 64 bits: {name: (value, bound before the value's own rounding)}."""
    u = half_step(dtype)
    tiny = (2.0 ** -25 * k.shape[0]) if dtype == torch.float16 else 0.0
    vmax = float(v.abs().max()) if v.numel() else 0.0
    s = (q @ k.t().contiguous() * sm).masked_fill(~seen, float("-inf"))
    some = seen.any(-1, keepdim=True)
    p = torch.where(some, torch.softmax(s, -1), torch.zeros_like(s)) if s.shape[1] else s
    p = torch.nan_to_num(p)
    a = p @ v.abs()
    o = p @ v
    got = {"o": (o, (u + FP32) * a + tiny * vmax)}
    if grad is None:
        return got
    dp = grad @ v.t().contiguous()
    delta = (o * grad).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    e = (grad.abs() * ((u + FP32) * a + tiny * vmax + u * o.abs())).sum(-1, keepdim=True)
    sums = p * (grad.abs() @ v.abs().t().contiguous() + (o * grad).abs().sum(-1, keepdim=True))   # |dS| before it cancels
    off = u * ds.abs() + p * e + FP32 * sums
    small = (2.0 ** -25) if dtype == torch.float16 else 0.0
    off = off + small * seen
    got["dv"] = (p.t().contiguous() @ grad, ((u + FP32) * p + small * seen).t().contiguous() @ grad.abs())
    got["dq"] = (sm * (ds @ k), sm * (off @ k.abs()))
    got["dk"] = (sm * (ds.t().contiguous() @ q), sm * (off.t().contiguous() @ q.abs()))
    return got


def reference(q, k, v, lengths, k_lengths, causal, sm, grad=None):
    """{name: (value, bound)} for packed tensors; zeros, and a bound of 0, outside every sequence."""
    dtype = q.dtype
    u, group = half_step(dtype), q.shape[0] // k.shape[0]
    qd, kd, vd = (t.detach().double() for t in (q, k, v))
    gd = None if grad is None else grad.double()
    shapes = {"o": qd, "dq": qd, "dk": kd, "dv": vd} if grad is not None else {"o": qd}
    value = {n: torch.zeros(t.shape, dtype=torch.float64, device=q.device) for n, t in shapes.items()}
    bound = {n: torch.zeros(t.shape, dtype=torch.float64, device=q.device) for n, t in shapes.items()}
    a = b = 0
    for nq, nk in zip(lengths, k_lengths):
        rows, keys = slice(a, a + nq), slice(b, b + nk)
        seen = sees(nq, nk, causal, q.device)
        for h in range(q.shape[0]):
            g = h // group
            got = one(qd[h, rows], kd[g, keys], vd[g, keys], None if gd is None else gd[h, rows], seen, sm, dtype)
            for n, (x, y) in got.items():
                hh, at = (h, rows) if n in ("o", "dq") else (g, keys)
                value[n][hh, at] += x
                bound[n][hh, at] += y
        a, b = a + nq, b + nk
    return {n: (value[n], 1.02 * bound[n] + (u + FP32) * value[n].abs() + 1e-30) for n in value}


def assert_within(got, want, name):
    value, bound = want
    off = (got.double() - value).abs()
    assert torch.isfinite(got.float()).all(), f"{name}: not finite"
    worst = float((off / bound.clamp_min(1e-300)).max()) if off.numel() else 0.0
    assert bool((off <= bound).all()), f"{name}: {worst:.2f} times the bound"
