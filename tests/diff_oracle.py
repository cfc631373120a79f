"""Differential attention in 64 bits, with elementwise bounds on what fp16 operands may cost a kernel.

u = 2^-11 is half a step of fp16.  A kernel rounds P (relative to a row reference), dS and its outputs to fp16 and sums in 32 bits;
values below fp16's normal range are off by at most 2^-25.  The bounds add these errors up with absolute values, nothing is measured.
"""
import math

import torch

U = 2.0 ** -11
TINY = 2.0 ** -25


def visible(sq, sk, causal, device):
    i, j = torch.arange(sq, device=device)[:, None], torch.arange(sk, device=device)[None]
    return j <= i + sk - sq if causal else torch.ones(sq, sk, dtype=torch.bool, device=device)


def maps(q, k, scale, seen):
    """A_1, A_2 of one head: q (sq, d), k (sk, d)."""
    out = []
    for a, b in zip(q.chunk(2, -1), k.chunk(2, -1)):
        s = torch.where(seen, a @ b.T * scale, torch.full((), -math.inf, dtype=q.dtype, device=q.device))
        out.append(torch.softmax(s, -1).nan_to_num(0.0))
    return out


def sequence(q, k, v, lam, causal, dout=None, scale=None):
    """One sequence: q (sq, h, d), k, v (sk, hk, d), lam (h,).  {name: (value, bound)} of out and, with dout, dq, dk, dv, dlam."""
    q, k, v, lam = (t.detach().double() for t in (q, k, v, lam))
    (sq, h, d), (sk, hk) = q.shape, k.shape[:2]
    scale = (d // 2) ** -0.5 if scale is None else scale
    seen = visible(sq, sk, causal, q.device)
    zero = torch.zeros_like
    val = {"out": zero(q), "dq": zero(q), "dk": zero(k), "dv": zero(v), "dlam": zero(lam)}
    tol = {n: zero(t) for n, t in val.items()}
    half = d // 2
    for i in range(h if sq and sk else 0):
        kk, vv, w = k[:, i // (h // hk)], v[:, i // (h // hk)], lam[i]
        a1, a2 = maps(q[:, i], kk, scale, seen)
        a, size = a1 - w * a2, a1 + w.abs() * a2
        # scores in 32 bits: products of d / 2 terms, the exponent's argument and the exponential
        s_err = 2.0 ** -21 * (1 + scale * (q[:, i].abs() @ kk.abs().T).amax(-1, keepdim=True))
        o, o2 = a @ vv, a2 @ vv
        tiny_v = (1 + w.abs()) * TINY * vv.abs().sum(0)
        o2_tol = (U + s_err) * (a2 @ vv.abs()) + TINY * vv.abs().sum(0)
        o_tol = (2 * U + s_err) * (size @ vv.abs()) + tiny_v  # 2 U: the maps' outputs may be rounded before the difference
        val["out"][:, i], tol["out"][:, i] = o, o_tol + U * o.abs() + TINY
        if dout is None:
            continue
        do = dout[:, i].double()
        dp = do @ vv.T
        b = i // (h // hk)
        val["dv"][:, b] += a.T @ do
        tol["dv"][:, b] += ((2 * U + s_err) * size).T @ do.abs() + (1 + w.abs()) * TINY * do.abs().sum(0)
        val["dlam"][i] = -(do * o2).sum()
        tol["dlam"][i] = (do.abs() * (o2_tol + U * o2.abs() + TINY)).sum() + 2.0 ** -20 * (do * o2).abs().sum()
        for m, (am, f) in enumerate(((a1, 1.0), (a2, -w))):
            at = slice(m * half, (m + 1) * half)
            delta = (am * dp).sum(-1, keepdim=True)
            # delta comes from rounded outputs: O_2, and O_1 = O + lam O_2
            o_m = o if m == 0 else o2
            off = o_tol + U * (o.abs() + o_m.abs()) + w.abs() * (o2_tol + U * o2.abs()) if m == 0 else o2_tol + U * o2.abs()
            d_delta = (do.abs() * (off + TINY)).sum(-1, keepdim=True) + 2.0 ** -20 * (do.abs() @ vv.abs().T).amax(-1, keepdim=True)
            ds = f * am * (dp - delta)
            fa = abs(f)
            # 4 U: dS, P, a weight folded into an operand, and the difference of two rounded terms
            ds_tol = (4 * U + s_err) * ds.abs() + fa * am * (d_delta + U * (do.abs() @ vv.abs().T)) + 4 * TINY * (1 + fa) * (1 + dp.abs())
            ds_tol = torch.where(seen, ds_tol, 0.0)
            val["dq"][:, i, at], tol["dq"][:, i, at] = scale * ds @ kk[:, at], scale * ds_tol @ kk[:, at].abs()
            val["dk"][:, b, at] += scale * ds.T @ q[:, i, at]
            tol["dk"][:, b, at] += scale * ds_tol.T @ q[:, i, at].abs()
    if dout is not None:
        for n in ("dq", "dk", "dv"):
            tol[n] += U * val[n].abs() + TINY
    return {n: (val[n], tol[n]) for n in (val if dout is not None else ("out",))}


def batch(q, k, v, lam, causal, dout=None, scale=None):
    """The same for (b, s, h, d); dlam is summed over the batch."""
    per = [sequence(q[i], k[i], v[i], lam, causal, None if dout is None else dout[i], scale) for i in range(q.shape[0])]
    return {n: tuple((torch.stack([p[n][e] for p in per]) if n != "dlam" else sum(p[n][e] for p in per)) for e in (0, 1)) for n in per[0]}


def check(got, want, name=""):
    value, bound = want
    assert got.shape == value.shape, (name, got.shape, value.shape)
    err = (got.double() - value).abs()
    assert torch.isfinite(got).all(), f"{name}: not finite"
    worst = (err / bound.clamp_min(1e-30)).max().item() if err.numel() else 0.0
    assert (err <= bound).all(), f"{name}: {worst:.2f} times the bound"
    return worst


def check_dlam(got, want):
    value, bound = want
    one = 2.0 ** -11 if got.dtype == torch.float16 else 2.0 ** -24
    if got.numel() == 1:
        value, bound = value.sum(), bound.sum()
    return check(got.reshape(value.shape), (value, bound + one * value.abs() + (TINY if got.dtype == torch.float16 else 0.0)), "dlam")
