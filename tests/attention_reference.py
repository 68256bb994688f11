"""Plain 64-bit attention with capped, biased and masked scores and its gradients, on the CPU, and the
error bounds that the GPU tests hold the kernels to.

Bounds (u: half a step of the input type, 2^-8 in bf16, 2^-11 in fp16; fp32 steps f = 2^-24), all of them
sums of the largest errors:

- scores x: D + 8 steps of sum |q||k| scale, as in cache_reference; a cap c adds its own evaluation, 16 f c; a
  bias its roundings, 8 f slope distance; the exponential 2^-16.  es is their sum.
- forward: P is rounded to the input type in numerator and denominator, u each; es in both; sums of n terms n f.
- lse: es, n f and a few steps of its magnitude.  P of the backward pass, exp(x - lse): r = 2 es + n f + ...
  relative.
- delta = go.o: the stored o's error (the forward bound) and D steps; go.v: D steps.
- gv = sum P go: (u + r) each, n f of sums, the output's rounding.
- dS = P (go.v - delta) (1 - t^2): P may be rounded once more on its way to gk: 2 u + r of itself, P times the
  errors of go.v and delta, and the derivative's own 16 f; then as a factor of q or k.
- fp16: P 2^12 and dS / top (the largest |go| of the rows that share the factor) are held with absolute errors
  of 2^-25 where they are small; results below 2^-14 likewise.
"""
from __future__ import annotations

import math

import torch

from cache_reference import F32, U


def visible(n, m, ranges=None, causal=False, window=None):
    """[B or 1, n, m]: which keys a row sees."""
    p = torch.arange(n)[:, None] + (m - n)
    j = torch.arange(m)[None]
    see = torch.ones(1, n, m, dtype=torch.bool)
    if ranges is not None:
        r = (ranges if ranges.dim() == 3 else ranges[None]).long()
        see = (j >= r[:, :, :1]) & (j < r[:, :, 1:])
    if causal:
        see = see & (j <= p)
    if window is not None:
        see = see & ((p - j).abs() < window)
    return see


def scores(q, k, *, scale, cap=None, slope=None):
    """x [n, m] in 64 bits, by steps that autograd can follow."""
    n, m = q.shape[0], k.shape[0]
    x = (q @ k.T) * scale
    if cap is not None:
        x = cap * torch.tanh(x / cap)
    if slope is not None:
        p = torch.arange(n)[:, None] + (m - n)
        x = x - slope * (p - torch.arange(m)).abs()
    return x


def head(q, k, v, see, **score):
    """(o, lse) of one head, differentiable; rows that see nothing: 0 and -inf."""
    x = scores(q, k, **score)
    top = torch.where(see, x.detach(), -math.inf).amax(1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, 0.0)
    # (rows and keys that do not see each other: their products are left out, whatever they are)
    e = torch.where(see, torch.exp(torch.where(see, x - top, 0.0)), 0.0)
    total = e.sum(1, keepdim=True)
    none = total == 0
    w = e / torch.where(none, 1.0, total)
    lse = torch.where(none[:, 0], -math.inf, torch.log(torch.where(none, 1.0, total))[:, 0] + top[:, 0])
    return w @ v, lse


def attend(q, k, v, see, *, scale, cap=None, slopes=None, go=None, glse=None):
    """Values and bounds: dicts of o, lse and, with go, gq, gk, gv."""
    B, H, N, D = q.shape
    KH, M = k.shape[1:3]
    g, u, half = H // KH, U[q.dtype], q.dtype == torch.float16
    qd, kd, vd = q.double(), k.double(), v.double()
    val = {"o": torch.zeros(B, H, N, D, dtype=torch.float64), "lse": torch.zeros(B, H, N, dtype=torch.float64)}
    if go is not None:
        val |= {"gq": torch.zeros_like(qd), "gk": torch.zeros_like(kd), "gv": torch.zeros_like(vd)}
    tol = {n: torch.zeros_like(x) for n, x in val.items()}
    for b in range(B):
        s = see[b % see.shape[0]]
        n_seen = s.sum(1, keepdim=True).double()
        for h in range(H):
            kh, slope = h // g, None if slopes is None else float(slopes[h])
            x = scores(qd[b, h], kd[b, kh], scale=scale, cap=cap, slope=slope)
            most = (qd[b, h].abs() @ kd[b, kh].abs().T) * scale
            es = (D + 8) * F32 * torch.where(s, most, 0.0).amax(1, keepdim=True) + 2.0 ** -16
            if cap is not None:
                es = es + 16 * F32 * cap
            if slope is not None:
                es = es + 8 * F32 * abs(slope) * max(M, N)
            o, lse = head(qd[b, h], kd[b, kh], vd[b, kh], s, scale=scale, cap=cap, slope=slope)
            w = torch.where(s, torch.exp(x - torch.where(torch.isfinite(lse), lse, 0.0)[:, None]), 0.0)
            val["o"][b, h], val["lse"][b, h] = o, lse
            tol_o = (2 * u + 2 * es + 2 * n_seen * F32) * (w @ vd[b, kh].abs()) + u * o.abs()
            if half:
                tol_o = tol_o + n_seen * F32 * vd[b, kh].abs().max() + 2.0 ** -25
            tol["o"][b, h] = tol_o
            el = es[:, 0] + n_seen[:, 0] * F32 + 4 * F32 * (1 + torch.where(torch.isfinite(lse), lse, 0.0).abs())
            tol["lse"][b, h] = el
            if go is None:
                continue
            gd = go[b, h].double()
            gl = torch.zeros(N, dtype=torch.float64) if glse is None else glse[b, h].double()
            r = es + el[:, None] + 2.0 ** -16
            dp = gd @ vd[b, kh].T
            delta = (gd * o).sum(1, keepdim=True) - gl[:, None]
            deriv = torch.ones_like(x)
            if cap is not None:
                deriv = 1 - torch.tanh((qd[b, h] @ kd[b, kh].T) * scale / cap) ** 2
            ds = torch.where(s, w * (dp - delta) * deriv, 0.0)
            e_dp = D * F32 * (gd.abs() @ vd[b, kh].abs().T)
            e_delta = (gd.abs() * (tol_o + D * F32 * o.abs())).sum(1, keepdim=True) + F32 * delta.abs()
            e_ds = ds.abs() * (2 * u + r) + w * (e_dp + e_delta + 16 * F32 * (dp - delta).abs())
            e_p = w * (u + r)
            row_top = gd.abs().amax(1, keepdim=True)
            e_q = e_ds + (2.0 ** -25 * row_top * s if half else 0.0)
            e_k = e_ds + (2.0 ** -25 * go[b, kh * g:(kh + 1) * g].double().abs().max() * s if half else 0.0)
            e_p = e_p + (2.0 ** -37 * s if half else 0.0)
            val["gq"][b, h] = scale * (ds @ kd[b, kh])
            val["gk"][b, kh] += scale * (ds.T @ qd[b, h])
            val["gv"][b, kh] += w.T @ gd
            tol["gq"][b, h] = scale * ((e_q + n_seen * F32 * ds.abs()) @ kd[b, kh].abs())
            tol["gk"][b, kh] += scale * ((e_k + 2 * N * g * F32 * ds.abs()).T @ qd[b, h].abs())
            tol["gv"][b, kh] += (e_p + 2 * N * g * F32 * w).T @ gd.abs()
    for n in ("gq", "gk", "gv"):
        if n in val:
            tol[n] += u * val[n].abs() + (2.0 ** -25 if half else 0.0)
    return val, tol
