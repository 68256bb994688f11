"""Plain 64-bit forms of the paged cache's operators and of the q/k norm with
rotation, on the CPU, and the error bounds that the GPU tests hold the kernels to.

Bounds (u: half a step of the output type relative to the value, 2^-8 in bf16,
2^-11 in fp16; fp32 steps 2^-24):

- scores: a dot product of D terms in fp32 is off by at most D 2^-24 sum |q||k|;
  its scaling, the offset's and the exponent's roundings add a few steps of the
  same magnitude.  score_error() is that, plus 2^-16 for the exponential.  A
  weight p is then off by that much relative to itself.
- attention: P is rounded to the input type (relative u each, numerator and
  denominator alike): at most 2 u sum w|v|; fp16 P below 2^-14 are off by up to
  2^-25 absolute against a sum of at least 1/2: n 2^-24 max|v|; the weights'
  own error twice; sums of n terms n 2^-24; the output's rounding u |o|.
- key weights: relative score error, plus a sum of n terms.
- norm: a few fp32 steps of the pair's magnitude, the output's rounding.
"""
from __future__ import annotations

import math

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
F32 = 2.0 ** -24


def keys_of(cache, row, n):
    """Keys 0..n-1 of a sequence: [KH, n, ...] and which of them have a page."""
    pages, kh, size = cache.shape[:3]
    ids = row[: -(-n // size)].long() if n else row[:0].long()
    there = (ids >= 0) & (ids < pages)
    rows = cache[ids.clamp(0, pages - 1)].transpose(0, 1)
    rows = rows.reshape(kh, -1, *cache.shape[3:])[:, :n]
    return rows, there.repeat_interleave(size)[:n]


def sequences(cu, lens, tokens, max_q=None, max_kv=None, capacity=None):
    """(sequence, first row, rows computed, length, index of the first new key)."""
    for b in range(len(lens)):
        c0 = min(max(int(cu[b]), 0), tokens)
        c1 = min(max(int(cu[b + 1]), c0), tokens)
        n = max(int(lens[b]), 0)
        for limit in (max_kv, capacity):
            n = n if limit is None else min(n, limit)
        nq = c1 - c0
        yield b, c0, nq if max_q is None else min(nq, max_q), n, n - nq


def attend(q, kc, vc, table, cu, lens, *, scale, causal=True, max_q=None, max_kv=None):
    """(o, lse, bound on o, bound on lse) for the rows that are computed, NaN elsewhere."""
    T, H, D = q.shape
    kh, size = kc.shape[1], kc.shape[2]
    g = H // kh
    u = U[q.dtype]
    o = torch.full((T, H, D), math.nan, dtype=torch.float64)
    lse = torch.full((T, H), math.nan, dtype=torch.float64)
    tol_o, tol_l = torch.zeros_like(o), torch.zeros_like(lse)
    for b, c0, nq, n, first in sequences(cu, lens, T, max_q, max_kv, table.shape[1] * size):
        k, there = keys_of(kc, table[b], n)
        v, _ = keys_of(vc, table[b], n)
        j = torch.arange(n)
        for i in range(nq):
            see = there & ((j <= first + i) if causal else torch.ones(n, dtype=torch.bool))
            kk, vv = k[:, see].double(), v[:, see].double()
            for h in range(H):
                x = q[c0 + i, h].double()
                s = kk[h // g] @ x * scale
                if s.numel() == 0:
                    o[c0 + i, h], lse[c0 + i, h] = 0.0, -math.inf
                    continue
                lse[c0 + i, h] = torch.logsumexp(s, 0)
                w = torch.exp(s - lse[c0 + i, h])
                o[c0 + i, h] = w @ vv[h // g]
                es = score_error(x, kk[h // g], scale)
                m = w @ vv[h // g].abs()
                tol = (2 * u + 2 * es + 2 * n * F32) * m + u * o[c0 + i, h].abs()
                if q.dtype == torch.float16:  # subnormal P and outputs
                    most = torch.where(torch.isfinite(vv[h // g]), vv[h // g].abs(), 0.0).max()
                    tol = tol + n * F32 * most + 2.0 ** -25
                tol_o[c0 + i, h] = tol
                tol_l[c0 + i, h] = es + n * F32 + 4 * F32 * (1 + lse[c0 + i, h].abs())
    return o, lse, tol_o, tol_l


def score_error(x, kk, scale):
    most = float((kk.abs() @ x.abs()).max()) * scale
    return (len(x) + 8) * F32 * most + 2.0 ** -16


def key_weights(q, lse, kc, table, cu, lens, w, *, scale, causal=True, max_q=None, max_kv=None):
    """(new weights, bound), every slot."""
    T, H, D = q.shape
    kh, size = kc.shape[1], kc.shape[2]
    g = H // kh
    out, tol = w.double().clone(), torch.zeros(w.shape, dtype=torch.float64)
    for b, c0, nq, n, first in sequences(cu, lens, T, max_q, max_kv, table.shape[1] * size):
        if nq == 0 or n == 0:
            continue
        k, there = keys_of(kc, table[b], n)
        add, err = torch.zeros(kh, n, dtype=torch.float64), torch.zeros(kh, n, dtype=torch.float64)
        j = torch.arange(n)
        for i in range(nq):
            see = there & ((j <= first + i) if causal else torch.ones(n, dtype=torch.bool))
            if not see.any():
                continue
            for h in range(H):
                l = lse[c0 + i, h].double()
                if torch.isinf(l):  # -inf adds nothing by definition; +inf: exp(-inf) is exactly 0
                    continue
                x = q[c0 + i, h].double()
                kk = k[h // g][see].double()
                p = torch.exp(kk @ x * scale - l)
                add[h // g][see] += p
                err[h // g][see] += p * (score_error(x, kk, scale) + 4 * F32 * l.abs())
        for t in range(n):
            page = int(table[b, t // size])
            if not 0 <= page < kc.shape[0]:
                continue
            old = out[page, :, t % size] if t < first else torch.zeros(kh, dtype=torch.float64)
            out[page, :, t % size] = old + add[:, t]
            tol[page, :, t % size] = err[:, t] + (nq * g + 8) * F32 * (add[:, t] + old)
    return out, tol


def evict(kc, vc, w, table, lens, new_table, *, keep, recent, max_kv=None):
    """New lengths, kept indices and the caches afterwards."""
    pages, kh, size = kc.shape[:3]
    kc, vc, w = kc.clone(), vc.clone(), w.clone()
    src = kc.clone(), vc.clone(), w.clone()
    B = table.shape[0]
    out_lens = torch.zeros(B, dtype=torch.int32)
    kept = torch.full((B, kh, keep), -1, dtype=torch.int32)
    for b in range(B):
        n = min(max(int(lens[b]), 0), table.shape[1] * size)
        n = n if max_kv is None else min(n, max_kv)
        m = min(n, keep)
        used = torch.cat([table[b, : -(-n // size)], new_table[b, : -(-m // size)]])
        if ((used < 0) | (used >= pages)).any():
            continue
        out_lens[b] = m
        for h in range(kh):
            if n <= keep:
                idx = list(range(n))
            else:
                wt = keys_of(src[2], table[b], n)[0][h].tolist()
                rank = [math.inf if math.isnan(x) else x for x in wt]
                nan = [math.isnan(x) for x in wt]
                old = sorted(range(n - recent), key=lambda i: (not nan[i], -rank[i], i))
                idx = sorted(old[: keep - recent]) + list(range(n - recent, n))
            for t, i in enumerate(idx):
                kept[b, h, t] = i
                here = (int(table[b, i // size]), h, i % size)
                there = (int(new_table[b, t // size]), h, t % size)
                kc[there], vc[there], w[there] = src[0][here], src[1][here], src[2][here]
    return out_lens, kept, kc, vc, w


def norm_rope(x, w, cos, sin, pos, *, eps, interleaved):
    """x [..., D] at positions pos broadcast to x.shape[:-1]: (y, bound)."""
    D, r = x.shape[-1], 2 * cos.shape[1]
    xd = x.double()
    n = xd * torch.rsqrt(xd.square().mean(-1, keepdim=True) + eps) * w.double()
    ok = (pos >= 0) & (pos < cos.shape[0])
    c = cos.double()[pos.clamp(0, cos.shape[0] - 1).long()]
    s = sin.double()[pos.clamp(0, cos.shape[0] - 1).long()]
    y, mag = n.clone(), n.abs()
    a, b = (n[..., 0:r:2], n[..., 1:r:2]) if interleaved else (n[..., : r // 2], n[..., r // 2: r])
    m = torch.sqrt(a * a + b * b)
    if interleaved:
        y[..., 0:r:2], y[..., 1:r:2] = a * c - b * s, b * c + a * s
        mag[..., 0:r:2] = mag[..., 1:r:2] = m
    else:
        y[..., : r // 2], y[..., r // 2: r] = a * c - b * s, b * c + a * s
        mag[..., : r // 2] = mag[..., r // 2: r] = m
    y[~ok] = math.nan
    u = U[x.dtype]
    # fp32: D steps of the mean square halved by the root, four of the products
    # and the rotation's three on a pair; fp16 outputs below 2^-14 are subnormal
    tol = u * y.abs() + (D / 2 + 8) * F32 * 2 * mag + (2.0 ** -25 if x.dtype == torch.float16 else 0.0)
    return y, tol


def norm_rope_grad(x, w, cos, sin, pos, dy, *, eps, interleaved):
    """Formula's gradients: (dx, bound, dw, bound); dw over all leading dims."""
    D, r = x.shape[-1], 2 * cos.shape[1]
    xd, g = x.double(), dy.double().clone()
    c, s = cos.double()[pos.long()], sin.double()[pos.long()]
    gd = dy.double()
    if interleaved:
        a, b = gd[..., 0:r:2], gd[..., 1:r:2]
        g[..., 0:r:2], g[..., 1:r:2] = a * c + b * s, b * c - a * s
    else:
        a, b = gd[..., : r // 2], gd[..., r // 2: r]
        g[..., : r // 2], g[..., r // 2: r] = a * c + b * s, b * c - a * s
    rstd = torch.rsqrt(xd.square().mean(-1, keepdim=True) + eps)
    xh, gw = xd * rstd, g * w.double()
    dx = rstd * (gw - xh * (gw * xh).mean(-1, keepdim=True))
    dims = tuple(range(x.dim() - 1))
    dw = (g * xh).sum(dims)
    # The inverse rotation leaves three steps of a pair of dy on g; D steps on
    # the mean and the root.
    pair = gd.abs().amax(-1, keepdim=True) * 2
    mag = rstd * (pair * w.double().abs() + xh.abs() * (pair * w.double().abs() * xh.abs()).mean(-1, keepdim=True))
    u = U[x.dtype]
    tol_x = u * dx.abs() + (D + 16) * F32 * mag + (2.0 ** -25 if x.dtype == torch.float16 else 0.0)
    rows = x.numel() // D
    tol_w = ((pair + g.abs()) * xh.abs()).sum(dims) * ((D + 16) * F32) + (g * xh).abs().sum(dims) * rows * F32
    tol_w = tol_w + (U[w.dtype] * dw.abs() if w.dtype != torch.float32 else 0.0)
    return dx, tol_x, dw, tol_w


def check(name, got, want, tol):
    """got within tol of want everywhere; NaN and infinities in the same places."""
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    odd = ~torch.isfinite(want)
    same = (got[odd] == want[odd]) | (torch.isnan(got[odd]) & torch.isnan(want[odd]))
    assert bool(same.all()), f"{name}: {int((~same).sum())} non-finite values differ"
    off = (got - want).abs()[~odd] - tol[~odd]
    if off.numel():
        worst = int(off.argmax())
        assert off[worst] <= 0, (f"{name}: off by {float((got - want).abs()[~odd][worst]):.3e}, "
                                 f"bound {float(tol[~odd][worst]):.3e} at a value of "
                                 f"{float(want[~odd][worst]):.3e}")
