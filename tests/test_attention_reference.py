"""The 64-bit gradients that the GPU tests compare with, against finite differences and autograd (CPU)."""
from __future__ import annotations

import pytest
import torch

import attention_reference as R

CASES = [
    # H, KH, N, M, causal, window, cap, slopes, ranges
    (2, 1, 7, 7, True, None, None, False, None),
    (4, 2, 6, 9, True, 4, 3.0, True, None),
    (2, 2, 8, 8, False, 3, None, True, None),
    (3, 1, 6, 6, False, None, 2.0, False, [[0, 3], [0, 3], [0, 3], [3, 3], [3, 5], [3, 6]]),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_gradients_against_differences_and_autograd(case):
    H, KH, N, M, causal, window, cap, with_slopes, ranges = case
    g = torch.Generator().manual_seed(1)
    q, go = (torch.randn(1, H, N, 8, generator=g, dtype=torch.float64) for _ in range(2))
    k, v = (torch.randn(1, KH, M, 8, generator=g, dtype=torch.float64) for _ in range(2))
    q, k, v, go = (x.half().double() for x in (q, k, v, go))
    glse = torch.randn(1, H, N, generator=g, dtype=torch.float64).float()
    slopes = torch.rand(H, generator=g).float() if with_slopes else None
    see = R.visible(N, M, None if ranges is None else torch.tensor(ranges), causal, window)
    val, _ = R.attend(q.half(), k.half(), v.half(), see, scale=0.3, cap=cap, slopes=slopes, go=go.half(), glse=glse)

    def loss(q, k, v):
        total = 0.0
        for h in range(H):
            o, lse = R.head(q[0, h], k[0, h // (H // KH)], v[0, h // (H // KH)], see[0], scale=0.3, cap=cap,
                            slope=None if slopes is None else float(slopes[h]))
            some = torch.isfinite(lse)
            total = total + (o * go[0, h]).sum() + (lse[some] * glse[0, h].double()[some]).sum()
        return total

    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    auto = torch.autograd.grad(loss(*leaves), leaves)
    for name, x, a in zip(("gq", "gk", "gv"), (q, k, v), auto):
        assert (val[name] - a).abs().max() < 1e-10, name
        for _ in range(3):
            d = torch.randn(x.shape, generator=g, dtype=torch.float64)
            args = {"gq": q, "gk": k, "gv": v}
            up, down = dict(args), dict(args)
            up[name], down[name] = x + 1e-5 * d, x - 1e-5 * d
            diff = (loss(*up.values()) - loss(*down.values())) / 2e-5
            assert abs(diff - (val[name] * d).sum()) < 1e-6 * (1 + abs(diff)), name
