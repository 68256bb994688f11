"""No bit of a document's results goes by what its neighbours in the row hold: zeros, loud or quiet values,
infinities, NaN, in q, k, v and both incoming gradients, for seeded shapes and masks."""
from __future__ import annotations

import math
import random

import pytest
import torch

from test_gpu_attention import call, documents

pytestmark = pytest.mark.gpu


def fill(x, others, r):
    """Other documents' rows, in place."""
    kind = r.choice(["zero", "loud", "quiet", "inf", "nan", "one"])
    if kind == "zero":
        x[:, :, others] = 0
    elif kind in ("loud", "quiet"):
        x[:, :, others] *= 2000.0 if kind == "loud" else 2.0 ** -10
    elif kind in ("inf", "nan"):
        x[:, :, others] = math.inf if kind == "inf" else math.nan
    else:
        row = int(others.nonzero()[r.randrange(int(others.sum())), 0])
        x[:, :, row, r.randrange(x.shape[3])] = r.choice([math.inf, -math.inf, math.nan, 60000.0])


@pytest.mark.parametrize("seed", range(16))
def test_a_document_among_others(fa, seed):
    print("case isolation", seed, flush=True)
    r, g = random.Random(seed), torch.Generator().manual_seed(seed)
    D, dt = (64, 128)[seed % 2], (torch.float16, torch.float16, torch.bfloat16)[seed % 3]
    KH = r.choice([1, 2, 3]) if seed % 4 else 150
    H, N = KH * (r.choice([1, 2, 4]) if KH < 10 else 1), r.choice([129, 200, 300, 700] if KH < 10 else [140, 300])
    ends = sorted(r.sample(range(1, N), r.choice([1, 2, 4]))) + [N]
    first = [0, *ends[:-1]]
    ranges = documents(fa, ends, N, causal=r.random() < 0.6)
    opt = {}
    if r.random() < 0.3:
        opt["softcap"] = 20.0
    if r.random() < 0.2:
        opt["window"] = 40
    slopes = 0.05 * torch.arange(1, H + 1).float() if r.random() < 0.3 else None
    tensors = [torch.randn(2, h, N, D, generator=g).to(dt) for h in (H, KH, KH, H)]
    glse = torch.randn(2, H, N, generator=g) if r.random() < 0.5 else None
    i = r.randrange(len(ends))
    mine = torch.zeros(N, dtype=torch.bool)
    mine[first[i]:ends[i]] = True
    got = []
    for _ in range(2):
        x = [t.clone() for t in tensors]
        for t in x:
            fill(t, ~mine, r)
        gl = None if glse is None else glse * torch.where(mine, 1.0, r.choice([1e4, 1e-6, math.inf]))
        got.append(call(fa, x, ranges, slopes, opt, gl))
    for n in got[0]:
        a, b = (y[n][:, :, mine] for y in got)
        assert torch.equal(a, b), n
        assert bool(torch.isfinite(a).all()), n
