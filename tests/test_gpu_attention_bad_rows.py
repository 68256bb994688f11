"""One infinity or NaN among the rows of a backward pass: every key that sees its row says so, in spans of rows
that are seen whole and in those at an edge of a mask; the other keys' results keep every bit."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_attention import DEV, DT, call, rows

pytestmark = pytest.mark.gpu
N, ROW, DIM = 300, 100, 3


def masks(fa):
    """Name, key ranges, options, the keys that see row ROW."""
    docs = fa.document_ranges(torch.tensor([0, 30, 180, N]), N)
    window = dict(causal=True, window=60)
    return {"causal": (None, dict(causal=True), (0, ROW + 1)), "docs": (docs, {}, (30, ROW + 1)),
            "window": (None, window, (ROW - 59, ROW + 1)), "full": (None, {}, (0, N))}


# heads: few workgroups, whose teams share them, and more than the GPU holds at once
@pytest.mark.parametrize("D,dtype,H", [(64, "fp16", 2), (128, "fp16", 2), (64, "bf16", 2), (128, "bf16", 2),
                                       (64, "bf16", 260), (128, "fp16", 260)])
@pytest.mark.parametrize("mask", ["causal", "docs", "window", "full"])
@pytest.mark.parametrize("bad", [math.nan, -math.inf])
def test_a_bad_incoming_gradient_reaches_the_keys_that_see_its_row(fa, D, dtype, H, mask, bad):
    print("case bad gradient", D, dtype, H, mask, bad, flush=True)
    g = torch.Generator().manual_seed(70)
    q, k, v, go = (rows(1, H, N, D, DT[dtype], g) for _ in range(4))
    ranges, opt, (first, end) = masks(fa)[mask]
    go[0, 0, ROW, DIM] = 0.0
    dirty = go.clone()
    dirty[0, 0, ROW, DIM] = bad
    want, got = (call(fa, (q, k, v, x), ranges, None, opt) for x in (go, dirty))
    assert not bool(torch.isfinite(got["gv"][0, 0, first:end, DIM]).any())
    assert not bool(torch.isfinite(got["gk"][0, 0, first:end]).any())
    assert not bool(torch.isfinite(got["gq"][0, 0, ROW]).any())
    unseen = torch.ones(N, dtype=torch.bool)
    unseen[first:end] = False
    assert torch.equal(got["gv"][0, 0, unseen], want["gv"][0, 0, unseen])
    other = torch.arange(N) != ROW
    assert torch.equal(got["gq"][0, 0, other], want["gq"][0, 0, other])
    for n in ("gq", "gk", "gv"):  # the other heads
        assert torch.equal(got[n][0, 1:], want[n][0, 1:]), n


@pytest.mark.parametrize("D,dtype,H", [(64, "fp16", 2), (128, "bf16", 2), (64, "bf16", 260), (128, "bf16", 260)])
@pytest.mark.parametrize("mask", ["causal", "docs", "window", "full"])
def test_an_infinite_query_of_capped_scores_reaches_the_keys_that_see_its_row(fa, D, dtype, H, mask):
    """Its scores are the cap and its logsumexp a number: dk is 0 times an infinity."""
    print("case bad query", D, dtype, H, mask, flush=True)
    g = torch.Generator().manual_seed(71)
    q, k, v, go = (rows(1, H, N, D, DT[dtype], g) for _ in range(4))
    ranges, opt, (first, end) = masks(fa)[mask]
    dirty = q.clone()
    dirty[0, 0, ROW, DIM] = math.inf
    got = call(fa, (dirty, k, v, go), ranges, None, dict(opt, softcap=20.0))
    want = call(fa, (q, k, v, go), ranges, None, dict(opt, softcap=20.0))
    assert bool(torch.isfinite(got["lse"]).all())
    assert not bool(torch.isfinite(got["gk"][0, 0, first:end, DIM]).any())
    unseen = torch.ones(N, dtype=torch.bool)
    unseen[first:end] = False
    for n in ("gk", "gv"):
        assert torch.equal(got[n][0, 0, unseen], want[n][0, 0, unseen]), n
        assert torch.equal(got[n][0, 1:], want[n][0, 1:]), n
