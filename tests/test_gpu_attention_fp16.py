"""fp16 gradients of attention over the type's range: what one key's or row's gradients are rounded to goes by what
it sees, and nothing overflows or is lost on the way to a result that is a number."""
from __future__ import annotations

import math

import pytest
import torch

import attention_reference as A
import cache_reference as R
from test_gpu_attention import DEV, call, rows

pytestmark = pytest.mark.gpu
HALF = torch.float16
EDGES = [0, 70, 150, 280]  # of documents; rows from 280 on belong to none
N = 300
# few workgroups, whose teams share them, and more than the GPU holds at once
SHAPES = [(64, 2, 1), (128, 4, 2), (64, 280, 140), (128, 280, 280)]


def inputs(D, H, KH, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    q, go = (rows(1, H, N, D, HALF, g, scale=s) for s in (1.0, scale))
    return [q, *(rows(1, KH, N, D, HALF, g) for _ in range(2)), go]


def documents(fa):
    return fa.document_ranges(torch.tensor(EDGES), N)


def inside(i):
    at = torch.zeros(N, dtype=torch.bool)
    at[EDGES[i]:EDGES[i + 1]] = True
    return at


@pytest.mark.parametrize("D,H,KH", SHAPES)
@pytest.mark.parametrize("cap", [None, 30.0])
@pytest.mark.parametrize("bad", [math.inf, math.nan, 60000.0])
def test_no_bit_goes_by_the_gradients_of_unseen_rows(fa, D, H, KH, cap, bad):
    """Another document's incoming gradients are infinities, NaN or as large as the type holds, beside some of
    deviation 512, whose dS overflows without a factor of their own."""
    print("case unseen", D, H, cap, bad, flush=True)
    tensors = inputs(D, H, KH, 81, 512.0)
    dirty = [x.clone() for x in tensors]
    tensors[3][:, :, inside(1)] = 0
    dirty[3][:, :, inside(1)] = bad
    dirty[3][:, :, EDGES[-1]:] = bad
    opt = {} if cap is None else dict(softcap=cap)
    a, b = (call(fa, x, documents(fa), None, opt) for x in (tensors, dirty))
    for n in ("gq", "gk", "gv"):
        for i in (0, 2):
            assert torch.equal(a[n][:, :, inside(i)], b[n][:, :, inside(i)]), (n, i)
            assert bool(torch.isfinite(b[n][:, :, inside(i)]).all()), (n, i)


@pytest.mark.parametrize("D,H,KH", SHAPES)
def test_no_bit_goes_by_the_gradients_of_earlier_rows(fa, D, H, KH):
    """A causal mask: keys behind row 100 are not seen by it."""
    print("case earlier", D, H, flush=True)
    tensors = inputs(D, H, KH, 82, 512.0)
    dirty = [x.clone() for x in tensors]
    tensors[3][:, :, 100] = 0
    dirty[3][:, :, 100] = math.inf
    a, b = (call(fa, x, None, None, dict(causal=True)) for x in (tensors, dirty))
    for n in ("gk", "gv"):
        assert torch.equal(a[n][:, :, 101:], b[n][:, :, 101:]), n
        assert bool(torch.isfinite(b[n][:, :, 101:]).all()), n


@pytest.mark.parametrize("D,H,KH", SHAPES)
@pytest.mark.parametrize("loud,quiet", [(2.0 ** 9, 2.0 ** -9), (2.0 ** 10, 2.0 ** -6), (2.0 ** 4, 2.0 ** -11)])
def test_a_quiet_document_beside_a_loud_one(fa, D, H, KH, loud, quiet):
    """Each document within the bounds that it has by itself."""
    print("case quiet", D, H, loud, quiet, flush=True)
    tensors = inputs(D, H, KH, 83)
    factor = torch.full((N, 1), quiet)
    factor[inside(1)] = loud
    tensors[3] = (tensors[3].float() * factor).to(HALF)
    got = call(fa, tensors, documents(fa), None, {})
    heads = slice(0, 2 * H // KH)  # (two of k and v's, to keep the 64-bit form short)
    for i in range(3):
        at = inside(i)
        part = [x[:, heads if x.shape[1] == H else slice(0, 2)][:, :, at] for x in tensors]
        see = A.visible(part[0].shape[2], part[0].shape[2], causal=True)
        val, tol = A.attend(*part[:3], see, scale=1 / math.sqrt(D), go=part[3])
        for n in ("gq", "gk", "gv"):
            x = got[n].cpu()[:, heads if n == "gq" else slice(0, 2)][:, :, at]
            R.check(f"{n} of document {i}", x, val[n], tol[n])
