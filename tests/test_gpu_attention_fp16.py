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


def lost(tensors, see, opt, glse, scale):
    """What dS may lose to fp16's least step, 2^-25 by its factor, beside A.attend's bounds: of a key's sum below
    2^-37 of the largest |go| |v| + |delta| of a row that sees it; of a row's 2^-37 of |go| 64 + |delta|, or 2^-26
    of its largest |dS| where that overflows."""
    q, k, v, go = (x.double() for x in tensors)
    H, KH = q.shape[1], k.shape[1]
    out = {"gq": torch.zeros_like(q), "gk": torch.zeros_like(k)}
    s = see[0].double()
    for h in range(H):
        kh = h // (H // KH)
        o, lse = A.head(q[0, h], k[0, kh], v[0, kh], see[0], scale=scale, cap=opt.get("softcap"))
        delta = (go[0, h] * o).sum(1) - (0.0 if glse is None else glse[0, h].double())
        bound = go[0, h].norm(dim=1)[:, None] * v[0, kh].norm(dim=1)[None] + delta.abs()[:, None]
        w = s * torch.exp(A.scores(q[0, h], k[0, kh], scale=scale, cap=opt.get("softcap")) - lse[:, None]).clamp(max=1.0)
        ds = (w * (go[0, h] @ v[0, kh].T - delta[:, None])).abs().amax(1, keepdim=True)
        most = torch.maximum(2.0 ** -37 * (64 * go[0, h].norm(dim=1) + delta.abs())[:, None], 2.0 ** -26 * ds)
        out["gq"][0, h] = scale * ((most * s) @ k[0, kh].abs())
        out["gk"][0, kh] += scale * (2.0 ** -37 * (bound * s).amax(0)[:, None] * (s.T @ q[0, h].abs()))
    return out


def check_against_64_bits(fa, tensors, opt, glse=None):
    D, n = tensors[0].shape[3], tensors[0].shape[2]
    see, scale = A.visible(n, n, causal=True, window=opt.get("window")), 1 / math.sqrt(D)
    got = call(fa, tensors, None, None, dict(opt, causal=True), glse)
    val, tol = A.attend(*tensors[:3], see, scale=scale, cap=opt.get("softcap"), go=tensors[3], glse=glse)
    more = lost(tensors, see, opt, glse, scale)
    for n in ("gq", "gk", "gv"):
        assert bool((val[n].abs() < 65000).all()), n
        R.check(n, got[n], val[n], tol[n] + more.get(n, 0.0))


@pytest.mark.parametrize("D,H,KH", [(64, 2, 1), (128, 4, 2)])
@pytest.mark.parametrize("cap", [None, 20.0])
@pytest.mark.parametrize("go,glse", [(0.0, 1.0), (0.0, 64.0), (0.0, 4096.0), (2.0 ** -14, 1.0), (2.0 ** -20, 3.0),
                                     (1.0, 1000.0), (2.0 ** 9, 2.0 ** -20)])
def test_gradients_of_the_logsumexp(fa, D, H, KH, cap, go, glse):
    """A loss on lse beside o's, of any size: dS is P (go.v - go.o + glse)."""
    print("case lse", D, H, cap, go, glse, flush=True)
    tensors = inputs(D, H, KH, 84, go)
    g = torch.Generator().manual_seed(85)
    check_against_64_bits(fa, tensors, {} if cap is None else dict(softcap=cap),
                          glse * torch.randn(1, H, N, generator=g))


@pytest.mark.parametrize("D,H,KH", [(64, 2, 1), (128, 4, 2)])
@pytest.mark.parametrize("cap", [None, 20.0])
@pytest.mark.parametrize("size,go", [(100.0, 1.0), (5000.0, 1.0), (60000.0, 2.0 ** -6), (2.0 ** -12, 1.0)])
def test_values_of_any_size(fa, D, H, KH, cap, size, go):
    """Rows of v of one sign and one size and rows of go of one sign: go.v is all of |go| |v|.  (Small keys and
    queries: dq and dk are numbers.)"""
    print("case values", D, H, cap, size, go, flush=True)
    tensors = inputs(D, H, KH, 86)
    g = torch.Generator().manual_seed(87)
    sign = [torch.randint(0, 2, (1, h, N, 1), generator=g) * 2.0 - 1 for h in (KH, H)]
    tensors[2] = (sign[0] * size * (1 + 0.05 * torch.randn(1, KH, N, D, generator=g))).clamp(-65000, 65000).to(HALF)
    tensors[3] = (sign[1] * go * (1 + 0.05 * torch.randn(1, H, N, D, generator=g))).to(HALF)
    small = min(1.0, 300.0 / (size * go * math.sqrt(D)))
    tensors[0], tensors[1] = ((x.float() * small).to(HALF) for x in tensors[:2])
    check_against_64_bits(fa, tensors, {} if cap is None else dict(softcap=cap))


@pytest.mark.parametrize("D,H,KH", SHAPES)
def test_no_bit_goes_by_rows_that_start_again(fa, D, H, KH):
    """One document's dS overflows its first factor: the rows of the others beside it, which start again with it,
    keep every bit."""
    print("case again", D, H, flush=True)
    tensors = inputs(D, H, KH, 88)
    loud = [x.clone() for x in tensors]
    tensors[2][:, :, inside(1)] = 0
    loud[2][:, :, inside(1)] *= 6000.0
    loud[3][:, :, inside(1)] *= 16.0
    loud[1][:, :, inside(1)] *= 0.01
    tensors[3], tensors[1] = loud[3], loud[1]
    a, b = (call(fa, x, documents(fa), None, {}) for x in (tensors, loud))
    for n in ("gq", "gk", "gv"):
        for i in (0, 2):
            assert torch.equal(a[n][:, :, inside(i)], b[n][:, :, inside(i)]), (n, i)
    # (in 64 bits the loud document's dq is up to 2.2e3, its dk up to 3.7e5, past what fp16 holds)
    assert bool(torch.isfinite(b["gq"]).all()) and not bool(torch.isnan(b["gk"]).any())


@pytest.mark.parametrize("D,H,KH", [(64, 2, 1), (128, 4, 2)])
@pytest.mark.parametrize("dims", [[0], [1], [2], [3], [5], [6, 15], [60], [63]])
def test_values_and_gradients_in_a_few_dims(fa, D, H, KH, dims):
    """One or two dims of v and go hold nearly all of their norms, as outlier channels do; rows see two keys of
    about the same weight and of opposite v there, so that go.o cancels and dS is half of |go| |v|."""
    print("case dims", D, H, dims, flush=True)
    tensors = inputs(D, H, KH, 89)
    sign = 1.0 - 2.0 * (torch.arange(N) % 2)
    tensors[2][..., dims] = (20000.0 * sign[:, None]).to(HALF)
    tensors[3][..., dims] = 4.0
    tensors[0], tensors[1] = ((x.float() * 0.01).to(HALF) for x in tensors[:2])
    check_against_64_bits(fa, tensors, dict(window=2))
