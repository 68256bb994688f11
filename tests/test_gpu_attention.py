"""Attention with gradients and with capped, biased and masked scores: against the 64-bit forms, through
autograd, in graphs and on other streams, and what masked rows and keys may hold."""
from __future__ import annotations

import math

import pytest
import torch

import attention_reference as A
import cache_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def rows(B, H, N, D, dt, g, layout="bhnd", scale=1.0):
    x = (scale * torch.randn(B, H, N, D, generator=g)).to(dt)
    if layout == "bnhd":
        x = x.transpose(1, 2).contiguous().transpose(1, 2)
    elif layout == "wide":  # rows inside larger ones
        x = torch.cat([torch.zeros_like(x), x], -1)[..., D:]
    return x


def dev(x):
    return torch.empty_strided(x.size(), x.stride(), dtype=x.dtype, device=DEV).copy_(x)


def documents(fa, ends, n, prefix=None, causal=True):
    cu = torch.tensor([0, *ends], dtype=torch.int32)
    return fa.document_ranges(cu, n, causal=causal, prefix_lens=None if prefix is None else torch.tensor(prefix))


def random_ranges(B, n, m, seed):
    """Any pairs: empty, reversed, negative and past the end among them."""
    g = torch.Generator().manual_seed(seed)
    r = torch.randint(-20, m + 20, (B, n, 2), generator=g, dtype=torch.int32)
    return torch.where(torch.rand(B, n, 1, generator=g) < 0.5, r.sort(-1).values, r)


# B, H, KH, N, M, D, type, layout, scale of q, options
CASES = {
    "one": (1, 1, 1, 1, 1, 64, "fp16", "bhnd", 1, {}),
    "one-of-many": (2, 4, 2, 1, 333, 128, "bf16", "bhnd", 1, dict(causal=True)),
    "many-of-one": (1, 2, 1, 70, 1, 64, "bf16", "bhnd", 1, {}),
    "full-odd": (2, 3, 3, 77, 130, 64, "fp16", "bnhd", 1, {}),
    "causal": (1, 4, 2, 300, 300, 128, "bf16", "bhnd", 1, dict(causal=True)),
    "causal-later-part": (1, 2, 1, 100, 420, 64, "fp16", "bhnd", 1, dict(causal=True)),
    "causal-more-rows-than-keys": (1, 2, 2, 200, 90, 128, "fp16", "bhnd", 1, dict(causal=True)),
    "group-5": (1, 5, 1, 150, 150, 128, "fp16", "wide", 1, dict(causal=True)),
    "window": (2, 2, 2, 400, 400, 64, "bf16", "bhnd", 1, dict(causal=True, window=50)),
    "window-one": (1, 2, 1, 130, 130, 128, "bf16", "bhnd", 1, dict(causal=True, window=1)),
    "window-both-ways": (1, 2, 1, 260, 300, 64, "fp16", "bhnd", 1, dict(window=33)),
    "window-larger-than-all": (1, 2, 1, 100, 100, 64, "fp16", "bhnd", 1, dict(causal=True, window=2 ** 40)),
    "cap": (1, 4, 2, 290, 290, 128, "bf16", "bhnd", 6, dict(causal=True, softcap=15.0)),
    "cap-fp16": (2, 2, 2, 129, 200, 64, "fp16", "bnhd", 6, dict(softcap=20.0)),
    "cap-largest": (1, 2, 2, 100, 100, 64, "fp16", "bhnd", 1, dict(softcap=1000.0)),
    "cap-all-at-it": (1, 2, 1, 90, 90, 64, "bf16", "bhnd", 400, dict(causal=True, softcap=5.0)),
    "slopes": (1, 8, 2, 257, 257, 64, "bf16", "bhnd", 1, dict(causal=True, slopes=0.3)),
    "slopes-both-ways": (1, 3, 1, 140, 200, 128, "fp16", "bhnd", 1, dict(slopes=0.1)),
    "all-options": (2, 6, 2, 350, 350, 128, "bf16", "bnhd", 4,
                    dict(causal=True, softcap=10.0, slopes=0.05, window=111, docs=[100, 101, 230, 350])),
    "docs": (2, 4, 4, 500, 500, 64, "bf16", "bhnd", 1, dict(docs=[3, 64, 200, 201, 470])),
    "docs-prefix": (1, 4, 1, 400, 400, 128, "fp16", "bhnd", 1, dict(docs=[150, 400], prefix=[90, 0])),
    "docs-whole": (1, 2, 2, 333, 333, 128, "bf16", "bhnd", 1, dict(docs=[20, 300, 333], whole=True)),
    "any-ranges": (2, 2, 1, 333, 200, 64, "bf16", "bhnd", 1, dict(random=5)),
    "any-ranges-128": (1, 4, 2, 200, 300, 128, "fp16", "bhnd", 1, dict(random=6, softcap=30.0, slopes=0.01)),
    "nothing-seen": (1, 2, 1, 100, 100, 64, "fp16", "bhnd", 1, dict(nothing=True)),
    "long": (1, 2, 1, 1500, 1500, 64, "fp16", "bhnd", 1, dict(causal=True)),
    "long-128": (1, 2, 2, 1100, 1100, 128, "bf16", "bhnd", 1, dict(docs=[700, 1100])),
    # more workgroups than compute units, so without teams (with ranges: ranked by their work)
    "many-full": (3, 100, 100, 90, 130, 64, "fp16", "bhnd", 1, {}),
    "many-causal": (3, 180, 180, 140, 140, 128, "bf16", "bnhd", 1, dict(causal=True)),
    "many-window": (2, 150, 150, 260, 260, 64, "bf16", "bhnd", 1, dict(window=50)),
    "many-docs": (2, 150, 150, 300, 300, 128, "fp16", "bhnd", 1, dict(docs=[20, 200, 290])),
    "many-ranges": (2, 320, 160, 300, 200, 64, "bf16", "bhnd", 1, dict(random=7)),
    "many-cap": (2, 150, 150, 200, 330, 64, "bf16", "bhnd", 4, dict(softcap=12.0, slopes=0.001)),
    "many-all-options": (2, 150, 150, 280, 280, 128, "fp16", "bhnd", 4,
                         dict(causal=True, softcap=20.0, slopes=0.002, window=100)),
}


def setup(fa, name):
    B, H, KH, N, M, D, dtype, layout, scale, opt = CASES[name]
    g = torch.Generator().manual_seed(50 + list(CASES).index(name))
    dt = DT[dtype]
    q, go = rows(B, H, N, D, dt, g, layout, scale), rows(B, H, N, D, dt, g, layout)
    k, v = rows(B, KH, M, D, dt, g, layout), rows(B, KH, M, D, dt, g, layout)
    opt, ranges = dict(opt), None
    if "docs" in opt:
        ranges = documents(fa, opt.pop("docs"), N, opt.pop("prefix", None), not opt.pop("whole", False))
    elif "random" in opt:
        ranges = random_ranges(B, N, M, opt.pop("random"))
    elif opt.pop("nothing", False):
        ranges = torch.zeros(N, 2, dtype=torch.int32)
    slopes = None
    if "slopes" in opt:
        slopes = opt.pop("slopes") * torch.arange(1, H + 1).float()
    return (q, k, v, go), ranges, slopes, opt


def reference(tensors, ranges, slopes, opt, glse=None, scale=None):
    q, k, v, go = tensors
    see = A.visible(q.shape[2], k.shape[2], ranges, opt.get("causal", False), opt.get("window"))
    return A.attend(q, k, v, see, scale=scale or 1 / math.sqrt(q.shape[3]), cap=opt.get("softcap"), slopes=slopes,
                    go=go, glse=glse)


def call(fa, tensors, ranges, slopes, opt, glse=None, scale=None):
    """Values on the GPU, through autograd."""
    q, k, v, go = (dev(x) for x in tensors)
    for x in (q, k, v):
        x.requires_grad_()
    o, lse = fa.attention(q, k, v, None if ranges is None else ranges.to(DEV),
                          slopes=None if slopes is None else slopes.to(DEV), softmax_scale=scale, return_lse=True, **opt)
    outs, grads = (o, go) if glse is None else ((o, lse), (go, glse.to(DEV)))
    gq, gk, gv = torch.autograd.grad(outs, (q, k, v), grads)
    return {"o": o.detach(), "lse": lse.detach(), "gq": gq, "gk": gk, "gv": gv}


def compare(got, val, tol):
    for n in val:
        R.check(n, got[n].cpu(), val[n], tol[n])


@pytest.mark.parametrize("name", list(CASES))
def test_against_64_bits(fa, name):
    print("case", name, flush=True)
    tensors, ranges, slopes, opt = setup(fa, name)
    got = call(fa, tensors, ranges, slopes, opt)
    for x, y in zip(tensors, (got["gq"], got["gk"], got["gv"])):
        assert x.shape == y.shape and (CASES[name][7] != "bnhd" or x.stride() == y.stride())
    compare(got, *reference(tensors, ranges, slopes, opt))
    plain = fa.attention(*(dev(x) for x in tensors[:3]), None if ranges is None else ranges.to(DEV),
                         slopes=None if slopes is None else slopes.to(DEV), **opt)
    assert torch.equal(plain, got["o"])


@pytest.mark.parametrize("D", [64, 128])
def test_gradient_of_the_logsumexp_and_a_scale(fa, D):
    print("case lse", D, flush=True)
    g = torch.Generator().manual_seed(3)
    tensors = [rows(1, h, 150, D, torch.bfloat16, g) for h in (4, 2, 2, 4)]
    glse = torch.randn(1, 4, 150, generator=g)
    opt = dict(causal=True)
    compare(call(fa, tensors, None, None, opt, glse, 0.05), *reference(tensors, None, None, opt, glse, 0.05))


@pytest.mark.parametrize("D,cap", [(64, None), (128, 4.0)])
def test_gradients_against_differences(fa, D, cap):
    """The kernel's gradients along random directions against differences of the 64-bit loss."""
    print("case differences", D, cap, flush=True)
    g = torch.Generator().manual_seed(9)
    q, k, v, go = (rows(1, h, 60, D, torch.float16, g) for h in (2, 1, 1, 2))
    got = call(fa, (q, k, v, go), None, None, dict(causal=True, softcap=cap))
    _, tol = reference((q, k, v, go), None, None, dict(causal=True, softcap=cap))
    see = A.visible(60, 60, None, True)[0]

    def loss(q, k, v):
        return sum((A.head(q[0, h], k[0, 0], v[0, 0], see, scale=1 / math.sqrt(D), cap=cap)[0] * go[0, h].double()).sum()
                   for h in range(2))

    args = {"gq": q.double(), "gk": k.double(), "gv": v.double()}
    for n, x in args.items():
        d = torch.randn(x.shape, generator=g, dtype=torch.float64)
        up, down = {**args, n: x + 1e-5 * d}, {**args, n: x - 1e-5 * d}
        diff = (loss(*up.values()) - loss(*down.values())) / 2e-5
        assert abs(diff - (got[n].cpu().double() * d).sum()) <= (tol[n] * d.abs()).sum() + 1e-6 * (1 + abs(diff)), n


@pytest.mark.parametrize("factor", [2.0 ** -14, 2.0 ** 9])
@pytest.mark.parametrize("D", [64, 128])
def test_small_and_large_incoming_gradients_in_fp16(fa, D, factor):
    """Gradients scale with the incoming one over fp16's range: dS itself would underflow or overflow."""
    print("case factor", D, factor, flush=True)
    g = torch.Generator().manual_seed(4)
    q, k, v, go = (rows(1, h, 260, D, torch.float16, g) for h in (2, 1, 1, 2))
    go = (go * factor).half()
    compare(call(fa, (q, k, v, go), None, None, dict(causal=True)),
            *reference((q, k, v, go), None, None, dict(causal=True)))


@pytest.mark.parametrize("D,dtype,heads", [(64, "fp16", 4), (128, "bf16", 4), (64, "bf16", 90), (128, "bf16", 180)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_masked_rows_and_keys_may_hold_anything(fa, D, dtype, heads, bad):
    """A document of infinities or NaN in the middle, and garbage rows that see and are seen by nothing:
    the other documents' results keep every bit that they have with zeros in its place."""
    print("case masked", D, dtype, heads, bad, flush=True)
    g = torch.Generator().manual_seed(8)
    N, dt = 300, DT[dtype]
    kv_heads = 2 if heads == 4 else heads
    good = [rows(1, h, N, D, dt, g) for h in (heads, kv_heads, kv_heads, heads)]
    cu = torch.tensor([0, 70, 150, 280], dtype=torch.int32)  # rows 280 .. 299 belong to none
    ranges = fa.document_ranges(cu, N)
    mine = torch.zeros(N, dtype=torch.bool)
    mine[:70] = mine[150:280] = True
    zero, dirty = [], []
    for x in good:
        z, w = x.clone(), x.clone()
        z[:, :, ~mine] = 0
        w[:, :, ~mine] = bad
        w[:, :, 75] = -bad
        zero.append(z)
        dirty.append(w)
    a, b = call(fa, zero, ranges, None, {}), call(fa, dirty, ranges, None, {})
    for n in a:
        if dt == torch.float16 and n in ("gk", "gv"):
            # (the factor of dS goes by the largest |go| of all documents)
            assert bool(torch.isfinite(b[n][:, :, mine]).all()), n
            continue
        assert torch.equal(a[n][:, :, mine], b[n][:, :, mine]), n
    for n in ("o", "gq", "gk", "gv"):
        assert bool((a[n][:, :, 280:] == 0).all()) and bool((b[n][:, :, 280:] == 0).all()), n
        assert not bool(torch.isfinite(b[n][:, :, 76:150]).any()), n


@pytest.mark.parametrize("D,H", [(64, 2), (128, 2), (64, 300), (128, 300)])
def test_one_bad_key_reaches_the_rows_that_see_it(fa, D, H):
    print("case bad key", D, H, flush=True)
    g = torch.Generator().manual_seed(18)
    q, k, v, go = (rows(1, H, 200, D, torch.bfloat16, g) for _ in range(4))
    for x in (k, v):
        y = [t.clone() for t in (q, k, v, go)]
        y[1 if x is k else 2][0, 0, 120, 3] = math.nan
        got = call(fa, y, None, None, dict(causal=True))
        want = call(fa, (q, k, v, go), None, None, dict(causal=True))
        assert torch.equal(got["o"][:, 1], want["o"][:, 1]) and torch.equal(got["gq"][:, 1], want["gq"][:, 1])
        assert torch.equal(got["o"][0, 0, :120], want["o"][0, 0, :120])
        assert torch.equal(got["gq"][0, 0, :120], want["gq"][0, 0, :120])
        assert bool(torch.isnan(got["gq"][0, 0, 120:]).any(-1).all())
        assert bool(torch.isnan(got["o"][0, 0, 120:]).any(-1).all())


@pytest.mark.parametrize("name", ["causal", "any-ranges-128", "all-options", "many-window"])
def test_attention_backward(fa, name):
    """By itself, from the o that attention returned."""
    print("case backward", name, flush=True)
    tensors, ranges, slopes, opt = setup(fa, name)
    q, k, v, go = (dev(x) for x in tensors)
    rest = dict(key_ranges=None if ranges is None else ranges.to(DEV), slopes=None if slopes is None else slopes.to(DEV), **opt)
    o, lse = fa.attention(q, k, v, return_lse=True, **rest)
    got = dict(zip(("gq", "gk", "gv"), fa.attention_backward(go, q, k, v, o, lse, **rest)), o=o, lse=lse)
    compare(got, *reference(tensors, ranges, slopes, opt))


def test_gradients_of_sharp_rows_take_what_rounding_left_of_o(fa):
    """Where few keys have most of the weight, go.v - delta cancels, and the rounding of o that
    attention_backward is given weighs as much as all others: without it the root mean square error is smaller."""
    print("case sharp", flush=True)
    g = torch.Generator().manual_seed(44)
    q, go = (rows(1, 2, 500, 128, torch.bfloat16, g, scale=s) for s in (4.0, 1.0))
    k, v = (rows(1, 2, 500, 128, torch.bfloat16, g) for _ in range(2))
    opt = dict(causal=True, softcap=50.0)
    got = call(fa, (q, k, v, go), None, None, opt)
    val, _ = reference((q, k, v, go), None, None, opt)
    x = [dev(t) for t in (q, k, v)]
    o, lse = fa.attention(*x, return_lse=True, **opt)
    plain = dict(zip(("gq", "gk"), fa.attention_backward(dev(go), *x, o, lse, **opt)))
    for n in plain:
        off = [float((y[n].cpu().double() - val[n]).norm()) for y in (got, plain)]
        assert off[0] < off[1], (n, off)


def test_gradients_with_expanded_and_odd_strides(fa):
    """sum().backward() hands in an expanded gradient; k and v of one head may be broadcast."""
    g = torch.Generator(device=DEV).manual_seed(2)
    q = torch.randn(2, 4, 90, 64, generator=g, device=DEV).half().requires_grad_()
    kv = torch.randn(1, 2, 90, 64, generator=g, device=DEV).half().requires_grad_()
    k = kv.expand(2, 2, 90, 64)
    fa.attention(q, k, k, causal=True).sum().backward()
    a, b = q.grad.clone(), kv.grad.clone()
    ones = torch.ones(2, 4, 90, 64, device=DEV).half()
    kc, vc = (k.detach().clone().requires_grad_() for _ in range(2))
    dq, dk, dv = torch.autograd.grad(fa.attention(q, kc, vc, causal=True), (q, kc, vc), ones)
    assert torch.equal(a, dq)
    want = (dk.float() + dv.float()).sum(0, keepdim=True)
    assert float((b.float() - want).abs().max()) <= 4 * 2.0 ** -11 * float(want.abs().max())


def test_same_bits_in_a_graph_and_on_another_stream(fa):
    g = torch.Generator(device=DEV).manual_seed(5)
    q, go = (torch.randn(1, 4, 500, 128, generator=g, device=DEV).bfloat16() for _ in range(2))
    k, v = (torch.randn(1, 2, 500, 128, generator=g, device=DEV).bfloat16() for _ in range(2))
    ranges = fa.document_ranges(torch.tensor([0, 200, 500], device=DEV), 500)
    slopes = torch.rand(4, device=DEV)
    opt = dict(softcap=20.0, slopes=slopes)

    def both():
        o, lse = fa.attention(q, k, v, ranges, return_lse=True, **opt)
        return (o, lse, *fa.attention_backward(go, q, k, v, o, lse, ranges, **opt))

    first = both()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = both()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(x, y) for x, y in zip(first, second))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = both()
    for step in range(3):
        cpu = torch.Generator().manual_seed(step)
        for t in (q, k, v, go):
            t.copy_(torch.randn(t.shape, generator=cpu))
        ranges.copy_(fa.document_ranges(torch.tensor([0, 50 + 100 * step, 500]), 500))
        graph.replay()
        eager = both()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(res, eager)), step


def test_autograd_in_a_graph(fa):
    """As qk_norm_rope: with an older eager graph of the same leaves alive a captured call is refused
    before it can end the capture."""
    g = torch.Generator(device=DEV).manual_seed(6)
    q, k, v = (torch.randn(1, 2, 100, 64, generator=g, device=DEV).half().requires_grad_() for _ in range(3))
    go = torch.randn(1, 2, 100, 64, generator=g, device=DEV).half()

    def step():
        return torch.autograd.grad(fa.attention(q, k, v, causal=True), (q, k, v), go)

    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    x = [t.detach() for t in (q, k, v)]
    o, lse = fa.attention(*x, causal=True, return_lse=True)
    want = fa.attention_backward(go, *x, o, lse, causal=True)
    alive = fa.attention(q, k, v, causal=True)  # holds the leaves' accumulators
    other = torch.cuda.CUDAGraph()
    with torch.cuda.graph(other):
        keep = q.detach() + 1
        with pytest.raises(RuntimeError, match="attention_backward"):
            fa.attention(q, k, v, causal=True)
        o, lse = fa.attention(q.detach(), k.detach(), v.detach(), causal=True, return_lse=True)
        grads = fa.attention_backward(go, q, k, v, o, lse, causal=True)
    for _ in range(2):
        other.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(grads, want))
    del alive, keep


def test_what_autograd_is_owed(fa):
    g = torch.Generator(device=DEV).manual_seed(7)
    q, k, v = (torch.randn(1, 2, 40, 64, generator=g, device=DEV).half() for _ in range(3))
    go = torch.randn(1, 2, 40, 64, generator=g, device=DEV).half()
    # one input alone; o alone and lse alone
    ref = call(fa, [x.cpu() for x in (q, k, v, go)], None, None, {})
    for i, n in enumerate(("gq", "gk", "gv")):
        x = [t.detach().clone() for t in (q, k, v)]
        x[i].requires_grad_()
        assert torch.equal(torch.autograd.grad(fa.attention(*x), x[i], go)[0], ref[n])
    x = q.clone().requires_grad_()
    o, lse = fa.attention(x, k, v, return_lse=True)
    (gl,) = torch.autograd.grad(lse.sum(), x)
    assert bool(torch.isfinite(gl).all()) and bool(gl.any())
    # a second derivative, tangents, gradients of slopes: refused
    o = fa.attention(x, k, v)
    (d,) = torch.autograd.grad(o, x, go.clone().requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        d.float().sum().backward()
    with pytest.raises(RuntimeError, match="slopes get no gradient"):
        fa.attention(x, k, v, slopes=torch.ones(2, device=DEV, requires_grad=True))
    import torch.autograd.forward_ad as fwad
    with fwad.dual_level():
        with pytest.raises(RuntimeError, match="tangent"):
            fa.attention(fwad.make_dual(q, q), k, v)
    # an input that is overwritten after the forward pass is noticed
    y = q.clone().requires_grad_()
    z = y * 1
    o = fa.attention(z, k, v)
    z.data.zero_()
    z.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()


@pytest.mark.parametrize("D,dt", [(64, torch.float16), (128, torch.bfloat16)])
def test_offsets_past_32_bits(fa, D, dt):
    """Rows 8 MiB apart: the last ones of each tensor are 5 GiB behind the first."""
    print("case far", D, flush=True)
    g = torch.Generator(device=DEV).manual_seed(33)
    N, apart = 700, 1 << 22

    def far():
        x = torch.empty(N * apart, dtype=dt, device=DEV).as_strided((1, 1, N, D), (N * apart, N * apart, apart, 1))
        return x.copy_(torch.randn(1, 1, N, D, generator=g, device=DEV).to(dt))

    q, k, v, go = (far() for _ in range(4))
    near = [x.contiguous() for x in (q, k, v, go)]
    assert q.stride(2) == apart and near[0].stride(2) == D
    got = []
    for a, b, c, d in ((q, k, v, go), near):
        o, lse = fa.attention(a, b, c, causal=True, return_lse=True)
        got.append((o, lse, *fa.attention_backward(d, a, b, c, o, lse, causal=True)))
    for x, y in zip(*got):
        assert torch.equal(x, y)


def test_other_documents_in_a_replayed_graph(fa):
    """Enough tiles that they are ranked by their work, whose order then changes between replays."""
    print("case documents in a graph", flush=True)
    g = torch.Generator(device=DEV).manual_seed(34)
    B, H, N, D = 2, 40, 1000, 64
    q, k, v, go = (torch.randn(B, H, N, D, generator=g, device=DEV).half() for _ in range(4))
    ends = [[0, 100, 1000], [0, 900, 950, 1000], [0, 333, 700, 990]]
    ranges = [fa.document_ranges(torch.tensor(e, device=DEV), N) for e in ends]

    def step(r):
        o, lse = fa.attention(q, k, v, r, return_lse=True)
        return (o, lse, *fa.attention_backward(go, q, k, v, o, lse, r))

    want = [step(r) for r in ranges]
    r = ranges[0].clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(r)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(r)
    for i in (1, 2, 0, 1):
        r.copy_(ranges[i])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want[i])), i
        step(ranges[i])


@pytest.mark.parametrize("H", [2, 150])
@pytest.mark.parametrize("D,opt", [(64, {}), (128, dict(softcap=30.0)), (64, dict(window=150)), (128, dict(biased=True))])
def test_no_bit_of_a_row_goes_by_other_rows(fa, H, D, opt):
    """The rows beside it have scores that raise their offsets again and again."""
    print("case alone", H, D, opt, flush=True)
    g = torch.Generator(device=DEV).manual_seed(31)
    q, k, v = (torch.randn(1, H, 300, D, generator=g, device=DEV).half() for _ in range(3))
    opt = dict(opt)
    if opt.pop("biased", False):
        opt["slopes"] = torch.rand(H, generator=g, device=DEV) * 0.2
    loud = q * torch.where(torch.arange(300, device=DEV) % 3 == 0, 1.0, 40.0).half()[:, None]
    a, b = (fa.attention(x, k, v, return_lse=True, **opt) for x in (q, loud))
    assert torch.equal(a[0][:, :, ::3], b[0][:, :, ::3]) and torch.equal(a[1][:, :, ::3], b[1][:, :, ::3])


def test_splits_of_the_rows_and_long_keys(fa):
    """Few keys and many rows are split over workgroups whose parts are joined in order."""
    print("case splits", flush=True)
    g = torch.Generator().manual_seed(12)
    q, go = (rows(1, 2, 2000, 64, torch.bfloat16, g) for _ in range(2))
    k, v = (rows(1, 1, 90, 64, torch.bfloat16, g) for _ in range(2))
    got = call(fa, (q, k, v, go), None, None, {})
    compare(got, *reference((q, k, v, go), None, None, {}))
    again = call(fa, (q, k, v, go), None, None, {})
    assert all(torch.equal(got[n], again[n]) for n in got)


def test_training_step_of_norm_and_attention(fa):
    """qk_norm_rope with axes in front of attention, gradients to the projections and weights, against the
    same chain in 64 bits.  Bound: the attention's own on its rounded inputs, carried through the norm's
    formula, which is linear in them, by its largest factor."""
    print("case step", flush=True)
    g = torch.Generator().manual_seed(30)
    N, D = 180, 64
    x = [rows(1, h, N, D, torch.float16, g) for h in (4, 2)]
    v, go = rows(1, 2, N, D, torch.float16, g), rows(1, 4, N, D, torch.float16, g)
    w = [1 + 0.1 * torch.randn(D, generator=g) for _ in range(2)]
    pos = torch.stack([torch.arange(N) // 60, torch.arange(N) % 60 // 8, torch.arange(N) % 8]).int()
    axes = [0] * 10 + [1] * 11 + [2] * 11
    freq = 100.0 ** (-torch.arange(32, dtype=torch.float64) / 32)
    angle = torch.arange(64, dtype=torch.float64)[:, None] * freq
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    ranges = fa.document_ranges(torch.tensor([0, 60, 180]), N, prefix_lens=torch.tensor([20, 50]))
    leaves = [t.to(DEV).requires_grad_() for t in (*x, *w, v)]
    qn, kn = fa.qk_norm_rope(leaves[0], leaves[1], leaves[2], leaves[3], cos.to(DEV), sin.to(DEV), pos.to(DEV), axes=axes)
    o = fa.attention(qn, kn, leaves[4], ranges.to(DEV), softcap=30.0)
    got = torch.autograd.grad(o, leaves, go.to(DEV))

    ref = [t.double().requires_grad_() for t in (*x, *w, v)]
    c, s = (torch.stack([t[pos[axes[i]].long(), i] for i in range(32)], 1).double() for t in (cos, sin))

    def norm(t, weight):
        y = t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * weight
        a, b = y[..., :32], y[..., 32:]
        return torch.cat((a * c - b * s, b * c + a * s), -1)

    q64, k64 = norm(ref[0], ref[2]), norm(ref[1], ref[3])
    see = A.visible(N, N, ranges)[0]
    o64 = torch.stack([A.head(q64[0, h], k64[0, h // 2], ref[4][0, h // 2], see, scale=0.125, cap=30.0)[0]
                       for h in range(4)])[None]
    want = torch.autograd.grad(o64, ref, go.double())
    # relative to a tensor's norm: roundings of q, k, P, dS, o and the results, each at most 2^-11 of
    # what it rounds, some 8 in a row, and sums of them by Cauchy-Schwarz
    for name, a, b in zip(("q", "k", "q_weight", "k_weight", "v"), got, want):
        assert (a.cpu().double() - b).norm() <= 16 * 2.0 ** -11 * b.norm(), name


def test_document_ranges(fa):
    r = fa.document_ranges(torch.tensor([1, 4, 4, 7]), 9, prefix_lens=torch.tensor([2, 5, 100]))
    assert r.dtype == torch.int32
    assert r.tolist() == [[0, 0], [1, 3], [1, 3], [1, 4], [4, 7], [4, 7], [4, 7], [0, 0], [0, 0]]
    assert fa.document_ranges(torch.tensor([0, 2, 3]), 3, causal=False).tolist() == [[0, 2], [0, 2], [2, 3]]
    assert fa.document_ranges(torch.tensor([0]), 2).tolist() == [[0, 0], [0, 0]]


def test_refusals(fa):
    g = torch.Generator(device=DEV).manual_seed(1)
    q, k, v = (torch.randn(2, h, 8, 64, generator=g, device=DEV).half() for h in (4, 2, 2))
    ok = dict(q=q, k=k, v=v)
    fa.attention(**ok)
    r = torch.zeros(2, 8, 2, dtype=torch.int32, device=DEV)
    bad = [
        (dict(q=q.float()), "float16 or bfloat16"), (dict(k=k.bfloat16()), "same dtype"),
        (dict(v=v[:, :, :4]), "same shape"), (dict(q=q[:1]), "same batch"), (dict(q=q[:, :3]), "multiple of kv_heads"),
        (dict(q=q.cpu()), "CUDA tensor"), (dict(q=q[0]), "4D"), (dict(q=q.transpose(2, 3)), "unit stride"),
        (dict(q=q[..., :32], k=k[..., :32], v=v[..., :32]), "head_dim 64 and 128"),
        (dict(k=k[:, :, :0], v=v[:, :, :0]), "must all be >= 1"),
        (dict(q=torch.zeros(2, 4, 8, 65, device=DEV).half()[..., 1:]), "multiple of 8"),
        (dict(key_ranges=r.long()), "int32"), (dict(key_ranges=r[:, :4]), r"\[N, 2\]"),
        (dict(key_ranges=r[:1]), r"\[N, 2\]"), (dict(key_ranges=r[..., :1]), r"\[N, 2\]"),
        (dict(key_ranges=torch.zeros(2, 8, 4, dtype=torch.int32, device=DEV)[..., :2]), "contiguous rows"),
        (dict(key_ranges=torch.zeros(17, dtype=torch.int32, device=DEV)[1:].view(8, 2)), "8-byte aligned"),
        (dict(window=0), "window"), (dict(window=-3), "window"), (dict(softcap=0.0), "softcap"),
        (dict(softcap=-1.0), "softcap"), (dict(softcap=2000.0), "softcap"), (dict(softcap=math.nan), "softcap"),
        (dict(softcap=math.inf), "softcap"), (dict(softmax_scale=0.0), "softmax_scale"),
        (dict(softmax_scale=1e38, softcap=0.01), "softmax_scale / softcap"),
        (dict(slopes=torch.ones(2, device=DEV)), "slopes"), (dict(slopes=torch.ones(4, device=DEV).half()), "slopes"),
        (dict(slopes=torch.ones(4)), "slopes"), (dict(slopes=torch.ones(8, device=DEV)[::2]), "slopes"),
    ]
    for change, text in bad:
        with pytest.raises(RuntimeError, match=text):
            fa.attention(**{**ok, **change})
    o, lse = fa.attention(**ok, return_lse=True)
    for change, text in [(dict(do=o[:, :2]), "shape"), (dict(do=o.float()), "dtype"), (dict(o=o[:, :2]), "shape"),
                         (dict(lse=lse[:, :2]), r"\[B, H, N\]"), (dict(lse=lse.double()), "float32"),
                         (dict(dlse=lse.cpu()), "same device")]:
        with pytest.raises(RuntimeError, match=text):
            fa.attention_backward(**{**dict(do=o, o=o, lse=lse), **ok, **change})
