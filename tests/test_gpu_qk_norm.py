"""The q/k norm with rotation and its gradients against the 64-bit formulas,
finite differences, and through autograd and graphs."""
from __future__ import annotations

import math

import pytest
import torch

import cache_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def tables(rows, r, seed=3):
    freq = 10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)
    a = torch.arange(rows, dtype=torch.float64)[:, None] * freq
    return torch.cos(a).float(), torch.sin(a).float()


def inputs(B, H, KH, N, D, dt, seed, layout="bhnd"):
    g = torch.Generator().manual_seed(seed)
    out = []
    for heads in (H, KH, H, KH):
        x = (1.5 * torch.randn(B, heads, N, D, generator=g)).to(dt)
        if layout == "bnhd":
            x = x.transpose(1, 2).contiguous().transpose(1, 2)
        elif layout == "wide":  # rows inside larger ones
            x = torch.cat([torch.zeros_like(x), x], -1)[..., D:]
        out.append(x)
    return out


def weights(D, dt, seed):
    g = torch.Generator().manual_seed(seed)
    return [(1 + 0.3 * torch.randn(D, generator=g)).to(dt) for _ in range(2)]


def to_dev(x):
    """x on the GPU with its strides."""
    y = torch.empty_strided(x.size(), x.stride(), dtype=x.dtype, device=DEV)
    return y.copy_(x)


CASES = [
    # B, H, KH, N, D, dtype, layout, rotated, interleaved, weights, positions
    (1, 1, 1, 1, 64, "fp16", "bhnd", 64, False, "fp32", None),
    (1, 1, 1, 1, 128, "bf16", "bhnd", 128, True, "same", None),
    (2, 5, 1, 33, 64, "bf16", "bnhd", 64, True, "fp32", "n"),
    (3, 4, 2, 17, 128, "fp16", "wide", 128, False, "same", "bn"),
    (2, 3, 3, 100, 128, "bf16", "bhnd", 32, False, "fp32", "n"),
    (2, 7, 2, 65, 64, "fp16", "bnhd", 16, True, "fp32", "bn"),
    (1, 32, 8, 500, 128, "bf16", "bnhd", 112, False, "same", None),
    (4, 8, 8, 301, 64, "fp16", "bhnd", 48, False, "fp32", "bn"),
    (1, 2, 1, 3001, 128, "fp16", "bhnd", 128, True, "fp32", "n"),
]


def setup(case):
    B, H, KH, N, D, dtype, layout, r, inter, wdt, posk = case
    dt = DT[dtype]
    q, k, dq, dk = inputs(B, H, KH, N, D, dt, 7 + N, layout)
    qw, kw = weights(D, torch.float32 if wdt == "fp32" else dt, 11)
    cos, sin = tables(2 * N + 5, r)
    g = torch.Generator().manual_seed(N)
    pos = None
    if posk == "n":
        pos = torch.randint(0, 2 * N + 5, (N,), generator=g, dtype=torch.int32)
    elif posk == "bn":
        pos = torch.randint(0, 2 * N + 5, (B, N), generator=g, dtype=torch.int32)
    full = torch.arange(N) if pos is None else pos
    full = (full if full.dim() == 2 else full[None].expand(B, N))[:, None]  # [B, 1, N]
    return q, k, dq, dk, qw, kw, cos, sin, pos, full


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_forward(fa, case):
    print("case", case, flush=True)
    q, k, _, _, qw, kw, cos, sin, pos, full = setup(case)
    qo, ko = fa.qk_norm_rope(to_dev(q), to_dev(k), qw.to(DEV), kw.to(DEV), cos.to(DEV), sin.to(DEV),
                             None if pos is None else pos.to(DEV), eps=1e-5, interleaved=case[8])
    for name, x, w, y in (("q", q, qw, qo), ("k", k, kw, ko)):
        assert y.dtype == x.dtype
        want, tol = R.norm_rope(x, w, cos, sin, full.expand(x.shape[:-1]), eps=1e-5, interleaved=case[8])
        R.check(name, y, want, tol)


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_gradients(fa, case):
    print("case", case, flush=True)
    q, k, dq, dk, qw, kw, cos, sin, pos, full = setup(case)
    leaves = [to_dev(q), to_dev(k), qw.to(DEV), kw.to(DEV)]
    for t in leaves:
        t.requires_grad_()
    p = None if pos is None else pos.to(DEV)
    qo, ko = fa.qk_norm_rope(*leaves, cos.to(DEV), sin.to(DEV), p, eps=1e-5, interleaved=case[8])
    got = torch.autograd.grad((qo, ko), leaves, (to_dev(dq), to_dev(dk)))
    with torch.no_grad():
        plain = fa.qk_norm_rope_backward(to_dev(dq), to_dev(dk), *leaves, cos.to(DEV), sin.to(DEV), p,
                                         eps=1e-5, interleaved=case[8])
    for a, b in zip(got, plain):
        assert torch.equal(a, b)
    for name, x, w, dy, gx, gw in (("q", q, qw, dq, got[0], got[2]), ("k", k, kw, dk, got[1], got[3])):
        dx, tx, dw, tw = R.norm_rope_grad(x, w, cos, sin, full.expand(x.shape[:-1]), dy, eps=1e-5,
                                          interleaved=case[8])
        assert gx.dtype == x.dtype and gw.dtype == w.dtype
        R.check("d" + name, gx, dx, tx)
        R.check("d" + name + "_weight", gw, dw, tw)


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradients_against_differences(fa, interleaved):
    """The 64-bit formula that the kernel is held to, against central
    differences of the 64-bit forward, and the kernel's gradient of the same
    sum against both (bf16 gradients: 2^-8 of the largest)."""
    D, N, r = 64, 3, 48
    g = torch.Generator().manual_seed(1)
    x = torch.randn(1, 1, N, D, generator=g).bfloat16()
    w = (1 + 0.2 * torch.randn(D, generator=g))
    dy = torch.randn(1, 1, N, D, generator=g).bfloat16()
    cos, sin = tables(N, r)
    pos = torch.arange(N)[None, None]

    def loss(xd, wd):
        n = xd * torch.rsqrt(xd.square().mean(-1, keepdim=True) + 1e-5) * wd
        y = n.clone()
        a, b = (n[..., 0:r:2], n[..., 1:r:2]) if interleaved else (n[..., : r // 2], n[..., r // 2: r])
        c, s = cos.double(), sin.double()
        if interleaved:
            y[..., 0:r:2], y[..., 1:r:2] = a * c - b * s, b * c + a * s
        else:
            y[..., : r // 2], y[..., r // 2: r] = a * c - b * s, b * c + a * s
        return float((y * dy.double()).sum())

    dx, _, dw, _ = R.norm_rope_grad(x, w, cos, sin, pos, dy, eps=1e-5, interleaved=interleaved)
    h = 1e-5
    for e in range(0, D, 7):
        step = torch.zeros(1, 1, N, D, dtype=torch.float64)
        step[0, 0, 1, e] = h
        d = (loss(x.double() + step, w.double()) - loss(x.double() - step, w.double())) / (2 * h)
        assert abs(d - float(dx[0, 0, 1, e])) <= 1e-7, e
        sw = torch.zeros(D, dtype=torch.float64)
        sw[e] = h
        d = (loss(x.double(), w.double() + sw) - loss(x.double(), w.double() - sw)) / (2 * h)
        assert abs(d - float(dw[e])) <= 1e-7, e
    gx, _, gw, _ = fa.qk_norm_rope_backward(dy.to(DEV), dy.to(DEV), x.to(DEV), x.to(DEV), w.to(DEV),
                                            w.to(DEV), cos.to(DEV), sin.to(DEV), eps=1e-5,
                                            interleaved=interleaved)
    assert float((gx.cpu().double() - dx).abs().max()) <= 2.0 ** -8 * float(dx.abs().max()) * 1.01
    assert float((gw.cpu().double() - dw).abs().max()) <= 1e-5


def test_gradients_of_one_result_and_of_expanded_ones(fa):
    """Only q's result is used; its gradient is an expanded scalar."""
    q, k, _, _ = inputs(2, 3, 1, 9, 64, torch.bfloat16, 21)
    qw, kw = weights(64, torch.float32, 22)
    cos, sin = tables(9, 64)
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, qw, kw)]
    qo, _ = fa.qk_norm_rope(*leaves, cos.to(DEV), sin.to(DEV))
    qo.float().sum().backward()
    ones = torch.ones_like(q)
    pos = torch.arange(9)[None, None].expand(2, 3, 9)
    dx, tx, dw, tw = R.norm_rope_grad(q, qw, cos, sin, pos, ones, eps=1e-6, interleaved=False)
    R.check("dq", leaves[0].grad, dx, tx)
    R.check("dqw", leaves[2].grad, dw, tw)
    assert not leaves[1].grad.any() and not leaves[3].grad.any()
    qo, _ = fa.qk_norm_rope(*leaves, cos.to(DEV), sin.to(DEV))
    g = torch.autograd.grad(qo.sum(), leaves[0])[0]  # expanded: strides of 0
    R.check("dq", g, dx, tx)


def test_shared_heads_and_weights(fa):
    """The same tensor as q and k, and one weight for both: gradients add up."""
    x, _, d1, d2 = inputs(1, 2, 2, 40, 128, torch.float16, 23)
    w = weights(128, torch.float32, 24)[0]
    cos, sin = tables(40, 128)
    xl, wl = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    a, b = fa.qk_norm_rope(xl, xl, wl, wl, cos.to(DEV), sin.to(DEV))
    assert torch.equal(a, b)
    torch.autograd.backward((a, b), (d1.to(DEV), d2.to(DEV)))
    pos = torch.arange(40)[None, None].expand(1, 2, 40)
    parts = [R.norm_rope_grad(x, w, cos, sin, pos, d, eps=1e-6, interleaved=False) for d in (d1, d2)]
    R.check("dw", wl.grad, parts[0][2] + parts[1][2], parts[0][3] + parts[1][3] + 2.0 ** -23)
    total = parts[0][0] + parts[1][0]
    R.check("dx", xl.grad, total, parts[0][1] + parts[1][1] + 2.0 ** -11 * total.abs())


def test_expanded_inputs(fa):
    """q expanded over the batch (stride 0): read as it is, its gradient summed by autograd."""
    q, k, dq, dk = inputs(1, 2, 1, 12, 64, torch.bfloat16, 25)
    qw, kw = (w.to(DEV) for w in weights(64, torch.float32, 26))
    cos, sin = (t.to(DEV) for t in tables(12, 64))
    ql = q.to(DEV).requires_grad_()
    qo, _ = fa.qk_norm_rope(ql.expand(3, -1, -1, -1), k.to(DEV).expand(3, -1, -1, -1), qw, kw, cos, sin)
    one, _ = fa.qk_norm_rope(q.to(DEV), k.to(DEV), qw, kw, cos, sin)
    assert torch.equal(qo, one.expand(3, -1, -1, -1))
    g = torch.autograd.grad(qo, ql, dq.to(DEV).expand(3, -1, -1, -1))[0]
    single = fa.qk_norm_rope_backward(dq.to(DEV), dk.to(DEV), q.to(DEV), k.to(DEV), qw, kw, cos, sin)[0]
    assert float((g.float() - 3 * single.float()).abs().max()) <= 3 * 2.0 ** -8 * float(single.float().abs().max()) * 2


def test_zero_rows_extreme_rows_and_positions_outside_the_tables(fa):
    D, N = 64, 6
    for dt in DT.values():
        q = torch.zeros(1, 1, N, D, dtype=dt)
        q[0, 0, 1] = 60000.0 if dt == torch.float16 else 1e18
        q[0, 0, 2] = 2.0 ** -20
        q[0, 0, 3, 5] = math.nan
        w = torch.ones(D)
        cos, sin = tables(4, D)
        pos = torch.tensor([0, 1, 2, 3, 4, -1], dtype=torch.int32)
        y, _ = fa.qk_norm_rope(q.to(DEV), q.to(DEV), w.to(DEV), w.to(DEV), cos.to(DEV), sin.to(DEV),
                               pos.to(DEV), eps=1e-12)
        want, tol = R.norm_rope(q, w, cos, sin, pos[None, None], eps=1e-12, interleaved=False)
        R.check("y", y[:, :, :3], want[:, :, :3], tol[:, :, :3])
        assert not y[0, 0, 0].any()
        assert bool(torch.isnan(y[0, 0, 3:]).all())


def test_second_derivatives_and_table_gradients_are_refused(fa):
    q, k, dq, _ = inputs(1, 1, 1, 4, 64, torch.bfloat16, 27)
    qw, kw = (w.to(DEV) for w in weights(64, torch.float32, 28))
    cos, sin = (t.to(DEV) for t in tables(4, 64))
    ql = q.to(DEV).requires_grad_()
    qo, _ = fa.qk_norm_rope(ql, k.to(DEV), qw, kw, cos, sin)
    (g,) = torch.autograd.grad(qo, ql, dq.to(DEV).requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.float().sum().backward()
    with pytest.raises(RuntimeError, match="cos and sin"):
        fa.qk_norm_rope(ql, k.to(DEV), qw, kw, cos.requires_grad_(), sin)


def test_same_bits_in_a_graph_and_on_another_stream(fa):
    case = CASES[6]
    q, k, dq, dk, qw, kw, cos, sin, pos, _ = setup(case)
    a = [to_dev(t) for t in (q, k, dq, dk)]
    c = [t.to(DEV) for t in (qw, kw, cos, sin)]

    def both():
        return (*fa.qk_norm_rope(a[0], a[1], *c), *fa.qk_norm_rope_backward(a[2], a[3], a[0], a[1], *c))

    first = both()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = both()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(x, y) for x, y in zip(first, second))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        res = both()
    for step in range(3):
        for t in a:
            t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(step)))
        g.replay()
        eager = both()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(res, eager)), step


def test_autograd_in_a_graph(fa):
    """Forward and backward captured through autograd; with an older eager graph
    of the same leaves alive, the captured call is refused before it can end the
    capture."""
    q, k, dq, dk = (t.to(DEV) for t in inputs(1, 4, 2, 50, 64, torch.bfloat16, 29))
    cos, sin = (t.to(DEV) for t in tables(50, 64))
    qw, kw = (w.to(DEV).requires_grad_() for w in weights(64, torch.float32, 30))
    q.requires_grad_()

    def step():
        qo, ko = fa.qk_norm_rope(q, k, qw, kw, cos, sin)
        return torch.autograd.grad((qo, ko), (q, qw, kw), (dq, dk))

    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    alive = fa.qk_norm_rope(q, k, qw, kw, cos, sin)  # holds the leaves' accumulators
    h = torch.cuda.CUDAGraph()
    with torch.cuda.graph(h):
        keep = q.detach() + 1
        with pytest.raises(RuntimeError, match="qk_norm_rope_backward"):
            fa.qk_norm_rope(q, k, qw, kw, cos, sin)
        grads = fa.qk_norm_rope_backward(dq, dk, q, k, qw, kw, cos, sin)
    for _ in range(2):
        h.replay()
        torch.cuda.synchronize()
        assert torch.equal(grads[0], want[0]) and torch.equal(grads[2], want[1])
    del alive, keep


def test_refusals(fa):
    q, k, _, _ = (t.to(DEV) for t in inputs(1, 2, 2, 8, 64, torch.float16, 31))
    qw, kw = (w.to(DEV) for w in weights(64, torch.float32, 32))
    cos, sin = (t.to(DEV) for t in tables(8, 64))
    ok = dict(q=q, k=k, q_weight=qw, k_weight=kw, cos=cos, sin=sin)
    fa.qk_norm_rope(**ok)
    bad = [
        (dict(q=q.float()), "float16 or bfloat16"),
        (dict(k=k.bfloat16()), "same dtype"),
        (dict(k=k[:, :, :4]), "same batch, length"),
        (dict(q=q.transpose(2, 3)), "unit stride"),
        (dict(q=q[..., :32], k=k[..., :32], q_weight=qw[:32], k_weight=kw[:32]), "head_dim 64 and 128"),
        (dict(q_weight=qw[:32]), r"shape \[head_dim\]"),
        (dict(q_weight=qw.double()), "float32 or have q's dtype"),
        (dict(q_weight=qw.half()), "same dtype"),
        (dict(cos=cos.half()), "contiguous float32"),
        (dict(sin=sin[:4]), "same shape"),
        (dict(cos=cos[:, :12].contiguous(), sin=sin[:, :12].contiguous()), "multiple of 16"),
        (dict(cos=torch.zeros(8, 40, device=DEV), sin=torch.zeros(8, 40, device=DEV)), "multiple of 16"),
        (dict(positions=torch.arange(8, device=DEV)), "int32"),
        (dict(positions=torch.arange(7, device=DEV, dtype=torch.int32)), r"\[N\] or \[B, N\]"),
        (dict(positions=torch.zeros(2, 8, device=DEV, dtype=torch.int32)), r"\[N\] or \[B, N\]"),
        (dict(eps=-1.0), "eps"),
        (dict(eps=math.nan), "eps"),
        (dict(q_weight=torch.ones(65, device=DEV)[1:]), "16-byte aligned"),
        (dict(q=torch.zeros(1, 2, 8, 65, device=DEV).half()[..., 1:]), "multiple of 8"),
    ]
    for change, text in bad:
        with pytest.raises(RuntimeError, match=text):
            fa.qk_norm_rope(**{**ok, **change})
    with pytest.raises(RuntimeError, match="shape"):
        fa.qk_norm_rope_backward(q[:, :, :4], k, **ok)
