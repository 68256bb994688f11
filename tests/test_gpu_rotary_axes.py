"""Rotation by positions of several axes: qk_norm_rope, its gradients and paged_store against the 64-bit formulas."""
from __future__ import annotations

import math

import pytest
import torch

import cache_reference as R
from test_gpu_paged_forward import Cache, cu_of
from test_gpu_qk_norm import inputs, tables, to_dev, weights

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}

CASES = [
    # B, H, KH, N, D, type, layout, rotated, interleaved, weights, axes, order, positions per batch entry
    (1, 1, 1, 1, 64, "fp16", "bhnd", 64, False, "fp32", 1, "blocks", False),
    (2, 3, 1, 37, 128, "bf16", "bhnd", 128, False, "fp32", 3, "blocks", False),
    (2, 3, 3, 50, 64, "fp16", "bnhd", 64, True, "same", 3, "cyclic", True),
    (1, 5, 1, 65, 128, "fp16", "wide", 96, True, "fp32", 2, "odd", True),
    (3, 4, 2, 33, 64, "bf16", "bhnd", 32, False, "same", 4, "cyclic", True),
    (1, 16, 4, 700, 128, "bf16", "bnhd", 128, False, "fp32", 4, "odd", False),
    (2, 7, 7, 100, 64, "fp16", "bhnd", 16, False, "fp32", 2, "blocks", False),
]


def pair_axes(pairs, axes, order, seed=0):
    if order == "cyclic":
        return [i % axes for i in range(pairs)]
    if order == "blocks":
        return [i * axes // pairs for i in range(pairs)]
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, axes, (pairs,), generator=g).tolist()


def setup(case):
    B, H, KH, N, D, dtype, layout, r, inter, wdt, A, order, per_batch = case
    dt = DT[dtype]
    q, k, dq, dk = inputs(B, H, KH, N, D, dt, 40 + N, layout)
    qw, kw = weights(D, torch.float32 if wdt == "fp32" else dt, 41)
    cos, sin = tables(90, r)
    g = torch.Generator().manual_seed(N)
    pos = torch.randint(0, 90, (A, B, N) if per_batch else (A, N), generator=g, dtype=torch.int32)
    axes = pair_axes(r // 2, A, order, N)
    return q, k, dq, dk, qw, kw, cos, sin, pos, axes


def token_tables(cos, sin, pos, axes, B, N):
    """The tables of each token, [B * N, r / 2] and the row of each, [B, 1, N]: one position a token."""
    p = pos if pos.dim() == 3 else pos[:, None].expand(-1, B, -1)
    a = torch.tensor(axes)
    row = p[a].permute(1, 2, 0).long()  # [B, N, pairs]
    pair = torch.arange(len(axes))
    ok = (row >= 0) & (row < cos.shape[0])
    c, s = (torch.where(ok, t[row.clamp(0, cos.shape[0] - 1), pair], math.nan).reshape(B * N, -1) for t in (cos, sin))
    return c, s, torch.arange(B * N).view(B, 1, N)


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_forward_and_gradients(fa, case):
    print("case", case, flush=True)
    q, k, dq, dk, qw, kw, cos, sin, pos, axes = setup(case)
    B, N, inter = case[0], case[3], case[8]
    leaves = [to_dev(q).requires_grad_(), to_dev(k).requires_grad_(), qw.to(DEV).requires_grad_(), kw.to(DEV).requires_grad_()]
    rest = (cos.to(DEV), sin.to(DEV), pos.to(DEV))
    qo, ko = fa.qk_norm_rope(*leaves, *rest, interleaved=inter, axes=axes)
    got = torch.autograd.grad((qo, ko), leaves, (to_dev(dq), to_dev(dk)))
    c, s, at = token_tables(cos, sin, pos, axes, B, N)
    for name, x, w, y, dy, dx, dw in (("q", q, qw, qo, dq, got[0], got[2]), ("k", k, kw, ko, dk, got[1], got[3])):
        want, tol = R.norm_rope(x, w, c, s, at.expand(-1, x.shape[1], -1), eps=1e-6, interleaved=inter)
        R.check(name, y, want, tol)
        wx, tx, ww, tw = R.norm_rope_grad(x, w, c, s, at, dy, eps=1e-6, interleaved=inter)
        R.check("d" + name, dx, wx, tx)
        R.check("d weight of " + name, dw, ww, tw)
    direct = fa.qk_norm_rope_backward(to_dev(dq), to_dev(dk), to_dev(q), to_dev(k), qw.to(DEV), kw.to(DEV), *rest,
                                      interleaved=inter, axes=bytes(axes))
    assert all(torch.equal(a, b) for a, b in zip(direct, got))


def test_gradients_against_differences(fa):
    case = (1, 1, 1, 5, 64, "fp16", "bhnd", 64, False, "fp32", 3, "cyclic", False)
    q, k, dq, dk, qw, kw, cos, sin, pos, axes = setup(case)
    got = fa.qk_norm_rope_backward(*(t.to(DEV) for t in (dq, dk, q, k, qw, kw, cos, sin, pos)), axes=axes)
    c, s, at = token_tables(cos, sin, pos, axes, 1, 5)

    def loss(x, w):
        n = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
        a, b = n[..., :32], n[..., 32:]
        y = torch.cat((a * c.double() - b * s.double(), b * c.double() + a * s.double()), -1)
        return (y * dq.double()).sum()

    g = torch.Generator().manual_seed(1)
    _, tx, _, tw = R.norm_rope_grad(q, qw, c, s, at, dq, eps=1e-6, interleaved=False)
    for x, w, got_x, tol in ((True, False, got[0], tx), (False, True, got[2], tw)):
        d = torch.randn(got_x.shape, generator=g, dtype=torch.float64)
        h = 1e-6
        args = lambda e: (q.double() + e * d * x if x else q.double(), qw.double() + e * d if w else qw.double())
        diff = (loss(*args(h)) - loss(*args(-h))) / (2 * h)
        assert abs(diff - (got_x.cpu().double() * d).sum()) <= (tol * d.abs()).sum() + 1e-6 * (1 + abs(diff))


def test_one_axis_is_the_plain_rotation(fa):
    q, k, _, _ = (t.to(DEV) for t in inputs(2, 3, 1, 40, 64, torch.bfloat16, 7))
    qw, kw = (w.to(DEV) for w in weights(64, torch.float32, 8))
    cos, sin = (t.to(DEV) for t in tables(40, 64))
    pos = torch.randperm(40, device=DEV).int()
    plain = fa.qk_norm_rope(q, k, qw, kw, cos, sin, pos)
    one = fa.qk_norm_rope(q, k, qw, kw, cos, sin, pos[None], axes=[0] * 32)
    same = fa.qk_norm_rope(q, k, qw, kw, cos, sin, pos.expand(3, -1), axes=[i % 3 for i in range(32)])
    for a, b, c in zip(plain, one, same):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_positions_outside_the_tables(fa):
    """NaN in the pairs of that axis alone, and where there is no such position the value itself."""
    q, k, _, _ = (t.to(DEV) for t in inputs(1, 1, 1, 4, 64, torch.float16, 9))
    one = torch.ones(64, device=DEV)
    cos, sin = (t.to(DEV) for t in tables(10, 32))
    pos = torch.tensor([[1, 2, 10, 3], [4, -1, 5, 6]], dtype=torch.int32, device=DEV)
    axes = [0] * 6 + [1] * 10
    y, _ = fa.qk_norm_rope(q, k, one, one, cos, sin, pos, axes=axes)
    nan = torch.isnan(y[0, 0])
    want = torch.zeros(4, 64, dtype=torch.bool, device=DEV)
    for t, axis in ((2, 0), (1, 1)):
        for i, a in enumerate(axes):
            want[t, [i, 16 + i]] |= a == axis
    assert torch.equal(nan, want)


def test_store(fa):
    """paged_store with axes is qk_norm_rope of the tokens, in their places; replayed with other positions."""
    c = Cache([40, 20, 7], 16, 2, 64, torch.bfloat16, 60)
    kc, vc, table = c.dev()
    new = [5, 1, 7]
    g = torch.Generator(device=DEV).manual_seed(2)
    q, k, v = (torch.randn(sum(new), h, 64, generator=g, device=DEV).bfloat16() for h in (6, 2, 2))
    qw, kw = (w.to(DEV) for w in weights(64, torch.bfloat16, 61))
    cos, sin = (t.to(DEV) for t in tables(50, 64))
    axes = bytes(i % 3 for i in range(32))
    pos = torch.randint(0, 50, (3, sum(new)), generator=g, device=DEV, dtype=torch.int32)
    cu, lens = cu_of(new).to(DEV), c.lens.to(DEV)
    graph, kg, vg = torch.cuda.CUDAGraph(), kc.clone(), vc.clone()
    with torch.cuda.graph(graph):
        qg = fa.paged_store(q, k, v, qw, kw, cos, sin, pos, kg, vg, table, cu, lens, axes=axes)
    for _ in range(3):
        pos.random_(0, 50, generator=g)
        qs = fa.paged_store(q, k, v, qw, kw, cos, sin, pos, kc, vc, table, cu, lens, axes=axes)
        graph.replay()
        qn, kn = fa.qk_norm_rope(q.transpose(0, 1)[None], k.transpose(0, 1)[None], qw, kw, cos, sin, pos, axes=axes)
        torch.cuda.synchronize()
        assert torch.equal(qs, qn[0].transpose(0, 1)) and torch.equal(qg, qs)
        assert torch.equal(kg.nan_to_num(), kc.nan_to_num()) and torch.equal(vg.nan_to_num(), vc.nan_to_num())
        at = 0
        for b, n in enumerate(new):
            for i in range(n):
                key = c.lens[b] - n + i
                page = c.table[b, key // 16]
                assert torch.equal(kc[page, :, key % 16], kn[0, :, at + i])
                assert torch.equal(vc[page, :, key % 16], v[at + i])
            at += n


def test_refusals(fa):
    q, k, dq, dk = (t.to(DEV) for t in inputs(2, 2, 2, 8, 64, torch.float16, 31))
    qw, kw = (w.to(DEV) for w in weights(64, torch.float32, 32))
    cos, sin = (t.to(DEV) for t in tables(8, 64))
    pos = torch.zeros(3, 8, dtype=torch.int32, device=DEV)
    axes = [i % 3 for i in range(32)]
    ok = dict(q=q, k=k, q_weight=qw, k_weight=kw, cos=cos, sin=sin, positions=pos, axes=axes)
    fa.qk_norm_rope(**ok)
    for change, text in [
        (dict(positions=None), "axes need positions"), (dict(positions=pos[0]), "dimension"),
        (dict(positions=pos.long()), "int32"), (dict(positions=pos[:, :7]), r"\[axes, N\]"),
        (dict(positions=torch.zeros(3, 3, 8, dtype=torch.int32, device=DEV)), r"\[axes, B, N\]"),
        (dict(axes=axes[:-1]), "one entry per pair"), (dict(axes=axes + [0]), "one entry per pair"),
        (dict(axes=[3] * 32), "axis 3 of 3"), (dict(positions=pos[:0]), "1 to 4"),
        (dict(positions=torch.zeros(5, 8, dtype=torch.int32, device=DEV)), "1 to 4"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            fa.qk_norm_rope(**{**ok, **change})
        with pytest.raises(RuntimeError, match=text):
            fa.qk_norm_rope_backward(dq, dk, **{**ok, **change})
    with pytest.raises((ValueError, TypeError)):
        fa.qk_norm_rope(**{**ok, "axes": [-1] * 32})
