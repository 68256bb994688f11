"""Tensors that share memory: views of one buffer that share no element are taken,
a result that would overwrite what the call still reads is refused."""
from __future__ import annotations

import pytest
import torch

import cache_reference as R
from test_gpu_paged_forward import Cache, cu_of
from test_gpu_qk_norm import tables

pytestmark = pytest.mark.gpu
DEV = "cuda"
H, KH, D, T = 4, 2, 64, 45


def setup():
    c = Cache([60, 33], 16, KH, D, torch.float16, 900)
    k, v, table = c.dev()
    return c, k, v, table, cu_of([40, 5]).to(DEV), c.lens.to(DEV)


def fused(seed=4, wide=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(T, 2 * H + 2 * KH + 2, D + wide, generator=g, device=DEV).half()


def test_forward_into_other_heads_of_the_same_buffer(fa):
    _, k, v, table, cu, ln = setup()
    for wide in (0, 8):
        buf = fused(wide=wide)[..., wide:]
        q = buf[:, :H].clone()
        want = fa.paged_forward(q, k, v, table, cu, ln, max_q=40)
        o = fa.paged_forward(buf[:, :H], k, v, table, cu, ln, buf[:, H:2 * H], max_q=40)
        assert torch.equal(o, want) and torch.equal(buf[:, :H], q)
    # every second head; the two halves of a row
    buf = fused()
    want = fa.paged_forward(buf[:, 0:2 * H:2].clone(), k, v, table, cu, ln, max_q=40)
    assert torch.equal(fa.paged_forward(buf[:, 0:2 * H:2], k, v, table, cu, ln, buf[:, 1:2 * H:2], max_q=40), want)
    buf = torch.randn(T, H, 2 * D, device=DEV).half()
    want = fa.paged_forward(buf[..., :D].clone(), k, v, table, cu, ln, max_q=40)
    assert torch.equal(fa.paged_forward(buf[..., :D], k, v, table, cu, ln, buf[..., D:], max_q=40), want)


def test_forward_refuses_results_over_its_inputs(fa):
    _, k, v, table, cu, ln = setup()
    buf = fused()
    rows = torch.randn(T + 1, H, D, device=DEV).half()
    flat = torch.zeros(T * H * D + 64, device=DEV).half()
    pool = torch.zeros(8, KH, 16, D, device=DEV).half()
    over = pool.view(-1)[:T * H * D].view(T, H, D) if pool.numel() >= T * H * D else None
    cases = [
        (buf[:, :H], buf[:, 1:H + 1]),                 # a head on
        (rows[:-1], rows[1:]),                         # a token on
        (rows[1:], rows[:-1]),
        (flat[:-64].view(T, H, D), flat[64:].view(T, H, D)),
        (flat[:-64].view(T, H, D), flat[32:-32].view(T, H, D)),  # half a row on
        (flat[:-64].view(T, H, D), flat[:-64].view(H, T, D).transpose(0, 1)),  # other strides
    ]
    for q, out in cases:
        with pytest.raises(RuntimeError, match="out must not|overlap"):
            fa.paged_forward(q, k, v, table, cu, ln, out, max_q=40)
    q = buf[:, :H]
    if over is not None:
        for kk, vv in ((pool, v[:8]), (k[:8], pool)):
            with pytest.raises(RuntimeError, match="overlap"):
                fa.paged_forward(q, kk, vv, table, cu, ln, over, max_q=40)


def store_args():
    c, k, v, table, cu, ln = setup()
    one = torch.ones(D, device=DEV)
    cos, sin = (t.to(DEV) for t in tables(60, D))
    return k, v, table, cu, ln, one, cos, sin, torch.arange(T, dtype=torch.int32, device=DEV)


def test_store_takes_views_of_one_pool_and_of_one_projection(fa):
    k, v, table, cu, ln, one, cos, sin, pos = store_args()
    for layout in ("pages, 2", "2, pages", "rows"):
        if layout == "pages, 2":
            pool = torch.zeros(k.shape[0], 2, KH, 16, D, device=DEV).half()
            kp, vp = pool[:, 0], pool[:, 1]
        elif layout == "2, pages":
            pool = torch.zeros(2, *k.shape, device=DEV).half()
            kp, vp = pool[0], pool[1]
        else:  # a key's K and V in one row
            pool = torch.zeros(k.shape[0], KH, 16, 2 * D, device=DEV).half()
            kp, vp = pool[..., :D], pool[..., D:]
        qkv = fused()
        q, kn, vn = qkv[:, :H], qkv[:, H:H + KH], qkv[:, H + KH:H + 2 * KH]
        ka, va = torch.zeros_like(k), torch.zeros_like(v)
        want = fa.paged_store(q, kn, vn, one, one, cos, sin, pos, ka, va, table, cu, ln)
        got = fa.paged_store(q, kn, vn, one, one, cos, sin, pos, kp, vp, table, cu, ln, q)  # in place
        assert torch.equal(got, want) and torch.equal(kp, ka) and torch.equal(vp, va), layout


def test_store_refuses_what_it_would_overwrite(fa):
    k, v, table, cu, ln, one, cos, sin, pos = store_args()
    qkv = fused()
    q, kn, vn = qkv[:, :H], qkv[:, H:H + KH], qkv[:, H + KH:H + 2 * KH]
    rows = torch.zeros(T + 1, H, D, device=DEV).half()
    call = lambda q, kn, vn, k, v, out=None: fa.paged_store(  # noqa: E731
        q, kn, vn, one, one, cos, sin, pos, k, v, table, cu, ln, out)
    for args in [
        (q, kn, vn, k, k),                                   # one pool for both
        (q, kn, vn, k[:-1], k[1:]),                          # shifted by a page
        (q, kn, vn, k, v, qkv[:, 1:H + 1]),                  # a head on: over q and k
        (q, kn, vn, k, v, qkv[:, H:2 * H]),                  # over k and v
        (q, kn, vn, k, v, qkv[:, H + KH:2 * H + KH]),        # over v
        (rows[:-1], kn, vn, k, v, rows[1:]),
        (rows[1:], kn, vn, k, v, rows[1:].view(-1).view(H, T, D).transpose(0, 1)),  # q in another order
        (q, k.view(-1)[:T * KH * D].view(T, KH, D), vn, k, v),  # new keys inside the pool
    ]:
        with pytest.raises(RuntimeError, match="overlap"):
            call(*args)
    call(q, kn, vn, k, v)


def test_evict_refuses_one_pool_for_keys_and_values(fa):
    _, k, v, table, _, ln = setup()
    w = torch.zeros(k.shape[:3], device=DEV)
    nt = torch.zeros(2, 1, dtype=torch.int32, device=DEV)
    for a, b in ((k, k), (k[1:], k[:-1])):
        with pytest.raises(RuntimeError, match="overlap"):
            fa.paged_evict(a, b, w[:a.shape[0]], table, ln, nt, keep=16)
