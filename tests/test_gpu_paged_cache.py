"""The paged cache's store, key weights and eviction against their 64-bit forms,
and a run of all operators as a server uses them."""
from __future__ import annotations

import math

import pytest
import torch

import cache_reference as R
from test_gpu_paged_forward import Cache, cu_of, DT, SHAPES
from test_gpu_qk_norm import tables

pytestmark = pytest.mark.gpu
DEV = "cuda"


# ---- store ----

STORES = [
    # lens, new, H, KH, D, page, dtype, rotated, interleaved, weights
    ([1], [1], 1, 1, 64, 16, "fp16", 64, False, "fp32"),
    ([15, 16, 17, 40], [1, 1, 1, 1], 8, 2, 128, 16, "bf16", 128, True, "same"),
    ([100, 3, 64, 200], [100, 3, 10, 70], 4, 4, 64, 64, "bf16", 32, False, "fp32"),
    ([50] * 100, [1, 0, 2, 1] * 25, 3, 1, 128, 32, "fp16", 128, False, "same"),
    ([2, 0, 30], [5, 4, 3], 2, 1, 64, 16, "fp16", 64, True, "fp32"),  # more tokens than keys
]


@pytest.mark.parametrize("case", STORES, ids=lambda c: f"B{len(c[0])}-T{sum(c[1])}-D{c[4]}-{c[6]}")
@pytest.mark.parametrize("layout", ["heads-first", "keys-first"])
def test_store(fa, case, layout):
    lens, new, H, KH, D, page, dtype, r, inter, wdt = case
    print("case store", case, layout, flush=True)
    dt = DT[dtype]
    c = Cache(lens, page, KH, D, dt, 500, wide=1, pages_first=layout == "heads-first")
    T = sum(new) + 3  # three rows of no sequence at the end
    g = torch.Generator().manual_seed(9)
    qkv = torch.randn(T, H + 2 * KH, D, generator=g).to(dt)  # a fused projection's output
    q, k, v = qkv[:, :H], qkv[:, H: H + KH], qkv[:, H + KH:]
    wt = torch.float32 if wdt == "fp32" else dt
    qw, kw = ((1 + 0.2 * torch.randn(D, generator=g)).to(wt) for _ in range(2))
    cos, sin = tables(400, r)
    pos = torch.randint(0, 400, (T,), generator=g, dtype=torch.int32)
    cu = cu_of(new)
    kc, vc, table = c.dev()
    out = torch.full((T, H, D), 9.0, dtype=dt, device=DEV)
    d = qkv.to(DEV)
    res = fa.paged_store(d[:, :H], d[:, H: H + KH], d[:, H + KH:], qw.to(DEV), kw.to(DEV), cos.to(DEV),
                         sin.to(DEV), pos.to(DEV), kc, vc, table, cu.to(DEV), c.lens.to(DEV), out,
                         eps=1e-5, interleaved=inter)
    assert res.data_ptr() == out.data_ptr()
    wq, tq = R.norm_rope(q, qw, cos, sin, pos[:, None].expand(T, H), eps=1e-5, interleaved=inter)
    wk, tk = R.norm_rope(k, kw, cos, sin, pos[:, None].expand(T, KH), eps=1e-5, interleaved=inter)
    n = sum(new)
    R.check("q", res[:n], wq[:n], tq[:n])
    assert bool((out[n:] == 9).all())
    want_k, want_v, tol = c.k.double(), c.v.double(), torch.zeros(c.k.shape, dtype=torch.float64)
    for b, c0, nq, L, first in R.sequences(cu, c.lens, T):
        for i in range(nq):
            j = first + i
            if j < 0:
                continue
            at = (int(c.table[b, j // page]), slice(None), j % page)
            want_k[at], tol[at], want_v[at] = wk[c0 + i], tk[c0 + i], v[c0 + i].double()
    R.check("k_cache", kc, want_k, tol)
    R.check("v_cache", vc, want_v, torch.zeros_like(tol))


def test_store_in_place_and_on_absent_pages(fa):
    c = Cache([40, 20], 16, 1, 64, torch.bfloat16, 510)
    full = c.table.clone()
    c.table[0, 1] = -1
    c.table[1, 0] = c.k.shape[0]
    T = 60
    g = torch.Generator().manual_seed(10)
    q, k, v = (torch.randn(T, h, 64, generator=g).bfloat16() for h in (2, 1, 1))
    w = torch.ones(64)
    cos, sin = tables(60, 64)
    pos = torch.arange(60, dtype=torch.int32)
    kc, vc, table = c.dev()
    before = kc.clone(), vc.clone()
    qd = q.to(DEV)
    res = fa.paged_store(qd, k.to(DEV), v.to(DEV), w.to(DEV), w.to(DEV), cos.to(DEV), sin.to(DEV),
                         pos.to(DEV), kc, vc, table, cu_of([40, 20]).to(DEV), c.lens.to(DEV), qd)
    assert res.data_ptr() == qd.data_ptr()
    wq, tq = R.norm_rope(q, w, cos, sin, pos[:, None].expand(T, 2), eps=1e-6, interleaved=False)
    R.check("q", res, wq, tq)
    for p in (int(full[0, 1]), int(full[1, 0]), 0):  # nothing reached these pages
        assert torch.equal(kc[p].view(torch.int16), before[0][p].view(torch.int16))
        assert torch.equal(vc[p].view(torch.int16), before[1][p].view(torch.int16))
    assert torch.equal(vc[int(full[0, 2]), 0, :8].cpu(), v[32:40, 0])


# ---- key weights ----


def weights_of(c, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.rand(c.k.shape[:3], generator=g)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("name", list(SHAPES))
def test_key_weights(fa, name, dtype):
    print(f"case weights {name} {dtype}", flush=True)
    lens, new, H, KH, D, page = SHAPES[name]
    c = Cache(lens, page, KH, D, DT[dtype], 520, wide=1)
    T = sum(new)
    q = torch.randn(T, H, D, generator=torch.Generator().manual_seed(21)).to(DT[dtype])
    k, v, table = c.dev()
    cu = cu_of(new)
    w = weights_of(c, 22)
    _, lse = fa.paged_forward(q.to(DEV), k, v, table, cu.to(DEV), c.lens.to(DEV), max_q=max(new),
                              return_lse=True)
    wd = w.to(DEV)
    res = fa.paged_key_weights(q.to(DEV), lse, k, table, cu.to(DEV), c.lens.to(DEV), wd, max_q=max(new))
    assert res is wd
    want, tol = R.key_weights(q, lse.cpu(), c.k, c.table, cu, c.lens, w, scale=D ** -0.5)
    R.check("weights", wd, want, tol)


@pytest.mark.parametrize("name", ["mixed", "mixed-long", "mixed-long-d128", "group-40-chunk-rows", "empty-sequences"])
def test_key_weights_of_a_cache_that_may_be_large(fa, name):
    """Limits of more than 384 MiB of K, by a wide table: sequences of few rows
    get a kernel of their own beside the others."""
    print(f"case weights large limits {name}", flush=True)
    lens, new, H, KH, D, page = SHAPES[name]
    keys = 384 * 2 ** 20 // (len(lens) * KH * D * 2) + 1
    c = Cache(lens, page, KH, D, torch.float16, 525, wide=-(-keys // page))
    T = sum(new)
    q = torch.randn(T, H, D, generator=torch.Generator().manual_seed(26)).half()
    lse = 6 + torch.randn(T, H, generator=torch.Generator().manual_seed(27))
    k, _, table = c.dev()
    cu = cu_of(new)
    w = weights_of(c, 28)
    wd = fa.paged_key_weights(q.to(DEV), lse.to(DEV), k, table, cu.to(DEV), c.lens.to(DEV), w.to(DEV),
                              max_q=max(new))
    want, tol = R.key_weights(q, lse, c.k, c.table, cu, c.lens, w, scale=D ** -0.5)
    R.check("weights", wd, want, tol)


@pytest.mark.parametrize("name", ["ragged-decode", "mixed", "few-tokens"])
def test_key_weights_with_limits_no_mask_and_absent_pages(fa, name):
    print(f"case weights limits {name}", flush=True)
    lens, new, H, KH, D, page = SHAPES[name]
    c = Cache(lens, page, KH, D, torch.bfloat16, 530)
    c.table[0, 0] = -1
    c.table[2, 0] = 2 ** 30
    T = sum(new)
    q = torch.randn(T, H, D, generator=torch.Generator().manual_seed(23)).bfloat16()
    k, v, table = c.dev()
    cu = cu_of(new)
    lse = (6 + torch.randn(T, H, generator=torch.Generator().manual_seed(24)))
    lse[0, 0] = -math.inf
    lse[-1, -1] = math.inf
    for causal in (True, False):
        for max_q, max_kv in ((max(new), None), (max(1, max(new) // 2), max(lens) - 30)):
            # (weights in a wider buffer: strides of its own)
            buf = torch.full((c.k.shape[0], KH + 1, 2 * page), 5.0)
            w = buf[:, 1:, page:]
            w.copy_(weights_of(c, 25))
            bd = buf.to(DEV)
            fa.paged_key_weights(q.to(DEV), lse.to(DEV), k, table, cu.to(DEV), c.lens.to(DEV),
                                 bd[:, 1:, page:], max_q=max_q, max_kv=max_kv, causal=causal,
                                 softmax_scale=0.07)
            want, tol = R.key_weights(q, lse, c.k, c.table, cu, c.lens, w, scale=0.07, causal=causal,
                                      max_q=max_q, max_kv=max_kv)
            R.check("weights", bd[:, 1:, page:], want, tol)
            assert bool((bd[:, 0] == 5).all()) and bool((bd[:, :, :page] == 5).all())


def test_key_weights_sum_to_the_rows(fa):
    """Every row gives away a weight of 1 per head."""
    lens, new, H, KH, D, page = SHAPES["chunks"]
    c = Cache(lens, page, KH, D, torch.float16, 540)
    q = torch.randn(sum(new), H, D, generator=torch.Generator().manual_seed(26)).half().to(DEV)
    k, v, table = c.dev()
    cu = cu_of(new).to(DEV)
    _, lse = fa.paged_forward(q, k, v, table, cu, c.lens.to(DEV), max_q=max(new), return_lse=True)
    w = torch.zeros(c.k.shape[:3], device=DEV)
    fa.paged_key_weights(q, lse, k, table, cu, c.lens.to(DEV), w, max_q=max(new))
    # sums of sums of 1 in fp32: 2^-13 relative holds scores' and sums' errors many times
    assert abs(float(w.double().sum()) - sum(new) * H) <= 2.0 ** -13 * sum(new) * H


def test_key_weights_same_bits_twice_in_graphs(fa):
    lens, new, H, KH, D, page = SHAPES["split-chunk"]
    c = Cache(lens, page, KH, D, torch.bfloat16, 550)
    q = torch.randn(sum(new), H, D, generator=torch.Generator().manual_seed(27)).bfloat16().to(DEV)
    k, v, table = c.dev()
    cu, ln = cu_of(new).to(DEV), c.lens.to(DEV)
    lse = torch.full((sum(new), H), 8.0, device=DEV)
    start = weights_of(c, 28).to(DEV)
    w = start.clone()
    call = lambda x: fa.paged_key_weights(q, lse, k, table, cu, ln, x, max_q=max(new))  # noqa: E731
    eager = call(start.clone())
    assert torch.equal(eager, call(start.clone()))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call(w)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(w)
    for n in (3000, 1700, 41):
        ln.fill_(n)
        w.copy_(start)
        g.replay()
        want = call(start.clone())
        torch.cuda.synchronize()
        assert torch.equal(w, want), n


# ---- eviction ----


def evict_setup(lens, page, kh, d, dt, keep, seed, max_kv=None):
    c = Cache(lens, page, kh, d, dt, seed)
    n_new = max(1, -(-min(keep, c.table.shape[1] * page) // page))
    old = c.k.shape[0]
    extra = torch.full((len(lens) * n_new, kh, page, d), 3.0, dtype=dt)
    c.k, c.v = torch.cat([c.k, extra]), torch.cat([c.v, extra])
    g = torch.Generator().manual_seed(seed)
    new_table = (old + torch.randperm(len(lens) * n_new, generator=g)).to(torch.int32).view(len(lens), n_new)
    w = torch.rand(c.k.shape[:3], generator=g)
    return c, new_table, w


def evict_compare(fa, c, new_table, w, *, keep, recent, max_kv=None):
    k, v, table = c.dev()
    wd = w.to(DEV)
    lens, kept = fa.paged_evict(k, v, wd, table, c.lens.to(DEV), new_table.to(DEV), keep=keep,
                                recent=recent, max_kv=max_kv)
    want = R.evict(c.k, c.v, w, c.table, c.lens, new_table, keep=keep, recent=recent, max_kv=max_kv)
    assert lens.dtype == torch.int32 and kept.dtype == torch.int32
    assert torch.equal(lens.cpu(), want[0])
    assert torch.equal(kept.cpu(), want[1])
    for got, ref in ((k, want[2]), (v, want[3]), (wd, want[4])):
        same = got.cpu().contiguous().view(torch.uint8) == ref.contiguous().view(torch.uint8)
        assert bool(same.all())
    return lens, kept


EVICTS = [
    # lens, page, KH, D, keep, recent
    ([1], 16, 1, 64, 1, 0),
    ([2], 16, 1, 64, 1, 1),
    ([100, 40, 41, 0, 300], 16, 2, 64, 40, 7),
    ([100, 40, 41, 0, 300], 32, 1, 128, 40, 0),
    ([100, 64, 65], 64, 3, 128, 64, 64),
    ([1024, 1025, 3000], 256, 1, 64, 1024, 100),
    ([20000], 64, 1, 64, 5000, 1000),  # more keys than a workgroup keeps in registers
    ([500, 700], 16, 2, 64, 1000, 3),  # nothing to evict
]


@pytest.mark.parametrize("case", EVICTS, ids=lambda c: f"L{max(c[0])}-page{c[1]}-D{c[3]}-keep{c[4]}-{c[5]}")
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_evict(fa, case, dtype):
    lens, page, kh, d, keep, recent = case
    print("case evict", case, dtype, flush=True)
    c, new_table, w = evict_setup(lens, page, kh, d, DT[dtype], keep, 600)
    evict_compare(fa, c, new_table, w, keep=keep, recent=recent)


@pytest.mark.parametrize("kind", ["ties", "zeros", "nan-inf-negative", "tiny", "all-nan", "steps"])
def test_evict_order_of_weights(fa, kind):
    print("case evict order", kind, flush=True)
    c, new_table, w = evict_setup([1500, 333], 16, 2, 64, torch.float16, 200, 610)
    g = torch.Generator().manual_seed(3)
    if kind == "ties":
        w = torch.randint(0, 3, w.shape, generator=g).float()
    elif kind == "zeros":
        w = torch.where(torch.rand(w.shape, generator=g) < 0.5, 0.0, -0.0)
    elif kind == "nan-inf-negative":
        w = torch.randn(w.shape, generator=g)
        pick = torch.randint(0, 12, w.shape, generator=g)
        for i, x in enumerate((math.nan, math.inf, -math.inf, -0.0, -math.nan)):
            w[pick == i] = x
    elif kind == "tiny":
        w = torch.rand(w.shape, generator=g) * 1e-40
    elif kind == "all-nan":
        w = torch.full(w.shape, math.nan)
    else:  # one bit apart
        w = (torch.randint(0, 5, w.shape, generator=g, dtype=torch.int32) + 0x3F800000).view(torch.float32)
    evict_compare(fa, c, new_table, w, keep=200, recent=30)


def test_evict_absent_pages_and_limits(fa):
    c, new_table, w = evict_setup([100, 90, 80, 70], 16, 2, 64, torch.float16, 50, 620)
    c.table[0, 2] = -1
    new_table[1, 0] = c.k.shape[0]
    c.table[2, 4] = -1  # holds keys 64 to 79: behind max_kv
    evict_compare(fa, c, new_table, w, keep=50, recent=5, max_kv=64)
    c.lens = torch.tensor([2 ** 31 - 1, -5, 3, 64], dtype=torch.int32)
    evict_compare(fa, c, new_table, w, keep=50, recent=5, max_kv=64)


def test_evict_keys_first_layout_and_graph(fa):
    c, new_table, w = evict_setup([400, 120], 16, 2, 128, torch.bfloat16, 100, 630)
    c.pages_first = False
    evict_compare(fa, c, new_table, w, keep=100, recent=10)
    k, v, table = c.dev()
    wd, nt, ln = w.to(DEV), new_table.to(DEV), c.lens.to(DEV)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        res = fa.paged_evict(k, v, wd, table, ln, nt, keep=100, recent=10)
    for a, b in ((400, 120), (99, 101), (300, 0)):
        ln.copy_(torch.tensor([a, b], dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        want = R.evict(c.k, c.v, w, c.table, ln.cpu(), new_table, keep=100, recent=10)
        assert torch.equal(res[0].cpu(), want[0]) and torch.equal(res[1].cpu(), want[1])
        n = int(want[0][0])
        got = R.keys_of(k.cpu(), new_table[0], n)[0]
        assert torch.equal(got, R.keys_of(want[2], new_table[0], n)[0])


# ---- all of them ----


def test_a_server_with_a_bounded_cache(fa):
    """Prompts, decode steps, eviction and more decode steps; each step's
    results against the 64-bit forms on the cache as the step found it."""
    D, H, KH, page, keep, recent = 64, 4, 2, 16, 48, 8
    dt = torch.bfloat16
    g = torch.Generator().manual_seed(77)
    pool = 64
    kc = torch.full((pool, KH, page, D), math.nan, dtype=dt, device=DEV)
    vc = kc.clone()
    w = torch.full((pool, KH, page), math.nan, device=DEV)
    free = list(range(pool))
    table = torch.full((2, 8), -1, dtype=torch.int32)
    lens, position = [0, 0], [0, 0]
    cos, sin = tables(300, D)
    qw, kw = 1 + 0.2 * torch.randn(D, generator=g), 1 + 0.2 * torch.randn(D, generator=g)
    for step, new in enumerate([[70, 33], [1, 1], [1, 5], "evict", [1, 1], [20, 0], "evict", [1, 1]]):
        before = kc.cpu(), vc.cpu(), w.cpu()
        ln = torch.tensor(lens, dtype=torch.int32)
        if new == "evict":
            nt = torch.tensor([[free.pop() for _ in range(3)] for _ in range(2)], dtype=torch.int32)
            got, kept = fa.paged_evict(kc, vc, w, table.to(DEV), ln.to(DEV), nt.to(DEV), keep=keep,
                                       recent=recent)
            want = R.evict(*before, table, ln, nt, keep=keep, recent=recent)
            assert torch.equal(got.cpu(), want[0]) and torch.equal(kept.cpu(), want[1])
            free += [p for p in table.flatten().tolist() if p >= 0]
            table = torch.full((2, 8), -1, dtype=torch.int32)
            table[:, :3] = nt
            lens = got.tolist()
            continue
        T = sum(new)
        pos = torch.cat([torch.arange(p, p + n) for p, n in zip(position, new)]).to(torch.int32)
        for b, n in enumerate(new):
            lens[b] += n
            position[b] += n
            for i in range(-(-lens[b] // page)):
                if table[b, i] < 0:
                    table[b, i] = free.pop(0)
        ln, cu = torch.tensor(lens, dtype=torch.int32), cu_of(new)
        q, k, v = (torch.randn(T, h, D, generator=g).to(dt) for h in (H, KH, KH))
        td, cd, ld = table.to(DEV), cu.to(DEV), ln.to(DEV)
        qn = fa.paged_store(q.to(DEV), k.to(DEV), v.to(DEV), qw.to(DEV), kw.to(DEV), cos.to(DEV),
                            sin.to(DEV), pos.to(DEV), kc, vc, td, cd, ld)
        wq, tq = R.norm_rope(q, qw, cos, sin, pos[:, None].expand(T, H), eps=1e-6, interleaved=False)
        R.check("q", qn, wq, tq)
        o, lse = fa.paged_forward(qn, kc, vc, td, cd, ld, max_q=max(new), return_lse=True)
        want_o, want_l, tol, tol_l = R.attend(qn.cpu(), kc.cpu(), vc.cpu(), table, cu, ln, scale=D ** -0.5)
        R.check(f"o, step {step}", o, want_o, tol)
        R.check(f"lse, step {step}", lse, want_l, tol_l)
        fa.paged_key_weights(qn, lse, kc, td, cd, ld, w, max_q=max(new))
        want_w, tol_w = R.key_weights(qn.cpu(), lse.cpu(), kc.cpu(), table, cu, ln, before[2], scale=D ** -0.5)
        R.check(f"weights, step {step}", w, want_w, tol_w)
    assert lens == [49, 41] and position == [94, 41]


def test_refusals(fa):
    c, new_table, w = evict_setup([40, 20], 16, 2, 64, torch.float16, 16, 640)
    k, v, table = c.dev()
    wd, nt, ln, cu = w.to(DEV), new_table.to(DEV), c.lens.to(DEV), cu_of([3, 2]).to(DEV)
    q = torch.zeros(5, 4, 64, device=DEV).half()
    lse = torch.zeros(5, 4, device=DEV)
    kv = torch.zeros(5, 2, 64, device=DEV).half()
    one, pos = torch.ones(64, device=DEV), torch.zeros(5, dtype=torch.int32, device=DEV)
    cos, sin = (t.to(DEV) for t in tables(40, 64))
    calls = {
        "paged_forward": dict(q=q, k_cache=k, v_cache=v, block_table=table, cu_seqlens=cu, seq_lens=ln, max_q=3),
        "paged_key_weights": dict(q=q, lse=lse, k_cache=k, block_table=table, cu_seqlens=cu, seq_lens=ln,
                                  key_weights=wd, max_q=3),
        "paged_evict": dict(k_cache=k, v_cache=v, key_weights=wd, block_table=table, seq_lens=ln,
                            new_table=nt, keep=16),
        "paged_store": dict(q=q, k=kv, v=kv, q_weight=one, k_weight=one, cos=cos, sin=sin, positions=pos,
                            k_cache=k, v_cache=v, block_table=table, cu_seqlens=cu, seq_lens=ln),
    }
    for name, ok in calls.items():
        getattr(fa, name)(**ok)
    paged = [
        (dict(block_table=table.long()), "int32"),
        (dict(block_table=table.T), "unit stride"),
        (dict(block_table=table[:1]), "one entry per row|one entry more|as many rows"),
        (dict(seq_lens=ln.cpu()), "CUDA tensor"),
        (dict(k_cache=k.float()), "float16 or bfloat16"),
        (dict(k_cache=k[:, :, :8]), "same shape|key_weights must have shape|page_size 8"),
    ]
    for name, ok in calls.items():
        for change, text in paged:
            with pytest.raises(RuntimeError, match=text):
                getattr(fa, name)(**{**ok, **change})
    more = {
        "paged_forward": [
            (dict(v_cache=v.bfloat16()), "same dtype"), (dict(q=q.bfloat16()), "same dtype"),
            (dict(q=q[:, :3]), "multiple of kv_heads"), (dict(q=q[:, :, :32]), "head_dim"),
            (dict(max_q=-1), "max_q"), (dict(max_kv=-1), "max_kv"), (dict(softmax_scale=0.0), "softmax_scale"),
            (dict(softmax_scale=math.inf), "softmax_scale"), (dict(out=q), "must not be q"),
            (dict(out=q[:4]), "as many tokens"), (dict(out=torch.zeros_like(q)[:, :1].expand(5, 4, 64)), "rows overlap"),
            (dict(q=torch.zeros(5, 4, 65, device=DEV).half()[..., 1:]), "multiple of 8"),
            (dict(q=q.clone().requires_grad_()), "no gradients"),
            (dict(out=torch.zeros_like(q).requires_grad_()), "no gradients"),
            (dict(cu_seqlens=cu[:2]), "one entry more"),
        ],
        "paged_key_weights": [
            (dict(lse=lse[:, :2]), "lse must"), (dict(lse=lse.double()), "float32"),
            (dict(key_weights=wd.half()), "float32"), (dict(key_weights=wd[:, :1]), "shape"),
            (dict(key_weights=wd[:, :1].expand_as(wd)), "rows overlap"),
        ],
        "paged_evict": [
            (dict(keep=0), "keep"), (dict(recent=17), "recent"), (dict(recent=-1), "recent"),
            (dict(keep=40), "hold fewer"), (dict(new_table=table), "pages of their own"),
            (dict(new_table=nt[:1]), "as many rows"), (dict(keep=2 ** 40), "32 bits"),
            (dict(k_cache=k[:, :1].expand_as(k)), "rows overlap"), (dict(keep=2 ** 30 + 1), "2\\^30"),
        ],
        "paged_store": [
            (dict(k=q), "number of heads"), (dict(v=kv[:4]), "as many tokens"),
            (dict(positions=pos.long()), "int32"), (dict(positions=pos[:4]), "one entry per token"),
            (dict(q_weight=one[:32]), "head_dim"), (dict(k_cache=k[:1].expand_as(k)), "rows overlap"),
            (dict(cos=cos.half()), "float32"), (dict(q_weight=one.clone().requires_grad_()), "no gradients"),
            (dict(out=torch.zeros_like(q).requires_grad_()), "no gradients"),
        ],
    }
    for name in ("paged_forward", "paged_key_weights", "paged_evict", "paged_store"):
        more[name].append((dict(k_cache=k.clone().requires_grad_()), "no gradients"))
    for name, changes in more.items():
        for change, text in changes:
            with pytest.raises(RuntimeError, match=text):
                getattr(fa, name)(**{**calls[name], **change})
