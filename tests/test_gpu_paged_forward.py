"""Attention of new tokens over a paged cache, against the 64-bit form.

Every slot of the cache that no visible key owns (rows past a sequence's end,
free pages, the page that absent ids read) holds NaN in K and V, so a masked
key that leaks into a result shows as NaN.
"""
from __future__ import annotations

import math

import pytest
import torch

import cache_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


class Cache:
    """A pool of shuffled pages (page 0 and one more are nobody's), tables and lengths."""

    def __init__(self, lens, page, kh, d, dt, seed, wide=0, pages_first=True, extra=2):
        g = torch.Generator().manual_seed(seed)
        counts = [-(-n // page) for n in lens]
        pool = sum(counts) + extra
        ids = (torch.randperm(pool - extra, generator=g) + 1).to(torch.int32)
        self.table = torch.full((len(lens), max([1, *counts]) + wide), -1, dtype=torch.int32)
        self.k = torch.full((pool, kh, page, d), math.nan, dtype=dt)
        self.v = torch.full((pool, kh, page, d), math.nan, dtype=dt)
        at = 0
        for b, n in enumerate(lens):
            mine = ids[at: at + counts[b]]
            at += counts[b]
            self.table[b, : counts[b]] = mine
            for i, p in enumerate(mine.tolist()):
                rows = min(page, n - i * page)
                self.k[p, :, :rows] = torch.randn(kh, rows, d, generator=g).to(dt)
                self.v[p, :, :rows] = torch.randn(kh, rows, d, generator=g).to(dt)
        self.lens = torch.tensor(lens, dtype=torch.int32)
        self.page = page
        self.pages_first = pages_first

    def dev(self):
        k, v = self.k.to(DEV), self.v.to(DEV)
        if not self.pages_first:  # [pages, page_size, kv_heads, head_dim] pools
            k, v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))
        return k, v, self.table.to(DEV)


def cu_of(new):
    return torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32)


def run(fa, c, q, cu, *, max_q, **kw):
    k, v, table = c.dev()
    return fa.paged_forward(q.to(DEV), k, v, table, cu.to(DEV), c.lens.to(DEV), max_q=max_q,
                            return_lse=True, **kw)


def compare(fa, c, q, cu, *, max_q, scale=None, causal=True, max_kv=None):
    s = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    o, lse = run(fa, c, q, cu, max_q=max_q, causal=causal, max_kv=max_kv, softmax_scale=scale)
    want, want_l, tol, tol_l = R.attend(q, c.k, c.v, c.table, cu, c.lens, scale=s, causal=causal,
                                        max_q=max_q, max_kv=max_kv)
    rows = torch.zeros(q.shape[0], dtype=torch.bool)
    for _, c0, nq, _, _ in R.sequences(cu, c.lens, q.shape[0], max_q):
        rows[c0: c0 + nq] = True
    R.check("o", o.cpu()[rows], want[rows], tol[rows])
    R.check("lse", lse.cpu()[rows], want_l[rows], tol_l[rows])
    return o, lse


# lens, new tokens, H, KH, D, page
SHAPES = {
    "one-key": ([1], [1], 1, 1, 64, 16),
    "one-token-page-edges": ([15, 16, 17, 31, 32, 33, 64, 65], [1] * 8, 4, 2, 128, 16),
    "ragged-decode": ([300, 1, 1024, 33, 700], [1] * 5, 8, 2, 64, 64),
    "empty-sequences": ([0, 5, 0, 40, 1], [0, 5, 0, 3, 1], 4, 4, 64, 32),
    "keys-without-tokens": ([30, 50], [0, 2], 2, 1, 128, 16),
    "more-tokens-than-keys": ([3, 0, 20], [5, 4, 40], 3, 1, 64, 16),
    "odd-group-3": ([77, 130], [4, 9], 9, 3, 128, 16),
    "group-17-two-blocks": ([90, 200], [1, 1], 17, 1, 64, 32),
    "group-40-chunk-rows": ([90, 200, 3], [1, 2, 1], 40, 1, 128, 16),
    "few-tokens": ([100, 65, 500], [2, 7, 3], 16, 4, 64, 128),
    "chunks": ([130, 300, 64, 257], [130, 1, 64, 200], 4, 2, 128, 16),
    "chunks-d64": ([130, 300, 64, 257], [130, 1, 64, 200], 4, 2, 64, 256),
    "prefill": ([193], [193], 3, 3, 128, 64),
    "mixed": ([260, 400, 17, 90], [150, 1, 1, 33], 8, 2, 64, 16),
    "many-sequences": ([(37 * i) % 150 for i in range(70)], [min((37 * i) % 150, (5 * i) % 47) for i in range(70)],
                       2, 1, 64, 16),
    "many-long-sequences": ([1100 + i for i in range(66)], [(i * 7) % 36 for i in range(66)], 2, 1, 64, 64),
    "last-round-of-one-head": ([1500, 1400], [200, 130], 2, 1, 128, 32),
    "mixed-long": ([2500, 3000, 1100, 40, 2049], [1, 90, 2, 3, 1], 8, 2, 64, 64),
    "mixed-long-d128": ([1700, 2300, 1], [130, 1, 1], 4, 2, 128, 16),
    "split-decode": ([5000], [1], 4, 2, 128, 64),
    "split-chunk": ([3000], [40], 1, 1, 64, 16),
}


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("name", list(SHAPES))
def test_against_64_bits(fa, name, dtype):
    print(f"case {name} {dtype}", flush=True)
    lens, new, H, KH, D, page = SHAPES[name]
    seed = 100 + list(SHAPES).index(name)
    c = Cache(lens, page, KH, D, DT[dtype], seed, wide=1)
    q = torch.randn(sum(new), H, D, generator=torch.Generator().manual_seed(seed)).to(DT[dtype])
    compare(fa, c, q, cu_of(new), max_q=max(new))


@pytest.mark.parametrize("name", ["ragged-decode", "few-tokens", "mixed", "more-tokens-than-keys"])
def test_without_causal_mask(fa, name):
    print(f"case not causal {name}", flush=True)
    lens, new, H, KH, D, page = SHAPES[name]
    c = Cache(lens, page, KH, D, torch.bfloat16, 300)
    q = torch.randn(sum(new), H, D, generator=torch.Generator().manual_seed(5)).bfloat16()
    compare(fa, c, q, cu_of(new), max_q=max(new), causal=False)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("sigma", [4.0, 30.0])
@pytest.mark.parametrize("name", ["ragged-decode", "chunks", "split-decode"])
def test_wide_scores(fa, name, sigma, dtype):
    """Scores whose maximum moves by hundreds between tiles: the offset is raised
    again and again, and most weights are 0."""
    print(f"case wide {name} {sigma} {dtype}", flush=True)
    lens, new, H, KH, D, page = SHAPES[name]
    c = Cache(lens, page, KH, D, DT[dtype], 310)
    q = (sigma * torch.randn(sum(new), H, D, generator=torch.Generator().manual_seed(6))).to(DT[dtype])
    compare(fa, c, q, cu_of(new), max_q=max(new))


@pytest.mark.parametrize("name", ["ragged-decode", "mixed"])
def test_rising_scores(fa, name):
    """Each key scores above all before it, by far more than fp16 P can hold."""
    print(f"case rising {name}", flush=True)
    lens, new, H, KH, D, page = SHAPES[name]
    c = Cache(lens, page, KH, D, torch.float16, 311)
    for b, n in enumerate(lens):
        for j in range(n):
            c.k[int(c.table[b, j // page]), :, j % page] = 0.02 * j
    q = torch.ones(sum(new), H, D).half()
    compare(fa, c, q, cu_of(new), max_q=max(new))


@pytest.mark.parametrize("name", ["ragged-decode", "mixed", "split-decode"])
def test_pages_last_layout_and_strided_queries(fa, name):
    print(f"case strides {name}", flush=True)
    lens, new, H, KH, D, page = SHAPES[name]
    c = Cache(lens, page, KH, D, torch.bfloat16, 320, pages_first=False)
    T = sum(new)
    wide = torch.randn(T, 2 * H + 1, D + 8, generator=torch.Generator().manual_seed(7)).bfloat16()
    q = wide[:, 1: H + 1, :D]
    k, v, table = c.dev()
    qd = wide.to(DEV)[:, 1: H + 1, :D]
    out = torch.full((T, H + 2, 2 * D), 7.0, dtype=torch.bfloat16, device=DEV)
    o, lse = fa.paged_forward(qd, k, v, table, cu_of(new).to(DEV), c.lens.to(DEV),
                              out[:, 2:, D:], max_q=max(new), return_lse=True)
    assert o.data_ptr() == out[:, 2:, D:].data_ptr()
    want, want_l, tol, tol_l = R.attend(q, c.k, c.v, c.table, cu_of(new), c.lens, scale=D ** -0.5)
    R.check("o", o, want, tol)
    R.check("lse", lse, want_l, tol_l)
    assert bool((out[:, :2] == 7).all()) and bool((out[:, :, :D] == 7).all())


@pytest.mark.parametrize("bad", [-1, -2 ** 31, 2 ** 31 - 1, "pages"])
@pytest.mark.parametrize("name", ["ragged-decode", "mixed", "split-decode"])
def test_absent_pages(fa, name, bad):
    print(f"case absent {name} {bad}", flush=True)
    lens, new, H, KH, D, page = SHAPES[name]
    c = Cache(lens, page, KH, D, torch.float16, 330)
    bad = c.k.shape[0] if bad == "pages" else bad
    c.table[0, 0] = bad       # the first page of the first sequence
    c.table[0, -(-lens[0] // page) - 1] = bad  # its last
    if len(lens) > 1:
        c.table[1, : -(-lens[1] // page)] = bad  # all of the second: its rows see nothing
    q = torch.randn(sum(new), H, D, generator=torch.Generator().manual_seed(8)).half()
    compare(fa, c, q, cu_of(new), max_q=max(new))


def test_absent_pages_of_a_single_sequence(fa):
    c = Cache([333], 32, 2, 64, torch.float16, 331)
    c.table[0, 1::2] = -1
    q = torch.randn(1, 2, 64, generator=torch.Generator().manual_seed(8)).half()
    compare(fa, c, q, cu_of([1]), max_q=1)


@pytest.mark.parametrize("name", ["few-tokens", "chunks", "mixed"])
def test_limits_on_tokens_and_keys(fa, name):
    """max_q below a sequence's tokens: the ones past it are left alone; max_kv
    below a length: taken as the length."""
    print(f"case limits {name}", flush=True)
    lens, new, H, KH, D, page = SHAPES[name]
    c = Cache(lens, page, KH, D, torch.bfloat16, 340)
    q = torch.randn(sum(new), H, D, generator=torch.Generator().manual_seed(9)).bfloat16()
    k, v, table = c.dev()
    cu = cu_of(new)
    max_q, max_kv = max(new) // 2, max(lens) - 40
    out = torch.full_like(q, 5.0).to(DEV)
    o, lse = fa.paged_forward(q.to(DEV), k, v, table, cu.to(DEV), c.lens.to(DEV), out, max_q=max_q,
                              max_kv=max_kv, return_lse=True)
    want, want_l, tol, tol_l = R.attend(q, c.k, c.v, c.table, cu, c.lens, scale=D ** -0.5, max_q=max_q,
                                        max_kv=max_kv)
    rows = ~torch.isnan(want_l[:, 0])
    R.check("o", o.cpu()[rows], want[rows], tol[rows])
    R.check("lse", lse.cpu()[rows], want_l[rows], tol_l[rows])
    assert bool((out.cpu()[~rows] == 5).all()) and int((~rows).sum()) > 0


def test_rows_of_no_sequence_are_left_alone(fa):
    c = Cache([100, 30], 16, 2, 64, torch.float16, 350)
    q = torch.randn(60, 4, 64, generator=torch.Generator().manual_seed(10)).half()
    k, v, table = c.dev()
    cu = torch.tensor([3, 4, 45], dtype=torch.int32)
    out = torch.full_like(q, 5.0).to(DEV)
    o, lse = fa.paged_forward(q.to(DEV), k, v, table, cu.to(DEV), c.lens.to(DEV), out, max_q=41,
                              return_lse=True)
    want, want_l, tol, tol_l = R.attend(q, c.k, c.v, c.table, cu, c.lens, scale=0.125)
    rows = ~torch.isnan(want_l[:, 0])
    assert rows.tolist() == [3 <= i < 45 for i in range(60)]
    R.check("o", o.cpu()[rows], want[rows], tol[rows])
    R.check("lse", lse.cpu()[rows], want_l[rows], tol_l[rows])
    assert bool((out.cpu()[~rows] == 5).all())


@pytest.mark.parametrize("cu", [[0, 200, 100, 150], [-5, 3, 1000, 2000], [0, 0, 0, 0], [90, 60, 30, 0]])
def test_offsets_that_make_no_sense_stay_in_bounds(fa, cu):
    c = Cache([100, 30, 64], 16, 2, 64, torch.float16, 351)
    q = torch.randn(100, 4, 64).half().to(DEV)
    k, v, table = c.dev()
    lens = torch.tensor([2 ** 31 - 1, -7, 64], dtype=torch.int32, device=DEV)
    out = torch.zeros_like(q)
    fa.paged_forward(q, k, v, table, torch.tensor(cu, dtype=torch.int32, device=DEV), lens, out, max_q=50)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
def test_infinities_and_nan_behind_the_mask(fa, D, dtype):
    """Token i's row must not see what later tokens hold, infinities and NaN
    included, and must see what its own keys hold."""
    print(f"case non-finite {D} {dtype}", flush=True)
    dt = DT[dtype]
    n, H = 150, 2
    c = Cache([n], 16, 1, D, dt, 360)
    q = torch.randn(n, H, D, generator=torch.Generator().manual_seed(11)).to(dt)

    def put(cache, j, d, x):
        cache[int(c.table[0, j // 16]), 0, j % 16, d] = x

    put(c.v, 140, 3, math.inf)
    put(c.v, 141, 3, math.inf)
    put(c.v, 142, 5, -math.inf)
    put(c.v, 145, 5, math.inf)
    put(c.v, 146, D - 1, math.nan)
    put(c.k, 148, 0, math.nan)
    o, lse = run(fa, c, q, cu_of([n]), max_q=n)
    want, want_l, tol, tol_l = R.attend(q, c.k, c.v, c.table, cu_of([n]), c.lens, scale=D ** -0.5)
    # rows 140..147 see infinities in some dims only; 148 on, a NaN score
    R.check("o", o[:148], want[:148], tol[:148])
    R.check("lse", lse[:148], want_l[:148], tol_l[:148])
    assert bool(torch.isfinite(o[:140]).all()) and bool((o[141, :, 3] == math.inf).all())
    assert bool(torch.isnan(o[145:148, :, 5]).all()) and bool(torch.isnan(o[148:]).all())


def test_nan_query_stays_in_its_row(fa):
    for new in ([1, 1, 1], [70, 1, 40]):
        c = Cache([100, 60, 200], 16, 1, 64, torch.bfloat16, 361)
        T = sum(new)
        q = torch.randn(T, 2, 64, generator=torch.Generator().manual_seed(12)).bfloat16()
        q[T - 1, 1, 7] = math.nan
        o, lse = run(fa, c, q, cu_of(new), max_q=max(new))
        want, want_l, tol, tol_l = R.attend(q, c.k, c.v, c.table, cu_of(new), c.lens, scale=0.125)
        assert bool(torch.isnan(o[T - 1, 1]).all()) and bool(torch.isnan(lse[T - 1, 1]))
        tol[T - 1, 1] = tol_l[T - 1, 1] = 0
        R.check("o", o, want, tol)
        R.check("lse", lse, want_l, tol_l)


def test_offsets_past_32_bits(fa):
    """The sequences' pages lie past 4 GiB of each pool."""
    pages, page, D = 1_100_000, 16, 128
    k = torch.empty((pages, 1, page, D), dtype=torch.bfloat16, device=DEV)
    v = torch.empty((pages, 1, page, D), dtype=torch.bfloat16, device=DEV)
    c = Cache([200, 90], page, 1, D, torch.bfloat16, 370)
    at = pages - c.k.shape[0]
    k[at:], v[at:] = c.k.to(DEV), c.v.to(DEV)
    far = torch.where(c.table >= 0, c.table + at, c.table)
    new = [1, 70]
    q = torch.randn(sum(new), 2, D, generator=torch.Generator().manual_seed(13)).bfloat16()
    o, lse = fa.paged_forward(q.to(DEV), k, v, far.to(DEV), cu_of(new).to(DEV), c.lens.to(DEV),
                              max_q=70, return_lse=True)
    want, want_l, tol, tol_l = R.attend(q, c.k, c.v, c.table, cu_of(new), c.lens, scale=D ** -0.5)
    R.check("o", o, want, tol)
    R.check("lse", lse, want_l, tol_l)


@pytest.mark.parametrize("name", ["split-decode", "mixed", "chunks"])
def test_same_bits_twice_and_on_another_stream(fa, name):
    lens, new, H, KH, D, page = SHAPES[name]
    c = Cache(lens, page, KH, D, torch.float16, 380)
    q = torch.randn(sum(new), H, D, generator=torch.Generator().manual_seed(14)).half().to(DEV)
    k, v, table = c.dev()
    cu, ln = cu_of(new).to(DEV), c.lens.to(DEV)
    o, lse = fa.paged_forward(q, k, v, table, cu, ln, max_q=max(new), return_lse=True)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        o2, lse2 = fa.paged_forward(q, k, v, table, cu, ln, max_q=max(new), return_lse=True)
    s.synchronize()
    assert torch.equal(o, o2) and torch.equal(lse, lse2)


def test_two_graphs_replayed_with_other_lengths(fa):
    """Two captured graphs (split decode and chunks) replayed in turn, with
    lengths, tables and queries changed between the replays, against eager."""
    D, H, KH, page = 128, 4, 2, 16
    lens = [2500, 900]
    c = Cache(lens, page, KH, D, torch.float16, 390)
    k, v, table = c.dev()
    ln = c.lens.to(DEV)
    jobs = []
    for new in ([1, 1], [60, 40]):
        q = torch.zeros(sum(new), H, D, dtype=torch.float16, device=DEV)
        cu = cu_of(new).to(DEV)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            fa.paged_forward(q, k, v, table, cu, ln, max_q=max(new), return_lse=True)
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = fa.paged_forward(q, k, v, table, cu, ln, max_q=max(new), return_lse=True)
        jobs.append((g, q, cu, max(new), res))
    for step, (a, b) in enumerate([(2500, 900), (70, 100), (64, 0), (2100, 899)]):
        ln.copy_(torch.tensor([a, b], dtype=torch.int32))
        for g, q, cu, max_q, res in jobs:
            q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(step)).half())
            g.replay()
        for g, q, cu, max_q, res in jobs:
            o, lse = fa.paged_forward(q, k, v, table, cu, ln, max_q=max_q, return_lse=True)
            torch.cuda.synchronize()
            assert torch.equal(res[0], o) and torch.equal(res[1], lse), step


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_agrees_with_the_contiguous_forward(fa, dtype):
    """A prompt in pages against forward(causal=True) on the same tensors: both
    within their bounds of the 64-bit form."""
    n, H, D = 700, 4, 128
    c = Cache([n], 64, H, D, DT[dtype], 395)
    q = torch.randn(n, H, D, generator=torch.Generator().manual_seed(15)).to(DT[dtype])
    o, lse = run(fa, c, q, cu_of([n]), max_q=n)
    kk, _ = R.keys_of(c.k, c.table[0], n)
    vv, _ = R.keys_of(c.v, c.table[0], n)
    of, lf = fa.forward(q.transpose(0, 1)[None].to(DEV), kk[None].to(DEV), vv[None].to(DEV), causal=True,
                        return_lse=True)
    # each within P's and the output's rounding (3 u of values of at most 4.5)
    assert float((o.float() - of[0].transpose(0, 1).float()).abs().max()) <= 6 * R.U[DT[dtype]] * 4.5
    assert float((lse - lf[0].T).abs().max()) <= 1e-3


@pytest.mark.parametrize("KH,N", [(1, 9000), (2, 3000), (3, 2500), (4, 2100), (8, 1500), (16, 1300), (24, 1100),
                                  (32, 1500), (64, 1500), (100, 1200)])
def test_grid_orders_against_the_contiguous_forward(fa, KH, N):
    """Head counts that take each order of the grid (whole heads per XCD in
    groups, heads shared by XCDs, all interleaved), with whole rounds and a last
    round in pieces, against forward(causal=True): every row written, each within
    its rounding (3 u of values of at most 5.5)."""
    print(f"case grid order KH {KH} N {N}", flush=True)
    D, page = 64, 64
    g = torch.Generator(device=DEV).manual_seed(KH)
    q, k, v = (torch.randn(1, KH, N, D, generator=g, device=DEV).half() for _ in range(3))
    n = -(-N // page)
    kc, vc = (torch.zeros(n, KH, page, D, dtype=torch.float16, device=DEV) for _ in range(2))
    for cache, x in ((kc, k), (vc, v)):
        pad = torch.zeros(KH, n * page, D, dtype=torch.float16, device=DEV)
        pad[:, :N] = x[0]
        cache.copy_(pad.view(KH, n, page, D).transpose(0, 1))
    table = torch.arange(n, dtype=torch.int32, device=DEV)[None]
    out = torch.full((N, KH, D), math.nan, dtype=torch.float16, device=DEV)
    o, lse = fa.paged_forward(q[0].transpose(0, 1), kc, vc, table,
                              torch.tensor([0, N], dtype=torch.int32, device=DEV),
                              torch.tensor([N], dtype=torch.int32, device=DEV), out, max_q=N, return_lse=True)
    of, lf = fa.forward(q, k, v, causal=True, return_lse=True)
    assert float((o.float() - of[0].transpose(0, 1).float()).abs().max()) <= 6 * 2.0 ** -11 * 5.5
    assert float((lse - lf[0].T).abs().max()) <= 1e-3


@pytest.mark.parametrize("name", ["ragged-decode", "chunks"])
def test_no_keys_allowed(fa, name):
    """max_kv = 0: every row is empty."""
    lens, new, H, KH, D, page = SHAPES[name]
    c = Cache(lens, page, KH, D, torch.float16, 397)
    q = torch.ones(sum(new), H, D).half()
    o, lse = run(fa, c, q, cu_of(new), max_q=max(new), max_kv=0)
    assert not o.any() and bool((lse == -math.inf).all())


@pytest.mark.parametrize("scale", [1.2e-38, 1e-20, 100.0])
@pytest.mark.parametrize("name", ["ragged-decode", "chunks"])
def test_extreme_scales(fa, name, scale):
    lens, new, H, KH, D, page = SHAPES[name]
    c = Cache(lens, page, KH, D, torch.bfloat16, 398)
    q = torch.randn(sum(new), H, D, generator=torch.Generator().manual_seed(16)).bfloat16()
    compare(fa, c, q, cu_of(new), max_q=max(new), scale=scale)


def test_empty_calls(fa):
    c = Cache([20], 16, 1, 64, torch.float16, 396)
    k, v, table = c.dev()
    q = torch.zeros(0, 2, 64, dtype=torch.float16, device=DEV)
    o, lse = fa.paged_forward(q, k, v, table, torch.zeros(2, dtype=torch.int32, device=DEV),
                              c.lens.to(DEV), max_q=0, return_lse=True)
    assert o.shape == (0, 2, 64) and lse.shape == (0, 2)
    q = torch.ones(3, 2, 64, dtype=torch.float16, device=DEV)
    out = torch.full_like(q, 3.0)
    fa.paged_forward(q, k, v, table[:0], torch.zeros(1, dtype=torch.int32, device=DEV),
                     c.lens.to(DEV)[:0], out, max_q=3)
    assert bool((out == 3).all())
