"""The paged cache's calls at the edges of what their documents allow: tables,
offsets and lengths that make no sense, limits, head counts."""
from __future__ import annotations

import ctypes

import pytest
import torch

import abi_ctypes as A
import cache_ctypes as C
import cache_reference as R
from test_gpu_paged_cache import evict_compare, evict_setup
from test_gpu_paged_forward import Cache, compare, cu_of
from test_gpu_qk_norm import tables

pytestmark = pytest.mark.gpu
DEV = "cuda"


def cache_of(k, v, table, cu, lens):
    c = C.PagedCache()
    c.k, c.v = k.data_ptr(), v.data_ptr()
    for i in range(3):
        c.k_stride[i], c.v_stride[i] = k.stride(i), v.stride(i)
    c.block_table, c.table_stride = table.data_ptr(), table.stride(0)
    c.cu_seqlens, c.seq_lens = None if cu is None else cu.data_ptr(), lens.data_ptr()
    c.batch, c.max_pages = table.shape
    c.num_pages, c.kv_heads, c.page_size, c.head_dim = k.shape
    c.dtype = int(k.dtype == torch.bfloat16)
    return c


@pytest.mark.parametrize("cu", [[0, 64, 0, 64], [64, 0, 64, 0], [0, 64, 0, 64, 0, 64, 0, 64]])
def test_nothing_behind_the_workspace_is_written(cu):
    """Descending offsets put two sequences on the same rows, more row tiles than
    the launch counts on, each long enough to be cut in 64 pieces of keys."""
    print("case workspace", cu, flush=True)
    H, D, page, n, T, B = 8, 64, 64, 40000, 64, len(cu) - 1
    pages = n // page
    g = torch.Generator(device=DEV).manual_seed(1)
    k, v = (torch.randn(pages, 1, page, D, generator=g, device=DEV).half() for _ in range(2))
    q = torch.randn(T, H, D, generator=g, device=DEV).half()
    table = torch.arange(pages, dtype=torch.int32, device=DEV).expand(B, -1).contiguous()
    offsets = torch.tensor(cu, dtype=torch.int32, device=DEV)
    lens = torch.full((B,), n, dtype=torch.int32, device=DEV)
    o = torch.zeros_like(q)
    L = C.load()
    p = C.PagedFwd()
    p.cache, p.q, p.o = cache_of(k, v, table, offsets, lens), q.data_ptr(), o.data_ptr()
    p.q_stride[0], p.q_stride[1] = p.o_stride[0], p.o_stride[1] = q.stride(0), q.stride(1)
    p.tokens, p.heads, p.max_q, p.max_kv, p.softmax_scale, p.causal = T, H, T, n, D ** -0.5, 1
    need = ctypes.c_uint64(0)
    assert L.fa_paged_fwd_workspace_size(ctypes.byref(p), ctypes.byref(need)) == A.FA_OK and need.value > 0
    behind = 64 << 20  # more than all pieces of all tiles would take
    ws = torch.full((need.value + behind,), 0x5A, dtype=torch.uint8, device=DEV)
    rc = L.fa_paged_fwd(ctypes.byref(p), ctypes.c_void_p(ws.data_ptr()), need.value,
                        ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == A.FA_OK, L.fa_last_error()
    torch.cuda.synchronize()
    assert bool((ws[need.value:] == 0x5A).all())


def store_and_compare(fa, c, lens, cu, T):
    """paged_store of T tokens against the 64-bit form, whose lengths are limited to
    the table and whose offsets to the rows, as in every other call."""
    H, KH, D, page = 2, c.k.shape[1], c.k.shape[3], c.page
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(T, h, D, generator=g).to(c.k.dtype) for h in (H, KH, KH))
    w = 1 + 0.2 * torch.randn(D, generator=g)
    cos, sin = tables(100, D)
    pos = torch.randint(0, 100, (T,), generator=g, dtype=torch.int32)
    kc, vc, table = c.dev()
    out = torch.full((T, H, D), 9.0, dtype=q.dtype, device=DEV)
    fa.paged_store(q.to(DEV), k.to(DEV), v.to(DEV), w.to(DEV), w.to(DEV), cos.to(DEV), sin.to(DEV),
                   pos.to(DEV), kc, vc, table, torch.tensor(cu, dtype=torch.int32, device=DEV),
                   torch.tensor(lens, dtype=torch.int32, device=DEV), out)
    wq, tq = R.norm_rope(q, w, cos, sin, pos[:, None].expand(T, H), eps=1e-6, interleaved=False)
    wk, tk = R.norm_rope(k, w, cos, sin, pos[:, None].expand(T, KH), eps=1e-6, interleaved=False)
    want_k, want_v, tol = c.k.double(), c.v.double(), torch.zeros(c.k.shape, dtype=torch.float64)
    rows = torch.zeros(T, dtype=torch.bool)
    for b, c0, nq, n, first in R.sequences(cu, lens, T, capacity=c.table.shape[1] * page):
        rows[c0:c0 + nq] = True
        for i in range(max(0, -first), nq):
            at = (int(c.table[b, (first + i) // page]), slice(None), (first + i) % page)
            want_k[at], tol[at], want_v[at] = wk[c0 + i], tk[c0 + i], v[c0 + i].double()
    R.check("q", out[rows.to(DEV)], wq[rows], tq[rows])
    assert bool((out.cpu()[~rows] == 9).all())
    R.check("k_cache", kc, want_k, tol)
    R.check("v_cache", vc, want_v, torch.zeros_like(tol))


@pytest.mark.parametrize("name,lens,cu", [
    ("length above the table", [70, 40], [0, 10, 15]),
    ("far above it", [2 ** 31 - 1, 64], [0, 10, 15]),
    ("more tokens than the table has keys", [200, 40], [0, 100, 110]),
    ("no keys", [-5, 0], [0, 10, 15]),
    ("last offset above the rows", [64, 40], [0, 10, 40]),
    ("every offset above the rows", [64, 40], [50, 60, 70]),
    ("offsets to both sides of the rows", [64, 40], [-7, 3, 2 ** 31 - 1]),
    ("rows before the first and behind the last", [64, 40], [2, 9, 11]),
])
def test_store_limits_lengths_and_offsets_as_the_other_calls(fa, name, lens, cu):
    print("case store limits", name, flush=True)
    c = Cache([64, 64], 16, 2, 64, torch.bfloat16, 700)
    store_and_compare(fa, c, lens, cu, 110 if cu[-1] == 110 else 15)


def test_store_then_forward_agree_on_a_length_above_the_table(fa):
    """Each token's own key is where its query looks for it: with values that name
    the token and a score that only its own key reaches, every row gets its token."""
    D, T, n = 64, 10, 64
    c = Cache([n], 16, 1, D, torch.float16, 701)
    kc, vc, table = c.dev()
    kc.zero_(), vc.zero_()
    # q and k of token i along axis i: a score of D against 0 for every other key
    q = torch.zeros(T, 1, D, device=DEV).half()
    q[torch.arange(T), 0, torch.arange(T)] = 1.0
    v = torch.arange(1, T + 1, device=DEV).half()[:, None, None].expand(T, 1, D).contiguous()
    w = torch.ones(D, device=DEV)
    cos, sin = torch.ones(1, D // 2, device=DEV), torch.zeros(1, D // 2, device=DEV)
    cu = torch.tensor([0, T], dtype=torch.int32, device=DEV)
    ln = torch.tensor([n + 6], dtype=torch.int32, device=DEV)
    pos = torch.zeros(T, dtype=torch.int32, device=DEV)
    qn = fa.paged_store(q, q, v, w, w, cos, sin, pos, kc, vc, table, cu, ln)
    o = fa.paged_forward(qn, kc, vc, table, cu, ln, max_q=T, softmax_scale=1.0)
    # weight of each other key: exp(-64), so that the row is its own value but for fp16's steps
    assert float((o[:, 0, 0].float() - torch.arange(1, T + 1, device=DEV)).abs().max()) <= T * 2.0 ** -10


def test_evict_may_update_the_lengths_in_place():
    """new_lens is seq_lens: no head may see the new length in place of the old one.
    Thousands of heads with the same keys and weights, beside a large product on
    another stream, so that many of them start after others have ended."""
    print("case evict in place", flush=True)
    kh, keep, recent, page, D, lens = 8192, 64, 8, 16, 64, [600, 500]
    c, new_table, w = evict_setup(lens, page, 1, D, torch.float16, keep, 710)
    want = R.evict(c.k, c.v, w, c.table, c.lens, new_table, keep=keep, recent=recent)
    table, nt = c.table.to(DEV), new_table.to(DEV)
    start = [t.to(DEV).expand(-1, kh, *t.shape[2:]) for t in (c.k, c.v, w)]
    k, v, wd = (t.contiguous() for t in start)
    big, side = torch.randn(8192, 8192, device=DEV).half(), torch.cuda.Stream()
    L = C.load()
    for trial in range(3):
        for t, x in zip((k, v, wd), start):
            t.copy_(x)
        ln = c.lens.to(DEV)
        kept = torch.full((2, kh, keep), -7, dtype=torch.int32, device=DEV)
        p = C.PagedEvict()
        p.cache = cache_of(k, v, table, None, ln)
        p.key_weights, p.w_stride[0], p.w_stride[1] = wd.data_ptr(), wd.stride(0), wd.stride(1)
        p.new_table, p.new_table_stride, p.new_pages = nt.data_ptr(), nt.stride(0), nt.shape[1]
        p.new_lens, p.kept, p.keep, p.recent, p.max_kv = ln.data_ptr(), kept.data_ptr(), keep, recent, max(lens)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.mm(big, big)
        rc = L.fa_paged_evict(ctypes.byref(p), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        assert rc == A.FA_OK, L.fa_last_error()
        torch.cuda.synchronize()
        assert torch.equal(ln.cpu(), want[0])
        assert bool((kept == want[1].to(DEV)).all()), trial  # (of one head: the same for all)
        for got, ref in ((k, want[2]), (v, want[3]), (wd, want[4])):
            kind = torch.int16 if got.dtype == torch.float16 else torch.int32
            assert bool((got.view(kind) == ref.to(DEV).view(kind)).all()), trial


@pytest.mark.parametrize("keep", [1, 16, 17, 5000])
def test_evict_lengths_at_the_edges_of_what_is_kept(fa, keep):
    """Lengths of zero, below, at and above keep; an absent page; a table of no keys."""
    lens = [0, 1, keep - 1, keep, keep + 1, 3 * keep, 40]
    c, new_table, w = evict_setup(lens, 16, 2, 64, torch.float16, keep, 711)
    c.table[6, 0] = -1
    evict_compare(fa, c, new_table, w, keep=keep, recent=min(keep, 3))
    evict_compare(fa, c, new_table, w, keep=keep, recent=0, max_kv=0)


@pytest.mark.parametrize("new", [[40, 3, 1, 0, 1, 2, 1, 1, 33], [35, 1]])
def test_more_kv_heads_than_compute_units(fa, new):
    """One workgroup of a kv head at a time: no rounds to cut, no join."""
    print("case many heads", new, flush=True)
    KH = torch.cuda.get_device_properties(0).multi_processor_count + 1
    lens = [n + 5 * i for i, n in enumerate(new)]
    c = Cache(lens, 16, KH, 64, torch.bfloat16, 720, wide=100)
    q = torch.randn(sum(new), KH, 64, generator=torch.Generator().manual_seed(5)).bfloat16()
    compare(fa, c, q, cu_of(new), max_q=max(new))


# cu, T: offsets past the rows, before them, and descending ones that leave no row
# to two sequences
SENSELESS = [([0, 200, 100, 150], 100), ([-5, 3, 1000, 2000], 100), ([0, 0, 0, 0], 100), ([90, 60, 30, 0], 100),
             ([40, 70, 2 ** 31 - 1, -2 ** 31], 100)]


@pytest.mark.parametrize("more", [0, 70])
@pytest.mark.parametrize("max_q", [50, 7])
@pytest.mark.parametrize("cu,T", SENSELESS)
def test_offsets_and_lengths_that_make_no_sense(fa, cu, T, max_q, more):
    """Each call against its 64-bit form under the same limits, rows and weights of
    no sequence untouched: decode and chunk kernels, lists of up to 64 sequences and
    of more (sequences without rows behind the others)."""
    print("case senseless", cu, max_q, more, flush=True)
    H, KH, D, page = 4, 2, 64, 16
    c = Cache([100, 30, 64], page, KH, D, torch.float16, 730)
    lens = torch.tensor([2 ** 31 - 1, -7, 64] + [20] * more, dtype=torch.int32)
    cu = torch.tensor(cu + [cu[-1]] * more, dtype=torch.int32)
    c.table = torch.cat([c.table, torch.full((more, c.table.shape[1]), -1, dtype=torch.int32)])
    g = torch.Generator().manual_seed(6)
    q = torch.randn(T, H, D, generator=g).half()
    k, v, table = c.dev()
    out = torch.full_like(q, 5.0).to(DEV)
    o, lse = fa.paged_forward(q.to(DEV), k, v, table, cu.to(DEV), lens.to(DEV), out, max_q=max_q, return_lse=True)
    want, want_l, tol, tol_l = R.attend(q, c.k, c.v, c.table, cu, lens, scale=D ** -0.5, max_q=max_q)
    # (the first sequence's length is the table's 112 keys: its rows see the NaN of keys 100 on)
    rows = torch.zeros(T, dtype=torch.bool)
    for _, c0, nq, _, _ in R.sequences(cu, lens, T, max_q):
        rows[c0:c0 + nq] = True
    R.check("o", o.cpu()[rows], want[rows], tol[rows])
    R.check("lse", lse.cpu()[rows], want_l[rows], tol_l[rows])
    assert bool((out.cpu()[~rows] == 5).all())
    w = torch.rand(c.k.shape[:3], generator=g)
    # (rows of no sequence: a logsumexp that would show)
    given = torch.where(rows[:, None], want_l.float(), torch.tensor(-20.0))
    wd = fa.paged_key_weights(q.to(DEV), given.to(DEV), k, table, cu.to(DEV), lens.to(DEV), w.to(DEV), max_q=max_q)
    want_w, tol_w = R.key_weights(q, given, c.k, c.table, cu, lens, w, scale=D ** -0.5, max_q=max_q)
    R.check("weights", wd, want_w, tol_w)
