"""The LDS-poison debug build (libfa_mi355x_poison.so) of the paged cache's
kernels: LDS is filled with NaN before every staging write, so a read ahead of
its wait or barrier shows; with correct synchronisation the results are the
product build's bit for bit."""
from __future__ import annotations

import ctypes
import math
import os

import pytest
import torch

import abi_ctypes as A
import cache_ctypes as C

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def libs():
    if not os.path.exists(A.POISON_LIB_PATH):
        pytest.fail("libfa_mi355x_poison.so is missing: run build() first")
    return C.load(A.LIB_PATH), C.load(A.POISON_LIB_PATH)


def call(L, name, p):
    ws_bytes, ws = ctypes.c_uint64(0), None
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert getattr(L, name + "_workspace_size")(ctypes.byref(p), ctypes.byref(ws_bytes)) == A.FA_OK
    ws = torch.empty(max(16, ws_bytes.value), dtype=torch.uint8, device=DEV)
    rc = getattr(L, name)(ctypes.byref(p), ctypes.c_void_p(ws.data_ptr()), ws_bytes.value, stream)
    assert rc == A.FA_OK, L.fa_last_error()
    torch.cuda.synchronize()


CASES = [
    # lens, new, H, KH, D, page, dtype
    ([300, 1, 1024, 33, 0], [1] * 5, 8, 2, 64, 64, torch.float16),
    ([5000, 700], [1, 1], 8, 2, 128, 16, torch.bfloat16),
    ([900, 77], [5, 7], 16, 4, 128, 32, torch.float16),
    ([1700, 400, 64], [300, 1, 64], 4, 2, 128, 16, torch.bfloat16),
    ([1500], [1500], 2, 1, 64, 256, torch.float16),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"L{max(c[0])}-n{max(c[1])}-D{c[4]}")
def test_poison_build_keeps_every_bit(libs, case):
    lens, new, H, KH, D, page, dt = case
    print("case poison", case, flush=True)
    g = torch.Generator(device=DEV).manual_seed(3)
    counts = [-(-n // page) for n in lens]
    pool = sum(counts) + 1
    k, v = (torch.randn(pool, KH, page, D, generator=g, device=DEV).to(dt) for _ in range(2))
    ids = (torch.randperm(pool - 1, generator=g, device=DEV) + 1).int()
    table = torch.zeros(len(lens), max(counts), dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = ids[at:at + n]
        at += n
    T = sum(new)
    cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=DEV)
    ln = torch.tensor(lens, dtype=torch.int32, device=DEV)
    q = (3 * torch.randn(T, H, D, generator=g, device=DEV)).to(dt)
    got = []
    for L in libs:
        c = C.PagedCache()
        c.k, c.v = k.data_ptr(), v.data_ptr()
        for i in range(3):
            c.k_stride[i], c.v_stride[i] = k.stride(i), v.stride(i)
        c.block_table, c.table_stride = table.data_ptr(), table.stride(0)
        c.cu_seqlens, c.seq_lens = cu.data_ptr(), ln.data_ptr()
        c.batch, c.num_pages, c.page_size, c.max_pages = len(lens), pool, page, table.shape[1]
        c.kv_heads, c.head_dim, c.dtype = KH, D, int(dt == torch.bfloat16)
        o = torch.full_like(q, math.nan)
        lse = torch.full((T, H), math.nan, device=DEV)
        p = C.PagedFwd()
        p.cache, p.q, p.o, p.lse = c, q.data_ptr(), o.data_ptr(), lse.data_ptr()
        w = torch.zeros(pool, KH, page, device=DEV)
        x = C.PagedWeights()
        x.cache, x.q, x.lse, x.key_weights = c, q.data_ptr(), lse.data_ptr(), w.data_ptr()
        for s in (p, x):
            s.q_stride[0], s.q_stride[1] = q.stride(0), q.stride(1)
            s.tokens, s.heads, s.max_q, s.max_kv = T, H, max(new), max(lens)
            s.softmax_scale, s.causal = D ** -0.5, 1
        p.o_stride[0], p.o_stride[1] = o.stride(0), o.stride(1)
        x.w_stride[0], x.w_stride[1] = w.stride(0), w.stride(1)
        call(L, "fa_paged_fwd", p)
        call(L, "fa_paged_key_weights", x)
        got.append((o, lse, w))
    for a, b in zip(*got):
        assert torch.equal(a, b) and not torch.isnan(a).any()
