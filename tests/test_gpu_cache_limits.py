"""The paged cache's calls at the edges of what their documents allow: tables,
offsets and lengths that make no sense, limits, head counts."""
from __future__ import annotations

import ctypes

import pytest
import torch

import abi_ctypes as A
import cache_ctypes as C

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
