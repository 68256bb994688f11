"""The LDS-poison debug build of the kernels of attention with gradients and of scored attention over the
cache: LDS is filled with NaN before every staging write, so a read ahead of its wait or barrier shows; with
correct synchronisation the results are the product build's bit for bit."""
from __future__ import annotations

import ctypes
import math
import os

import pytest
import torch

import abi_ctypes as A
import attention_ctypes as T

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def libs():
    if not os.path.exists(A.POISON_LIB_PATH):
        pytest.fail("libfa_mi355x_poison.so is missing: run build() first")
    return T.load(A.LIB_PATH), T.load(A.POISON_LIB_PATH)


def call(L, name, *structs):
    refs = [ctypes.byref(s) for s in structs]
    stream, workspace = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream), ()
    if T.ENTRIES[name][1]:
        n = ctypes.c_uint64(0)
        assert getattr(L, name + "_workspace_size")(*refs, ctypes.byref(n)) == A.FA_OK, L.fa_last_error()
        ws = torch.empty(max(16, n.value), dtype=torch.uint8, device=DEV)
        workspace = (ctypes.c_void_p(ws.data_ptr()), n.value)
    assert getattr(L, name)(*refs, *workspace, stream) == A.FA_OK, L.fa_last_error()
    torch.cuda.synchronize()


def strides(field, x):
    for i in range(len(field)):
        field[i] = x.stride(i)


# B, H, KH, N, M, D, type, causal, softcap, window, slopes, ranges: of few workgroups and of many, with each mask
CASES = [
    (1, 4, 2, 700, 700, 128, "bf16", 0, 0.0, 0, False, False),
    (1, 4, 2, 700, 700, 64, "fp16", 1, 0.0, 0, True, False),
    (2, 2, 2, 300, 420, 128, "fp16", 1, 30.0, 0, False, False),
    (1, 8, 2, 900, 900, 64, "bf16", 1, 20.0, 100, True, False),
    (2, 3, 1, 500, 500, 128, "bf16", 0, 0.0, 0, False, True),
    (3, 100, 100, 300, 300, 128, "fp16", 0, 0.0, 0, False, False),
    (3, 100, 100, 300, 300, 64, "bf16", 0, 0.0, 0, False, False),
    (3, 120, 120, 260, 260, 128, "bf16", 1, 40.0, 0, False, False),
    (3, 120, 120, 260, 260, 64, "fp16", 0, 0.0, 0, False, True),
    (1, 2, 1, 3000, 70, 64, "bf16", 0, 0.0, 0, False, False),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_attention_keeps_every_bit(libs, case):
    B, H, KH, N, M, D, dtype, causal, cap, window, biased, ranged = case
    print("case poison", case, flush=True)
    dt = {"fp16": torch.float16, "bf16": torch.bfloat16}[dtype]
    g = torch.Generator(device=DEV).manual_seed(21)
    q, go = (torch.randn(B, H, N, D, generator=g, device=DEV).to(dt) for _ in range(2))
    k, v = (torch.randn(B, KH, M, D, generator=g, device=DEV).to(dt) for _ in range(2))
    slopes = torch.rand(H, generator=g, device=DEV) * 0.1
    at = torch.arange(N, device=DEV)
    ranges = torch.stack((at // 97 * 97, at + 1), -1).clamp(max=M).int().contiguous()
    got = []
    for L in libs:
        o, low, gq = (torch.full_like(q, math.nan) for _ in range(3))
        gk, gv = (torch.full_like(k, math.nan) for _ in range(2))
        lse = torch.full((B, H, N), math.nan, device=DEV)
        p = T.Attn()
        for name, x in (("q", q), ("k", k), ("v", v), ("o", o)):
            setattr(p, name, x.data_ptr())
            strides(getattr(p, name + "_stride"), x)
        p.lse, p.o_low, p.ranges = lse.data_ptr(), low.data_ptr(), ranges.data_ptr() if ranged else None
        p.batch, p.heads, p.kv_heads, p.seq_len, p.keys, p.head_dim = B, H, KH, N, M, D
        p.dtype, p.causal, p.softmax_scale = int(dt == torch.bfloat16), causal, D ** -0.5
        p.score.softcap, p.score.window, p.score.slopes = cap, window, slopes.data_ptr() if biased else None
        x = T.AttnBwd()
        x.fwd, x.go = p, go.data_ptr()
        strides(x.go_stride, go)
        for name, y in (("gq", gq), ("gk", gk), ("gv", gv)):
            setattr(x, name, y.data_ptr())
            strides(getattr(x, name + "_stride"), y)
        call(L, "fa_attn_fwd", p)
        call(L, "fa_attn_bwd", x)
        got.append((o, low, lse, gq, gk, gv))
    for a, b in zip(*got):
        assert torch.equal(a, b) and not torch.isnan(a).any()


# lengths, new tokens, H, KH, D, page, type, softcap, window, slopes
PAGED = [
    ([300, 1, 1024, 33], [1] * 4, 8, 2, 64, 64, "fp16", 30.0, 0, False),
    ([5000, 700], [1, 1], 8, 2, 128, 16, "bf16", 0.0, 600, True),
    ([900, 77], [5, 7], 16, 4, 128, 32, "fp16", 20.0, 40, True),
    ([1700, 400, 64], [300, 1, 64], 4, 2, 128, 16, "bf16", 50.0, 500, False),
    ([1500], [1500], 2, 1, 64, 256, "fp16", 0.0, 0, True),
]


@pytest.mark.parametrize("case", PAGED, ids=lambda c: f"L{max(c[0])}-n{max(c[1])}-D{c[4]}")
def test_scored_paged_attention_keeps_every_bit(libs, case):
    lens, new, H, KH, D, page, dtype, cap, window, biased = case
    print("case poison", case, flush=True)
    dt = {"fp16": torch.float16, "bf16": torch.bfloat16}[dtype]
    g = torch.Generator(device=DEV).manual_seed(22)
    counts = [-(-n // page) for n in lens]
    pool = sum(counts) + 1
    k, v = (torch.randn(pool, KH, page, D, generator=g, device=DEV).to(dt) for _ in range(2))
    ids = (torch.randperm(pool - 1, generator=g, device=DEV) + 1).int()
    table = torch.zeros(len(lens), max(counts), dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = ids[at:at + n]
        at += n
    tokens = sum(new)
    cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=DEV)
    ln = torch.tensor(lens, dtype=torch.int32, device=DEV)
    q = (3 * torch.randn(tokens, H, D, generator=g, device=DEV)).to(dt)
    slopes = torch.rand(H, generator=g, device=DEV) * 0.1
    got = []
    for L in libs:
        o = torch.full_like(q, math.nan)
        lse = torch.full((tokens, H), math.nan, device=DEV)
        p = T.C.PagedFwd()
        c = p.cache
        c.k, c.v = k.data_ptr(), v.data_ptr()
        strides(c.k_stride, k)
        strides(c.v_stride, v)
        c.block_table, c.table_stride = table.data_ptr(), table.stride(0)
        c.cu_seqlens, c.seq_lens = cu.data_ptr(), ln.data_ptr()
        c.batch, c.num_pages, c.page_size, c.max_pages = len(lens), pool, page, table.shape[1]
        c.kv_heads, c.head_dim, c.dtype = KH, D, int(dt == torch.bfloat16)
        p.q, p.o, p.lse = q.data_ptr(), o.data_ptr(), lse.data_ptr()
        strides(p.q_stride, q)
        strides(p.o_stride, o)
        p.tokens, p.heads, p.max_q, p.max_kv = tokens, H, max(new), max(lens)
        p.softmax_scale, p.causal = D ** -0.5, 1
        call(L, "fa_paged_fwd_scored", p, T.Score(softcap=cap, window=window, slopes=slopes.data_ptr() if biased else None))
        got.append((o, lse))
    for a, b in zip(*got):
        assert torch.equal(a, b) and not torch.isnan(a).any()
