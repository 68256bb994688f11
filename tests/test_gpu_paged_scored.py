"""paged_forward with capped and biased scores and windows, against the 64-bit forms; a server of such a model
against attention on its whole sequences."""
from __future__ import annotations

import math

import pytest
import torch

import attention_reference as A
import cache_reference as R
from test_gpu_paged_forward import DT, SHAPES, Cache, cu_of

pytestmark = pytest.mark.gpu
DEV = "cuda"

OPTIONS = {
    "cap": dict(softcap=3.0),
    "slopes": dict(slopes=0.02),
    "window": dict(window=40),
    "window-one": dict(window=1),
    "all": dict(softcap=5.0, slopes=0.01, window=100),
}
SOME = ["one-key", "one-token-page-edges", "ragged-decode", "empty-sequences", "more-tokens-than-keys", "odd-group-3",
        "group-17-two-blocks", "few-tokens", "chunks", "chunks-d64", "prefill", "mixed", "many-sequences",
        "last-round-of-one-head", "mixed-long", "split-decode", "split-chunk"]


def reference(q, c, cu, *, causal=True, slopes=None, softcap=None, window=None, max_q=None, max_kv=None):
    T, H, D = q.shape
    val = {"o": torch.full((T, H, D), math.nan, dtype=torch.float64), "lse": torch.full((T, H), math.nan, dtype=torch.float64)}
    tol = {n: torch.zeros_like(x) for n, x in val.items()}
    for b, c0, nq, n, first in R.sequences(cu, c.lens, T, max_q, max_kv, c.table.shape[1] * c.page):
        if nq == 0:
            continue
        new = n - first
        rows = slice(c0, c0 + nq)
        if n == 0:
            val["o"][rows], val["lse"][rows] = 0.0, -math.inf
            continue
        k, there = R.keys_of(c.k, c.table[b], n)
        v, _ = R.keys_of(c.v, c.table[b], n)
        see = A.visible(new, n, None, causal, window)[:, :nq] & there
        # (a masked key's row may hold anything)
        k, v = (torch.where(there[:, None], x, 0.0) for x in (k, v))
        pad = torch.zeros(new, H, D, dtype=q.dtype)
        pad[:nq] = q[rows]
        full = torch.zeros(1, new, n, dtype=torch.bool)
        full[:, :nq] = see
        a, t = A.attend(pad.transpose(0, 1)[None], k[None], v[None], full, scale=1 / math.sqrt(D), cap=softcap, slopes=slopes)
        val["o"][rows], val["lse"][rows] = a["o"][0].transpose(0, 1)[:nq], a["lse"][0].T[:nq]
        tol["o"][rows], tol["lse"][rows] = t["o"][0].transpose(0, 1)[:nq], t["lse"][0].T[:nq]
    return val, tol


def run(fa, c, q, cu, *, max_q, max_kv=None, causal=True, slopes=None, **opt):
    k, v, table = c.dev()
    slopes_dev = None if slopes is None else slopes.to(DEV)
    o, lse = fa.paged_forward(q.to(DEV), k, v, table, cu.to(DEV), c.lens.to(DEV), max_q=max_q, max_kv=max_kv,
                              causal=causal, return_lse=True, slopes=slopes_dev, **opt)
    val, tol = reference(q, c, cu, causal=causal, slopes=slopes, max_q=max_q, max_kv=max_kv, **opt)
    rows = ~torch.isnan(val["lse"][:, 0])
    R.check("o", o.cpu()[rows], val["o"][rows], tol["o"][rows])
    R.check("lse", lse.cpu()[rows], val["lse"][rows], tol["lse"][rows])
    return o, lse


def setup(name, dtype, seed):
    lens, new, H, KH, D, page = SHAPES[name]
    c = Cache(lens, page, KH, D, DT[dtype], seed, wide=1)
    q = (2 * torch.randn(sum(new), H, D, generator=torch.Generator().manual_seed(seed))).to(DT[dtype])
    return c, q, cu_of(new), max(new)


@pytest.mark.parametrize("option", list(OPTIONS))
@pytest.mark.parametrize("name", SOME)
def test_against_64_bits(fa, name, option):
    dtype = "fp16" if (SOME.index(name) + list(OPTIONS).index(option)) % 2 else "bf16"
    print(f"case {name} {option} {dtype}", flush=True)
    c, q, cu, max_q = setup(name, dtype, 700 + SOME.index(name))
    opt = dict(OPTIONS[option])
    if "slopes" in opt:
        opt["slopes"] = opt["slopes"] * torch.arange(1, q.shape[1] + 1).float()
    run(fa, c, q, cu, max_q=max_q, **opt)


@pytest.mark.parametrize("name", ["ragged-decode", "chunks", "mixed", "more-tokens-than-keys"])
@pytest.mark.parametrize("option", ["all", "window"])
def test_without_causal_mask(fa, name, option):
    print(f"case not causal {name} {option}", flush=True)
    c, q, cu, max_q = setup(name, "bf16", 760)
    opt = dict(OPTIONS[option])
    if "slopes" in opt:
        opt["slopes"] = opt["slopes"] * torch.arange(1, q.shape[1] + 1).float()
    run(fa, c, q, cu, max_q=max_q, causal=False, **opt)


@pytest.mark.parametrize("window", [1, 16, 63, 64, 65, 127, 500, 4999, 5000, 2 ** 31 - 1, 2 ** 40])
def test_windows_of_a_split_decode(fa, window):
    print("case window", window, flush=True)
    c = Cache([5000, 40, 3000], 16, 2, 64, torch.float16, 780)
    q = torch.randn(3, 4, 64, generator=torch.Generator().manual_seed(1)).half()
    run(fa, c, q, cu_of([1, 1, 1]), max_q=1, window=window)


def test_keys_before_the_window_and_absent_pages_may_hold_anything(fa):
    """NaN before the window, in pages that are gone from the table or still listed, in K and V."""
    for D, new, window in ((64, 1, 100), (128, 40, 50), (128, 3, 17)):
        print("case behind the window", D, new, window, flush=True)
        c = Cache([700], 16, 2, D, torch.bfloat16, 790)
        q = torch.randn(new, 4, D, generator=torch.Generator().manual_seed(2)).bfloat16()
        first = 700 - new - window + 1  # the first key that any token sees
        for key in range(first):
            c.k[c.table[0, key // 16], :, key % 16] = math.nan
            c.v[c.table[0, key // 16], :, key % 16] = math.inf
        c.table[0, : (first // 16) // 2] = -1
        clean = Cache([700], 16, 2, D, torch.bfloat16, 790)
        kv = [x.clone() for x in (c.k, c.v)]
        c.k, c.v = clean.k, clean.v
        val, tol = reference(q, c, cu_of([new]), window=window)
        c.k, c.v = kv
        k, v, table = c.dev()
        o = fa.paged_forward(q.to(DEV), k, v, table, cu_of([new]).to(DEV), c.lens.to(DEV), max_q=new, window=window)
        R.check("o", o.cpu(), val["o"], tol["o"])


def test_no_options_are_the_plain_call(fa):
    c, q, cu, max_q = setup("mixed", "bf16", 795)
    k, v, table = c.dev()
    args = (q.to(DEV), k, v, table, cu.to(DEV), c.lens.to(DEV))
    plain = fa.paged_forward(*args, max_q=max_q, return_lse=True)
    none = fa.paged_forward(*args, max_q=max_q, return_lse=True, softcap=None, window=None, slopes=None)
    zero = fa.paged_forward(*args, max_q=max_q, return_lse=True, window=2 ** 40,
                            slopes=torch.zeros(q.shape[1], device=DEV))
    assert torch.equal(plain[0].nan_to_num(), none[0].nan_to_num())
    u = 2.0 ** -8
    assert float((plain[0].float() - zero[0].float()).abs().nan_to_num().max()) <= 4 * u * float(
        plain[0].float().abs().nan_to_num().max())


def test_a_server_against_attention_on_whole_sequences(fa):
    """Prompts in chunks and single tokens through paged_store with axes and paged_forward with capped scores
    and a window, eager and replayed, against qk_norm_rope and attention on each whole sequence."""
    g = torch.Generator(device=DEV).manual_seed(5)
    H, KH, D, page, B = 4, 2, 64, 16, 2
    total = [150, 90]
    q, k, v = ([torch.randn(1, h, n, D, generator=g, device=DEV).half() for n in total] for h in (H, KH, KH))
    qw, kw = (1 + 0.1 * torch.randn(D, generator=g, device=DEV) for _ in range(2))
    angle = torch.arange(200, dtype=torch.float64)[:, None] * 50.0 ** (-torch.arange(32) / 32)
    cos, sin = torch.cos(angle).float().to(DEV), torch.sin(angle).float().to(DEV)
    axes = bytes(i % 3 for i in range(32))
    pos = [torch.stack([torch.arange(n) // 9, torch.arange(n) % 9, torch.arange(n)]).int().to(DEV) for n in total]
    opt = dict(softcap=10.0, window=64, slopes=torch.tensor([0.0, 0.01, 0.02, 0.03], device=DEV))
    want = []
    for b in range(B):
        qn, kn = fa.qk_norm_rope(q[b], k[b], qw, kw, cos, sin, pos[b], axes=axes)
        want.append(fa.attention(qn, kn, v[b], causal=True, **opt)[0].transpose(0, 1))
    kc, vc = (torch.full((20, KH, page, D), math.nan, device=DEV).half() for _ in range(2))
    table = torch.arange(20, dtype=torch.int32, device=DEV).view(2, 10)
    have = [0, 0]
    got = [[], []]

    def step(tokens, cu, lens, p, max_q):
        qs = fa.paged_store(*tokens, qw, kw, cos, sin, p, kc, vc, table, cu, lens, axes=axes)
        return fa.paged_forward(qs, kc, vc, table, cu, lens, max_q=max_q, **opt)

    def inputs(new):
        tokens = [torch.cat([x[b][0, :, have[b]:have[b] + new[b]].transpose(0, 1) for b in range(B)]).contiguous()
                  for x in (q, k, v)]
        p = torch.cat([pos[b][:, have[b]:have[b] + new[b]] for b in range(B)], 1).contiguous()
        lens = torch.tensor([have[b] + new[b] for b in range(B)], dtype=torch.int32, device=DEV)
        return tokens, cu_of(new).to(DEV), lens, p

    graph = static = None
    for new in ([100, 50], [40, 0], [1, 30], [1, 1], [1, 1], [1, 1]):
        args = inputs(new)
        if new == [1, 1] and graph is None:
            static = ([t.clone() for t in args[0]], *(t.clone() for t in args[1:]))
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step(*static, 1)
        if new == [1, 1]:
            for a, b in zip((*static[0], *static[1:]), (*args[0], *args[1:])):
                a.copy_(b)
            graph.replay()
            o = out.clone()
        else:
            o = step(*args, max(new))
        at = 0
        for b in range(B):
            got[b].append(o[at:at + new[b]])
            at += new[b]
            have[b] += new[b]
    u = 2.0 ** -11
    for b in range(B):
        x = torch.cat(got[b])
        y = want[b][:len(x)]
        # both are off by at most 2 u sum P |v| + u |o| + ..., sum P |v| <= the largest |v|
        assert float((x.float() - y.float()).abs().max()) <= 2 * 4 * u * float(v[b].float().abs().max())


def test_refusals(fa):
    c, q, cu, max_q = setup("ragged-decode", "fp16", 799)
    k, v, table = c.dev()
    args = (q.to(DEV), k, v, table, cu.to(DEV), c.lens.to(DEV))
    for change, text in [(dict(softcap=0.0), "softcap"), (dict(softcap=5e3), "softcap"), (dict(window=0), "window"),
                         (dict(slopes=torch.ones(3, device=DEV)), "slopes"),
                         (dict(slopes=torch.ones(8, device=DEV).double()), "slopes"),
                         (dict(slopes=torch.ones(8, device=DEV, requires_grad=True)), "computes no gradients")]:
        with pytest.raises(RuntimeError, match=text):
            fa.paged_forward(*args, max_q=max_q, **change)
