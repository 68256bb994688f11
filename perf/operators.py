"""Timed cases of the operators around a paged key/value cache and of the q/k norm with rotation.

`op` says which operator a case runs:

  attend   paged_forward: attention of each sequence's new tokens over its pages of the cache
  store    paged_store: norm and rotation of new q and k, k and v written to their pages
  norm     qk_norm_rope on [B, H, N, D] tensors, with its gradients where `train` is set
  weights  paged_key_weights: adds up the attention weight that each cached key has received
  evict    paged_evict: keeps the newest and the heaviest keys of each head, in other pages

Sizes: B sequences, H query heads on KH key/value heads of D dims, pages of `page` keys.  The first
sequence has `new` new tokens and `kv` keys (new ones included), the others up to that many by `mix`:
"one" (one new token each), "chunk" (ragged chunks), "prefill" (every key is new).
"""
import math
import os
import random
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
_EPS = 1e-6
_BASE = 10000.0


def _fa():
    path = os.path.join(_ROOT, "flash-attention_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import flash_attention_runtime as fa

    return fa


def _attend(name, B, H, KH, D, dtype, page, new, kv, mix, lse):
    return {"name": name, "op": "attend", "B": B, "H": H, "KH": KH, "D": D, "dtype": dtype,
            "page": page, "new": new, "kv": kv, "mix": mix, "lse": lse}


def _store(name, B, H, KH, D, dtype, page, new, kv, mix, interleaved):
    return {"name": name, "op": "store", "B": B, "H": H, "KH": KH, "D": D, "dtype": dtype,
            "page": page, "new": new, "kv": kv, "mix": mix, "interleaved": interleaved}


def _norm(name, B, H, KH, N, D, dtype, layout, interleaved, train):
    return {"name": name, "op": "norm", "B": B, "H": H, "KH": KH, "N": N, "D": D, "dtype": dtype,
            "layout": layout, "interleaved": interleaved, "train": train}


def _weights(name, B, H, KH, D, dtype, page, new, kv, mix):
    return {"name": name, "op": "weights", "B": B, "H": H, "KH": KH, "D": D, "dtype": dtype,
            "page": page, "new": new, "kv": kv, "mix": mix}


def _evict(name, B, KH, D, dtype, page, kv, keep, recent):
    return {"name": name, "op": "evict", "B": B, "KH": KH, "D": D, "dtype": dtype, "page": page,
            "kv": kv, "keep": keep, "recent": recent}


def listed():
    return [
        # Two short conversations on a small model: the latency of a call.
        _attend("decode-tiny", 2, 8, 2, 64, "fp16", 16, 1, 300, "one", False),
        # A serving batch that generates one token per sequence, at ragged lengths.
        _attend("decode-batch", 32, 32, 8, 128, "bf16", 64, 1, 8192, "one", False),
        # One very long conversation: only its keys can be split over the GPU.
        _attend("decode-long", 1, 32, 8, 128, "fp16", 64, 1, 131072, "one", False),
        # Prompts read in chunks behind long prefixes; the logsumexp feeds the key weights.
        _attend("chunk-ragged", 3, 32, 8, 128, "bf16", 16, 2048, 12288, "chunk", True),
        # The new tokens of a decode step enter the cache.
        _store("store-decode", 64, 32, 8, 128, "bf16", 64, 1, 4096, "one", False),
        # Whole prompts of ragged lengths enter the cache.
        _store("store-prompts", 8, 16, 16, 64, "fp16", 16, 3000, 3000, "prefill", True),
        # A prompt's q and k, views of the projections' [B, N, H, D] tensors.
        _norm("norm-prompt", 2, 16, 16, 1000, 64, "fp16", "bnhd", True, False),
        # A training step on long sequences: norm, rotation and all gradients.
        _norm("norm-train", 2, 32, 8, 8192, 128, "bf16", "bhnd", False, True),
        # Decode steps of a batch whose key weights are tracked.
        _weights("weights-decode", 32, 32, 8, 128, "bf16", 64, 1, 8192, "one"),
        # A chunk of a prompt whose key weights are tracked.
        _weights("weights-chunk", 1, 16, 4, 128, "fp16", 16, 1000, 8192, "chunk"),
        # A few conversations lose half of their keys.
        _evict("evict-half", 4, 8, 64, "fp16", 16, 2048, 1024, 64),
        # Long conversations are cut to a fixed budget.
        _evict("evict-long", 8, 8, 128, "bf16", 64, 16384, 4096, 512),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """1 to 64 sequences of 1 to 131072 keys, 1 to 2048 new tokens, all head counts of a group, both
    types and head dims; at most the work of the largest listed case of the same operator."""
    limits = {"attend": (1.0e9, 5e11, 1.2e9), "store": (2.5e8, 1e99, 1e99), "norm": (3.5e8, 1e99, 1e99),
              "weights": (5e8, 1.5e11, 1.2e9), "evict": (3e8, 1e99, 1e99)}
    while True:
        op = rng.choice(["attend", "attend", "store", "norm", "weights", "evict"])
        kh = rng.choice([1, 2, 3, 4, 8])
        h = kh * rng.choice([1, 1, 2, 3, 4, 5, 8])
        d, dtype = rng.choice([64, 128]), rng.choice(["fp16", "bf16"])
        page = rng.choice([16, 32, 64, 128, 256])
        b = _log(rng, 1, 64)
        kv = _log(rng, 1, 131072)
        mix = rng.choice(["one", "chunk", "prefill"])
        new = {"one": 1, "chunk": min(kv, _log(rng, 2, 2048)), "prefill": kv}[mix]
        if op == "norm":
            case = _norm("", b, h, kh, _log(rng, 1, 16384), d, dtype, rng.choice(["bhnd", "bnhd"]),
                         rng.random() < 0.5, rng.random() < 0.5)
        elif op == "evict":
            keep = max(1, int(kv * rng.uniform(0.1, 1.1)))
            case = _evict("", b, kh, d, dtype, page, kv, keep, int(keep * rng.uniform(0.0, 0.5)))
        elif op == "attend":
            case = _attend("", b, h, kh, d, dtype, page, new, kv, mix, rng.random() < 0.5)
        elif op == "weights":
            case = _weights("", b, h, kh, d, dtype, page, new, kv, mix)
        else:
            case = _store("", b, h, kh, d, dtype, page, new, kv, mix, rng.random() < 0.5)
        del case["name"]
        w = work(case)
        most = limits[op]
        scores = b * h * new * kv if op in ("attend", "weights") else 0  # of the plain form
        pool = b * kv * kh * d * 4 if op != "norm" else 0                # the whole cache
        if w["bytes"] <= most[0] and w["flops"] <= most[1] and scores <= most[2] and pool <= 4e9:
            return case


def _lengths(case):
    """New tokens and keys of each sequence, by the case alone."""
    rng = random.Random("%(B)d %(kv)d %(page)d" % case)
    kv = [case["kv"]] + [max(1, int(case["kv"] * rng.uniform(0.25, 1.0))) for _ in range(case["B"] - 1)]
    mix = case.get("mix", "one")
    if mix == "one":
        new = [1] * case["B"]
    elif mix == "prefill":
        new = list(kv)
    else:
        new = [case["new"]] + [max(1, int(case["new"] * rng.uniform(0.05, 1.0))) for _ in range(case["B"] - 1)]
    return [min(n, m) for n, m in zip(new, kv)], kv


def _pairs(case):
    return sum(n * m - n * (n - 1) // 2 for n, m in zip(*_lengths(case)))


def work(case):
    op, d = case["op"], case["D"]
    if op == "norm":
        rows = case["B"] * (case["H"] + case["KH"]) * case["N"]
        tables = case["N"] * d * 4
        # forward: rows read and written; backward: gradients read, rows read again, gradients written
        return {"bytes": rows * d * 2 * (5 if case["train"] else 2) + tables * (2 if case["train"] else 1),
                "flops": rows * d * (30 if case["train"] else 10)}
    new, kv = _lengths(case)
    tokens, keys = sum(new), sum(kv)
    if op == "store":
        return {"bytes": tokens * ((case["H"] + 2 * case["KH"]) * d * 2 * 2 + d * 4),
                "flops": tokens * (case["H"] + case["KH"]) * d * 10}
    if op == "attend":
        return {"bytes": keys * case["KH"] * d * 2 * 2 + tokens * case["H"] * (d * 4 + 4 * case["lse"]),
                "flops": 4.0 * case["H"] * d * _pairs(case)}
    if op == "weights":
        return {"bytes": keys * case["KH"] * (d * 2 + 8) + tokens * case["H"] * (d * 2 + 4),
                "flops": 2.0 * case["H"] * d * _pairs(case)}
    kept = sum(min(n, case["keep"]) for n in kv)
    return {"bytes": case["KH"] * (keys * 4 + kept * (2 * (2 * d * 2 + 4) + 4)),
            "flops": case["KH"] * keys * 4}


def _cos_sin(rows, dim):
    """Rotation tables: angles in 64 bits, held in 32."""
    freq = _BASE ** (-torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim)
    angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * freq
    return torch.cos(angle).float(), torch.sin(angle).float()


def _randn(g, *shape, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale


def _paged(case, g, null=1):
    """A pool of shuffled pages, the page table (rows padded with page 0, which no sequence owns)
    and the lengths, all as int32 on the GPU."""
    new, kv = _lengths(case)
    page = case["page"]
    counts = [-(-n // page) for n in kv]
    pages = torch.randperm(sum(counts), generator=g, device="cuda").to(torch.int32) + null
    table = torch.zeros((case["B"], max(counts)), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(counts):
        table[i, :n] = pages[at:at + n]
        at += n
    cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    return table, cu, torch.tensor(kv, dtype=torch.int32, device="cuda"), sum(counts) + null, new, kv


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt, op, d = _DTYPES[case["dtype"]], case["op"], case["D"]
    s = {"op": op, "D": d}
    if op == "norm":
        b, n = case["B"], case["N"]
        for x, heads in (("q", case["H"]), ("k", case["KH"]), ("dq", case["H"]), ("dk", case["KH"])):
            if x[0] == "d" and not case["train"]:
                continue
            shape = (b, heads, n, d) if case["layout"] == "bhnd" else (b, n, heads, d)
            t = _randn(g, *shape, scale=1.5).to(dt)
            s[x] = t if case["layout"] == "bhnd" else t.permute(0, 2, 1, 3)
        s["qw"], s["kw"] = 1.0 + _randn(g, d, scale=0.1), 1.0 + _randn(g, d, scale=0.1)
        s["cos"], s["sin"] = _cos_sin(n, d)
        s["interleaved"], s["train"] = case["interleaved"], case["train"]
        if case["train"]:
            for x in ("q", "k", "qw", "kw"):
                s[x].requires_grad_()
        return s
    kh, page = case["KH"], case["page"]
    s["table"], s["cu"], s["lens"], pages, new, kv = _paged(case, g)
    s["max_q"], s["max_kv"] = max(new), max(kv)
    s["kc"], s["vc"] = (_randn(g, pages, kh, page, d).to(dt) for _ in range(2))
    if op == "evict":
        # accumulated weights are heavy-tailed: a few keys hold most of a head's weight
        s["wts"] = torch.exp(_randn(g, pages, kh, page, scale=2.0))
        s["keep"], s["recent"] = case["keep"], case["recent"]
        out = -(-min(case["keep"], max(kv)) // page)
        s["kc"], s["vc"] = (torch.cat([c, torch.zeros((case["B"] * out, kh, page, d), dtype=dt, device="cuda")])
                            for c in (s["kc"], s["vc"]))
        s["wts"] = torch.cat([s["wts"], torch.zeros((case["B"] * out, kh, page), device="cuda")])
        s["to"] = (pages + torch.arange(case["B"] * out, device="cuda", dtype=torch.int32)).view(case["B"], out)
        return s
    h, tokens = case["H"], sum(new)
    # q after its norm has weights of about one: scores of unit spread
    s["q"] = _randn(g, tokens, h, d).to(dt)
    if op == "store":
        s["k"], s["v"] = (_randn(g, tokens, kh, d).to(dt) for _ in range(2))
        s["qw"], s["kw"] = 1.0 + _randn(g, d, scale=0.1), 1.0 + _randn(g, d, scale=0.1)
        s["cos"], s["sin"] = _cos_sin(max(kv), d)
        s["pos"] = torch.cat([torch.arange(m - n, m, device="cuda") for n, m in zip(new, kv)]).to(torch.int32)
        s["interleaved"] = case["interleaved"]
    elif op == "weights":
        s["wts"] = torch.exp(_randn(g, pages, kh, page))
        # the logsumexp that attention returns with these queries, about ln(keys) + 1/2
        last = torch.cat([torch.arange(m - n, m, device="cuda") for n, m in zip(new, kv)]).float()
        s["lse_in"] = torch.log(last + 1.0)[:, None] + 0.5 + _randn(g, tokens, h, scale=0.05)
    else:
        s["lse"] = case["lse"]
    return s


# ---- plain forms ----


def _rotate(x, cos, sin, interleaved, sign):
    """x [..., D] in 32 bits; cos, sin broadcast to [..., D / 2]; sign -1: the inverse rotation."""
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
    else:
        a, b = x.chunk(2, dim=-1)
    sin = sign * sin
    y, z = a * cos - b * sin, b * cos + a * sin
    return torch.stack((y, z), dim=-1).flatten(-2) if interleaved else torch.cat((y, z), dim=-1)


def _norm_rope(x, w, cos, sin, interleaved):
    x = x.float()
    x = x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + _EPS)
    return _rotate(x * w.float(), cos, sin, interleaved, 1.0)


def _norm_rope_grad(dy, x, w, cos, sin, interleaved):
    x, g = x.float(), _rotate(dy.float(), cos, sin, interleaved, -1.0)
    r = torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + _EPS)
    xh, gw = x * r, g * w.float()
    dx = r * (gw - xh * (gw * xh).mean(dim=-1, keepdim=True))
    return dx, (g * xh).sum(dim=(0, 1, 2))


def _gather(cache, table):
    """The keys of each sequence's pages: [B, KH, M * page, ...] in 32 bits."""
    x = cache[table.long()].transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], x.shape[2] * x.shape[3], *x.shape[4:]).float()


def _scores(s, q):
    """Scores [B, KH, G * max_q, keys] of the padded new tokens (masked: -inf) and the rows' tokens."""
    lens, cu, d = s["lens"].long(), s["cu"].long(), s["D"]
    b, kh, h, n = lens.shape[0], s["kc"].shape[1], q.shape[1], s["max_q"]
    i = torch.arange(n, device=q.device)
    new = cu[1:] - cu[:-1]
    token = (cu[:-1, None] + i).clamp(max=q.shape[0] - 1)  # [B, n]
    k = _gather(s["kc"], s["table"])
    qp = q[token].float().reshape(b, n, kh, h // kh, d).permute(0, 2, 3, 1, 4)
    sc = torch.matmul(qp.reshape(b * kh, (h // kh) * n, d), k.reshape(b * kh, -1, d).transpose(1, 2).contiguous())
    sc = sc.view(b, kh, h // kh, n, -1) / math.sqrt(d)
    j = torch.arange(sc.shape[-1], device=q.device)
    last = torch.where(i < new[:, None], (lens - new)[:, None] + i, -1)  # last visible key of a row
    return sc.masked_fill_((j > last[:, :, None])[:, None, None], -math.inf), token


def _rows(x, s, tokens):
    """[B, KH, G, n, ...] of the padded tokens -> [tokens, H, ...] of the packed ones."""
    cu = s["cu"].long()
    t = torch.arange(tokens, device=x.device)
    b = torch.searchsorted(cu, t, right=True) - 1
    x = x[b, :, :, t - cu[b]]
    return x.reshape(tokens, x.shape[1] * x.shape[2], *x.shape[3:])


def _plain_attend(s):
    q = s["q"]
    sc, _ = _scores(s, q)
    b, kh, g, n, m = sc.shape
    top = sc.amax(dim=-1, keepdim=True).clamp(min=-1e30)
    p = sc.sub_(top).exp_()
    total = p.sum(dim=-1)
    o = torch.matmul(p.view(b * kh, g * n, m), _gather(s["vc"], s["table"]).view(b * kh, m, s["D"]))
    o = o.view(b, kh, g, n, s["D"]) / total[..., None]
    o = _rows(o, s, q.shape[0]).to(q.dtype)
    return (o, _rows(top[..., 0] + torch.log(total), s, q.shape[0])) if s["lse"] else o


def _plain_weights(s):
    q = s["q"]
    sc, token = _scores(s, q)
    b, kh, g, n, m = sc.shape
    lse = s["lse_in"][token].reshape(b, n, kh, g).permute(0, 2, 3, 1)
    add = sc.sub_(lse[..., None]).exp_().sum(dim=(2, 3))  # [B, KH, keys]
    old = _gather(s["wts"], s["table"])
    lens = s["lens"].long()[:, None, None]
    new = (s["cu"][1:] - s["cu"][:-1]).long()[:, None, None]
    j = torch.arange(m, device=q.device)
    w = torch.where(j < lens - new, old + add, torch.where(j < lens, add, old))
    page = s["wts"].shape[2]
    s["wts"][s["table"].long()] = w.view(b, kh, m // page, page).transpose(1, 2)
    return s["wts"]


def _plain_store(s):
    cos, sin = s["cos"][s["pos"].long()][:, None], s["sin"][s["pos"].long()][:, None]
    q = _norm_rope(s["q"], s["qw"], cos, sin, s["interleaved"]).to(s["q"].dtype)
    k = _norm_rope(s["k"], s["kw"], cos, sin, s["interleaved"]).to(s["k"].dtype)
    cu, page = s["cu"].long(), s["kc"].shape[2]
    t = torch.arange(q.shape[0], device=q.device)
    b = torch.searchsorted(cu, t, right=True) - 1
    at = s["lens"].long()[b] - cu[b + 1] + t
    where = s["table"].long()[b, at // page]
    s["kc"][where, :, at % page] = k
    s["vc"][where, :, at % page] = s["v"]
    return q, s["kc"], s["vc"]


def _plain_norm(s):
    with torch.no_grad():
        c = (s["cos"], s["sin"], s["interleaved"])
        q = _norm_rope(s["q"], s["qw"], *c).to(s["q"].dtype)
        k = _norm_rope(s["k"], s["kw"], *c).to(s["k"].dtype)
        if not s["train"]:
            return q, k
        dq, dqw = _norm_rope_grad(s["dq"], s["q"], s["qw"], *c)
        dk, dkw = _norm_rope_grad(s["dk"], s["k"], s["kw"], *c)
        return q, k, dq.to(q.dtype), dk.to(k.dtype), dqw, dkw


def _plain_evict(s):
    page, lens = s["kc"].shape[2], s["lens"].long()
    w = _gather(s["wts"], s["table"])  # [B, KH, keys]
    b, kh, m = w.shape
    j = torch.arange(m, device=w.device)
    n = lens[:, None, None]
    rank = torch.where(j >= n, -math.inf, torch.where(j >= n - s["recent"], math.inf, w))
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices
    t = torch.arange(min(s["keep"], m), device=w.device)
    have = torch.clamp(lens, max=s["keep"])[:, None, None]
    kept = torch.where(t < have, order[:, :, :t.shape[0]], m).sort(dim=-1).values
    kept = torch.where(t < have, kept, -1)
    src = kept.clamp(min=0)
    rows = torch.arange(b, device=w.device)[:, None, None]
    heads = torch.arange(kh, device=w.device)[None, :, None]
    here = (s["table"].long()[rows, src // page], heads, src % page)
    there = (s["to"].long()[:, None, t // page].expand(b, kh, -1), heads.expand(b, kh, t.shape[0]),
             (t % page).expand(b, kh, -1))
    put = t < have
    s["kc"][there] = torch.where(put[..., None], s["kc"][here], s["kc"][there])
    s["vc"][there] = torch.where(put[..., None], s["vc"][here], s["vc"][there])
    s["wts"][there] = torch.where(put, s["wts"][here], s["wts"][there])
    full = torch.full((b, kh, s["keep"]), -1, dtype=torch.int32, device=w.device)
    full[:, :, :t.shape[0]] = kept.to(torch.int32)
    return have.view(b).to(torch.int32), full, s["kc"], s["vc"], s["wts"]


_PLAIN = {"attend": _plain_attend, "store": _plain_store, "norm": _plain_norm,
          "weights": _plain_weights, "evict": _plain_evict}


# ---- the framework's calls ----


def _own(s):
    fa = _fa()
    op = s["op"]
    if op == "attend":
        return fa.paged_forward(s["q"], s["kc"], s["vc"], s["table"], s["cu"], s["lens"],
                                max_q=s["max_q"], max_kv=s["max_kv"], return_lse=s["lse"])
    if op == "store":
        q = fa.paged_store(s["q"], s["k"], s["v"], s["qw"], s["kw"], s["cos"], s["sin"], s["pos"],
                           s["kc"], s["vc"], s["table"], s["cu"], s["lens"], eps=_EPS,
                           interleaved=s["interleaved"])
        return q, s["kc"], s["vc"]
    if op == "norm":
        q, k = fa.qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], s["cos"], s["sin"], eps=_EPS,
                               interleaved=s["interleaved"])
        if not s["train"]:
            return q, k
        dq, dk, dqw, dkw = torch.autograd.grad((q, k), (s["q"], s["k"], s["qw"], s["kw"]),
                                               (s["dq"], s["dk"]))
        return q, k, dq, dk, dqw, dkw
    if op == "weights":
        return fa.paged_key_weights(s["q"], s["lse_in"], s["kc"], s["table"], s["cu"], s["lens"],
                                    s["wts"], max_q=s["max_q"], max_kv=s["max_kv"])
    lens, kept = fa.paged_evict(s["kc"], s["vc"], s["wts"], s["table"], s["lens"], s["to"],
                                keep=s["keep"], recent=s["recent"])
    return lens, kept, s["kc"], s["vc"], s["wts"]


def run(state):
    return _own(state) if own else _PLAIN[state["op"]](state)


# ---- the definitions in 64 bits ----


def _exact_rows(x, w, pos, s, interleaved):
    """Rows x [..., n, D] at positions pos [n]: unit rms, weights, then a rotation as complex numbers."""
    x = x.detach().double()
    y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + _EPS) * w.detach().double()
    turn = torch.complex(s["cos"].double(), s["sin"].double())[pos]
    half = y.shape[-1] // 2
    z = torch.complex(y[..., 0::2], y[..., 1::2]) if interleaved else torch.complex(y[..., :half], y[..., half:])
    z = z * turn
    return torch.view_as_real(z).flatten(-2) if interleaved else torch.cat((z.real, z.imag), -1)


def _exact_norm(s):
    out, grads, wgrads = [], [], []
    pos = torch.arange(s["q"].shape[2], device="cuda")
    for x, w, dy in (("q", "qw", "dq"), ("k", "kw", "dk")):
        out.append(torch.empty(s[x].shape, dtype=torch.float64, device="cuda"))
        if s["train"]:
            grads.append(torch.empty_like(out[-1]))
            wgrads.append(torch.zeros(s["D"], dtype=torch.float64, device="cuda"))
        for i in range(s[x].shape[0]):
            for j in range(s[x].shape[1]):
                xd = s[x][i, j].detach().double().requires_grad_(s["train"])
                wd = s[w].detach().double().requires_grad_(s["train"])
                r = xd / torch.sqrt((xd * xd).mean(-1, keepdim=True) + _EPS) * wd
                half = s["D"] // 2
                a, b = (r[:, 0::2], r[:, 1::2]) if s["interleaved"] else (r[:, :half], r[:, half:])
                c, t = s["cos"].double(), s["sin"].double()
                y = (a * c - b * t, a * t + b * c)
                y = torch.stack(y, -1).flatten(-2) if s["interleaved"] else torch.cat(y, -1)
                out[-1][i, j] = y.detach()
                if s["train"]:
                    gx, gw = torch.autograd.grad(y, (xd, wd), s[dy][i, j].double())
                    grads[-1][i, j] = gx
                    wgrads[-1] += gw
    return (*out, *grads, *wgrads)


def _exact_keys(cache, s, i, h, n):
    page = cache.shape[2]
    ids = s["table"][i, :-(-n // page)].long()
    return cache[ids, h].reshape(-1, *cache.shape[3:])[:n].double()


def _exact_blocks(s):
    """(sequence, head, first token, keys, row block) of the packed rows, at most 2^25 scores each."""
    cu, lens = s["cu"].tolist(), s["lens"].tolist()
    for i in range(len(lens)):
        step = max(1, (1 << 25) // max(1, lens[i]))
        for h in range(s["q"].shape[1]):
            for r in range(cu[i], cu[i + 1], step):
                yield i, h, cu[i + 1], lens[i], slice(r, min(r + step, cu[i + 1]))


def _exact_scores(s, i, h, end, n, rows):
    g = s["q"].shape[1] // s["kc"].shape[1]
    kt = _exact_keys(s["kc"], s, i, h // g, n).t().contiguous()
    sc = torch.mm(s["q"][rows, h].double().contiguous(), kt) / math.sqrt(s["D"])
    own_key = torch.arange(rows.start, rows.stop, device="cuda") + n - end
    return sc.masked_fill_(torch.arange(n, device="cuda") > own_key[:, None], -math.inf)


def _exact_attend(s):
    g = s["q"].shape[1] // s["kc"].shape[1]
    o = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    for i, h, end, n, rows in _exact_blocks(s):
        sc = _exact_scores(s, i, h, end, n, rows)
        lse[rows, h] = torch.logsumexp(sc, dim=1)
        o[rows, h] = torch.mm(torch.exp(sc - lse[rows, h, None]), _exact_keys(s["vc"], s, i, h // g, n))
    return (o, lse) if s["lse"] else o


def _exact_weights(s):
    g, page = s["q"].shape[1] // s["kc"].shape[1], s["wts"].shape[2]
    w = s["wts"].double()
    cu = s["cu"].tolist()
    fresh = torch.zeros(w.shape, dtype=torch.bool, device="cuda")
    for i, n in enumerate(s["lens"].tolist()):
        at = torch.arange(n - (cu[i + 1] - cu[i]), n, device="cuda")
        fresh[s["table"][i].long()[at // page], :, at % page] = True
    w[fresh] = 0.0
    for i, h, end, n, rows in _exact_blocks(s):
        p = torch.exp(_exact_scores(s, i, h, end, n, rows) - s["lse_in"][rows, h, None].double()).sum(0)
        at = torch.arange(n, device="cuda")
        w.index_put_((s["table"][i].long()[at // page], torch.full_like(at, h // g), at % page), p, accumulate=True)
    return w


def _exact_store(s):
    q = _exact_rows(s["q"].transpose(0, 1), s["qw"], s["pos"].long(), s, s["interleaved"]).transpose(0, 1)
    k = _exact_rows(s["k"].transpose(0, 1), s["kw"], s["pos"].long(), s, s["interleaved"]).transpose(0, 1)
    kc, vc = s["kc"].double(), s["vc"].double()
    cu, page = s["cu"].tolist(), s["kc"].shape[2]
    for i, n in enumerate(s["lens"].tolist()):
        at = torch.arange(n - (cu[i + 1] - cu[i]), n, device="cuda")
        ids = s["table"][i].long()[at // page]
        kc[ids, :, at % page] = k[cu[i]:cu[i + 1]]
        vc[ids, :, at % page] = s["v"][cu[i]:cu[i + 1]].double()
    return q, kc, vc


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "evict":
        return None  # whole numbers and moved values: the plain form is their definition
    return {"attend": _exact_attend, "weights": _exact_weights, "store": _exact_store,
            "norm": _exact_norm}[s["op"]](s)
