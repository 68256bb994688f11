"""Timed cases of attention with capped, biased and masked scores, in training and over the paged
cache, and of the q/k norm with a rotation by several axes.

`op` says which operator a case runs:

  train    attention and its gradients on [B, H, N, D] tensors
  attend   attention alone (a prompt that nothing is learned from)
  serve    paged_forward with the same scores: new tokens of sequences over a paged cache
  norm     qk_norm_rope with positions of several axes, with its gradients where `train` is set
  store    paged_store with positions of several axes

Sizes: H query heads on KH key/value heads of D dims.  train, attend: N queries, the last of M keys
(N = M but for the later part of a context); `mask` is "full", "causal", "window", "docs" (documents
packed in a row) or "prefix" (the same, each with a first part that all of it sees).  serve and store: B sequences, the
first with `new` new tokens and `kv` keys, the others up to that many.  `cap` and `window` 0: none.
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


def _attend(name, op, B, H, KH, N, M, D, dtype, mask, docs, window, cap, slopes):
    return {"name": name, "op": op, "B": B, "H": H, "KH": KH, "N": N, "M": M, "D": D, "dtype": dtype,
            "mask": mask, "docs": docs, "window": window, "cap": cap, "slopes": slopes}


def _serve(name, B, H, KH, D, dtype, page, new, kv, window, cap, slopes):
    return {"name": name, "op": "serve", "B": B, "H": H, "KH": KH, "D": D, "dtype": dtype, "page": page,
            "new": new, "kv": kv, "window": window, "cap": cap, "slopes": slopes}


def _norm(name, B, H, KH, N, D, dtype, axes, order, interleaved, train):
    return {"name": name, "op": "norm", "B": B, "H": H, "KH": KH, "N": N, "D": D, "dtype": dtype,
            "axes": axes, "order": order, "interleaved": interleaved, "train": train}


def _store(name, B, H, KH, D, dtype, page, new, kv, axes, order):
    return {"name": name, "op": "store", "B": B, "H": H, "KH": KH, "D": D, "dtype": dtype, "page": page,
            "new": new, "kv": kv, "axes": axes, "order": order}


def listed():
    return [
        # A step on three short documents in one row: launches and latency.
        _attend("train-tiny", "train", 1, 4, 2, 300, 300, 64, "fp16", "docs", 3, 0, 0.0, False),
        # A small model whose positions are a bias by distance.
        _attend("train-slopes", "train", 4, 16, 16, 1024, 1024, 64, "fp16", "causal", 1, 0, 0.0, True),
        # Image and text: each example's first part sees itself both ways.
        _attend("train-prefix", "train", 2, 16, 16, 2000, 2000, 128, "bf16", "prefix", 2, 0, 0.0, False),
        # Documents packed in long rows.
        _attend("train-docs", "train", 1, 32, 8, 16384, 16384, 128, "bf16", "docs", 12, 0, 0.0, False),
        # A layer with capped scores that sees the whole of a long row.
        _attend("train-cap", "train", 2, 32, 8, 8192, 8192, 128, "bf16", "causal", 1, 0, 50.0, False),
        # A layer of a sliding window reads a long prompt.
        _attend("prompt-window", "attend", 1, 16, 16, 16384, 16384, 128, "fp16", "window", 1, 1024, 0.0, False),
        # One token each of two short conversations, positions as a bias.
        _serve("serve-tiny", 2, 8, 2, 64, "fp16", 16, 1, 300, 0, 0.0, True),
        # A batch that generates, capped scores.
        _serve("serve-cap", 32, 32, 8, 128, "bf16", 64, 1, 8192, 0, 50.0, False),
        # Prompts read in chunks behind long prefixes, capped scores in a window.
        _serve("serve-chunk", 3, 32, 8, 128, "bf16", 16, 2048, 12288, 4096, 50.0, False),
        # New tokens enter the cache, their positions of time, height and width.
        _store("axes-store", 64, 32, 8, 128, "bf16", 64, 1, 4096, 3, "blocks"),
        # An image's patches before attention: height and width.
        _norm("axes-image", 2, 16, 16, 1000, 64, "fp16", 2, "blocks", True, False),
        # A training step on long rows of video and text.
        _norm("axes-train", 2, 32, 8, 8192, 128, "bf16", 3, "cyclic", False, True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Rows of 1 to 16384 queries, 1 to 24 documents, windows of 1 to all, caps of 5 to 60, sequences of
    1 to 131072 keys, all head counts of a group, both types and head dims; at most the work of the
    largest listed case of the same operator."""
    most = {"train": 3.0e12, "attend": 1.2e12, "serve": 5e11, "norm": 1e99, "store": 1e99}
    while True:
        op = rng.choice(["train", "train", "train", "attend", "serve", "serve", "norm", "store"])
        kh = rng.choice([1, 2, 3, 4, 8])
        h = kh * rng.choice([1, 1, 2, 3, 4, 5, 8])
        d, dtype = rng.choice([64, 128]), rng.choice(["fp16", "bf16"])
        cap, slopes = rng.choice([0.0, 0.0, float(rng.randint(5, 60))]), rng.random() < 0.3
        if op in ("train", "attend"):
            n = _log(rng, 1, 16384)
            mask = rng.choice(["full", "causal", "window", "docs", "docs", "prefix"])
            m = n + (_log(rng, 1, 4096) if mask in ("full", "causal", "window") and rng.random() < 0.3 else 0)
            window = _log(rng, 1, n) if mask == "window" or rng.random() < 0.1 else 0
            docs = min(n, _log(rng, 1, 24)) if mask in ("docs", "prefix") else 1
            case = _attend("", op, rng.choice([1, 1, 2, 3, 4]), h, kh, n, m, d, dtype, mask, docs, window, cap, slopes)
            if case["B"] * h * n * m > 4.4e9:  # scores of the plain form
                continue
        elif op == "norm":
            case = _norm("", rng.choice([1, 2, 3, 4]), h, kh, _log(rng, 1, 16384), d, dtype, rng.choice([2, 3, 4]),
                         rng.choice(["blocks", "cyclic"]), rng.random() < 0.5, rng.random() < 0.5)
        else:
            b, kv, page = _log(rng, 1, 64), _log(rng, 1, 131072), rng.choice([16, 32, 64, 128, 256])
            new = rng.choice([1, 1, min(kv, _log(rng, 2, 2048))])
            if op == "store":
                case = _store("", b, h, kh, d, dtype, page, new, kv, rng.choice([2, 3, 4]), rng.choice(["blocks", "cyclic"]))
            else:
                window = _log(rng, 1, kv) if rng.random() < 0.5 else 0
                case = _serve("", b, h, kh, d, dtype, page, new, kv, window, cap, slopes)
            if b * h * new * kv > 1.2e9 or b * kv * kh * d * 4 > 4e9:  # the plain form's scores, the cache
                continue
        del case["name"]
        w = work(case)
        if w["bytes"] <= 1.2e9 and w["flops"] <= most[op]:
            return case


# ---- masks and lengths, by the case alone ----


def _documents(case):
    """Ends of the documents of each row of a batch, and the ends of their prefixes."""
    rng = random.Random("%(B)d %(N)d %(docs)d" % case)
    ends, prefixes = [], []
    for _ in range(case["B"]):
        e = sorted(rng.sample(range(1, case["N"]), case["docs"] - 1)) + [case["N"]]
        ends.append(e)
        prefixes.append([a + int((b - a) * rng.uniform(0.1, 0.6)) for a, b in zip([0] + e[:-1], e)])
    return ends, prefixes


def _ranges(case, device="cpu"):
    """First key and end of the keys that each row sees, [B, N] each; window and causal order left out
    where the call takes them by themselves."""
    n = case["N"]
    i = torch.arange(n, device=device)
    lo, hi = [], []
    for ends, prefixes in zip(*_documents(case)):
        e = torch.tensor(ends, device=device)
        doc = torch.searchsorted(e, i, right=True)
        first = torch.cat([torch.zeros(1, dtype=e.dtype, device=device), e[:-1]])[doc]
        lo.append(first)
        hi.append(torch.maximum(i + 1, torch.tensor(prefixes, device=device)[doc]) if case["mask"] == "prefix" else i + 1)
    return torch.stack(lo), torch.stack(hi)


def _limits(case, device="cpu"):
    """The same with all of the mask."""
    n, m = case["N"], case["M"]
    p = torch.arange(n, device=device) + (m - n)
    if case["mask"] in ("docs", "prefix"):
        lo, hi = _ranges(case, device)
    else:
        lo = torch.zeros((case["B"], n), dtype=torch.int64, device=device)
        hi = torch.full((case["B"], n), m, dtype=torch.int64, device=device)
    if case["mask"] in ("causal", "window"):
        hi = torch.minimum(hi, p + 1)
    if case["window"]:
        lo = torch.maximum(lo, p - case["window"] + 1)
        hi = torch.minimum(hi, p + case["window"])
    return lo, hi


def _lengths(case):
    """New tokens and keys of each sequence."""
    rng = random.Random("%(B)d %(kv)d %(page)d" % case)
    kv = [case["kv"]] + [max(1, int(case["kv"] * rng.uniform(0.25, 1.0))) for _ in range(case["B"] - 1)]
    new = [case["new"]] + [max(1, int(case["new"] * rng.uniform(0.05, 1.0))) for _ in range(case["B"] - 1)]
    return [min(n, m) for n, m in zip(new, kv)], kv


def work(case):
    op, d, h, kh = case["op"], case["D"], case["H"], case["KH"]
    if op in ("train", "attend"):
        lo, hi = _limits(case)
        pairs = int((hi - lo).clamp(min=0).sum()) * h
        q, k = case["B"] * case["N"] * h * d * 2, case["B"] * case["M"] * kh * d * 2
        # forward: q, k, v read, o written; backward: q, k, v, o, do read, dq, dk, dv written
        return {"bytes": 2 * q + 2 * k + (4 * q + 4 * k if op == "train" else 0),
                "flops": pairs * d * (14.0 if op == "train" else 4.0)}
    if op == "norm":
        rows = case["B"] * (h + kh) * case["N"]
        return {"bytes": rows * d * 2 * (5 if case["train"] else 2) + case["axes"] * case["N"] * 4,
                "flops": rows * d * (30 if case["train"] else 10)}
    new, kv = _lengths(case)
    tokens = sum(new)
    if op == "store":
        return {"bytes": tokens * ((h + 2 * kh) * d * 2 * 2 + d * 4), "flops": tokens * (h + kh) * d * 10}
    keys = pairs = 0
    for n, m in zip(new, kv):
        w = case["window"] or m
        keys += min(m, n + w - 1)  # seen by some token
        pairs += sum(min(m - n + i + 1, w) for i in range(n))
    return {"bytes": keys * kh * d * 2 * 2 + tokens * h * d * 4, "flops": 4.0 * h * d * pairs}


# ---- inputs ----


def _randn(g, *shape, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale


def _slopes(heads):
    """2^(-8 / heads), its square, and so on: the usual geometric slopes."""
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / heads) for i in range(heads)], device="cuda")


def _pair_axes(case):
    """The axis of each of D / 2 pairs of dims: in blocks, or in turn."""
    pairs, a = case["D"] // 2, case["axes"]
    if case["order"] == "cyclic":
        return [p % a for p in range(pairs)]
    return [min(p * a // pairs, a - 1) for p in range(pairs)]


def _tables(rows, dim):
    """Rotation tables: angles in 64 bits, held in 32."""
    freq = _BASE ** (-torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim)
    angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * freq
    return torch.cos(angle).float(), torch.sin(angle).float()


def _positions(axes, tokens):
    """Positions [axes, tokens] of frames of 16 x 16 patches: the first axis counts frames, the others
    run within them, ahead of the frames before."""
    t = torch.arange(tokens, device="cuda")
    frame, at = t // 256, t % 256
    pos = [frame * 16, frame * 16 + at // 16, frame * 16 + at % 16, frame * 16 + at % 7]
    return torch.stack(pos[:axes]).to(torch.int32)


def _paged(case, g):
    """A pool of shuffled pages, the page table (rows padded with page 0, which no sequence owns) and the
    lengths, all as int32 on the GPU."""
    new, kv = _lengths(case)
    counts = [-(-n // case["page"]) for n in kv]
    pages = torch.randperm(sum(counts), generator=g, device="cuda").to(torch.int32) + 1
    table = torch.zeros((case["B"], max(counts)), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(counts):
        table[i, :n] = pages[at:at + n]
        at += n
    cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    return table, cu, torch.tensor(kv, dtype=torch.int32, device="cuda"), sum(counts) + 1, new, kv


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt, op, d, h, kh = _DTYPES[case["dtype"]], case["op"], case["D"], case["H"], case["KH"]
    s = {"op": op, "case": dict(case)}
    if op in ("train", "attend"):
        b, n, m = case["B"], case["N"], case["M"]
        # capped scores are large ones
        s["q"] = _randn(g, b, h, n, d, scale=4.0 if case["cap"] else 1.0).to(dt)
        s["k"], s["v"] = (_randn(g, b, kh, m, d).to(dt) for _ in range(2))
        s["slopes"] = _slopes(h) if case["slopes"] else None
        s["ranges"] = None
        if case["mask"] in ("docs", "prefix"):
            s["ranges"] = torch.stack(_ranges(case, "cuda"), dim=-1).to(torch.int32).contiguous()
        if op == "train":
            s["do"] = _randn(g, b, h, n, d).to(dt)
            for x in ("q", "k", "v"):
                s[x].requires_grad_()
        return s
    if op in ("norm", "store"):
        s["qw"], s["kw"] = 1.0 + _randn(g, d, scale=0.1), 1.0 + _randn(g, d, scale=0.1)
        s["axes"] = bytes(_pair_axes(case))
    if op == "norm":
        b, n = case["B"], case["N"]
        for x, heads in (("q", h), ("k", kh), ("dq", h), ("dk", kh)):
            if x[0] != "d" or case["train"]:
                s[x] = _randn(g, b, heads, n, d, scale=1.5).to(dt)
        s["pos"] = _positions(case["axes"], n)
        s["cos"], s["sin"] = _tables(n // 16 + 48, d)
        s["interleaved"] = case["interleaved"]
        if case["train"]:
            for x in ("q", "k", "qw", "kw"):
                s[x].requires_grad_()
        return s
    page = case["page"]
    s["table"], s["cu"], s["lens"], pages, new, kv = _paged(case, g)
    s["max_q"], s["max_kv"] = max(new), max(kv)
    s["kc"], s["vc"] = (_randn(g, pages, kh, page, d).to(dt) for _ in range(2))
    s["q"] = _randn(g, sum(new), h, d, scale=4.0 if case.get("cap") else 1.0).to(dt)
    if op == "store":
        s["k"], s["v"] = (_randn(g, sum(new), kh, d).to(dt) for _ in range(2))
        s["cos"], s["sin"] = _tables(max(kv) // 16 + 48, d)
        last = torch.cat([torch.arange(m - n, m, device="cuda") for n, m in zip(new, kv)])
        s["pos"] = _positions(case["axes"], max(kv))[:, last].contiguous()
        s["interleaved"] = False
    else:
        s["slopes"] = _slopes(h) if case["slopes"] else None
    return s


# ---- plain forms ----


def _scores(s, q, k, p, j, lo, hi, slopes):
    """Final scores (masked: -inf) of rows q [..., n, D] at positions p against keys k [..., m, D] at j, and
    the slope of the cap (1 - tanh^2); p, lo, hi broadcast to [..., n, 1], j to [m], slopes to [..., 1, 1]."""
    case = s["case"]
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()).div_(math.sqrt(case["D"]))
    grad = None
    if case["cap"]:
        t = x.div_(case["cap"]).tanh_()
        grad = 1.0 - t * t
        x = t.mul_(case["cap"])
    if slopes is not None:
        x -= slopes * (p - j).abs().float()
    return x.masked_fill_((j < lo) | (j >= hi), -math.inf), grad


def _plain_attend(s):
    """Blocks of heads of one batch entry, as many as make 2^28 scores."""
    with torch.no_grad():
        case = s["case"]
        b, h, kh, n, m = (case[x] for x in ("B", "H", "KH", "N", "M"))
        g = h // kh
        lo, hi = (x[:, None, :, None] for x in _limits(case, "cuda"))
        p = (torch.arange(n, device="cuda") + (m - n))[:, None]
        j = torch.arange(m, device="cuda")
        outs = [torch.empty_like(s["q"])]
        if s["op"] == "train":
            outs += [torch.empty_like(s["q"]), torch.empty_like(s["k"]), torch.empty_like(s["v"])]
        step = max(1, (1 << 28) // (g * n * m))
        for i in range(b):
            for k0 in range(0, kh, step):
                ks, qs = slice(k0, min(kh, k0 + step)), slice(k0 * g, min(kh, k0 + step) * g)
                q = s["q"][i, qs].float()
                k = s["k"][i, ks].float().repeat_interleave(g, 0)
                v = s["v"][i, ks].float().repeat_interleave(g, 0)
                slopes = None if s["slopes"] is None else s["slopes"][qs, None, None]
                x, grad = _scores(s, q, k, p, j, lo[i], hi[i], slopes)
                x = x.sub_(x.amax(dim=-1, keepdim=True).clamp(min=-1e30)).exp_()
                x = x.div_(x.sum(dim=-1, keepdim=True).clamp(min=1e-30))
                o = torch.matmul(x, v)
                outs[0][i, qs] = o.to(outs[0].dtype)
                if s["op"] != "train":
                    continue
                do = s["do"][i, qs].float()
                outs[3][i, ks] = torch.matmul(x.transpose(-1, -2).contiguous(), do).view(-1, g, m, case["D"]).sum(1).to(outs[3].dtype)
                ds = torch.matmul(do, v.transpose(-1, -2).contiguous())
                ds = ds.sub_((do * o).sum(dim=-1, keepdim=True)).mul_(x)
                if grad is not None:
                    ds = ds.mul_(grad)
                ds = ds.div_(math.sqrt(case["D"]))
                outs[1][i, qs] = torch.matmul(ds, k).to(outs[1].dtype)
                outs[2][i, ks] = torch.matmul(ds.transpose(-1, -2).contiguous(), q).view(-1, g, m, case["D"]).sum(1).to(outs[2].dtype)
        return outs[0] if s["op"] != "train" else tuple(outs)


def _gather(cache, table):
    """The keys of each sequence's pages: [B, KH, M * page, D] in 32 bits."""
    x = cache[table.long()].transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[4]).float()


def _plain_serve(s):
    case, q = s["case"], s["q"]
    lens, cu, d = s["lens"].long(), s["cu"].long(), case["D"]
    b, kh, h, n = case["B"], case["KH"], case["H"], s["max_q"]
    g = h // kh
    i = torch.arange(n, device=q.device)
    new = cu[1:] - cu[:-1]
    token = (cu[:-1, None] + i).clamp(max=q.shape[0] - 1)  # [B, n]
    k, v = _gather(s["kc"], s["table"]), _gather(s["vc"], s["table"])
    qp = q[token].float().view(b, n, kh, g, d).permute(0, 2, 3, 1, 4).reshape(b, kh, g * n, d)
    p = (lens - new)[:, None] + i  # [B, n]
    hi = torch.where(i < new[:, None], p + 1, 0)
    lo = p - (case["window"] or s["max_kv"]) + 1
    rows = lambda x: x[:, None, None, :].expand(b, 1, g, n).reshape(b, 1, g * n, 1)
    slopes = None if s["slopes"] is None else s["slopes"].view(1, kh, g, 1).expand(1, kh, g, n).reshape(1, kh, g * n, 1)
    x, _ = _scores(s, qp, k, rows(p), torch.arange(k.shape[2], device=q.device), rows(lo), rows(hi), slopes)
    x = x.sub_(x.amax(dim=-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = x.sum(dim=-1, keepdim=True)
    o = (torch.matmul(x, v) / total).view(b, kh, g, n, d)
    t = torch.arange(q.shape[0], device=q.device)
    seq = torch.searchsorted(cu, t, right=True) - 1
    return o[seq, :, :, t - cu[seq]].reshape(q.shape).to(q.dtype)


def _rotate(x, cos, sin, interleaved, sign):
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else x.chunk(2, dim=-1)
    sin = sign * sin
    y, z = a * cos - b * sin, b * cos + a * sin
    return torch.stack((y, z), dim=-1).flatten(-2) if interleaved else torch.cat((y, z), dim=-1)


def _angles(s):
    """Cosines and sines [tokens, D / 2]: each pair's by the position on its own axis."""
    axis = torch.tensor(list(s["axes"]), device="cuda")
    pos = s["pos"].long()[axis]  # [D / 2, tokens]
    pair = torch.arange(axis.shape[0], device="cuda")[:, None]
    return s["cos"][pos, pair].t(), s["sin"][pos, pair].t()


def _norm_rope(x, w, cos, sin, interleaved):
    x = x.float()
    x = x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + _EPS)
    return _rotate(x * w, cos, sin, interleaved, 1.0)


def _norm_rope_grad(dy, x, w, cos, sin, interleaved):
    x, g = x.float(), _rotate(dy.float(), cos, sin, interleaved, -1.0)
    r = torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + _EPS)
    xh, gw = x * r, g * w
    return r * (gw - xh * (gw * xh).mean(dim=-1, keepdim=True)), (g * xh).sum(dim=(0, 1, 2))


def _plain_norm(s):
    with torch.no_grad():
        c = (*_angles(s), s["interleaved"])
        q = _norm_rope(s["q"], s["qw"], *c).to(s["q"].dtype)
        k = _norm_rope(s["k"], s["kw"], *c).to(s["k"].dtype)
        if not s["case"]["train"]:
            return q, k
        dq, dqw = _norm_rope_grad(s["dq"], s["q"], s["qw"], *c)
        dk, dkw = _norm_rope_grad(s["dk"], s["k"], s["kw"], *c)
        return q, k, dq.to(q.dtype), dk.to(k.dtype), dqw, dkw


def _places(s):
    """Page and row of each new token in the cache."""
    cu, page = s["cu"].long(), s["case"]["page"]
    t = torch.arange(s["q"].shape[0], device="cuda")
    b = torch.searchsorted(cu, t, right=True) - 1
    at = s["lens"].long()[b] - cu[b + 1] + t
    return s["table"].long()[b, at // page], at % page


def _plain_store(s):
    cos, sin = (x[:, None] for x in _angles(s))
    q = _norm_rope(s["q"], s["qw"], cos, sin, s["interleaved"]).to(s["q"].dtype)
    k = _norm_rope(s["k"], s["kw"], cos, sin, s["interleaved"]).to(s["k"].dtype)
    where, row = _places(s)
    s["kc"][where, :, row] = k
    s["vc"][where, :, row] = s["v"]
    return q, s["kc"], s["vc"]


_PLAIN = {"train": _plain_attend, "attend": _plain_attend, "serve": _plain_serve, "norm": _plain_norm,
          "store": _plain_store}


# ---- the framework's calls ----


def _own(s):
    fa, case, op = _fa(), s["case"], s["op"]
    if op in ("train", "attend"):
        o = fa.attention(s["q"], s["k"], s["v"], s["ranges"], causal=case["mask"] in ("causal", "window"),
                         window=case["window"] or None, softcap=case["cap"] or None, slopes=s["slopes"])
        if op == "attend":
            return o
        return (o, *torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"]))
    if op == "serve":
        return fa.paged_forward(s["q"], s["kc"], s["vc"], s["table"], s["cu"], s["lens"], max_q=s["max_q"],
                                max_kv=s["max_kv"], window=case["window"] or None,
                                softcap=case["cap"] or None, slopes=s["slopes"])
    if op == "store":
        q = fa.paged_store(s["q"], s["k"], s["v"], s["qw"], s["kw"], s["cos"], s["sin"], s["pos"], s["kc"],
                           s["vc"], s["table"], s["cu"], s["lens"], eps=_EPS, interleaved=s["interleaved"],
                           axes=s["axes"])
        return q, s["kc"], s["vc"]
    q, k = fa.qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], s["cos"], s["sin"], s["pos"], eps=_EPS,
                           interleaved=s["interleaved"], axes=s["axes"])
    if not case["train"]:
        return q, k
    return (q, k, *torch.autograd.grad((q, k), (s["q"], s["k"], s["qw"], s["kw"]), (s["dq"], s["dk"])))


def run(state):
    return _own(state) if own else _PLAIN[state["op"]](state)


# ---- the definitions in 64 bits ----


def _exact_head(case, q, k, v, p, lo, hi, slope):
    """Attention of rows q [n, D] at positions p over k, v [m, D], by autograd-friendly steps."""
    z = torch.mm(q, k.t().contiguous()) * (1.0 / math.sqrt(case["D"]))
    if case["cap"]:
        z = case["cap"] * torch.tanh(z / case["cap"])
    j = torch.arange(k.shape[0], device=q.device)
    if slope is not None:
        z = z - slope * (p[:, None] - j).abs().double()
    see = (j >= lo[:, None]) & (j < hi[:, None])
    top = torch.where(see, z.detach(), -math.inf).amax(1, keepdim=True)
    e = torch.where(see, torch.exp(torch.where(see, z - top, 0.0)), 0.0)
    return torch.mm(e / e.sum(1, keepdim=True).clamp(min=0.5), v)


def _exact_attend(s):
    case = s["case"]
    b, h, kh, n, m = (case[x] for x in ("B", "H", "KH", "N", "M"))
    lo, hi = _limits(case, "cuda")
    p = torch.arange(n, device="cuda") + (m - n)
    new = lambda x: torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    o, dq, dk, dv = new(s["q"]), new(s["q"]), new(s["k"]), new(s["v"])
    step = max(1, (1 << 26) // m)
    for i in range(b):
        for c in range(h):
            slope = None if s["slopes"] is None else s["slopes"][c].double()
            for r in range(0, n, step):
                rows = slice(r, r + step)
                # (the keys that some row of the block sees)
                k0 = max(0, int(lo[i, rows].min()))
                k1 = max(k0 + 1, min(m, int(hi[i, rows].max())))
                q, k, v = (x.detach().double().requires_grad_(s["op"] == "train") for x in
                           (s["q"][i, c, rows], s["k"][i, c * kh // h, k0:k1], s["v"][i, c * kh // h, k0:k1]))
                y = _exact_head(case, q, k, v, p[rows] - k0, lo[i, rows] - k0, hi[i, rows] - k0, slope)
                o[i, c, rows] = y.detach()
                if s["op"] == "train":
                    gq, gk, gv = torch.autograd.grad(y, (q, k, v), s["do"][i, c, rows].double())
                    dq[i, c, rows] = gq
                    dk[i, c * kh // h, k0:k1] += gk
                    dv[i, c * kh // h, k0:k1] += gv
    return (o, dq, dk, dv) if s["op"] == "train" else o


def _exact_serve(s):
    case = s["case"]
    o = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    g, page, cu = case["H"] // case["KH"], case["page"], s["cu"].tolist()
    for i, n in enumerate(s["lens"].tolist()):
        ids = s["table"][i, :-(-n // page)].long()
        step = max(1, (1 << 25) // n)
        for c in range(case["H"]):
            k, v = (x[ids, c // g].reshape(-1, case["D"])[:n].double() for x in (s["kc"], s["vc"]))
            for r in range(cu[i], cu[i + 1], step):
                rows = torch.arange(r, min(r + step, cu[i + 1]), device="cuda")
                p = rows + n - cu[i + 1]
                lo = p - case["window"] + 1 if case["window"] else torch.zeros_like(p)
                slope = None if s["slopes"] is None else s["slopes"][c].double()
                o[rows, c] = _exact_head(case, s["q"][rows, c].double(), k, v, p, lo, p + 1, slope)
    return o


def _exact_rows(s, x, w, cos, sin):
    """Rows x [..., tokens, D] in 64 bits: unit rms, weights, and the rotation as complex numbers."""
    y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + _EPS) * w
    half = y.shape[-1] // 2
    a, b = (y[..., 0::2], y[..., 1::2]) if s["interleaved"] else (y[..., :half], y[..., half:])
    a, b = a * cos - b * sin, a * sin + b * cos
    return torch.stack((a, b), -1).flatten(-2) if s["interleaved"] else torch.cat((a, b), -1)


def _exact_angles(s):
    cos = torch.empty((s["pos"].shape[1], len(s["axes"])), dtype=torch.float64, device="cuda")
    sin = torch.empty_like(cos)
    for pair, axis in enumerate(s["axes"]):
        cos[:, pair] = s["cos"][s["pos"][axis].long(), pair].double()
        sin[:, pair] = s["sin"][s["pos"][axis].long(), pair].double()
    return cos, sin


def _exact_norm(s):
    cos, sin = _exact_angles(s)
    train = s["case"]["train"]
    out, grads, wgrads = [], [], []
    for x, w, dy in (("q", "qw", "dq"), ("k", "kw", "dk")):
        out.append(torch.empty(s[x].shape, dtype=torch.float64, device="cuda"))
        if train:
            grads.append(torch.empty_like(out[-1]))
            wgrads.append(torch.zeros(s["case"]["D"], dtype=torch.float64, device="cuda"))
        for i in range(s[x].shape[0]):
            for c in range(s[x].shape[1]):
                xd = s[x][i, c].detach().double().requires_grad_(train)
                wd = s[w].detach().double().requires_grad_(train)
                y = _exact_rows(s, xd, wd, cos, sin)
                out[-1][i, c] = y.detach()
                if train:
                    gx, gw = torch.autograd.grad(y, (xd, wd), s[dy][i, c].double())
                    grads[-1][i, c] = gx
                    wgrads[-1] += gw
    return (*out, *grads, *wgrads)


def _exact_store(s):
    cos, sin = _exact_angles(s)
    q, k = (_exact_rows(s, s[x].double().transpose(0, 1), s[w].double(), cos, sin).transpose(0, 1)
            for x, w in (("q", "qw"), ("k", "kw")))
    kc, vc = s["kc"].double(), s["vc"].double()
    cu, page = s["cu"].tolist(), s["case"]["page"]
    for i, n in enumerate(s["lens"].tolist()):
        at = torch.arange(n - (cu[i + 1] - cu[i]), n, device="cuda")
        ids = s["table"][i].long()[at // page]
        kc[ids, :, at % page] = k[cu[i]:cu[i + 1]]
        vc[ids, :, at % page] = s["v"][cu[i]:cu[i + 1]].double()
    return q, kc, vc


def exact(case, seed):
    s = prepare(case, seed)
    return {"train": _exact_attend, "attend": _exact_attend, "serve": _exact_serve, "norm": _exact_norm,
            "store": _exact_store}[s["op"]](s)
