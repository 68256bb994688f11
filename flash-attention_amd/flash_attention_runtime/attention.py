"""Attention with gradients, whose scores may be capped, biased by distance and masked.

``attention`` takes whole tensors [B, H, N, D] as ``forward`` does, with fewer key/value heads, other
key lengths and these options, in autograd or without; a training step runs ``qk_norm_rope`` in front of
it.  ``paged_forward`` takes the same ``softcap``, ``window`` and ``slopes`` over a paged cache.

    ranges = fa.document_ranges(cu_seqlens, n)            # documents packed in a row, once per batch
    q, k = fa.qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions)
    o = fa.attention(q, k, v, ranges, softcap=50.0)
    o.backward(do)
"""
from __future__ import annotations

import torch

from . import _C as _EXT


def attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    key_ranges: torch.Tensor | None = None,
    *,
    causal: bool = False,
    window: int | None = None,
    softcap: float | None = None,
    slopes: torch.Tensor | None = None,
    softmax_scale: float | None = None,
    return_lse: bool = False,
):
    """Attention of ``q`` [B, H, N, D] over ``k`` and ``v`` [B, H', M, D] (fp16 or bf16, D 64 or 128, H a
    multiple of H', unit stride along D and other strides multiples of 8).

    Row i stands at p = i + M - N among the keys.  Its score of key j is z = scale q.k, then
    ``softcap * tanh(z / softcap)``, then less ``slopes[h] * |p - j|`` (fp32 [H] on the GPU).  It sees

    - the keys ``key_ranges[b, i, 0] <= j < key_ranges[b, i, 1]`` (int32 [N, 2] or [B, N, 2] on the
      GPU, read by the kernels: any values; see ``document_ranges``),
    - with ``causal`` those up to p, with ``window`` those at |p - j| < window.

    Returns ``o`` like q, or ``(o, lse)`` with the natural-log logsumexp, fp32 [B, H, N].  A row that
    sees no key has o = 0, lse = -inf and no gradients; keys that a row does not see contribute
    nothing to it, whatever they hold.

    Differentiable once in q, k and v, through o and lse; slopes get no gradient.  Besides its
    arguments and results a graph holds one more tensor like o, what rounding left out of it.  The
    same call gives the same bits, gradients included.  In a graph capture a backward pass through leaves that
    an older autograd graph still holds is refused (of q, k and v that are leaves themselves: what made others
    of them is not looked at); ``attention_backward`` can always be captured.
    """
    return _EXT.attention(q, k, v, key_ranges, causal, window, softcap, slopes, softmax_scale, return_lse)


def attention_backward(
    do: torch.Tensor,
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    o: torch.Tensor,
    lse: torch.Tensor,
    key_ranges: torch.Tensor | None = None,
    *,
    causal: bool = False,
    window: int | None = None,
    softcap: float | None = None,
    slopes: torch.Tensor | None = None,
    softmax_scale: float | None = None,
    dlse: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The gradients ``(dq, dk, dv)`` of ``attention`` for o's gradient ``do`` (and lse's, ``dlse``), without
    autograd; ``o`` and ``lse`` as it returned them for the same arguments.  With the rounded o alone dq
    and dk are up to a third less exact than autograd's where few keys have most of the weight."""
    return _EXT.attention_backward(do, q, k, v, o, lse, key_ranges, causal, window, softcap, slopes,
                                   softmax_scale, dlse)


def document_ranges(
    cu_seqlens: torch.Tensor,
    n: int,
    *,
    causal: bool = True,
    prefix_lens: torch.Tensor | None = None,
) -> torch.Tensor:
    """``key_ranges`` [n, 2] of documents packed in a row of n tokens, document d from ``cu_seqlens[d]`` to
    ``cu_seqlens[d + 1]`` (ascending, on any device; the result is on the same).  A token sees the tokens
    of its document up to itself (all of them with ``causal=False``), and the first ``prefix_lens[d]`` ones.
    Tokens outside the documents see nothing.  Computed once per batch, for all layers."""
    if cu_seqlens.dim() != 1:
        raise RuntimeError("cu_seqlens must have one dimension")
    if prefix_lens is not None and (prefix_lens.dim() != 1 or prefix_lens.shape[0] < cu_seqlens.shape[0] - 1):
        raise RuntimeError("prefix_lens must have one entry per document")
    cu = cu_seqlens.to(torch.int64)
    i = torch.arange(n, device=cu.device)
    if cu.shape[0] < 2:
        return torch.zeros((n, 2), dtype=torch.int32, device=cu.device)
    doc = torch.searchsorted(cu[1:].contiguous(), i, right=True)
    inside = (doc < cu.shape[0] - 1) & (i >= cu[0])
    doc = doc.clamp(max=cu.shape[0] - 2)
    start, end = cu[doc], cu[doc + 1]
    hi = torch.minimum(i + 1, end) if causal else end
    if prefix_lens is not None:
        hi = torch.maximum(hi, torch.minimum(start + prefix_lens.to(cu)[doc], end))
    ranges = torch.stack((start, hi), dim=1)
    return torch.where(inside[:, None], ranges, 0).to(torch.int32)
