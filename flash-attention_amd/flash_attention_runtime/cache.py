"""Operators around a paged key/value cache, and the q/k norm with rotation.

The cache is a pool of pages, ``[pages, kv_heads, page_size, head_dim]`` for
keys and for values (fp16 or bf16, head_dim 64 or 128, page_size a power of two
from 16 to 4096, any strides that are multiples of 8 with unit stride along
head_dim: a pool ``[pages, page_size, kv_heads, head_dim]`` is passed as
``pool.transpose(1, 2)``).  Key j of sequence b is row ``j % page_size`` of page
``block_table[b, j // page_size]``.

New tokens of all sequences are packed along the first dimension, oldest first:
rows ``cu_seqlens[b]`` to ``cu_seqlens[b + 1]`` are sequence b's, and
``seq_lens[b]`` counts its keys, these new ones included.  ``block_table``
[B, M], ``cu_seqlens`` [B + 1] and ``seq_lens`` [B] are int32 on the GPU; the
kernels check them as they read (a page id outside the pool is an absent page,
whose keys are masked; lengths are limited to ``max_kv`` and the table, offsets to
the rows).  ``cu_seqlens`` must not descend.  Rows that belong to no sequence are
left as they are.

A step of a server with a bounded cache::

    q = fa.paged_store(q, k, v, qw, kw, cos, sin, positions, kc, vc, table, cu, lens)
    o, lse = fa.paged_forward(q, kc, vc, table, cu, lens, max_q=n, return_lse=True)
    fa.paged_key_weights(q, lse, kc, table, cu, lens, weights, max_q=n)
    # now and then, for sequences that grew too long:
    lens, kept = fa.paged_evict(kc, vc, weights, table, lens, new_table, keep=4096, recent=256)

No call waits for the GPU; each may be captured into a graph and replayed with
other lengths and tables.  The cache's calls compute no gradients, and no call
carries forward-mode tangents on: inputs that ask for them are refused.
"""
from __future__ import annotations

import operator
from collections.abc import Sequence

import torch

from . import _C as _EXT


def paged_forward(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_table: torch.Tensor,
    cu_seqlens: torch.Tensor,
    seq_lens: torch.Tensor,
    out: torch.Tensor | None = None,
    *,
    max_q: int,
    max_kv: int | None = None,
    causal: bool = True,
    softmax_scale: float | None = None,
    return_lse: bool = False,
    softcap: float | None = None,
    window: int | None = None,
    slopes: torch.Tensor | None = None,
):
    """Attention of the new tokens ``q`` [T, H, D] over their sequences' keys.

    Query head h reads kv head ``h // (H / kv_heads)``.  With ``causal`` a token
    sees the keys up to its own, else all of its sequence.  ``max_q``: the most
    new tokens of any sequence (tokens past it are not computed); ``max_kv``:
    the most keys (default: what ``block_table`` holds).  They size the launch:
    decode splits sequences for ``max_kv`` keys, and one of 4000 takes 10.9 us
    with that limit, 32.8 with 131072.  A sequence of few tokens and far more
    keys than the others is not split where another has more than 32 rows (new
    tokens times heads per kv head): pass it in a call of its own.

    ``softcap``, ``window`` and ``slopes`` as in ``attention``, p being the token's key: scores
    become ``softcap * tanh(z / softcap)``, keys at a distance of ``window`` or more are neither
    seen nor read, and ``slopes`` (fp32 [H] on the GPU) times the distance is taken off.

    Returns ``o`` like q, or ``(o, lse)`` with the natural-log logsumexp, fp32
    [T, H], of these scores: ``paged_key_weights`` takes that of plain ones only.  A row
    without visible keys has o = 0 and lse = -inf.
    """
    res = _EXT.paged_forward(q, k_cache, v_cache, block_table, cu_seqlens, seq_lens, out, max_q,
                             max_kv, causal, softmax_scale, return_lse, softcap, window, slopes)
    if return_lse and (softcap is not None or slopes is not None or window is not None):
        # (plain scores where a window leaves all keys; a token without a place lies before the first)
        keys = block_table.shape[1] * k_cache.shape[2] if max_kv is None else max_kv
        if softcap is not None or slopes is not None or window < keys + (0 if causal else q.shape[0]):
            res[1]._fa_scores = "capped, biased or windowed"
    return res


def paged_key_weights(
    q: torch.Tensor,
    lse: torch.Tensor,
    k_cache: torch.Tensor,
    block_table: torch.Tensor,
    cu_seqlens: torch.Tensor,
    seq_lens: torch.Tensor,
    key_weights: torch.Tensor,
    *,
    max_q: int,
    max_kv: int | None = None,
    causal: bool = True,
    softmax_scale: float | None = None,
) -> torch.Tensor:
    """Adds to ``key_weights`` (fp32 [pages, kv_heads, page_size], in place) the
    attention weight each key receives from the new tokens: the sum over the
    query heads of its kv head and the tokens that see it of
    ``exp(scale q.k - lse)``.  ``q``, ``lse`` and the limits as given to and
    returned by ``paged_forward`` without ``softcap``, ``window`` and ``slopes``: there are no weights
    of such scores.  The ``lse`` that it returned with them is refused; nothing tells a copy or
    a part of it from another tensor.  The new tokens' own keys are set, not added
    to, so a reused page needs no clearing.  A page must belong to one sequence of
    the call only (sequences that share a prefix need weights of their own).  Returns ``key_weights``."""
    if getattr(lse, "_fa_scores", None) is not None:
        raise RuntimeError(f"paged_key_weights has plain scores only: this lse is of {lse._fa_scores} ones")
    _EXT.paged_key_weights(q, lse, k_cache, block_table, cu_seqlens, seq_lens, key_weights, max_q,
                           max_kv, causal, softmax_scale)
    return key_weights


def paged_evict(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    key_weights: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    new_table: torch.Tensor,
    *,
    keep: int,
    recent: int = 0,
    max_kv: int | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Keeps, per sequence and kv head, the ``recent`` last keys and of the others
    those of largest weight, ``keep`` in all; a shorter sequence keeps every
    key.  Equal weights: the lower index stays; NaN counts as the largest.

    The kept keys, values and weights are copied, in their order, to the pages
    of ``new_table`` [B, M'], each listed once and none read by this call; the old
    pages stay as they are, for the caller to reuse.  Pass the rows of the
    sequences to shorten.  Returns ``(new_lens, kept)``: int32 [B], and int32
    [B, kv_heads, keep] with the former index of the key now at each place (-1
    behind the last).  A sequence with an absent page is not copied (length 0).
    The two caches share no memory.
    """
    return _EXT.paged_evict(k_cache, v_cache, key_weights, block_table, seq_lens, new_table, keep,
                            recent, max_kv)


def _axes(axes) -> bytes | None:
    # (bytes(axes) would be an array's memory, and a number's many zeros)
    return axes if axes is None or isinstance(axes, bytes) else bytes(operator.index(a) for a in axes)


def paged_store(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    q_weight: torch.Tensor,
    k_weight: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    positions: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_table: torch.Tensor,
    cu_seqlens: torch.Tensor,
    seq_lens: torch.Tensor,
    out: torch.Tensor | None = None,
    *,
    eps: float = 1e-6,
    interleaved: bool = False,
    axes: bytes | Sequence[int] | None = None,
) -> torch.Tensor:
    """``qk_norm_rope`` of packed new tokens, ``q`` [T, H, D], ``k`` and ``v``
    [T, kv_heads, D], with k's result and v written to the tokens' places in the
    cache.  ``positions`` int32 [T] are the rows of the rotation's tables (after
    an eviction they run ahead of the places).  The pages that receive tokens
    must belong to one sequence only; tokens without a place (more tokens than
    keys, absent pages) are not stored.  ``axes`` as in ``qk_norm_rope``, with
    ``positions`` [A, T].  Returns q's result (``out`` if given, which may be q
    itself, row for row)."""
    return _EXT.paged_store(q, k, v, q_weight, k_weight, cos, sin, positions, k_cache, v_cache,
                            block_table, cu_seqlens, seq_lens, out, eps, interleaved, _axes(axes))


def qk_norm_rope(
    q: torch.Tensor,
    k: torch.Tensor,
    q_weight: torch.Tensor,
    k_weight: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    positions: torch.Tensor | None = None,
    *,
    eps: float = 1e-6,
    interleaved: bool = False,
    axes: bytes | Sequence[int] | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of each head's row of ``q`` [B, H, N, D] and ``k`` [B, H', N, D]
    with the weights [D] (fp32 or q's dtype), then the position rotation, in one
    pass: fp32 inside, one rounding at the end.

    ``cos`` and ``sin`` are fp32 [rows, r / 2] tables, r the rotated dims (a
    multiple of 16 up to D; the others keep their normed value).  The rotation
    turns the pairs (i, i + r/2), or (2i, 2i + 1) with ``interleaved``, by row
    ``positions`` (int32 [N] or [B, N]; default 0, 1, ...).  A position outside
    the tables gives NaN.

    ``axes``: a token has a position on each of A <= 4 axes (time, height, width),
    ``positions`` [A, N] or [A, B, N], and pair i turns by the position on axis
    ``axes[i]`` (r / 2 small integers; ``bytes`` are taken as they are).  It still
    uses column i of the tables: axes in blocks, in turn, or with frequencies of their
    own are a matter of ``axes`` and the tables.

    Returns new q and k in the layout of the inputs.  Differentiable once in q,
    k and the weights; cos and sin get no gradients.  (``forward`` computes none:
    a training step has ``attention`` behind this.)  In a graph capture a
    backward pass through leaves that an older autograd graph still holds is
    refused; ``qk_norm_rope_backward`` can always be captured.
    """
    return _EXT.qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, _axes(axes))


def qk_norm_rope_backward(
    dq_out: torch.Tensor,
    dk_out: torch.Tensor,
    q: torch.Tensor,
    k: torch.Tensor,
    q_weight: torch.Tensor,
    k_weight: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    positions: torch.Tensor | None = None,
    *,
    eps: float = 1e-6,
    interleaved: bool = False,
    axes: bytes | Sequence[int] | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """The gradients of ``qk_norm_rope`` for the gradients of its results, without
    autograd: ``(dq, dk, dq_weight, dk_weight)``.  The weights' gradients are
    summed in fp32 in a fixed order and have the weights' dtype."""
    return _EXT.qk_norm_rope_backward(dq_out, dk_out, q, k, q_weight, k_weight, cos, sin, positions,
                                      eps, interleaved, _axes(axes))
