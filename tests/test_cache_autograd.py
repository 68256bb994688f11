"""CPU tests: derivatives that a call would drop are refused, before anything else
is looked at (the tensors here are on the CPU, which is refused next)."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd

z = torch.zeros


def arguments():
    half = lambda *s: z(*s).half()  # noqa: E731
    i32 = lambda *s: z(*s).int()  # noqa: E731
    cache = dict(block_table=i32(1, 1), seq_lens=i32(1))
    packed = dict(cu_seqlens=i32(2), **cache)
    pools = dict(k_cache=half(1, 1, 16, 64), v_cache=half(1, 1, 16, 64))
    norm = dict(q_weight=z(64), k_weight=z(64), cos=z(4, 32), sin=z(4, 32))
    heads = dict(q=half(1, 1, 4, 64), k=half(1, 1, 4, 64))
    return {
        "paged_forward": dict(q=half(1, 1, 64), out=half(1, 1, 64), max_q=1, **pools, **packed),
        "paged_key_weights": dict(q=half(1, 1, 64), lse=z(1, 1), k_cache=half(1, 1, 16, 64), key_weights=z(1, 1, 16),
                                  max_q=1, **packed),
        "paged_evict": dict(key_weights=z(1, 1, 16), new_table=i32(1, 1), keep=16, **pools, **cache),
        "paged_store": dict(q=half(1, 1, 64), k=half(1, 1, 64), v=half(1, 1, 64), out=half(1, 1, 64), positions=i32(1),
                            **norm, **pools, **packed),
        "qk_norm_rope": dict(**heads, **norm),
        "qk_norm_rope_backward": dict(dq_out=half(1, 1, 4, 64), dk_out=half(1, 1, 4, 64), **heads, **norm),
    }


CASES = [(n, a) for n, args in arguments().items() for a, t in args.items()
         if torch.is_tensor(t) and t.is_floating_point()]


@pytest.mark.parametrize("name,arg", CASES)
def test_forward_mode_tangents_are_refused(fa, name, arg):
    args = arguments()[name]
    with fwd.dual_level():
        args[arg] = fwd.make_dual(args[arg], torch.ones_like(args[arg]))
        for grad in (True, False):  # no_grad does not stop forward mode
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                getattr(fa, name)(**args)
        with torch.inference_mode(), pytest.raises(RuntimeError, match="CUDA tensor"):
            getattr(fa, name)(**args)
        args[arg] = fwd.unpack_dual(args[arg]).primal
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            getattr(fa, name)(**args)


@pytest.mark.parametrize("name,arg", [(n, a) for n, a in CASES if n.startswith("paged")])
def test_gradients_that_a_call_would_drop_are_refused(fa, name, arg):
    args = arguments()[name]
    args[arg].requires_grad_()
    with pytest.raises(RuntimeError, match="no gradients"):
        getattr(fa, name)(**args)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA tensor"):
        getattr(fa, name)(**args)
