"""What the calls that write in place owe autograd: a tensor that a graph has saved
and that a call then overwrites is noticed by that graph's backward pass."""
from __future__ import annotations

import pytest
import torch

from test_gpu_paged_forward import Cache, cu_of
from test_gpu_qk_norm import tables

pytestmark = pytest.mark.gpu
DEV = "cuda"


def setup():
    c = Cache([40, 20], 16, 1, 64, torch.float16, 800)
    k, v, table = c.dev()
    nt = torch.tensor([[int(c.k.shape[0])], [int(c.k.shape[0]) + 1]], dtype=torch.int32, device=DEV)
    k, v = (torch.cat([x, torch.zeros(2, 1, 16, 64, device=DEV).half()]).nan_to_num() for x in (k, v))
    w = torch.rand(k.shape[:3], device=DEV)
    g = torch.Generator(device=DEV).manual_seed(3)
    q, kn, vn = (torch.randn(5, h, 64, generator=g, device=DEV).half() for h in (2, 1, 1))
    one, (cos, sin) = torch.ones(64, device=DEV), (t.to(DEV) for t in tables(40, 64))
    pos = torch.arange(5, dtype=torch.int32, device=DEV)
    return dict(k=k, v=v, w=w, q=q, kn=kn, vn=vn, one=one, cos=cos, sin=sin, pos=pos, table=table, nt=nt,
                cu=cu_of([3, 2]).to(DEV), lens=c.lens.to(DEV), out=torch.zeros_like(q))


def call(fa, name, s):
    """Runs an operator; the tensors that it writes."""
    cache = (s["k"], s["v"], s["table"], s["cu"], s["lens"])
    if name == "paged_forward":
        fa.paged_forward(s["q"], *cache, s["out"], max_q=3)
        return [s["out"]]
    if name == "paged_store":
        fa.paged_store(s["q"], s["kn"], s["vn"], s["one"], s["one"], s["cos"], s["sin"], s["pos"], *cache, s["out"])
        return [s["k"], s["v"], s["out"]]
    if name == "paged_key_weights":
        fa.paged_key_weights(s["q"], torch.ones(5, 2, device=DEV), s["k"], s["table"], s["cu"], s["lens"], s["w"],
                             max_q=3)
        return [s["w"]]
    fa.paged_evict(s["k"], s["v"], s["w"], s["table"], s["lens"], s["nt"], keep=16)
    return [s["k"], s["v"], s["w"]]


CALLS = ["paged_forward", "paged_store", "paged_key_weights", "paged_evict"]


@pytest.mark.parametrize("name", CALLS)
def test_written_tensors_get_a_new_version(fa, name):
    s = setup()
    before = {n: t._version for n, t in s.items()}
    written = call(fa, name, s)
    for n, t in s.items():
        assert (t._version > before[n]) == any(t is x for x in written), n


@pytest.mark.parametrize("name", CALLS)
def test_a_graph_notices_that_what_it_saved_was_overwritten(fa, name):
    s = setup()
    for n in ("k", "out", "w"):
        x = torch.ones_like(s[n], requires_grad=True)
        y = (x * s[n]).float().sum()  # saves s[n]
        if any(t is s[n] for t in call(fa, name, s)):
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                y.backward()
        else:
            y.backward()


def test_a_store_in_place_is_noticed_by_the_norm_before_it(fa):
    """qk_norm_rope saves q; paged_store(out=q) then overwrites it."""
    s = setup()
    w = torch.ones(64, device=DEV, requires_grad=True)
    q4, k4 = s["q"].transpose(0, 1)[None], s["kn"].transpose(0, 1)[None]
    y, _ = fa.qk_norm_rope(q4, k4, w, w, s["cos"], s["sin"])
    fa.paged_store(s["q"], s["kn"], s["vn"], s["one"], s["one"], s["cos"], s["sin"], s["pos"], s["k"], s["v"],
                   s["table"], s["cu"], s["lens"], s["q"])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.float().sum().backward()


@pytest.mark.parametrize("name", CALLS)
def test_tensors_made_in_inference_mode_are_written_outside_it(fa, name):
    """They have no versions; a cache made in inference mode serves both ways."""
    with torch.inference_mode():
        s = setup()
        call(fa, name, s)
    with torch.no_grad():
        call(fa, name, s)
    torch.cuda.synchronize()
