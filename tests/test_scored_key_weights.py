"""paged_key_weights has plain scores only: a logsumexp of capped, biased or windowed ones would make weights
of any size out of them, by which paged_evict then decides."""
from __future__ import annotations

import pytest
import torch


def test_a_marked_logsumexp_is_refused_before_anything_is_read(fa):
    lse = torch.zeros(3, 2)
    lse._fa_scores = "capped, biased or windowed"
    with pytest.raises(RuntimeError, match="plain scores only"):
        fa.paged_key_weights(None, lse, None, None, None, None, None, max_q=1)


@pytest.mark.gpu
def test_the_logsumexp_of_other_scores_is_refused(fa):
    print("case scored key weights", flush=True)
    g = torch.Generator(device="cuda").manual_seed(60)
    H, KH, D, page, n = 4, 2, 64, 16, 40
    k, v = (torch.randn(4, KH, page, D, generator=g, device="cuda").half() for _ in range(2))
    q = torch.randn(2, H, D, generator=g, device="cuda").half()
    table = torch.tensor([[1, 2, 3]], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")

    def weights(**scores):
        w = torch.zeros(4, KH, page, device="cuda")
        o, lse = fa.paged_forward(q, k, v, table, cu, lens, max_q=2, return_lse=True, **scores)
        return fa.paged_key_weights(q, lse, k, table, cu, lens, w, max_q=2)

    want = weights()
    # each of two tokens and two heads gives its keys a weight of 1 in all
    assert torch.allclose(want[1:].sum((0, 2)), torch.full((KH,), 4.0, device="cuda"), atol=1e-3)
    for scores in (dict(softcap=2.0), dict(window=8), dict(slopes=torch.ones(H, device="cuda")),
                   dict(softcap=50.0, window=4096), dict(window=47)):
        with pytest.raises(RuntimeError, match="plain scores only"):
            weights(**scores)
    # a window of all keys leaves plain scores
    for window in (48, 2 ** 40):
        assert torch.equal(weights(window=window), want)
