"""The layout of positions with axes, [A, B, N], also where there are as many axes as batch entries."""
from __future__ import annotations

import pytest
import torch

from test_gpu_qk_norm import inputs, tables, weights

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_the_axes_come_before_the_batch_entries(fa):
    print("case order", flush=True)
    q, k, *_ = (t.to(DEV) for t in inputs(2, 2, 1, 8, 64, torch.float16, 33))
    qw, kw = (w.to(DEV) for w in weights(64, torch.float32, 34))
    cos, sin = (t.to(DEV) for t in tables(40, 64))
    pos = torch.arange(32, dtype=torch.int32, device=DEV).view(2, 2, 8)
    axes = [i % 2 for i in range(32)]
    both = fa.qk_norm_rope(q, k, qw, kw, cos, sin, pos, axes=axes)
    for b in range(2):
        one = fa.qk_norm_rope(q[b:b + 1], k[b:b + 1], qw, kw, cos, sin, pos[:, b].contiguous(), axes=axes)
        for x, y in zip(both, one):
            assert torch.equal(x[b], y[0])
