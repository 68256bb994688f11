"""What attention's and the rotation's Python entry points make of their arguments before any kernel: CPU only."""
from __future__ import annotations

import pytest
import torch


@pytest.mark.parametrize("prefix", [[], [1], [1, 2], [[1, 2, 3]], 1])
def test_prefix_lens_has_one_entry_per_document(fa, prefix):
    """Too few of them would be an index past their end, on the GPU an assertion that ends the process."""
    cu = torch.tensor([0, 4, 6, 9])
    with pytest.raises(RuntimeError, match="one entry per document"):
        fa.document_ranges(cu, 9, prefix_lens=torch.tensor(prefix))
    want = fa.document_ranges(cu, 9, prefix_lens=torch.tensor([2, 0, 3]))
    assert torch.equal(fa.document_ranges(cu, 9, prefix_lens=torch.tensor([2, 0, 3, 7])), want)  # (and more, unused)


@pytest.mark.parametrize("cu", [[[0, 4], [0, 5]], 3])
def test_cu_seqlens_has_one_dimension(fa, cu):
    with pytest.raises(RuntimeError, match="one dimension"):
        fa.document_ranges(torch.tensor(cu), 5)


def test_no_documents(fa):
    for cu in ([], [0]):
        assert fa.document_ranges(torch.tensor(cu, dtype=torch.int32), 2).tolist() == [[0, 0], [0, 0]]


def test_axes_are_read_one_by_one(fa):
    """Integers of any sequence, an entry each: never the bytes of an array's memory, nor a number of zeros."""
    import numpy as np

    from flash_attention_runtime import cache

    want = bytes([0, 2, 1, 3, 0, 1, 2, 3])
    for axes in (list(want), tuple(want), want, bytearray(want), torch.tensor(list(want)),
                 *(np.array(list(want), dtype=t) for t in (np.int64, np.int32, np.uint8))):
        assert cache._axes(axes) == want, type(axes)
    assert cache._axes(None) is None
    for bad, error in ((8, TypeError), ("0213", TypeError), ([0.5] * 8, TypeError), ([-1] * 8, ValueError),
                       ([256] * 8, ValueError)):
        with pytest.raises(error):
            cache._axes(bad)
