"""CPU tests of the largest sizes that the cache's calls take: row numbers of whole
tiles past the last row stay below 2^31 in the kernels."""
from __future__ import annotations

import pytest

import abi_ctypes as A
import cache_ctypes as C
from test_cache_abi import make, put, validate


@pytest.fixture(scope="module")
def lib():
    return C.load()


@pytest.mark.parametrize("name", ["fa_paged_fwd", "fa_paged_key_weights"])
@pytest.mark.parametrize("tokens,expect", [(2 ** 31 - 256, A.FA_OK), (2 ** 31 - 255, A.FA_ERR_UNSUPPORTED),
                                           (2 ** 31 - 1, A.FA_ERR_UNSUPPORTED)])
def test_rows_of_packed_queries(lib, name, tokens, expect):
    s = make(name)
    s.heads = s.cache.kv_heads = 1
    s.tokens = tokens
    assert validate(lib, name, s)[0] == expect


@pytest.mark.parametrize("name,prefix", [("fa_qk_norm_rope", ""), ("fa_qk_norm_rope_bwd", "fwd.")])
@pytest.mark.parametrize("seq_len,expect", [(2 ** 31 - 256, A.FA_OK), (2 ** 31 - 255, A.FA_ERR_UNSUPPORTED),
                                            (2 ** 31 - 1, A.FA_ERR_UNSUPPORTED)])
def test_tokens_of_the_norm(lib, name, prefix, seq_len, expect):
    s = make(name)
    for field, v in (("batch", 1), ("heads", 1), ("kv_heads", 1), ("seq_len", seq_len)):
        put(s, prefix + field, v)
    assert validate(lib, name, s)[0] == expect
