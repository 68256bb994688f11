"""CPU tests of the C ABI in include/fa_mi355x_cache.h: exports, struct layouts and
every refusal of the host-side checks, on addresses that are never read."""
from __future__ import annotations

import ctypes
import math
import os
import re
import subprocess

import pytest

import abi_ctypes as A
import cache_ctypes as C

PTR = 0x10000


@pytest.fixture(scope="module")
def lib():
    return C.load()


def test_exports_and_header(lib):
    names = A.declared_functions(C.HEADER)
    assert set(names) >= set(C.ENTRIES) | {n + "_validate" for n in C.ENTRIES}
    out = subprocess.run(["nm", "-D", "--defined-only", A.LIB_PATH], capture_output=True, text=True,
                         check=True).stdout
    exported = {line.split()[-1] for line in out.splitlines() if " T " in line}
    assert set(names) <= exported


def test_struct_layouts(tmp_path):
    """Sizes and field offsets of the ctypes structs against the C compiler's."""
    text = open(C.HEADER).read()
    lines = []
    for struct, cname, _ in list(C.ENTRIES.values()) + [(C.PagedCache, "fa_paged_cache", False)]:
        assert re.search(r"\}\s*" + cname + ";", text)
        lines.append(f'printf("{cname} %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname}.{f} %zu\\n", offsetof({cname}, {f}));' for f, _ in struct._fields_]
    src = tmp_path / "probe.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "fa_mi355x_cache.h"\nint main(void){'
                   + "\n".join(lines) + "return 0;}\n")
    exe = tmp_path / "probe"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(A.REPO_ROOT, "include"),
                    str(src), "-o", str(exe)], check=True)
    got = dict(x.split() for x in subprocess.run([str(exe)], capture_output=True, text=True,
                                                 check=True).stdout.splitlines())
    for struct, cname, _ in list(C.ENTRIES.values()) + [(C.PagedCache, "fa_paged_cache", False)]:
        assert int(got[cname]) == ctypes.sizeof(struct), cname
        for f, _ in struct._fields_:
            assert int(got[f"{cname}.{f}"]) == getattr(struct, f).offset, (cname, f)


def fill(s, **kw):
    """Every pointer set, then the given fields (dotted names reach into structs)."""
    def pointers(x):
        for f, t in x._fields_:
            if t is ctypes.c_void_p:
                setattr(x, f, PTR)
            elif isinstance(getattr(x, f), ctypes.Structure):
                pointers(getattr(x, f))

    pointers(s)
    for name, v in kw.items():
        put(s, name.replace("__", "."), v)
    return s


def put(s, name, v):
    *path, last = name.split(".")
    for p in path:
        s = getattr(s, p)
    if "[" in last:
        f, i = last[:-1].split("[")
        getattr(s, f)[int(i)] = v
    elif isinstance(v, (list, tuple)):
        for i, x in enumerate(v):
            getattr(s, last)[i] = x
    else:
        setattr(s, last, v)


CACHE = dict(cache__k_stride=(2 * 16 * 64, 16 * 64, 64), cache__v_stride=(2 * 16 * 64, 16 * 64, 64),
             cache__table_stride=4, cache__batch=3, cache__num_pages=9, cache__page_size=16,
             cache__max_pages=4, cache__kv_heads=2, cache__head_dim=64, cache__dtype=1)
NORM = dict(rot=64, table_rows=10, interleaved=0, weight_fp32=1, eps=1e-6)
ROWS4 = (4 * 8 * 64, 8 * 64, 64)


def make(name):
    if name == "fa_paged_fwd":
        return fill(C.PagedFwd(), **CACHE, q_stride=(256, 64), o_stride=(256, 64), tokens=5, heads=4,
                    max_q=2, max_kv=64, softmax_scale=0.125, causal=1)
    if name == "fa_paged_key_weights":
        return fill(C.PagedWeights(), **CACHE, q_stride=(256, 64), w_stride=(32, 16), tokens=5, heads=4,
                    max_q=2, max_kv=64, softmax_scale=0.125, causal=1)
    if name == "fa_paged_evict":
        s = fill(C.PagedEvict(), **CACHE, w_stride=(32, 16), new_table_stride=2, new_pages=2, keep=20,
                 recent=4, max_kv=64)
        s.new_table = PTR + 64
        return s
    if name == "fa_paged_store":
        return fill(C.PagedStore(), **CACHE, **NORM, q_stride=(256, 64), k_stride=(128, 64),
                    v_stride=(128, 64), q_out_stride=(256, 64), tokens=5, heads=4)
    norm = dict(q_stride=ROWS4, k_stride=ROWS4, q_out_stride=ROWS4, k_out_stride=ROWS4, pos_stride=0,
                batch=2, heads=4, kv_heads=4, seq_len=8, head_dim=64, dtype=0, **NORM)
    if name == "fa_qk_norm_rope":
        return fill(C.QkNorm(), **norm)
    return fill(C.QkNormBwd(), **{"fwd__" + k: v for k, v in norm.items()}, dq_stride=ROWS4, dk_stride=ROWS4)


def validate(lib, name, s):
    rc = getattr(lib, name + "_validate")(ctypes.byref(s) if s is not None else None)
    return rc, lib.fa_last_error().decode()


@pytest.mark.parametrize("name", list(C.ENTRIES))
def test_valid_and_null(lib, name):
    assert validate(lib, name, make(name)) == (A.FA_OK, "")
    assert validate(lib, name, None)[0] == A.FA_ERR_NULL


CACHE_BAD = [
    ("cache.dtype", 2, A.FA_ERR_DTYPE), ("cache.head_dim", 96, A.FA_ERR_HEADDIM),
    ("cache.batch", -1, A.FA_ERR_SHAPE), ("cache.num_pages", 0, A.FA_ERR_SHAPE),
    ("cache.max_pages", 0, A.FA_ERR_SHAPE), ("cache.kv_heads", 0, A.FA_ERR_SHAPE),
    ("cache.page_size", 8, A.FA_ERR_SHAPE), ("cache.page_size", 24, A.FA_ERR_SHAPE),
    ("cache.page_size", 8192, A.FA_ERR_SHAPE), ("cache.max_pages", 2 ** 27, A.FA_ERR_UNSUPPORTED),
    ("cache.k", None, A.FA_ERR_NULL), ("cache.k", PTR + 8, A.FA_ERR_STRIDE),
    ("cache.k_stride[0]", -64, A.FA_ERR_STRIDE), ("cache.k_stride[1]", 1028, A.FA_ERR_STRIDE),
    ("cache.k_stride[2]", 56, A.FA_ERR_STRIDE), ("cache.k_stride[2]", 2 ** 24 + 8, A.FA_ERR_UNSUPPORTED),
    ("cache.block_table", None, A.FA_ERR_NULL), ("cache.block_table", PTR + 2, A.FA_ERR_STRIDE),
    ("cache.seq_lens", None, A.FA_ERR_NULL), ("cache.table_stride", 3, A.FA_ERR_STRIDE),
]
VALUES_BAD = [
    ("cache.v", None, A.FA_ERR_NULL), ("cache.v", PTR + 2, A.FA_ERR_STRIDE),
    ("cache.v_stride[1]", -8, A.FA_ERR_STRIDE), ("cache.v_stride[2]", 2 ** 24 + 8, A.FA_ERR_UNSUPPORTED),
]
WRITTEN_BAD = [("cache.k_stride[0]", 0, A.FA_ERR_STRIDE), ("cache.v_stride[1]", 56, A.FA_ERR_STRIDE),
               # heads' last rows overlap the next page's first, though every stride spans a row
               ("cache.k_stride[0]", 2 * 16 * 64 - 64, A.FA_ERR_STRIDE), ("cache.v_stride[1]", 64, A.FA_ERR_STRIDE)]
QUERY_BAD = [
    ("cache.cu_seqlens", None, A.FA_ERR_NULL), ("tokens", -1, A.FA_ERR_SHAPE), ("heads", 0, A.FA_ERR_SHAPE),
    ("heads", 3, A.FA_ERR_SHAPE), ("max_q", -1, A.FA_ERR_ARG), ("max_kv", -1, A.FA_ERR_ARG),
    ("causal", 2, A.FA_ERR_ARG), ("softmax_scale", 0.0, A.FA_ERR_ARG), ("softmax_scale", 1e-39, A.FA_ERR_ARG),
    ("softmax_scale", math.nan, A.FA_ERR_ARG), ("softmax_scale", 2e38, A.FA_ERR_ARG),
    ("tokens", 2 ** 30, A.FA_ERR_UNSUPPORTED), ("cache.batch", 2 ** 23, A.FA_ERR_UNSUPPORTED),
    ("q", None, A.FA_ERR_NULL), ("q", PTR + 4, A.FA_ERR_STRIDE), ("q_stride[0]", 100, A.FA_ERR_STRIDE),
    ("lse", PTR + 2, A.FA_ERR_STRIDE),
]
TABLES_BAD = [
    ("q_weight", None, A.FA_ERR_NULL), ("k_weight", PTR + 8, A.FA_ERR_STRIDE), ("cos", None, A.FA_ERR_NULL),
    ("sin", PTR + 4, A.FA_ERR_STRIDE), ("rot", 0, A.FA_ERR_ARG), ("rot", 24, A.FA_ERR_ARG),
    ("rot", 80, A.FA_ERR_ARG), ("table_rows", 0, A.FA_ERR_SHAPE), ("interleaved", 2, A.FA_ERR_ARG),
    ("weight_fp32", -1, A.FA_ERR_ARG), ("eps", -1.0, A.FA_ERR_ARG), ("eps", math.inf, A.FA_ERR_ARG),
]
NORM_BAD = [
    ("dtype", 3, A.FA_ERR_DTYPE), ("head_dim", 32, A.FA_ERR_HEADDIM), ("batch", 0, A.FA_ERR_SHAPE),
    ("kv_heads", 0, A.FA_ERR_SHAPE), ("seq_len", 0, A.FA_ERR_SHAPE), ("batch", 2 ** 29, A.FA_ERR_UNSUPPORTED),
    ("q", None, A.FA_ERR_NULL), ("k_stride[2]", 68, A.FA_ERR_STRIDE), ("k_out", PTR + 8, A.FA_ERR_STRIDE),
    ("q_out", None, A.FA_ERR_NULL), ("positions", PTR + 1, A.FA_ERR_STRIDE), ("pos_stride", -1, A.FA_ERR_STRIDE),
]
BAD = {
    "fa_paged_fwd": CACHE_BAD + VALUES_BAD + QUERY_BAD + [("o", None, A.FA_ERR_NULL), ("o_stride[1]", 0, A.FA_ERR_STRIDE)],
    "fa_paged_key_weights": CACHE_BAD + QUERY_BAD + [
        ("lse", None, A.FA_ERR_NULL), ("key_weights", None, A.FA_ERR_NULL), ("key_weights", PTR + 2, A.FA_ERR_STRIDE),
        ("w_stride[0]", 8, A.FA_ERR_STRIDE), ("w_stride[1]", 15, A.FA_ERR_STRIDE), ("w_stride[0]", 16, A.FA_ERR_STRIDE),
        ("q_stride[0]", 2 ** 24 + 8, A.FA_ERR_UNSUPPORTED), ("q_stride[1]", 2 ** 28 + 8, A.FA_ERR_UNSUPPORTED)],
    "fa_paged_evict": CACHE_BAD + VALUES_BAD + WRITTEN_BAD + [
        ("key_weights", None, A.FA_ERR_NULL), ("w_stride[1]", 8, A.FA_ERR_STRIDE), ("keep", 0, A.FA_ERR_ARG),
        ("keep", 2 ** 30 + 1, A.FA_ERR_UNSUPPORTED),
        ("recent", 21, A.FA_ERR_ARG), ("recent", -1, A.FA_ERR_ARG), ("max_kv", -1, A.FA_ERR_ARG),
        ("keep", 33, A.FA_ERR_SHAPE), ("new_pages", 0, A.FA_ERR_SHAPE), ("new_table", None, A.FA_ERR_NULL),
        ("new_lens", None, A.FA_ERR_NULL), ("kept", PTR + 2, A.FA_ERR_STRIDE), ("new_table_stride", 1, A.FA_ERR_STRIDE),
        ("new_table", PTR, A.FA_ERR_ARG), ("cache.batch", 2 ** 23, A.FA_ERR_UNSUPPORTED)],
    "fa_paged_store": CACHE_BAD + VALUES_BAD + WRITTEN_BAD + TABLES_BAD + [
        ("cache.cu_seqlens", None, A.FA_ERR_NULL), ("tokens", -1, A.FA_ERR_SHAPE), ("heads", 0, A.FA_ERR_SHAPE),
        ("q", None, A.FA_ERR_NULL), ("k_stride[0]", 4, A.FA_ERR_STRIDE), ("v", PTR + 2, A.FA_ERR_STRIDE),
        ("q_out_stride[0]", 32, A.FA_ERR_STRIDE), ("positions", None, A.FA_ERR_NULL)],
    "fa_qk_norm_rope": NORM_BAD + TABLES_BAD + [("q_out_stride[0]", 0, A.FA_ERR_STRIDE)],
    "fa_qk_norm_rope_bwd": [("fwd." + f, v, e) for f, v, e in NORM_BAD + TABLES_BAD] + [
        ("dq", None, A.FA_ERR_NULL), ("dk_stride[1]", 0, A.FA_ERR_STRIDE), ("dq_weight", None, A.FA_ERR_NULL),
        ("dk_weight", PTR + 2, A.FA_ERR_STRIDE)],
}


@pytest.mark.parametrize("name,field,value,expect", [(n, *b) for n, bad in BAD.items() for b in bad],
                         ids=lambda x: str(x))
def test_refusals(lib, name, field, value, expect):
    s = make(name)
    put(s, field, value)
    rc, text = validate(lib, name, s)
    assert rc == expect and text, (rc, text)
    # the call itself refuses the same way, before any HIP call
    ws = C.ENTRIES[name][2]
    f = getattr(lib, name)
    assert (f(ctypes.byref(s), None, 0, None) if ws else f(ctypes.byref(s), None)) == expect
    if ws:
        n = ctypes.c_uint64(7)
        assert getattr(lib, name + "_workspace_size")(ctypes.byref(s), ctypes.byref(n)) == expect
        assert n.value == 0


@pytest.mark.parametrize("name", ["fa_paged_fwd", "fa_paged_key_weights", "fa_paged_evict", "fa_paged_store"])
def test_no_sequences_need_no_tables(lib, name):
    s = make(name)
    s.cache.batch = 0
    s.cache.block_table = s.cache.seq_lens = s.cache.cu_seqlens = None
    assert validate(lib, name, s)[0] == A.FA_OK
    ws = C.ENTRIES[name][2]
    f = getattr(lib, name)  # nothing to do: no HIP call
    assert (f(ctypes.byref(s), None, 0, None) if ws else f(ctypes.byref(s), None)) == A.FA_OK


@pytest.mark.parametrize("name", ["fa_paged_fwd", "fa_paged_key_weights", "fa_paged_store"])
def test_no_tokens_need_no_rows(lib, name):
    s = make(name)
    s.tokens = 0
    s.q = None
    ws = C.ENTRIES[name][2]
    f = getattr(lib, name)
    assert (f(ctypes.byref(s), None, 0, None) if ws else f(ctypes.byref(s), None)) == A.FA_OK


def test_strides_of_single_entries_do_not_matter(lib):
    s = make("fa_paged_store")
    s.cache.num_pages = s.cache.kv_heads = 1
    s.cache.k_stride[0] = s.cache.k_stride[1] = s.cache.v_stride[0] = s.cache.v_stride[1] = 0
    assert validate(lib, "fa_paged_store", s)[0] == A.FA_OK


def test_workspace_needs_a_place_for_its_size(lib):
    for name, (_, _, ws) in C.ENTRIES.items():
        if ws:
            s = make(name)
            assert getattr(lib, name + "_workspace_size")(ctypes.byref(s), None) == A.FA_ERR_NULL


def test_calls_on_the_cpu_are_refused_by_the_package(fa):
    import torch

    z = torch.zeros
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        fa.paged_forward(z(1, 1, 64).half(), z(1, 1, 16, 64).half(), z(1, 1, 16, 64).half(),
                         z(1, 1).int(), z(2).int(), z(1).int(), max_q=1)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        fa.qk_norm_rope(z(1, 1, 4, 64).half(), z(1, 1, 4, 64).half(), z(64), z(64), z(4, 32), z(4, 32))
