"""CPU tests of the C ABI in include/fa_mi355x_attention.h: exports, struct layouts and every refusal of
the host-side checks, on addresses that are never read."""
from __future__ import annotations

import ctypes
import math
import os
import subprocess

import pytest

import abi_ctypes as A
import attention_ctypes as T
from test_cache_abi import PTR, ROWS4, fill, make as make_cache, put


@pytest.fixture(scope="module")
def lib():
    return T.load()


def test_exports_and_header(lib):
    names = A.declared_functions(T.HEADER)
    sized = {n + "_workspace_size" for n, (_, _, s) in T.ENTRIES.items() if s}
    assert set(names) == set(T.ENTRIES) | {n + "_validate" for n in T.ENTRIES} | sized
    out = subprocess.run(["nm", "-D", "--defined-only", A.LIB_PATH], capture_output=True, text=True, check=True).stdout
    assert set(names) <= {line.split()[-1] for line in out.splitlines() if " T " in line}


def test_struct_layouts(tmp_path):
    lines = []
    for cname, struct in T.STRUCTS.items():
        lines.append(f'printf("{cname} %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname}.{f} %zu\\n", offsetof({cname}, {f}));' for f, _ in struct._fields_]
    src = tmp_path / "probe.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "fa_mi355x_attention.h"\nint main(void){'
                   + "\n".join(lines) + "return 0;}\n")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(A.REPO_ROOT, "include"), str(src),
                    "-o", str(tmp_path / "probe")], check=True)
    got = dict(x.split() for x in subprocess.run([str(tmp_path / "probe")], capture_output=True, text=True,
                                                 check=True).stdout.splitlines())
    for cname, struct in T.STRUCTS.items():
        assert int(got[cname]) == ctypes.sizeof(struct), cname
        for f, _ in struct._fields_:
            assert int(got[f"{cname}.{f}"]) == getattr(struct, f).offset, (cname, f)


ATTN = dict(q_stride=ROWS4, k_stride=ROWS4, v_stride=ROWS4, o_stride=ROWS4, range_stride=16, batch=2, heads=4,
            kv_heads=2, seq_len=8, keys=8, head_dim=64, dtype=0, causal=1, softmax_scale=0.125,
            score__softcap=30.0, score__window=5)


def make(name):
    """The structs of a valid call."""
    if name == "fa_attn_fwd":
        return [fill(T.Attn(), **ATTN)]
    if name == "fa_attn_bwd":
        return [fill(T.AttnBwd(), **{"fwd__" + k: v for k, v in ATTN.items()}, go_stride=ROWS4, gq_stride=ROWS4,
                     gk_stride=ROWS4, gv_stride=ROWS4)]
    if name == "fa_paged_fwd_scored":
        return [make_cache("fa_paged_fwd"), fill(T.Score(), softcap=30.0, window=5)]
    axes = T.Axes(axes=3, axis_stride=10)
    for i in range(32):
        axes.axis[i] = i % 3
    plain = {"fa_qk_norm_rope_axes": "fa_qk_norm_rope", "fa_qk_norm_rope_bwd_axes": "fa_qk_norm_rope_bwd",
             "fa_paged_store_axes": "fa_paged_store"}[name]
    return [make_cache(plain), axes]


def refs(structs):
    return [None if s is None else ctypes.byref(s) for s in structs]


def validate(lib, name, structs):
    rc = getattr(lib, name + "_validate")(*refs(structs))
    return rc, lib.fa_last_error().decode()


@pytest.mark.parametrize("name", list(T.ENTRIES))
def test_valid_and_null(lib, name):
    assert validate(lib, name, make(name)) == (A.FA_OK, "")
    for i in range(len(make(name))):
        structs = make(name)
        structs[i] = None
        assert validate(lib, name, structs)[0] == A.FA_ERR_NULL


def test_valid_edges(lib):
    """What the header allows at its limits."""
    for field, value in [("ranges", None), ("range_stride", 0), ("score.slopes", None), ("score.window", 0),
                         ("score.window", 2 ** 31 - 1), ("score.softcap", 0.0), ("score.softcap", 1000.0), ("lse", None), ("o_low", None),
                         ("keys", 2 ** 22), ("k_stride", (0, 0, 0)), ("seq_len", 1), ("kv_heads", 4)]:
        s = make("fa_attn_fwd")[0]
        put(s, field, value)
        assert validate(lib, "fa_attn_fwd", [s])[0] == A.FA_OK, field


SCORE_BAD = [
    ("softcap", -1.0, A.FA_ERR_ARG), ("softcap", 1e-4, A.FA_ERR_ARG), ("softcap", 1001.0, A.FA_ERR_ARG),
    ("softcap", math.nan, A.FA_ERR_ARG), ("softcap", math.inf, A.FA_ERR_ARG), ("window", -1, A.FA_ERR_ARG),
    ("slopes", PTR + 2, A.FA_ERR_STRIDE),
]
ATTN_BAD = [
    ("dtype", 2, A.FA_ERR_DTYPE), ("head_dim", 96, A.FA_ERR_HEADDIM), ("batch", 0, A.FA_ERR_SHAPE),
    ("heads", 0, A.FA_ERR_SHAPE), ("kv_heads", 0, A.FA_ERR_SHAPE), ("kv_heads", 3, A.FA_ERR_SHAPE),
    ("seq_len", 0, A.FA_ERR_SHAPE), ("keys", 0, A.FA_ERR_SHAPE), ("seq_len", 2 ** 28 + 1, A.FA_ERR_UNSUPPORTED),
    ("keys", 2 ** 28 + 1, A.FA_ERR_UNSUPPORTED), ("batch", 2 ** 30, A.FA_ERR_UNSUPPORTED),
    ("q", None, A.FA_ERR_NULL), ("k", PTR + 8, A.FA_ERR_STRIDE), ("v", None, A.FA_ERR_NULL), ("o", None, A.FA_ERR_NULL),
    ("q_stride[0]", -64, A.FA_ERR_STRIDE), ("k_stride[2]", 68, A.FA_ERR_STRIDE),
    ("v_stride[2]", 2 ** 24 + 8, A.FA_ERR_UNSUPPORTED), ("q_stride[2]", 2 ** 24 + 8, A.FA_ERR_UNSUPPORTED),
    ("lse", PTR + 2, A.FA_ERR_STRIDE), ("o_low", PTR + 8, A.FA_ERR_STRIDE), ("ranges", PTR + 4, A.FA_ERR_STRIDE), ("range_stride", 3, A.FA_ERR_STRIDE),
    ("range_stride", -2, A.FA_ERR_STRIDE), ("causal", 2, A.FA_ERR_ARG), ("softmax_scale", 0.0, A.FA_ERR_ARG),
    ("softmax_scale", math.nan, A.FA_ERR_ARG), ("softmax_scale", 2e38, A.FA_ERR_ARG),
    ("softmax_scale", 1.5e-38, A.FA_OK),
    *[("score." + f, v, e) for f, v, e in SCORE_BAD],
]
AXES_BAD = [(1, "axes", 0, A.FA_ERR_ARG), (1, "axes", 5, A.FA_ERR_ARG), (1, "axes", 2, A.FA_ERR_ARG),
            (1, "axis[31]", 3, A.FA_ERR_ARG), (1, "axis_stride", -1, A.FA_ERR_STRIDE)]
BAD = {
    "fa_attn_fwd": [(0, *b) for b in ATTN_BAD] + [(0, "o_stride[1]", 0, A.FA_ERR_STRIDE)],
    "fa_attn_bwd": [(0, "fwd." + f, v, e) for f, v, e in ATTN_BAD] + [(0, *b) for b in [
        ("fwd.lse", None, A.FA_ERR_NULL), ("go", None, A.FA_ERR_NULL), ("go_stride[1]", 4, A.FA_ERR_STRIDE),
        ("go_stride[2]", 2 ** 24 + 8, A.FA_ERR_UNSUPPORTED), ("gq", None, A.FA_ERR_NULL), ("gk", PTR + 2, A.FA_ERR_STRIDE),
        ("gv_stride[2]", 0, A.FA_ERR_STRIDE), ("gq_stride[0]", 0, A.FA_ERR_STRIDE), ("glse", PTR + 2, A.FA_ERR_STRIDE)]],
    "fa_paged_fwd_scored": [(1, *b) for b in SCORE_BAD] + [
        (0, "softmax_scale", 0.0, A.FA_ERR_ARG), (0, "cache.page_size", 24, A.FA_ERR_SHAPE)],
    "fa_qk_norm_rope_axes": AXES_BAD + [(0, "positions", None, A.FA_ERR_NULL), (0, "rot", 24, A.FA_ERR_ARG)],
    "fa_qk_norm_rope_bwd_axes": AXES_BAD + [(0, "fwd.positions", None, A.FA_ERR_NULL), (0, "dq", None, A.FA_ERR_NULL)],
    "fa_paged_store_axes": AXES_BAD + [(0, "positions", None, A.FA_ERR_NULL), (0, "cache.k", None, A.FA_ERR_NULL)],
}


@pytest.mark.parametrize("name,i,field,value,expect", [(n, *b) for n, bad in BAD.items() for b in bad], ids=str)
def test_refusals(lib, name, i, field, value, expect):
    structs = make(name)
    put(structs[i], field, value)
    rc, text = validate(lib, name, structs)
    if expect == A.FA_OK:  # out of the plain scale's range with a cap beside it only
        assert rc == A.FA_ERR_ARG and "softcap" in text
        put(structs[i], field.replace("softmax_scale", "score.softcap"), 0.0)
        assert validate(lib, name, structs)[0] == A.FA_OK
        return
    assert rc == expect and text, (rc, text)
    # the call itself refuses the same way, before any HIP call
    _, ws, sizes = T.ENTRIES[name]
    f = getattr(lib, name)
    assert (f(*refs(structs), None, 0, None) if ws else f(*refs(structs), None)) == expect
    if sizes:
        n = ctypes.c_uint64(7)
        assert getattr(lib, name + "_workspace_size")(*refs(structs), ctypes.byref(n)) == expect and n.value == 0
