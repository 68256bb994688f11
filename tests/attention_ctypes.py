"""ctypes binding of include/fa_mi355x_attention.h, beside abi_ctypes and cache_ctypes."""
from __future__ import annotations

import ctypes
import os

import abi_ctypes as A
import cache_ctypes as C
from cache_ctypes import _struct

HEADER = os.path.join(A.REPO_ROOT, "include", "fa_mi355x_attention.h")
_p, _i32, _i64, _f = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float

Score = _struct("Score", [("softcap", _f), ("window", _i32), ("slopes", _p)])
Attn = _struct("Attn", [
    ("q", _p), ("k", _p), ("v", _p), ("o", _p), ("lse", _p), ("o_low", _p), ("q_stride", _i64 * 3), ("k_stride", _i64 * 3),
    ("v_stride", _i64 * 3), ("o_stride", _i64 * 3), ("ranges", _p), ("range_stride", _i64), ("batch", _i32),
    ("heads", _i32), ("kv_heads", _i32), ("seq_len", _i32), ("keys", _i32), ("head_dim", _i32), ("dtype", _i32),
    ("causal", _i32), ("softmax_scale", _f), ("score", Score)])
AttnBwd = _struct("AttnBwd", [
    ("fwd", Attn), ("go", _p), ("glse", _p), ("gq", _p), ("gk", _p), ("gv", _p), ("go_stride", _i64 * 3),
    ("gq_stride", _i64 * 3), ("gk_stride", _i64 * 3), ("gv_stride", _i64 * 3)])
Axes = _struct("Axes", [("axis", ctypes.c_uint8 * 64), ("axes", _i32), ("axis_stride", _i64)])

STRUCTS = {"fa_score_params": Score, "fa_attn_params": Attn, "fa_attn_bwd_params": AttnBwd, "fa_rotary_axes": Axes}
# entry point: its parameter structs, whether it takes a workspace, whether it sizes one
ENTRIES = {
    "fa_attn_fwd": ((Attn,), False, False),
    "fa_attn_bwd": ((AttnBwd,), True, True),
    "fa_paged_fwd_scored": ((C.PagedFwd, Score), True, True),
    "fa_qk_norm_rope_axes": ((C.QkNorm, Axes), False, False),
    "fa_qk_norm_rope_bwd_axes": ((C.QkNormBwd, Axes), True, False),
    "fa_paged_store_axes": ((C.PagedStore, Axes), False, False),
}


def load(path: str = A.LIB_PATH):
    L = C.load(path)
    for name, (structs, ws, sizes) in ENTRIES.items():
        P = [ctypes.POINTER(s) for s in structs]
        getattr(L, name + "_validate").argtypes = P
        getattr(L, name).argtypes = [*P, _p, ctypes.c_uint64, _p] if ws else [*P, _p]
        if sizes:
            getattr(L, name + "_workspace_size").argtypes = [*P, ctypes.POINTER(ctypes.c_uint64)]
    return L
