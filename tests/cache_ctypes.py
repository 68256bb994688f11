"""ctypes binding of include/fa_mi355x_cache.h, beside abi_ctypes."""
from __future__ import annotations

import ctypes
import os

import abi_ctypes as A

HEADER = os.path.join(A.REPO_ROOT, "include", "fa_mi355x_cache.h")
_p, _i32, _i64, _f = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float


def _struct(name, fields):
    return type(name, (ctypes.Structure,), {"_fields_": fields})


PagedCache = _struct("PagedCache", [
    ("k", _p), ("v", _p), ("k_stride", _i64 * 3), ("v_stride", _i64 * 3), ("block_table", _p),
    ("table_stride", _i64), ("cu_seqlens", _p), ("seq_lens", _p), ("batch", _i32), ("num_pages", _i32),
    ("page_size", _i32), ("max_pages", _i32), ("kv_heads", _i32), ("head_dim", _i32), ("dtype", _i32),
    ("reserved", _i32)])
PagedFwd = _struct("PagedFwd", [
    ("cache", PagedCache), ("q", _p), ("o", _p), ("lse", _p), ("q_stride", _i64 * 2),
    ("o_stride", _i64 * 2), ("tokens", _i32), ("heads", _i32), ("max_q", _i32), ("max_kv", _i32),
    ("softmax_scale", _f), ("causal", _i32)])
PagedWeights = _struct("PagedWeights", [
    ("cache", PagedCache), ("q", _p), ("lse", _p), ("key_weights", _p), ("q_stride", _i64 * 2),
    ("w_stride", _i64 * 2), ("tokens", _i32), ("heads", _i32), ("max_q", _i32), ("max_kv", _i32),
    ("softmax_scale", _f), ("causal", _i32)])
PagedEvict = _struct("PagedEvict", [
    ("cache", PagedCache), ("key_weights", _p), ("w_stride", _i64 * 2), ("new_table", _p),
    ("new_table_stride", _i64), ("new_lens", _p), ("kept", _p), ("new_pages", _i32), ("keep", _i32),
    ("recent", _i32), ("max_kv", _i32)])
QkNorm = _struct("QkNorm", [
    ("q", _p), ("k", _p), ("q_out", _p), ("k_out", _p), ("q_stride", _i64 * 3), ("k_stride", _i64 * 3),
    ("q_out_stride", _i64 * 3), ("k_out_stride", _i64 * 3), ("q_weight", _p), ("k_weight", _p),
    ("cos", _p), ("sin", _p), ("positions", _p), ("pos_stride", _i64), ("batch", _i32), ("heads", _i32),
    ("kv_heads", _i32), ("seq_len", _i32), ("head_dim", _i32), ("rot", _i32), ("table_rows", _i32),
    ("interleaved", _i32), ("dtype", _i32), ("weight_fp32", _i32), ("eps", _f)])
QkNormBwd = _struct("QkNormBwd", [
    ("fwd", QkNorm), ("dq", _p), ("dk", _p), ("dq_stride", _i64 * 3), ("dk_stride", _i64 * 3),
    ("dq_weight", _p), ("dk_weight", _p)])
PagedStore = _struct("PagedStore", [
    ("cache", PagedCache), ("q", _p), ("k", _p), ("v", _p), ("q_out", _p), ("q_stride", _i64 * 2),
    ("k_stride", _i64 * 2), ("v_stride", _i64 * 2), ("q_out_stride", _i64 * 2), ("q_weight", _p),
    ("k_weight", _p), ("cos", _p), ("sin", _p), ("positions", _p), ("tokens", _i32), ("heads", _i32),
    ("rot", _i32), ("table_rows", _i32), ("interleaved", _i32), ("weight_fp32", _i32), ("eps", _f)])

# C struct name, entry point's stem, whether it takes a workspace
ENTRIES = {
    "fa_paged_fwd": (PagedFwd, "fa_paged_fwd_params", True),
    "fa_paged_key_weights": (PagedWeights, "fa_paged_weights_params", True),
    "fa_paged_evict": (PagedEvict, "fa_paged_evict_params", False),
    "fa_qk_norm_rope": (QkNorm, "fa_qk_norm_params", False),
    "fa_qk_norm_rope_bwd": (QkNormBwd, "fa_qk_norm_bwd_params", True),
    "fa_paged_store": (PagedStore, "fa_paged_store_params", False),
}


def load(path: str = A.LIB_PATH):
    L = A.load(path)
    for name, (struct, _, ws) in ENTRIES.items():
        P = ctypes.POINTER(struct)
        getattr(L, name + "_validate").argtypes = [P]
        getattr(L, name).argtypes = [P, _p, ctypes.c_uint64, _p] if ws else [P, _p]
        if ws:
            getattr(L, name + "_workspace_size").argtypes = [P, ctypes.POINTER(ctypes.c_uint64)]
    return L
