"""Build properties of the kernels of attention with gradients and of scored attention over the cache, from
the device assembly that hipcc emits with the library's flags (CPU only): no scratch, no VGPR spills, the
registers and LDS of the workgroups per CU that their comments count on, m0 used by the staging copies alone, no
packed fp32 arithmetic."""
from __future__ import annotations

import os
import re
import subprocess
import sys

import pytest

from test_cache_kernel_occupancy import GRANULE, LDS, REGS, SIMDS
from test_kernel_resources import REPO, _kernel_metadata

sys.path.insert(0, os.path.join(REPO, "flash-attention_amd"))

# kernels (template arguments as in the mangled name): threads, workgroups per CU
WANT = {
    "fa_attention_fwd.hip": [(r"fa_attn_fwd_kernel.*ELi1EEE", 256, 2), (r"fa_attn_fwd_kernel.*ELi2EEE", 512, 1)],
    "fa_attention_bwd.hip": [(r"fa_attn_rows_kernel", 256, 4), (r"fa_attn_order_kernel", 1024, 1),
                             (r"fa_attn_dkv_kernelILi128.*ELi1EEE", 256, 2), (r"fa_attn_dkv_kernelILi128.*ELi2EEE", 512, 1),
                             (r"fa_attn_dkv_kernelILi64.*ELi1EEE", 256, 3), (r"fa_attn_dkv_kernelILi64.*ELi3EEE", 768, 1),
                             (r"fa_attn_dq_kernelILi128.*ELi1EEE", 256, 2), (r"fa_attn_dq_kernelILi64.*ELi1EEE", 256, 3),
                             (r"fa_attn_dq_kernel.*ELi2EEE", 512, 1),
                             (r"fa_attn_join_kernel", 256, 4)],
    "fa_paged_scored.hip": [(r"fa_paged_chunk_kernel", 256, 2), (r"fa_paged_decode_kernelILi\d+ELb\dELi\dELi2E", 128, 2),
                            (r"fa_paged_decode_kernelILi\d+ELb\dELi\dELi4E", 256, 1), (r"fa_paged_merge_kernel", 256, 4)],
}


@pytest.fixture(scope="module", params=list(WANT))
def asm(request, tmp_path_factory):
    import build as fa_build

    try:
        hipcc = fa_build._hipcc()
    except RuntimeError:
        pytest.skip("hipcc not available")
    out = str(tmp_path_factory.mktemp("asm") / "k.s")
    flags = [f for f in fa_build.HIP_FLAGS if f not in ("-fPIC", "-Wall")]
    r = subprocess.run([hipcc, *flags, "-I", fa_build.INCLUDE, "-I", fa_build.CSRC, "-x", "hip", "--cuda-device-only",
                        "-S", os.path.join(fa_build.CSRC, request.param), "-o", out], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    return request.param, open(out).read()


def test_registers_lds_and_workgroups_per_cu(asm):
    name, text = asm
    kernels = _kernel_metadata(text)
    matched = set()
    for pattern, threads, workgroups in WANT[name]:
        found = [(k, f) for k, f in kernels if re.search(pattern, k)]
        assert found, pattern
        waves = -(-threads // 64 * workgroups // SIMDS)
        for k, f in found:
            matched.add(k)
            assert int(f["private_segment_fixed_size"]) == 0, (k, "scratch")
            assert int(f["vgpr_spill_count"]) == 0, (k, "VGPR spills")
            assert int(f["max_flat_workgroup_size"]) == threads, k
            assert int(f["vgpr_count"]) <= REGS // waves // GRANULE * GRANULE, (k, f["vgpr_count"])
            assert int(f["group_segment_fixed_size"]) * workgroups <= LDS, k
    assert matched == {k for k, _ in kernels}


def test_m0_and_packed_fp32(asm):
    _, text = asm
    code = [ln.strip() for ln in text.splitlines()]
    code = [ln for ln in code if ln and not ln.startswith((";", "."))]
    for i, ln in enumerate(code):
        assert not re.match(r"v_pk_(add|mul|fma)_f32", ln), ln
        if re.search(r"\bm0\b", ln):
            assert re.fullmatch(r"s_mov_b32 m0, s\d+", ln), ln
            assert code[i + 1].startswith("global_load_lds_dwordx4"), code[i + 1]
