"""Build properties of the cache's and the norm's gfx950 kernels, from the device
assembly that hipcc emits with the library's flags (CPU only): no scratch, no
VGPR spills, registers and LDS for the occupancy their comments count on, m0
used by the staging DMA alone, no packed fp32 arithmetic."""
from __future__ import annotations

import os
import re
import subprocess
import sys

import pytest

from test_kernel_resources import REPO, _kernel_metadata

sys.path.insert(0, os.path.join(REPO, "flash-attention_amd"))


@pytest.fixture(scope="module", params=["fa_paged_fwd.hip", "fa_paged_cache.hip", "fa_qk_norm.hip"])
def asm(request, tmp_path_factory):
    import build as fa_build

    try:
        hipcc = fa_build._hipcc()
    except RuntimeError:
        pytest.skip("hipcc not available")
    out = str(tmp_path_factory.mktemp("asm") / "k.s")
    flags = [f for f in fa_build.HIP_FLAGS if f not in ("-fPIC", "-Wall")]
    r = subprocess.run([hipcc, *flags, "-I", fa_build.INCLUDE, "-I", fa_build.CSRC, "-x", "hip",
                        "--cuda-device-only", "-S", os.path.join(fa_build.CSRC, request.param), "-o", out],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    return request.param, open(out).read()


def test_registers_and_lds(asm):
    name, text = asm
    kernels = _kernel_metadata(text)
    assert kernels
    for k, f in kernels:
        assert int(f["private_segment_fixed_size"]) == 0, (k, "scratch")
        assert int(f["vgpr_spill_count"]) == 0, (k, "VGPR spills")
        if "chunk_kernel" in k:  # two waves per SIMD, two workgroups per CU
            assert int(f["vgpr_count"]) <= 256 and int(f.get("agpr_count", 0)) == 0, k
            assert int(f["group_segment_fixed_size"]) <= 80 * 1024, k
        else:
            assert int(f["vgpr_count"]) <= 512, k
            assert int(f["group_segment_fixed_size"]) <= 160 * 1024, k


def test_m0_and_packed_fp32(asm):
    _, text = asm
    code = [ln.strip() for ln in text.splitlines()]
    code = [ln for ln in code if ln and not ln.startswith((";", "."))]
    for i, ln in enumerate(code):
        assert not re.match(r"v_pk_(add|mul|fma)_f32", ln), ln
        if re.search(r"\bm0\b", ln):
            assert re.fullmatch(r"s_mov_b32 m0, s\d+", ln), ln
            assert code[i + 1].startswith("global_load_lds_dwordx4"), code[i + 1]
