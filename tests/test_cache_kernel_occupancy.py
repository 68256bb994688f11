"""The registers and LDS that each of the cache's and the norm's kernels may take for
the workgroups per CU that its comments and the launch plans count on (CPU only,
from the device assembly)."""
from __future__ import annotations

import re

from test_cache_kernel_resources import asm  # noqa: F401  (the fixture)
from test_kernel_resources import _kernel_metadata

LDS, REGS, GRANULE, SIMDS = 160 * 1024, 512, 8, 4

# kernels (template arguments as in the mangled name): threads, workgroups per CU
WANT = {
    "fa_paged_fwd.hip": [
        (r"fa_paged_chunk_kernel", 256, 2),
        (r"fa_paged_decode_kernelILi\d+ELb\dELi\dELi2E", 128, 2),
        (r"fa_paged_decode_kernelILi\d+ELb\dELi\dELi4E", 256, 1),
        (r"fa_paged_merge_kernel", 256, 4),
    ],
    "fa_paged_cache.hip": [
        (r"fa_weights_kernel", 256, 3),
        (r"fa_weights_few_kernel", 128, 4),
        (r"fa_weights_sum_kernel", 256, 4),
        (r"fa_select_kernel", 1024, 1),
        (r"fa_move_kernel", 256, 4),
    ],
    "fa_qk_norm.hip": [
        (r"fa_norm_kernel", 256, 4),
        (r"fa_norm_bwd_kernel", 256, 4),
        (r"fa_norm_dw_kernel", 256, 1),
    ],
}


def test_workgroups_per_cu(asm):  # noqa: F811
    name, text = asm
    kernels = _kernel_metadata(text)
    matched = set()
    for pattern, threads, workgroups in WANT[name]:
        found = [(k, f) for k, f in kernels if re.search(pattern, k)]
        assert found, pattern
        waves = -(-threads // 64 * workgroups // SIMDS)  # of a SIMD
        regs = REGS // waves // GRANULE * GRANULE
        for k, f in found:
            matched.add(k)
            assert int(f["max_flat_workgroup_size"]) == threads, k
            assert int(f["vgpr_count"]) <= regs, (k, f["vgpr_count"], regs)
            assert int(f["group_segment_fixed_size"]) * workgroups <= LDS, k
    assert matched == {k for k, _ in kernels}
