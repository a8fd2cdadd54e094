"""Build-time guard of the register budgets that the paged cache's kernels are tuned to (CPU only: hipcc cross-compiles for gfx950)."""
from concurrent.futures import ThreadPoolExecutor

import pytest

from test_kernel_resources import _compile, _pick

UNITS = ["fa_paged_decode.hip", "fa_paged_chunk.hip", "fa_paged_weights.hip", "fa_norm.hip", "fa_paged_append.hip", "fa_paged_evict.hip"]


@pytest.mark.timeout(600)
def test_paged_kernels_keep_their_waves_per_simd():
    with ThreadPoolExecutor(len(UNITS)) as pool:
        units = dict(zip(UNITS, pool.map(_compile, UNITS)))
    want = [  # unit, kernel, waves per SIMD, most spilled registers
        ("fa_paged_decode.hip", "fa_paged_decode_kernelIDF16_Li64ELi2E", 3, 0), ("fa_paged_decode.hip", "fa_paged_decode_kernelIDF16_Li64ELi8E", 2, 0),
        ("fa_paged_decode.hip", "fa_paged_decode_kernelIDF16bLi128ELi2E", 1, 0), ("fa_paged_decode.hip", "fa_paged_decode_kernelIDF16_Li32ELi4E", 4, 0),
        # (without lse: the last wave for a few registers that are parked across the main loop)
        ("fa_paged_chunk.hip", "fa_paged_chunk_kernelIDF16bLi128ELb0E", 3, 10), ("fa_paged_chunk.hip", "fa_paged_chunk_kernelIDF16_Li64ELb0E", 4, 6),
        ("fa_paged_chunk.hip", "fa_paged_chunk_kernelIDF16bLi128ELb1E", 2, 0), ("fa_paged_chunk.hip", "fa_paged_chunk_kernelIDF16_Li64ELb1E", 3, 0),
        ("fa_paged_weights.hip", "fa_paged_weights_kernelIDF16_Li64ELi128E", 4, 8), ("fa_paged_weights.hip", "fa_paged_weights_few_kernelIDF16_Li64E", 4, 0),
        ("fa_paged_weights.hip", "fa_paged_weights_kernelIDF16bLi128ELi64E", 4, 8), ("fa_paged_weights.hip", "fa_paged_weights_few_kernelIDF16bLi128E", 2, 0),
        ("fa_norm.hip", "qk_norm_rotary_kernelIDF16bLi128ELb1ELi4E", 5, 0), ("fa_norm.hip", "qk_norm_rotary_bwd_kernelIDF16bLi128ELb1E", 4, 0),
        ("fa_paged_append.hip", "paged_append_kernelIDF16_Li64ELi4E", 5, 0)]
    for unit, kernel, waves, spilled in want:
        k = _pick(units[unit], kernel)
        assert k["Occupancy"] >= waves and k["VGPRs Spill"] <= spilled, (kernel, k)
    # matrix products stay out of the accumulation registers where there is room beside them
    for unit, kernel in (("fa_paged_decode.hip", "fa_paged_decode_kernelIDF16_Li64ELi2E"), ("fa_paged_weights.hip", "fa_paged_weights_kernelIDF16_Li64ELi128E"),
                         ("fa_paged_weights.hip", "fa_paged_weights_few_kernelIDF16bLi128E")):
        assert _pick(units[unit], kernel)["AGPRs"] == 0, kernel
    for k in units["fa_paged_evict.hip"].values():
        assert k["VGPRs Spill"] == 0
