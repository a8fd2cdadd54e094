"""Build-time guard of the register budgets that the kernels over pages in 8 bits and over shared prefixes are tuned to (CPU only: hipcc cross-compiles for gfx950)."""
from concurrent.futures import ThreadPoolExecutor

import pytest

from test_kernel_resources import _compile, _pick

UNITS = ["fa_paged_decode_8bit.hip", "fa_paged_chunk_8bit.hip", "fa_paged_prefix.hip", "fa_paged_prefix_8bit.hip", "fa_paged_append.hip", "fa_paged_read.hip"]


@pytest.mark.timeout(600)
def test_kernels_over_8_bits_and_prefixes_keep_their_waves_per_simd():
    with ThreadPoolExecutor(len(UNITS)) as pool:
        units = dict(zip(UNITS, pool.map(_compile, UNITS)))
    want = [  # unit, kernel, waves per SIMD, most spilled registers
        ("fa_paged_decode_8bit.hip", "fa_paged_decode_8bit_kernelIDF16bLi128ELi4E", 2, 0), ("fa_paged_decode_8bit.hip", "fa_paged_decode_8bit_kernelIDF16_Li64ELi8E", 2, 0),
        ("fa_paged_decode_8bit.hip", "fa_paged_decode_8bit_kernelIDF16_Li64ELi4E", 3, 0), ("fa_paged_decode_8bit.hip", "fa_paged_decode_8bit_kernelIDF16bLi32ELi4E", 4, 0),
        ("fa_paged_chunk_8bit.hip", "fa_paged_chunk_8bit_kernelIDF16bLi128ELb0E", 2, 0), ("fa_paged_chunk_8bit.hip", "fa_paged_chunk_8bit_kernelIDF16bLi128ELb1E", 2, 0),
        ("fa_paged_chunk_8bit.hip", "fa_paged_chunk_8bit_kernelIDF16_Li64ELb0E", 3, 0), ("fa_paged_chunk_8bit.hip", "fa_paged_chunk_8bit_kernelIDF16_Li64ELb1E", 2, 0),
        ("fa_paged_prefix.hip", "fa_paged_prefix_kernelIDF16bLi128ELb0ELb0E", 2, 0), ("fa_paged_prefix.hip", "fa_paged_prefix_kernelIDF16_Li64ELb1ELb0E", 2, 0),
        ("fa_paged_prefix_8bit.hip", "fa_paged_prefix_kernelIDF16bLi128ELb0ELb1E", 2, 0), ("fa_paged_prefix_8bit.hip", "fa_paged_prefix_kernelIDF16_Li64ELb0ELb1E", 3, 0),
        # (the second sum, for lse: the third wave for some registers parked across the main loop)
        ("fa_paged_prefix_8bit.hip", "fa_paged_prefix_kernelIDF16_Li64ELb1ELb1E", 3, 10),
        ("fa_paged_append.hip", "paged_append_8bit_kernelIDF16_Li64ELi4E", 5, 0), ("fa_paged_read.hip", "paged_read_kernelIDF16bLi128ELi4ELb1E", 7, 0)]
    for unit, kernel, waves, spilled in want:
        k = _pick(units[unit], kernel)
        assert k["Occupancy"] >= waves and k["VGPRs Spill"] <= spilled, (kernel, k)
