"""Build-time guard of what the attention kernels over pages are compiled into (CPU only: hipcc cross-compiles for gfx950): every route's registers, and nothing twice."""
from concurrent.futures import ThreadPoolExecutor

import pytest

from test_kernel_resources import _compile, _pick

UNITS = ["fa_paged_chunk.hip", "fa_paged_chunk_8bit.hip", "fa_paged_decode.hip", "fa_paged_decode_8bit.hip"]


@pytest.fixture(scope="module")
def units():
    with ThreadPoolExecutor(len(UNITS)) as pool:
        return dict(zip(UNITS, pool.map(_compile, UNITS)))


@pytest.mark.timeout(600)
def test_the_parts_of_a_chunk_are_joined_by_one_kernel(units):
    """it joins fp32 parts, whatever the cache holds: compiled once for each dtype and head dim"""
    joins = [k for unit in ("fa_paged_chunk.hip", "fa_paged_chunk_8bit.hip") for k in units[unit] if "join" in k]
    assert len(joins) == 8 and all(k in units["fa_paged_chunk.hip"] for k in joins)


@pytest.mark.timeout(600)
def test_wide_workgroups_that_read_past_the_caches_keep_their_waves_per_simd(units):
    want = [  # unit, kernel, waves per SIMD; nothing spilled
        ("fa_paged_decode.hip", "paged_decode_wide_stream_kernelIDF16_Li64E", 2), ("fa_paged_decode.hip", "paged_decode_wide_stream_kernelIDF16bLi128E", 1),
        ("fa_paged_decode.hip", "paged_decode_wide_stream_kernelIDF16bLi32E", 2), ("fa_paged_decode.hip", "paged_decode_wide_stream_kernelIDF16_Li16E", 2),
        ("fa_paged_decode_8bit.hip", "paged_decode_wide_stream_8bit_kernelIDF16_Li128E", 2), ("fa_paged_decode_8bit.hip", "paged_decode_wide_stream_8bit_kernelIDF16bLi128E", 2),
        ("fa_paged_decode_8bit.hip", "paged_decode_wide_stream_8bit_kernelIDF16bLi64E", 3), ("fa_paged_decode_8bit.hip", "paged_decode_wide_stream_8bit_kernelIDF16_Li32E", 4),
        ("fa_paged_decode_8bit.hip", "paged_decode_wide_stream_8bit_kernelIDF16bLi16E", 4)]
    for unit, kernel, waves in want:
        k = _pick(units[unit], kernel)
        assert k["Occupancy"] >= waves and k["VGPRs Spill"] == 0, (kernel, k)
