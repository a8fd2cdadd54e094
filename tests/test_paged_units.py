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
