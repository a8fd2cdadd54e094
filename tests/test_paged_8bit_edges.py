"""The paged cache in 8 bits and shared prefixes: bits of scores, layouts of partial results, where prefixes are shared.

Tolerances are counted, not measured: u half a step of the element type, e = 2^-24 a rounding in fp32 (see test_paged.py)."""
import ctypes
import math

import pytest
import torch

from test_paged import E32, Cache, cumulative
from test_paged import _args as paged_args
from test_paged_8bit import DTYPES, Cache8, _prefix, _scales, check_attention, randn, ref_quantise, share


# ---- GPU: bits of scores

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [16, 32, 64, 128])
@pytest.mark.parametrize("sizes", [[300.0], [2.0 ** -8, 1.0, 2.0 ** 14]])
def test_lse_of_one_key_over_8_bits(lib, D, dtype, sizes):
    """lse = scale q.k, whatever the value's exponent is: a score loses no bits to it.  q has one element that is not 0, a power of two, so that q.k is exact."""
    from flash_attn import flash_attn_paged_interface as p
    B, HK, scale = 96, 2, 0.5
    c = Cache8([1] * B, HK, D, 16, dtype, 3)
    v = torch.tensor(sizes, dtype=torch.float64)[torch.arange(c.n_pages * 16 * HK) % len(sizes)].view(c.n_pages, 16, HK, 1).expand(-1, -1, -1, D)
    y, e = ref_quantise(v, dtype)
    c.v, c.vc, c.vs = y.to(dtype), (y * (2.0 ** -e.double())[..., None]).float().to(torch.float8_e4m3fn).view(torch.uint8), (e + 127).to(torch.uint8).transpose(1, 2).contiguous()
    c.v, c.vc = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (c.v, c.vc))
    c.gpu()
    q = torch.zeros(B, HK, D, dtype=dtype)
    q[torch.arange(B), :, torch.arange(B) % D] = 4.0
    out, lse = p.flash_attn_paged_func(q.cuda(), c.dk, c.dv, c.dtable, cumulative([1] * B).cuda(), c.dlens, 1, 1, softmax_scale=scale, return_softmax_lse=True, **c.scales)
    page = c.table[:, 0].long()
    s = (q.double() * c.k[page, 0].double()).sum(-1) * scale
    assert torch.equal(out.cpu().double(), c.v[page, 0].double())
    # In log2 units, x = |s log2 e|, E = the exponent's distance from the one that is added as 0 (16 at most in fp16, none in bf16): log2 e and its product with the scale (2
    # roundings), the argument (1), the maximum's way back (1), the sum with log2 of 2^E, itself off by a step of E at most (2), ln 2 and its product (2)
    far = 16 if dtype == torch.float16 else 0
    x = s.abs() * math.log2(math.e)
    bound = math.log(2) * E32 * (2 * x + (x + far) + (x + far + 1) + (x + 1) + 2 * far + 2 * x)
    err = (lse[:, :, 0].cpu().double() - s).abs()
    assert (err <= bound).all(), (err / bound).max()


# ---- parts of a shared prefix: rows that are no multiple of four

def prefix_call(be, batch, H, HK, D, total, prefix, max_k, groups=1, new=1, always=1):
    """A call's structs, of which nothing is read but the numbers"""
    a = paged_args(be, "fwd")
    c = a.cache
    c.head_dim, c.nheads_k, c.nheads_q, c.page_size, c.batch, c.total_q, c.max_seqlen_q, c.max_seqlen_k = D, HK, H, 64, batch, total, new, max_k
    c.table_cols = c.table_row_stride = 4000
    return a, _prefix(be, n_groups=groups, max_prefix_len=prefix, always=always)


@pytest.mark.parametrize("D", [16, 32, 64, 128])
def test_parts_of_a_prefix_begin_at_16_bytes(lib, D):
    """a row's part is D + 3 floats: a split's rows are counted up to a multiple of four"""
    from flash_attn import flash_attn_gfx950 as be

    def scratch(total, HK=1):
        a, x = prefix_call(be, 5, HK, HK, D, total, 1024, 1100, new=4)
        return lib.fa_paged_fwd_with_workspace_bytes(ctypes.byref(a), None, ctypes.byref(x))

    assert scratch(5) == scratch(6) == scratch(8) and scratch(9) > scratch(8)
    assert scratch(7, HK=3) == scratch(8, HK=3) and scratch(8) % 16 == 0


def test_parts_of_pairs_behind_a_prefix_have_the_rows_of_the_call(lib):
    """a part for every pair, of as many rows as a pair has and not of the 32 that it may have; a row is D elements, m, l, u and what brings the next one to 16 bytes"""
    from flash_attn import flash_attn_gfx950 as be

    def scratch(batch, HK=32, G=1, new=1, D=128):
        a, x = prefix_call(be, batch, HK * G, HK, D, 64, 2048, 2100, new=new)  # (64 rows whatever the batch is: only the pairs' parts grow with it)
        return lib.fa_paged_fwd_with_workspace_bytes(ctypes.byref(a), None, ctypes.byref(x))

    for more, rows in ((dict(), 1), (dict(new=5), 5), (dict(HK=8, G=4), 4), (dict(HK=8, G=4, new=3), 12), (dict(HK=4, G=8, new=4), 32), (dict(D=16, G=3, new=3), 9)):
        each = more.get("HK", 32) * rows * (more.get("D", 128) + 4) * 4
        assert scratch(1024, **more) - scratch(256, **more) == 768 * each, more


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("H, HK, D, new", [(1, 1, 128, [1, 1, 1, 1, 1]), (3, 3, 64, [1, 2, 1, 1]), (6, 2, 16, [1, 1, 1]), (5, 5, 32, [2, 1, 0, 2]), (1, 1, 64, [3, 4])])
def test_parts_of_a_prefix_of_odd_numbers_of_rows(lib, H, HK, D, new, eight, dtype):
    from flash_attn import flash_attn_gfx950 as be
    B = len(new)
    c = share((Cache8 if eight else Cache)([1024 + 20 * i + 5 for i in range(B)], HK, D, 64, dtype, 3, **(dict(spread=0.5) if eight else {})), [B], [1024]).gpu()
    q = randn(sum(new), H, D, dtype=dtype, seed=5)
    pl = torch.full((B,), 1024, dtype=torch.int32).cuda()
    out, lse = be.paged_fwd(q.cuda(), c.dk, c.dv, c.dtable, cumulative(new).cuda(), c.dlens, max(new), max(c.lens), D ** -0.5, True, True, cu_groups=cumulative([B]).cuda(),
                            prefix_lens=pl, max_prefix_len=1024, always=True, **(c.scales if eight else {}))
    check_attention(q, c, new, True, out, lse)


# ---- where prefixes are shared

@pytest.mark.parametrize("eight, HK, G, D, batch, groups, prefix, shares", [
    # each line: what was measured, us shared / alone
    (False, 12, 1, 64, 16, 1, 2048, False),   # 18.5 / 15.9, 19.7 / 17.3
    (False, 12, 1, 64, 2, 1, 8192, False),    # 18.1 / 16.3, 17.6 / 17.1
    (False, 12, 1, 64, 4, 1, 8192, True),     # 17.8 / 21.6
    (False, 12, 1, 64, 48, 1, 2048, True),    # 29.3 / 38.0
    (False, 12, 1, 64, 16, 1, 1024, False),   # 18.6 / 12.5
    (False, 12, 1, 64, 32, 16, 2048, False),  # 48.5 / 32.9
    (True, 12, 1, 64, 16, 1, 2048, True),     # 16.6 / 20.4
    (True, 12, 1, 64, 4, 1, 8192, True),      # 14.9 / 20.8
    (False, 4, 3, 64, 48, 1, 1024, False),    # 15.8 / 12.6
    (False, 4, 3, 64, 16, 1, 8192, True),     # 16.2 / 22.1
    (False, 1, 8, 128, 4, 1, 8192, False),    # 20.2 / 15.9
    (False, 1, 8, 128, 48, 1, 8192, True),    # 21.5 / 33.6
    (True, 1, 8, 128, 16, 1, 8192, False),    # 22.4 / 17.9
    (True, 1, 8, 128, 16, 1, 32768, False),   # 37.9 / 31.2
    (False, 8, 4, 128, 2, 1, 2048, True),     # 12.4 / 14.2
    (False, 8, 4, 128, 48, 1, 1024, True),    # 24.2 / 36.1
    (True, 8, 4, 128, 32, 16, 2048, False),   # 42.8 / 32.4
    (False, 2, 16, 128, 2, 1, 8192, False),   # 20.9 / 17.0
    (False, 2, 16, 128, 16, 1, 8192, True),   # 22.4 / 26.6
    (False, 8, 1, 32, 32, 16, 2048, False),   # 19.5 / 13.8
    (False, 8, 1, 32, 16, 1, 8192, True),     # 12.3 / 24.1
    (False, 12, 4, 32, 16, 1, 1024, False),   # 13.3 / 9.9
    (True, 8, 1, 32, 64, 32, 1024, False),    # 26.2 / 18.6
    (False, 8, 2, 16, 64, 32, 1024, False),   # 20.8 / 15.4
    (True, 8, 2, 16, 16, 1, 8192, True),      # 14.0 / 31.2
])
def test_prefixes_are_shared_where_that_was_measured_to_be_quicker(lib, eight, HK, G, D, batch, groups, prefix, shares):
    """one new token, 300 keys of each sequence's own"""
    from flash_attn import flash_attn_gfx950 as be
    a, x = prefix_call(be, batch, HK * G, HK, D, batch, prefix, prefix + 300, groups=groups, always=0)
    scales = ctypes.byref(_scales(be)) if eight else None
    asked = lib.fa_paged_fwd_with_workspace_bytes(ctypes.byref(a), scales, ctypes.byref(x))
    assert (asked != lib.fa_paged_fwd_with_workspace_bytes(ctypes.byref(a), scales, None)) == shares
