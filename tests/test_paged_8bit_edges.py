"""The paged cache in 8 bits and shared prefixes: bits of scores, layouts of partial results, where prefixes are shared, every route of a decode step.

Tolerances are counted, not measured: u half a step of the element type, e = 2^-24 a rounding in fp32 (see test_paged.py)."""
import ctypes
import math

import pytest
import torch

from test_paged import E32, Cache, cumulative, half_step
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


# ---- GPU: every route of a decode step, each element within what its own keys allow

def mark_tiles(c, keys=32):
    """The upper half of a key's value says which `keys` of its sequence it belongs to: an element there is those keys' weight, so that a lost, doubled or exchanged tile shows"""
    D = c.v.shape[-1]
    eight = hasattr(c, "vc")
    half = D // 2
    for b, n in enumerate(c.lens):
        page, slot = c.where(b, n)
        x = c.v[page, slot].double()
        x[..., half:] = 2.0 * (torch.arange(half)[None] == (torch.arange(n)[:, None] // keys) % half).double()[:, None]
        if eight:
            x, e = ref_quantise(x, c.v.dtype)
            c.vc[page, slot] = (x * (2.0 ** -e.double())[..., None]).float().to(torch.float8_e4m3fn).view(torch.uint8)
            c.vs[page, :, slot] = (e + 127).to(torch.uint8)
        c.v[page, slot] = x.to(c.v.dtype)
    return c


def check_elements(q, c, new, got, lse=None):
    """causal attention against 64 bits.  A probability is rounded by u of itself, in the numerator and in the denominator, and where it is below the type's normal numbers by
    2^-25 (fp16) of the largest (times its value's scale): an element is off by 2 u of the sum of the magnitudes that it is made of, and by those."""
    D, G, u = q.shape[2], q.shape[1] // c.k.shape[2], half_step(q.dtype)
    at = 0
    for b, n in enumerate(new):
        Lk = c.lens[b]
        page, slot = c.where(b, Lk)
        for h in range(q.shape[1]):
            qh, k, v = q[at:at + n, h].double(), c.k[page, slot, h // G].double(), c.v[page, slot, h // G].double()
            s = qh @ k.t() * D ** -0.5
            s = s.masked_fill(torch.arange(Lk)[None] >= (Lk - n + 1 + torch.arange(n))[:, None], -math.inf)
            p = torch.softmax(s, 1)
            o, parts = p @ v, p @ v.abs()
            ds = (D + 12) * E32 * (qh.abs() @ k.abs().t()).max() * D ** -0.5
            small = Lk * 2.0 ** -25 * p.amax(1, keepdim=True) * v.abs().max() * (4 if q.dtype == torch.float16 else 0)  # (a scale is less than 4 / 448 of the largest value)
            tol = (2 * u + 2 * ds + 2 * (Lk + 8) * E32) * parts + u * o.abs() + small + 2.0 ** -24
            err = (got[at:at + n, h].cpu().double() - o).abs()
            assert (err <= tol).all(), (b, h, (err / tol).max(), (err > tol).nonzero()[:5])
            if lse is not None:
                t = torch.logsumexp(s, 1)
                assert ((lse[b, h, :n].cpu().double() - t).abs() <= ds + (Lk + 8) * E32 + 8 * E32 * (1 + t.abs())).all(), (b, h)
        at += n


ROUTES = [  # lens, new, H, HK, D, PS, whether the keys lie on one line for all workgroups (which takes scratch)
    # wide workgroups, a pair each, past the caches: 8 MB of keys
    ([200 + 25 * i for i in range(32)], 1, 16, 8, 128, 64, False),
    ([40 + 26 * i for i in range(25)], 2, 4, 4, 64, 16, False),
    ([17 + 20 * i for i in range(32)], 1, 8, 8, 32, 32, False),
    ([65 * i % 1061 + 1 for i in range(31)] + [1100], 1, 16, 8, 16, 128, False),
    # more pairs than the device holds at once: the usual workgroups, a pair each
    ([1 + 37 * i % 300 for i in range(70)], 1, 8, 4, 64, 16, False),
    ([1 + 41 * i % 210 for i in range(70)], 3, 4, 4, 128, 32, False),
    ([1 + 43 * i % 170 for i in range(130)], 1, 4, 4, 32, 16, False),
    ([1 + 29 * i % 150 for i in range(130)], 2, 8, 4, 16, 16, False),
    # few long pairs
    ([2500, 1030, 1], 1, 4, 2, 16, 16, True),
    ([1777, 3000], 2, 6, 2, 32, 64, True),
    ([1500, 2049], 1, 2, 2, 64, 32, True),
    ([900, 3001], 1, 8, 1, 128, 16, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens, new, H, HK, D, PS, line", ROUTES)
@pytest.mark.parametrize("eight, want_lse", [(True, False), (True, True), (False, True)])
def test_every_route_of_a_decode_step(lib, lens, new, H, HK, D, PS, line, dtype, eight, want_lse):
    from flash_attn import flash_attn_gfx950 as be
    from flash_attn import flash_attn_paged_interface as p
    lens = [max(n, new) for n in lens]
    c = mark_tiles((Cache8 if eight else Cache)(lens, HK, D, PS, dtype, 3)).gpu()
    if eight:
        a = be.PagedFwdArgs()
        a.struct_bytes = ctypes.sizeof(a)
        a.cache.head_dim, a.cache.nheads_k, a.cache.nheads_q, a.cache.page_size, a.cache.batch, a.cache.n_pages = D, HK, H, PS, len(lens), c.n_pages
        a.cache.total_q, a.cache.max_seqlen_q, a.cache.max_seqlen_k, a.cache.table_cols = len(lens) * new, new, max(lens), c.table.shape[1]
        a.cache.page_table = a.cache.seqlens_k = a.cache.cu_seqlens_q = 1 << 20
        a.cache.table_row_stride = c.table.shape[1]
        assert (lib.fa_paged_fwd_with_workspace_bytes(ctypes.byref(a), ctypes.byref(_scales(be)), None) > 0) == line
    q = randn(len(lens) * new, H, D, dtype=dtype, seed=5)
    r = p.flash_attn_paged_func(q.cuda(), c.dk, c.dv, c.dtable, cumulative([new] * len(lens)).cuda(), c.dlens, new, max(lens), return_softmax_lse=want_lse,
                                **(c.scales if eight else {}))
    out, lse = r if want_lse else (r, None)
    check_elements(q, c, [new] * len(lens), out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("eight, new", [(False, 1), (True, 1), (True, 3), (False, 2)])
def test_shared_prefixes_by_the_rule_against_64_bits(lib, eight, new, dtype):
    from flash_attn import flash_attn_paged_interface as p
    lens, groups, prefix = [2048 + 60 + 31 * i for i in range(7)] + [1408 + 33 + 40 * i for i in range(5)], [7, 5], [2048, 1408]
    c = mark_tiles(share((Cache8 if eight else Cache)(lens, 4, 128, 128, dtype, 3), groups, prefix)).gpu()
    scales = c.scales if eight else {}
    q, cu = randn(12 * new, 16, 128, dtype=dtype, seed=5), cumulative([new] * 12).cuda()
    pl = torch.tensor(prefix, dtype=torch.int32).repeat_interleave(torch.tensor(groups)).cuda()
    where = (q.cuda(), c.dk, c.dv, c.dtable, cu, c.dlens, new, max(lens))
    out, lse = p.flash_attn_paged_prefix_func(*where, cumulative(groups).cuda(), pl, max(prefix), return_softmax_lse=True, **scales)
    check_elements(q, c, [new] * 12, out, lse)
    alone, _ = p.flash_attn_paged_func(*where, return_softmax_lse=True, **scales)
    check_elements(q, c, [new] * 12, alone)
    assert not torch.equal(out, alone)  # (the rule shares here)
