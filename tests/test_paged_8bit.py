"""The paged cache in 8 bits and shared prefixes: what the entry points refuse and the format (CPU), and the kernels against the definitions in 64 bits (GPU).

Tolerances are counted, not measured: u half a step of the element type, e = 2^-24 a rounding in fp32 (see test_paged.py, whose bounds of attention hold here for the
values that the rows stand for)."""
import ctypes
import math

import pytest
import torch

from test_paged import E32, Cache, cumulative, half_step, ref_attention, ref_norm_rotary, tables
from test_paged import _args as paged_args

DTYPES = [torch.float16, torch.bfloat16]
RANGE = {torch.float16: (-15, 8), torch.bfloat16: (-100, 120)}


# ---- the format, in 64 bits on the CPU

def _grid():
    """The numbers of e4m3 that are not negative, in order: code i is grid[i]"""
    return torch.tensor([m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16) for m in range(8)][:127], dtype=torch.float64)


def ref_quantise(x, dtype):
    """x (..., D) float64 -> what the rows stand for (float64), and their exponents"""
    grid = _grid()
    least, most = RANGE[dtype]
    fine = x.isfinite()
    top = torch.where(fine, x.abs(), 0.0).amax(-1)
    e = torch.full(top.shape, least, dtype=torch.int64)
    for k in range(least, most):
        e += (top > 448.0 * 2.0 ** k).long()
    y = torch.where(fine, x, 0.0) * (2.0 ** -e.double())[..., None]
    mag = torch.minimum(y.abs(), torch.where(e == most, 240.0, 448.0).double()[..., None])
    hi = torch.searchsorted(grid, mag).clamp(max=126)  # the first that is not below
    lo = (hi - 1).clamp(min=0)
    up, down = grid[hi] - mag, mag - grid[lo]
    code = torch.where((up < down) | ((up == down) & (hi % 2 == 0)) | (grid[hi] == mag), hi, lo)
    value = torch.where(y < 0, -grid[code], grid[code]) * (2.0 ** e.double())[..., None]
    return torch.where(fine, value, math.nan), e


def decode(codes, exps):
    """What a cache's rows stand for: codes (pages, PS, HK, D) float8, exps (pages, HK, PS) bytes"""
    c = codes.cpu().contiguous().view(torch.uint8).long()
    mag = torch.cat([_grid(), torch.tensor([math.nan], dtype=torch.float64)])[c & 127]
    return torch.where(c >= 128, -mag, mag) * (2.0 ** (exps.cpu().transpose(1, 2).double() - 127))[..., None]


class Cache8(Cache):
    """A cache in 8 bits of the given sequences: `k` and `v` hold what the rows stand for (exact in dtype), NaN where nothing was stored; on the GPU the
    bytes there are 255, NaN under the largest exponent that a byte can have."""

    def __init__(self, *a, **kw):
        spread, v_sizes = kw.pop("spread", 0.0), kw.pop("v_sizes", None)
        super().__init__(*a, **kw)
        g = torch.Generator().manual_seed(7)
        dtype, out = self.k.dtype, []
        for name in ("k", "v"):
            x = getattr(self, name).double()
            x = x * torch.exp(spread * torch.randn(x.shape[:-1], generator=g, dtype=torch.float64))[..., None]
            there = ~x.isnan().all(-1)
            if name == "v" and v_sizes is not None:
                x = x * torch.tensor(v_sizes, dtype=torch.float64)[torch.randint(len(v_sizes), x.shape[:-1], generator=g)][..., None]
            y, e = ref_quantise(torch.where(there[..., None], x.to(dtype).double(), 0.0), dtype)
            codes = torch.where(there[..., None], (y * (2.0 ** -e.double())[..., None]).float().to(torch.float8_e4m3fn).view(torch.uint8), 255)
            setattr(self, name, torch.where(there[..., None], y, math.nan).to(dtype))
            out.append((codes.to(torch.uint8), torch.where(there, e + 127, 255).to(torch.uint8).transpose(1, 2).contiguous()))
        (self.kc, self.ks), (self.vc, self.vs) = out

    def gpu(self):
        head_major = self.k.stride(1) < self.k.stride(2)
        def put(t):
            t = t.transpose(1, 2).contiguous().cuda().transpose(1, 2) if head_major else t.contiguous().cuda()
            return t.view(torch.float8_e4m3fn)
        self.dk, self.dv, self.dks, self.dvs = put(self.kc), put(self.vc), self.ks.cuda(), self.vs.cuda()
        self.dtable, self.dlens = self.table.cuda(), torch.tensor(self.lens, dtype=torch.int32).cuda()
        self.scales = dict(k_scales=self.dks, v_scales=self.dvs)
        return self


def randn(*shape, dtype=torch.float16, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def same(a, b):
    return a.shape == b.shape and bool(((a == b) | (a.isnan() & b.isnan())).all())


def test_the_reference_format_is_what_it_says():
    g = _grid()
    assert g[0] == 0 and g[1] == 2.0 ** -9 and g[8] == 2.0 ** -6 and g[126] == 448 and (g[1:] > g[:-1]).all()
    x = torch.tensor([[448.0, 1.0625, 1.1875, -17.0, 2.0 ** -10, 3 * 2.0 ** -10, 0.0, -448.0]], dtype=torch.float64)
    y, e = ref_quantise(x, torch.float16)
    assert e == 0 and y[0].tolist() == [448, 1.0, 1.25, -16, 0, 2.0 ** -8, 0, -448]
    assert ref_quantise(2 * x, torch.float16)[1] == 1 and ref_quantise(x * 448.5 / 448, torch.float16)[1] == 1
    for dtype in DTYPES:
        big = torch.full((1, 8), torch.finfo(dtype).max, dtype=torch.float64)
        y, e = ref_quantise(big, dtype)
        assert e == RANGE[dtype][1] and torch.equal(y.to(dtype).double(), y) and (y.abs() <= big).all() and ((big - y) <= big / 16).all()
        x = randn(4000, 32, dtype=dtype, seed=1).double() * torch.exp(3 * torch.randn(4000, 1, dtype=torch.float64, generator=torch.Generator().manual_seed(2)))
        x = x.to(dtype).double()
        y, e = ref_quantise(x, dtype)
        assert same(y.to(dtype).double(), y)  # exact in the dtype
        assert torch.equal(y.isnan(), ~x.isfinite())  # (a few of the fp16 rows have infinities)
        assert (((y - x).abs() <= x.abs() / 16 + (2.0 ** (e.double() - 10))[:, None]) | ~x.isfinite()).all()
        assert same(ref_quantise(y, dtype)[0], y)  # stored again, nothing changes


# ---- what the entry points refuse (CPU: nothing is enqueued)

def _scales(be, **kw):
    s = be.PagedScales(ctypes.sizeof(be.PagedScales), 0, 1 << 20, 1 << 20)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def _prefix(be, **kw):
    x = be.PagedPrefix(ctypes.sizeof(be.PagedPrefix), 1, 32, 0, 1 << 20, 1 << 20)
    for k, v in kw.items():
        setattr(x, k, v)
    return x


def _set(a, change):
    for k, v in change.items():
        at, *rest = k.split(".")
        setattr(getattr(a, at) if rest else a, rest[0] if rest else at, v)
    return a


@pytest.mark.parametrize("scales, change, says", [
    (dict(struct_bytes=8), {}, "struct size"), (dict(k_scales=None), {}, "k_scales"), (dict(v_scales=None), {}, "v_scales"), (dict(k_scales=(1 << 20) + 8), {}, "16-byte"),
    ({}, {"cache.k_slot_stride": 72}, "multiples of 16"), ({}, {"cache.v_head_stride": 1032}, "multiples of 16"), ({}, {"cache.k_page_stride": 2056}, "multiples of 16"),
    ({}, {"cache.head_dim": 48}, "head_dim"), ({}, {"dtype": 2}, "dtype")])
def test_a_cache_in_8_bits_is_refused(lib, scales, change, says):
    from flash_attn import flash_attn_gfx950 as be
    s = _scales(be, **scales)
    for kind, call in (("append", lambda a: lib.fa_paged_append_with(ctypes.byref(a), ctypes.byref(s))),
                       ("fwd", lambda a: lib.fa_paged_fwd_with(ctypes.byref(a), ctypes.byref(s), None))):
        assert call(_set(paged_args(be, kind), change)) == -1 and says in lib.fa_last_error().decode(), kind
    r = be.PagedReadArgs()
    r.struct_bytes = ctypes.sizeof(r)
    r.cache = paged_args(be, "fwd").cache
    assert lib.fa_paged_read(ctypes.byref(_set(r, change)), ctypes.byref(s)) == -1 and says in lib.fa_last_error().decode()


@pytest.mark.parametrize("change, says", [
    (dict(struct_bytes=8), "struct size"), (dict(n_groups=0), "group"), (dict(n_groups=3), "group"), (dict(max_prefix_len=-1), "max_prefix_len"), (dict(cu_groups=None), "cu_groups"),
    (dict(prefix_lens=None), "prefix_lens"), (dict(cu_groups=(1 << 20) + 2), "4-byte")])
def test_a_prefix_is_refused(lib, change, says):
    from flash_attn import flash_attn_gfx950 as be
    a, x = paged_args(be, "fwd"), _prefix(be, **change)
    assert lib.fa_paged_fwd_with(ctypes.byref(a), None, ctypes.byref(x)) == -1 and says in lib.fa_last_error().decode()
    assert lib.fa_paged_fwd_with_workspace_bytes(ctypes.byref(a), None, ctypes.byref(x)) == 0


def test_calls_without_rows_pass_and_ask_for_nothing_more(lib):
    from flash_attn import flash_attn_gfx950 as be
    s, x = _scales(be), _prefix(be)
    assert lib.fa_paged_append_with(ctypes.byref(paged_args(be, "append")), ctypes.byref(s)) == 0
    assert lib.fa_paged_fwd_with(ctypes.byref(paged_args(be, "fwd")), ctypes.byref(s), ctypes.byref(x)) == 0
    r = be.PagedReadArgs()
    r.struct_bytes = ctypes.sizeof(r)
    r.cache = paged_args(be, "fwd").cache
    assert lib.fa_paged_read(ctypes.byref(r), ctypes.byref(s)) == 0
    r.cache.total_q = 3
    assert lib.fa_paged_read(ctypes.byref(r), ctypes.byref(s)) == -1 and b"k_out" in lib.fa_last_error()
    # the struct alone decides about the scratch, and a call without it is refused before anything is enqueued
    a = paged_args(be, "fwd")
    a.q = a.o = 1 << 20
    a.q_row_stride = a.o_row_stride = 256
    a.q_head_stride = a.o_head_stride = 64
    a.cache.total_q, a.cache.max_seqlen_q, a.cache.max_seqlen_k, a.cache.table_cols, a.cache.table_row_stride = 2, 1, 4096, 300, 300
    x.always, x.max_prefix_len = 1, 2048
    need = lib.fa_paged_fwd_with_workspace_bytes(ctypes.byref(a), None, ctypes.byref(x))
    assert need > 0 and need != lib.fa_paged_fwd_workspace_bytes(ctypes.byref(a))
    assert lib.fa_paged_fwd_with(ctypes.byref(a), None, ctypes.byref(x)) == -2 and str(need) in lib.fa_last_error().decode()


def test_prefixes_are_shared_where_it_pays(lib):
    """on both sides of the rule, by the scratch that a call asks for: 8 x 4 heads, d = 128, pages of 64"""
    from flash_attn import flash_attn_gfx950 as be

    def shares(batch, prefix, new=1, groups=1, eight=False, heads=8):
        a = paged_args(be, "fwd")
        c = a.cache
        c.head_dim, c.nheads_k, c.nheads_q, c.page_size, c.batch, c.total_q, c.max_seqlen_q, c.max_seqlen_k = 128, heads, 32, 64, batch, batch * new, new, prefix + 300
        c.table_cols = c.table_row_stride = 1000
        x = _prefix(be, n_groups=groups, max_prefix_len=prefix)
        scales = ctypes.byref(_scales(be)) if eight else None
        return lib.fa_paged_fwd_with_workspace_bytes(ctypes.byref(a), scales, ctypes.byref(x)) != lib.fa_paged_fwd_with_workspace_bytes(ctypes.byref(a), scales, None)

    assert shares(4, 2048) and shares(2, 8192) and shares(48, 1024) and shares(16, 8192, 8) and shares(16, 8192, groups=3)
    # ... and by how long a workgroup is at its part of the prefix
    assert shares(2, 60000) and not shares(2, 60000, eight=True) and not shares(2, 60000, heads=1) and shares(64, 60000, eight=True, heads=1) and shares(2, 2048)
    assert shares(128, 4096, groups=32, eight=True) and not shares(32, 2048, groups=16, eight=True)
    assert not shares(2, 1984) and not shares(48, 512) and not shares(48, 1023) and not shares(1, 100000) and not shares(16, 8192, 9) and not shares(16, 8192, groups=16)


def test_index_arithmetic_of_prefixes(tmp_path):
    import os
    import subprocess
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(r"""
#include <cassert>
#include <climits>
#include <initializer_list>
#include "fa_paged_index.h"
using namespace fa;
int main() {
  const int v[] = {INT_MIN, -1, 0, 1, 15, 16, 17, 1000, 1 << 20, INT_MAX};
  for (int a : v)
    for (int m : {0, 1, 16, 40, 1 << 30, INT_MAX})
      for (int n : {1, 16, 100, 1 << 30})
        for (int g = 4; g <= 10; g++) {
          const int k = shared_keys(a, m, n, g);
          assert(k >= 0 && k <= n && k <= m && k % (1 << g) == 0);
          if (a >= 0) assert(k <= a && (k + (1 << g) > a || k + (1 << g) > m || k + (1 << g) > n));
        }
}
""")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", os.path.join(root, "flash-attention_amd", "csrc"), str(src), "-o", str(exe)], check=True)
    subprocess.run([str(exe)], check=True)


def test_the_book_of_forks():
    from flash_attn.flash_attn_paged_interface import PagedKVCache
    c = PagedKVCache(2, 40, 16, 2, 32, dtype=torch.bfloat16, device="cpu", store_dtype=torch.float8_e4m3fn)
    a = c.add()
    assert c.step([a], [100]).prefix == () and c.free_pages() == 33
    c._k.view(torch.uint8)[1, 6] = 5  # (a page's bytes, in the last layer)
    c._scales[1][1, 6] = 9
    b, d = c.fork(a), c.fork(a, 64)
    e = c.fork(b, 33)
    assert [c.length(s) for s in (a, b, d, e)] == [100, 100, 64, 33] and c.free_pages() == 31  # two part pages were copied
    page = c._pages[b][6]
    assert page != c._pages[a][6] and (c._k.view(torch.uint8)[1, page] == 5).all() and (c._scales[1][1, page] == 9).all() and (c._k.view(torch.uint8)[0, page] == 0).all()
    st = c.step([a, b, d, e], [1, 2, 3, 4])
    assert [x if isinstance(x, int) else x.tolist() for x in st.prefix] == [[0, 3, 4], [64, 64, 64, 0], 64]  # (with e three would save 32 each)
    assert c.step([d, a], [1, 1]).prefix[1].tolist() == [64, 64]
    assert c.step([d, c.add(), a, b], [1, 1, 1, 1]).prefix[0].tolist() == [0, 1, 2, 4]
    assert c.step([e], [1]).prefix == ()
    f = c.fork(c.fork(a, 16), 5)  # a fork of a fork, and one that shares no whole page
    assert c._pages[f][0] not in c._pages[a] and c.step([f, a], [1, 1]).prefix == ()
    for s in list(c._pages):
        c.remove(s)
    assert sorted(c._free) == list(range(40)) and not c._users and not c._shared
    g = c.add()
    c.step([g], [39 * 16])
    with pytest.raises(RuntimeError, match="tokens"):
        c.fork(g, 39 * 16 + 1)
    with pytest.raises(RuntimeError, match="tokens"):
        c.fork(g, -1)
    h = c.fork(g, 17)  # the last free page
    with pytest.raises(RuntimeError, match="free page"):
        c.fork(g, 17)
    c.remove(h)
    h = c.fork(g, 32)
    assert c.length(c.fork(g, 32)) == 32 and c.length(h) == 32
    with pytest.raises(RuntimeError, match="different sequences"):
        c.fork(77)
    with pytest.raises(RuntimeError, match="16 bits"):
        PagedKVCache(1, 4, 16, 2, 32, device="cpu", store_dtype=torch.float8_e4m3fn, key_weights=True)
    with pytest.raises(RuntimeError, match="store_dtype"):
        PagedKVCache(1, 4, 16, 2, 32, device="cpu", store_dtype=torch.float8_e5m2)
    x = torch.zeros(1, 4, 32, dtype=torch.float16)
    st = c.step([c.fork(g, 16)], [1])
    for call in (lambda: st.append(0, x, x[:, :2], x[:, :2]), lambda: st.attend(0, x)):
        with pytest.raises(RuntimeError, match="made for torch.bfloat16"):
            call()
    w = PagedKVCache(1, 4, 16, 2, 32, device="cpu", key_weights=True)
    with pytest.raises(RuntimeError, match="not shared"):
        w.fork(w.add())


# ---- GPU: attention

def check_attention(q, c, new, causal, got, lse=None, scale=None):
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    want, top, _, tol, ds = ref_attention(q, c, new, causal, scale)
    err = (got.cpu().double() - want).abs()
    assert (err <= tol).all(), ((err / tol).max(), (err > tol).nonzero()[:5])
    if lse is not None:
        for (b, h), t in top.items():
            x = lse[b, h, :new[b]].cpu().double()
            assert torch.equal(x.isinf(), t.isinf())
            n = max(c.lens[b], 1)
            bound = ds + (n + 8) * E32 + 8 * E32 * (1 + t[~t.isinf()].abs())
            assert ((x - t)[~t.isinf()].abs() <= bound).all()


ATTEND = [  # lens, new, H, HK, D, PS, causal
    ([1], [1], 1, 1, 16, 16, True),
    ([17, 1, 300], [1, 1, 1], 8, 2, 32, 16, True),
    ([500], [1], 12, 12, 64, 16, True),
    ([33, 129, 4000, 31], [1, 1, 1, 1], 8, 8, 64, 32, True),
    ([700, 2500], [1, 1], 32, 8, 128, 64, True),
    ([260, 64, 100], [5, 1, 3], 8, 2, 64, 16, True),
    ([260, 64, 100], [5, 1, 3], 8, 2, 128, 128, False),
    ([90, 17, 2], [8, 0, 2], 4, 1, 16, 16, True),
    ([3, 40], [5, 7], 4, 4, 32, 16, True),      # new tokens that see nothing
    ([0, 40], [2, 1], 4, 2, 64, 16, True),
    ([300, 77], [64, 77], 4, 2, 64, 16, True),  # many rows
    ([1000, 129, 40], [100, 129, 40], 8, 2, 128, 32, True),
    ([700], [33], 12, 12, 32, 64, True),
    ([515, 90], [70, 60], 6, 2, 16, 16, False),
    ([2000], [40], 8, 1, 128, 16, True),
    ([3, 200], [50, 50], 4, 4, 64, 16, True),
    ([1500, 33], [1, 1], 32, 1, 128, 1024, True),  # 32 rows a pair
    ([40] * 70, [1] * 70, 2, 2, 64, 16, True),
    ([90, 2000], [1, 2], 40, 1, 16, 512, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens, new, H, HK, D, PS, causal", ATTEND)
@pytest.mark.parametrize("want_lse", [False, True])
def test_attention_over_8_bits(lib, lens, new, H, HK, D, PS, causal, dtype, want_lse):
    from flash_attn import flash_attn_paged_interface as p
    c = Cache8(lens, HK, D, PS, dtype, 3, head_major=D != 32, spread=0.7).gpu()
    q = randn(sum(new) + 3, H, D, dtype=dtype, seed=5)  # (three rows behind the last sequence)
    cu = cumulative(new).cuda()
    r = p.flash_attn_paged_func(q.cuda(), c.dk, c.dv, c.dtable, cu, c.dlens, max(new), max(max(lens), 1), causal=causal, return_softmax_lse=want_lse, **c.scales)
    out, lse = r if want_lse else (r, None)
    check_attention(q[:sum(new)], c, new, causal, out[:sum(new)], lse)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [1, 4, 40])
@pytest.mark.parametrize("D", [16, 128])
@pytest.mark.parametrize("sizes", [1, 0, -1])
def test_values_of_all_sizes(lib, D, new, dtype, sizes):
    """Rows of values as far apart as the format has them, zeros among them: each counts in the denominator for what its key says, whatever its value's size"""
    from flash_attn import flash_attn_gfx950 as be
    from flash_attn import flash_attn_paged_interface as p
    most = 2.0 ** (118 if dtype == torch.bfloat16 else 10)
    v_sizes = {1: [0.0, 1 / most if dtype == torch.float16 else 2.0 ** -95, 1.0, most], 0: [0.0, most], -1: [0.0, 2.0 ** -100 if dtype == torch.bfloat16 else 2.0 ** -14]}[sizes]
    lens, groups, prefix = [700, 690, 40, 60], [2, 2], [512, 32]
    news = [new, 1, 1, new]
    c = share(Cache8(lens, 2, D, 32, dtype, 3, v_sizes=v_sizes), groups, prefix).gpu()
    q = randn(sum(news), 4, D, dtype=dtype, seed=5)
    cu, cg = cumulative(news).cuda(), cumulative(groups).cuda()
    pl = torch.tensor([512, 512, 32, 32], dtype=torch.int32).cuda()
    where = (q.cuda(), c.dk, c.dv, c.dtable, cu, c.dlens, new, max(lens))
    out, lse = p.flash_attn_paged_func(*where, return_softmax_lse=True, **c.scales)
    check_attention(q, c, news, True, out, lse)
    for want_lse in (False, True):
        r = be.paged_fwd(*where, D ** -0.5, True, want_lse, cu_groups=cg, prefix_lens=pl, max_prefix_len=512, always=True, **c.scales)
        check_attention(q, c, news, True, r[0], r[1] if want_lse else None)


# ---- GPU: storing and reading

STORE = [  # lens (with the new tokens), new, H, HK, D, PS
    ([1], [1], 1, 1, 16, 16),
    ([40, 17, 90], [1, 1, 1], 8, 2, 32, 16),
    ([260, 64, 100], [5, 0, 100], 8, 2, 64, 32),
    ([700, 33], [300, 33], 4, 4, 128, 128),
    ([2500], [2400], 12, 12, 64, 16),
    ([30, 900, 50], [7, 888, 50], 32, 8, 128, 16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens, new, H, HK, D, PS", STORE)
def test_rows_stored_as_they_are(lib, lens, new, H, HK, D, PS, dtype):
    """without a norm and rotation nothing but the rounding to 8 bits happens: bit for bit the nearest values, of rows of every size, with zeros, infinities and NaN"""
    from flash_attn import flash_attn_paged_interface as p
    c = Cache8(lens, HK, D, PS, dtype, 3, head_major=D != 32).gpu()
    before = decode(c.dk, c.dks), decode(c.dv, c.dvs)
    total = sum(new)
    g = torch.Generator().manual_seed(4)
    k, v = (randn(total + 2, HK, D, dtype=torch.float32, seed=i) * torch.exp(4 * torch.randn(total + 2, HK, 1, generator=g)) for i in (1, 2))
    fin = torch.finfo(dtype)
    k, v = k.clamp(fin.min, fin.max).to(dtype), v.clamp(fin.min, fin.max).to(dtype)
    k[0, 0] = 0.0
    k[0, -1] = fin.max
    v[0, 0] = fin.tiny * 2.0 ** -4 if dtype == torch.float16 else fin.tiny
    if total > 3:
        v[1, 0, 3], v[2, 0, 0], v[3, 0] = math.inf, math.nan, -math.inf
        k[1, 0, ::2], k[2, 0, 5 % D] = fin.min, -math.inf
    cu = cumulative(new).cuda()
    assert p.paged_append_func(None, k.cuda(), v.cuda(), c.dk, c.dv, c.dtable, cu, c.dlens, **c.scales) is None
    after = decode(c.dk, c.dks), decode(c.dv, c.dvs)
    at = 0
    for b, n in enumerate(new):
        page, slot = c.where(b, lens[b])
        page, slot = page[lens[b] - n:], slot[lens[b] - n:]
        for i, x in enumerate((k, v)):
            assert same(after[i][page, slot], ref_quantise(x[at:at + n].double(), dtype)[0]), (b, i)
            after[i][page, slot] = before[i][page, slot]
        at += n
    assert same(after[0], before[0]) and same(after[1], before[1])  # nothing else was written


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens, new, H, HK, D, PS", STORE)
def test_rows_stored_normalised_and_turned(lib, lens, new, H, HK, D, PS, dtype):
    from flash_attn import flash_attn_paged_interface as p
    c = Cache8(lens, HK, D, PS, dtype, 3).gpu()
    c16 = Cache(lens, HK, D, PS, dtype, 3).gpu()
    total = sum(new)
    q, k, v = randn(total, H, D, dtype=dtype, seed=0), randn(total, HK, D, dtype=dtype, seed=1), randn(total, HK, D, dtype=dtype, seed=2)
    qw, kw = (1 + 0.3 * randn(D, dtype=torch.float32, seed=i) for i in (3, 4))
    cos, sin = tables(max(lens), D, dtype)
    cu = cumulative(new).cuda()
    more = dict(q_weight=qw.cuda(), k_weight=kw.cuda(), cos_half=cos.cuda(), sin_half=sin.cuda(), eps=1e-5)
    w, pos = torch.ones(c.n_pages, HK, PS, device="cuda"), torch.zeros(c.n_pages, HK, PS, dtype=torch.int32, device="cuda")
    gq = p.paged_append_func(q.cuda(), k.cuda(), v.cuda(), c.dk, c.dv, c.dtable, cu, c.dlens, **more, **c.scales, key_weights=w, key_positions=pos)
    assert torch.equal(gq, p.paged_append_func(q.cuda(), k.cuda(), v.cuda(), c16.dk, c16.dv, c16.dtable, cu, c16.dlens, **more))
    kk, vv = decode(c.dk, c.dks), decode(c.dv, c.dvs)
    at = 0
    for b, n in enumerate(new):
        t = torch.arange(lens[b] - n, lens[b])
        page, slot = c.where(b, lens[b])
        page, slot = page[lens[b] - n:], slot[lens[b] - n:]
        want = ref_norm_rotary(k[at:at + n].double(), kw.double(), cos.double(), sin.double(), t, 1e-5)
        top = want.abs().amax(-1, keepdim=True) if n else want
        # one rounding to e4m3: half a step, 2^-4 of the value, or 2^-10 of the scale, which is at most 1/224 of the largest; before it the norm's
        # and the rotation's roundings in fp32, (D + 12) of them at most, of the largest value
        bound = (want.abs() + (D + 12) * E32 * top) * 2.0 ** -4 + top * 2.0 ** -10 / 224 + (D + 12) * E32 * top
        assert ((kk[page, slot] - want).abs() <= bound).all()
        assert same(vv[page, slot], ref_quantise(v[at:at + n].double(), dtype)[0])
        assert (w.cpu()[page, :, slot] == 0).all() and (pos.cpu()[page, :, slot] == t[:, None].int()).all()
        at += n


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens, new, H, HK, D, PS", STORE)
@pytest.mark.parametrize("eight", [True, False])
def test_reading(lib, lens, new, H, HK, D, PS, dtype, eight):
    """the last tokens of each sequence, and whole sequences, bit for bit; rows of no sequence and in front of a sequence's first key are zeros"""
    from flash_attn import flash_attn_paged_interface as p
    c = (Cache8 if eight else Cache)(lens, HK, D, PS, dtype, 3, head_major=D != 32).gpu()
    scales = c.scales if eight else {}
    more = [n + 4 if i == 0 else n for i, n in enumerate(lens)]  # four rows more than the first sequence has keys
    for rows, total in ((new, sum(new)), (lens, sum(lens) + 3), (more, sum(more))):
        k, v = p.paged_read_func(c.dk, c.dv, c.dtable, cumulative(rows).cuda(), c.dlens, total, dtype=dtype if eight else None, **scales)
        assert k.shape == v.shape == (total, HK, D) and k.dtype == v.dtype == dtype
        at = 0
        for b, n in enumerate(rows):
            have = min(n, lens[b])
            page, slot = c.where(b, lens[b])
            page, slot = page[lens[b] - have:], slot[lens[b] - have:]
            for x, y in ((k, c.k), (v, c.v)):
                assert torch.equal(x[at + n - have:at + n].cpu(), y[page, slot]) and (x[at:at + n - have] == 0).all()
            at += n
        assert (k[at:] == 0).all() and (v[at:] == 0).all()


# ---- GPU: shared prefixes

def share(c, groups, prefix):
    """The sequences of each group get the first one's pages for the prefix's whole pages; c: before gpu()"""
    b = 0
    for n, m in zip(groups, prefix):
        for i in range(b + 1, b + n):
            c.table[i, :m // c.PS] = c.table[b, :m // c.PS]
        b += n
    return c


PREFIX = [  # lens, new, groups, prefix, H, HK, D, PS, causal
    ([40, 50], [1, 1], [2], [32], 2, 2, 64, 16, True),
    ([33, 34, 35, 40], [1, 1, 1, 1], [4], [33], 4, 2, 16, 16, True),       # a prefix of two pages and a token
    ([600, 520, 700], [1, 1, 1], [3], [512], 12, 12, 32, 32, True),
    ([300, 290, 700, 640, 650], [1, 2, 3, 0, 1], [2, 3], [256, 512], 8, 2, 64, 64, True),
    ([300, 290, 90, 640, 650], [1, 1, 1, 1, 1], [2, 1, 2], [272, 0, 512], 8, 8, 128, 16, False),
    ([2100] * 9, [1] * 9, [9], [2048], 32, 8, 128, 128, True),
    ([1030] * 40, [3] * 40, [40], [1000], 4, 1, 64, 32, True),             # more than one tile of rows
    ([700, 690, 560], [40, 50, 33], [3], [500], 8, 2, 128, 16, True),      # many rows
    ([300, 280], [17, 1], [1, 1], [256, 256], 8, 4, 32, 16, True),         # groups of one
    ([64, 80, 65], [64, 80, 65], [3], [0], 4, 4, 64, 16, True),            # nothing shared
    ([257, 260], [1, 4], [2], [256], 4, 4, 16, 256, True),                 # nothing but the prefix and the new tokens
    ([400, 410], [150, 140], [2], [240], 4, 2, 64, 16, True),
    ([520] * 70, [1] * 70, [1] * 30 + [40], [496] * 31, 2, 2, 32, 16, True),
    ([150, 140] * 66, [1, 2] * 66, [2] * 66, [128] * 66, 2, 1, 64, 16, True),  # more groups than lanes
    ([2100, 3000], [1, 1], [2], [2048], 64, 2, 64, 1024, True),               # 32 rows a pair, pages of 1024
    ([520, 530, 540], [2, 2, 2], [3], [512], 48, 3, 16, 512, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens, new, groups, prefix, H, HK, D, PS, causal", PREFIX)
@pytest.mark.parametrize("eight, want_lse", [(False, True), (True, False), (True, True)])
def test_shared_prefix(lib, lens, new, groups, prefix, H, HK, D, PS, causal, dtype, eight, want_lse):
    from flash_attn import flash_attn_gfx950 as be
    from flash_attn import flash_attn_paged_interface as p
    c = share((Cache8 if eight else Cache)(lens, HK, D, PS, dtype, 3, head_major=D != 32), groups, prefix).gpu()
    q = randn(sum(new) + 3, H, D, dtype=dtype, seed=5)
    cu, cg = cumulative(new).cuda(), cumulative(groups).cuda()
    pl = torch.tensor(prefix, dtype=torch.int32).repeat_interleave(torch.tensor(groups)).cuda()
    where = (q.cuda(), c.dk, c.dv, c.dtable, cu, c.dlens, max(max(new), 1), max(lens))
    scales = c.scales if eight else {}
    # prefixes read once wherever that is possible, and as the rule has it (these are too small for it)
    for r in (be.paged_fwd(*where, D ** -0.5, causal, want_lse, cu_groups=cg, prefix_lens=pl, max_prefix_len=max(prefix), always=True, **scales),
              p.flash_attn_paged_prefix_func(*where, cg, pl, max(prefix), causal=causal, return_softmax_lse=want_lse, **scales)):
        out, lse = r if want_lse else (r if isinstance(r, torch.Tensor) else r[0], None)
        check_attention(q[:sum(new)], c, new, causal, out[:sum(new)], lse)


@pytest.mark.gpu
@pytest.mark.parametrize("eight, new", [(False, 1), (True, 1), (True, 3)])
def test_shared_prefix_of_a_serving_batch(lib, eight, new):
    """sizes at which prefixes are read once by the rule: the same as when every sequence reads its own"""
    from flash_attn import flash_attn_paged_interface as p
    lens, groups, prefix = [2500 + 13 * i for i in range(21)] + [1500 + 7 * i for i in range(11)], [21, 11], [2304, 1408]
    c = share((Cache8 if eight else Cache)(lens, 4, 128, 128, torch.bfloat16, 3), groups, prefix).gpu()
    scales = c.scales if eight else {}
    q, cu = randn(32 * new, 16, 128, dtype=torch.bfloat16, seed=5).cuda(), cumulative([new] * 32).cuda()
    pl = torch.tensor(prefix, dtype=torch.int32).repeat_interleave(torch.tensor(groups)).cuda()
    where = (q, c.dk, c.dv, c.dtable, cu, c.dlens, new, max(lens))
    a, la = p.flash_attn_paged_prefix_func(*where, cumulative(groups).cuda(), pl, max(prefix), return_softmax_lse=True, **scales)
    b, lb = p.flash_attn_paged_func(*where, return_softmax_lse=True, **scales)
    # each is within 2 u of the largest value (probabilities), u of the result and the scores' errors, a few fp32 roundings of sums of 128 products
    vmax, u = c.v.float().nan_to_num(0).abs().max().item(), half_step(torch.bfloat16)
    assert ((a.float() - b.float()).abs() <= (4 * u + 1e-3) * vmax + 2 * u * b.float().abs()).all() and not torch.equal(a, b)
    assert ((la - lb)[:, :, :new].abs() <= 1e-3).all()


# ---- GPU: refusals, bad tables, streams, graphs, large pools

@pytest.mark.gpu
def test_python_refusals(lib):
    from flash_attn import flash_attn_paged_interface as p
    c, c16 = Cache8([40, 20], 2, 64, 16, torch.float16, 1).gpu(), Cache([40, 20], 2, 64, 16, torch.float16, 1).gpu()
    q, cu, cg = randn(2, 4, 64).cuda(), cumulative([1, 1]).cuda(), cumulative([2]).cuda()
    pl = torch.full((2,), 16, dtype=torch.int32, device="cuda")
    k = randn(2, 2, 64).cuda()

    def attend(q=q, k=c.dk, v=c.dv, ks=c.dks, vs=c.dvs):
        p.flash_attn_paged_func(q, k, v, c.dtable, cu, c.dlens, 1, 40, k_scales=ks, v_scales=vs)

    def shared(cg=cg, pl=pl, most=16):
        p.flash_attn_paged_prefix_func(q, c.dk, c.dv, c.dtable, cu, c.dlens, 1, 40, cg, pl, most, **c.scales)

    def store(k=k, v=k, **more):
        p.paged_append_func(None, k, v, c.dk, c.dv, c.dtable, cu, c.dlens, **{**c.scales, **more})

    def read(total=2, dtype=torch.float16, kc=c.dk, vc=c.dv, **more):
        p.paged_read_func(kc, vc, c.dtable, cu, c.dlens, total, dtype=dtype, **{**c.scales, **more})

    bad = [
        (attend, dict(ks=None)), (attend, dict(ks=None, vs=None)), (attend, dict(k=c16.dk, v=c16.dv)), (attend, dict(v=c16.dv)), (attend, dict(q=q.float())), (attend, dict(q=q[:, :3])),
        (attend, dict(ks=c.dks.int())), (attend, dict(ks=c.dks[:-1])), (attend, dict(ks=c.dks.transpose(1, 2))), (attend, dict(vs=c.dvs.cpu())), (attend, dict(k=c.dk.view(torch.float8_e5m2), v=c.dv.view(torch.float8_e5m2))),
        (shared, dict(cg=None)), (shared, dict(pl=None)), (shared, dict(cg=None, pl=None)), (shared, dict(cg=cg.long())), (shared, dict(cg=cg[:1])), (shared, dict(cg=torch.zeros(4, dtype=torch.int32, device="cuda"))),
        (shared, dict(pl=pl[:1])), (shared, dict(pl=pl.cpu())), (shared, dict(most=-1)), (shared, dict(most=2 ** 40)),
        (store, dict(k=k.to(torch.float8_e4m3fn))), (store, dict(k=k.float())), (store, dict(v=k.bfloat16())), (store, dict(k_scales=None)), (store, dict(k_scales=None, v_scales=None)),
        (store, dict(key_weights=c.dks)), (read, dict(total=-1)), (read, dict(dtype=None)), (read, dict(dtype=torch.float32)), (read, dict(v_scales=None)),
        (read, dict(kc=c16.dk, vc=c16.dv)), (read, dict(kc=c16.dk, vc=c16.dv, k_scales=None, v_scales=None, dtype=torch.bfloat16)), (read, dict(vc=None)), (read, dict(total=2 ** 40)),
    ]
    for i, (call, change) in enumerate(bad):
        print(i, sorted(change))  # (shown with a failure)
        with pytest.raises(RuntimeError):
            call(**change)
    for call in (lambda: p.paged_key_weights_func(q, torch.zeros(2, 4, 16, device="cuda"), c.dk, torch.zeros(c.n_pages, 2, 16, device="cuda"), c.dtable, cu, c.dlens, 1, 40),
                 lambda: p.paged_evict_func(c.dk, c.dv, torch.zeros(c.n_pages, 2, 16, device="cuda"), torch.zeros(c.n_pages, 2, 16, dtype=torch.int32, device="cuda"), c.dtable, c.dlens,
                                            c.dlens, 8, 2, 40),
                 lambda: attend(q=q.clone().requires_grad_()), lambda: store(k=k.clone().requires_grad_())):
        with pytest.raises(RuntimeError):
            call()
    with torch.no_grad():
        attend(), shared(), store(), read()
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 40])
def test_tables_lengths_and_prefixes_that_are_none(lib, new):
    """entries of the tables outside the pool, lengths beyond the table and below zero, prefixes and groups that make no sense: whatever comes out, calls end and sequences whose
    numbers are right get their results; what cannot be stored is not"""
    from flash_attn import flash_attn_gfx950 as be
    from flash_attn import flash_attn_paged_interface as p
    c = Cache8([200, 90, 130, 77], 2, 64, 16, torch.float16, 5, cols=14).gpu()
    q, cu = randn(4 * new, 4, 64, seed=1).cuda(), cumulative([new] * 4).cuda()
    table, lens = c.dtable.clone(), c.dlens.clone()
    c.dk.view(torch.uint8)[:] = torch.where(c.dk.view(torch.uint8) & 127 == 127, 3, c.dk.view(torch.uint8))  # (no NaN where bad entries may point)
    c.dv.view(torch.uint8)[:] = torch.where(c.dv.view(torch.uint8) & 127 == 127, 3, c.dv.view(torch.uint8))
    c.dks.clamp_(max=130)
    c.dvs.clamp_(max=130)
    want = p.flash_attn_paged_func(q, c.dk, c.dv, table, cu, lens, new, 224, **c.scales)
    table[0, :4] = torch.tensor([-5, 2 ** 31 - 1, c.n_pages, -2 ** 31], dtype=torch.int32)
    lens[1], lens[2] = 2 ** 31 - 1, -7
    got = p.flash_attn_paged_func(q, c.dk, c.dv, table, cu, lens, new, 224, **c.scales)
    assert torch.equal(got[3 * new:], want[3 * new:]) and (got[2 * new:3 * new] == 0).all() and got.isfinite().all()
    for groups, prefix in (([0, 2, 4], [64, 64, 2 ** 31 - 1, -3]), ([0, 9, 4], [-2 ** 31, 16, 32, 48]), ([3, 1, 4], [224, 224, 224, 224]), ([-1, 2, 2 ** 31 - 1], [17, 1, 0, 5])):
        cg, pl = torch.tensor(groups, dtype=torch.int32).cuda(), torch.tensor(prefix, dtype=torch.int32).cuda()
        be.paged_fwd(q, c.dk, c.dv, table, cu, lens, new, 224, 0.125, True, True, cu_groups=cg, prefix_lens=pl, max_prefix_len=224, always=True, **c.scales)
    k, v = p.paged_read_func(c.dk, c.dv, table, cu, lens, 4 * new + 2, dtype=torch.float16, **c.scales)
    assert (k[2 * new:3 * new] == 0).all() and (v[4 * new:] == 0).all() and k.isfinite().all()
    before = [t.clone() for t in (c.dk.view(torch.uint8), c.dks)]
    bad = table.clone()
    bad[:] = torch.tensor([-1, c.n_pages], dtype=torch.int32).repeat(7)
    p.paged_append_func(None, q[:, :2], q[:, 2:], c.dk, c.dv, bad, cu, lens, **c.scales)
    assert torch.equal(c.dk.view(torch.uint8), before[0]) and torch.equal(c.dks, before[1])
    for cu_bad in ([0, -3, 5, 2 ** 31 - 1, 1], [7, 3, 2, 1, 0], [0, 0, 0, 0, 0]):
        x = torch.tensor(cu_bad, dtype=torch.int32).cuda()
        p.paged_append_func(None, q[:, :2], q[:, 2:], c.dk, c.dv, table, x, lens, **c.scales)
        p.paged_read_func(c.dk, c.dv, table, x, lens, 4 * new, dtype=torch.float16, **c.scales)
        be.paged_fwd(q, c.dk, c.dv, table, x, lens, new, 224, 0.125, True, True, cu_groups=cumulative([2, 2]).cuda(), prefix_lens=lens, max_prefix_len=64, always=True, **c.scales)
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 128])
def test_values_that_are_no_numbers_and_rows_without_keys(lib, D):
    """an infinity stored becomes NaN and reaches who sees it, and nobody else's sequence; tokens that see nothing give zeros and -inf"""
    from flash_attn import flash_attn_gfx950 as be
    from flash_attn import flash_attn_paged_interface as p
    c = Cache8([60, 60, 3], 2, D, 16, torch.float16, 2).gpu()
    k = randn(3, 2, D, seed=3)
    v = k.clone()
    v[1, 0, 4] = math.inf
    cu = cumulative([1, 1, 1]).cuda()
    p.paged_append_func(None, k.cuda(), v.cuda(), c.dk, c.dv, c.dtable, cu, c.dlens, **c.scales)
    q = randn(7, 4, D, seed=4).cuda()
    cu = cumulative([1, 1, 5]).cuda()
    for always in (False, True):
        more = dict(cu_groups=cumulative([1, 1, 1]).cuda(), prefix_lens=torch.tensor([16, 16, 0], dtype=torch.int32).cuda(), max_prefix_len=16, always=True) if always else {}
        out, lse = be.paged_fwd(q, c.dk, c.dv, c.dtable, cu, c.dlens, 5, 60, D ** -0.5, True, True, **more, **c.scales)
        assert out[0].isfinite().all() and out[1, :2, 4].isnan().all() and out[1, 2:].isfinite().all() and out[3:].isfinite().all()
        assert (out[2:4] == 0).all() and (lse[2, :, :2] == -math.inf).all() and (out[4:] != 0).any(-1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 40])
def test_a_captured_step_over_8_bits_and_a_prefix(lib, new):
    """store, attend, attend behind a prefix and read in one graph: replayed with other tokens, lengths, tables and prefixes in the same tensors, with eager calls in between"""
    from flash_attn import flash_attn_gfx950 as be
    from flash_attn import flash_attn_paged_interface as p
    lens = [[200, 177], [190, 300], [141, 140], [299, 301], [200, 177]]
    prefix = [96, 128, 0, 240, 96]
    caches = [share(Cache8(n, 2, 64, 16, torch.float16, i, cols=20, spare=60 - sum(-(-x // 16) for x in n)), [2], [m]).gpu() for i, (n, m) in enumerate(zip(lens, prefix))]
    qkvs = [randn(2 * new, 8, 64, seed=i).cuda() for i in range(len(lens))]
    cu, cg = cumulative([new, new]).cuda(), cumulative([2]).cuda()
    w = torch.ones(64, dtype=torch.float16, device="cuda")
    cos, sin = (t.cuda() for t in tables(400, 64, torch.float16))

    def step(c, qkv):
        s = dict(k_scales=c["ks"], v_scales=c["vs"])
        q = p.paged_append_func(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], c["k"], c["v"], c["table"], cu, c["lens"], q_weight=w, k_weight=w, cos_half=cos, sin_half=sin, **s)
        a, la = p.flash_attn_paged_func(q, c["k"], c["v"], c["table"], cu, c["lens"], new, 310, return_softmax_lse=True, **s)
        b, lb = be.paged_fwd(q, c["k"], c["v"], c["table"], cu, c["lens"], new, 310, 0.125, True, True, cu_groups=cg, prefix_lens=c["prefix"], max_prefix_len=256, always=True, **s)
        return a, la[..., :new], b, lb[..., :new], *p.paged_read_func(c["k"], c["v"], c["table"], cu, c["lens"], 2 * new, dtype=torch.float16, **s)

    def fresh(i):
        c = caches[i]
        return dict(k=c.dk.clone(), v=c.dv.clone(), ks=c.dks.clone(), vs=c.dvs.clone(), table=c.dtable.clone(), lens=c.dlens.clone(),
                    prefix=torch.full((2,), prefix[i], dtype=torch.int32, device="cuda"))

    with torch.no_grad():
        static, qkv = fresh(0), qkvs[0].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(static, qkv)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step(static, qkv)
        for i in range(len(lens)):
            eager = fresh(i)
            want = step(eager, qkvs[i])
            for k, v in fresh(i).items():
                static[k].copy_(v)
            qkv.copy_(qkvs[i])
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(got, want)), i
            assert all(torch.equal(static[k].view(torch.uint8), eager[k].view(torch.uint8)) for k in ("k", "v", "ks", "vs")), i


@pytest.mark.gpu
def test_two_threads_share_prefixes_on_their_own_streams(lib):
    import threading
    from flash_attn import flash_attn_gfx950 as be
    jobs = []
    for i, (lens, eight) in enumerate((([3000, 2900, 2100], True), ([1200, 1300], False))):
        c = share((Cache8 if eight else Cache)(lens, 2, 64, 64, torch.float16, 30 + i), [len(lens)], [1024]).gpu()
        q, cu, cg = randn(len(lens), 8, 64, seed=i).cuda(), cumulative([1] * len(lens)).cuda(), cumulative([len(lens)]).cuda()
        pl, scales = torch.full((len(lens),), 1024, dtype=torch.int32, device="cuda"), c.scales if eight else {}
        jobs.append(lambda q=q, c=c, cu=cu, cg=cg, pl=pl, n=max(lens), s=scales: be.paged_fwd(q, c.dk, c.dv, c.dtable, cu, c.dlens, 1, n, 0.125, True, cu_groups=cg, prefix_lens=pl,
                                                                                               max_prefix_len=1024, always=True, **s)[0])
    want = [job() for job in jobs]
    torch.cuda.synchronize()
    wrong = []

    def work(job, want):
        with torch.cuda.stream(torch.cuda.Stream()):
            outs = [job() for _ in range(30)]
            torch.cuda.current_stream().synchronize()
        wrong.extend(i for i, x in enumerate(outs) if not torch.equal(x, want))

    threads = [threading.Thread(target=work, args=a) for a in zip(jobs, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 50])
def test_8_bits_beyond_32_bit_offsets(lib, new):
    """pages whose offsets pass 2^32 give what pages at the front give, and so do pools inside larger ones"""
    from flash_attn import flash_attn_gfx950 as be
    from flash_attn import flash_attn_paged_interface as p
    PS, HK, D, lens = 64, 2, 128, [500, 411]
    pages = -(-(5 << 30) // (PS * HK * D))
    small = share(Cache8(lens, HK, D, PS, torch.float16, 5), [2], [256]).gpu()
    big = [torch.empty(pages, HK, PS, D, dtype=torch.uint8, device="cuda").transpose(1, 2) for _ in range(2)]
    exps = [torch.empty(pages, HK, PS, dtype=torch.uint8, device="cuda") for _ in range(2)]
    far = pages - small.n_pages
    for b, x, e, y in zip(big, (small.dk, small.dv), exps, (small.dks, small.dvs)):
        b[far:], e[far:] = x.view(torch.uint8), y
    table = torch.where(small.dtable >= 0, small.dtable + far, -1).to(torch.int32)
    qkv, cu, cg = randn(2 * new, 8, D, seed=6).cuda(), cumulative([new, new]).cuda(), cumulative([2]).cuda()
    pl = torch.full((2,), 256, dtype=torch.int32, device="cuda")
    got = []
    for k, v, t, ks, vs in ((*(b.view(torch.float8_e4m3fn) for b in big), table, *exps), (small.dk, small.dv, small.dtable, small.dks, small.dvs)):
        s = dict(k_scales=ks, v_scales=vs)
        q = p.paged_append_func(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], k, v, t, cu, small.dlens, **s)
        out = p.flash_attn_paged_func(q, k, v, t, cu, small.dlens, new, 500, **s)
        two = be.paged_fwd(q, k, v, t, cu, small.dlens, new, 500, 0.1, True, cu_groups=cg, prefix_lens=pl, max_prefix_len=256, always=True, **s)[0]
        got.append((out, two, *p.paged_read_func(k, v, t, cu, small.dlens, 2 * new, dtype=torch.float16, **s)))
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 40])
def test_queries_that_are_views(lib, new):
    """q, k and v as parts of a packed projection, tables and integers as parts of larger tensors"""
    from flash_attn import flash_attn_paged_interface as p
    c = Cache8([300, 280], 2, 64, 16, torch.bfloat16, 3).gpu()
    packed = randn(2 * new, 3, 4, 64, dtype=torch.bfloat16, seed=5)
    d = packed.cuda()
    cu = torch.cat([cumulative([new, new]).cuda()] * 2)[:3]
    table = torch.cat([c.dtable, c.dtable], 1)[:, :c.dtable.shape[1]]
    where = (c.dk, c.dv, table, cu, c.dlens)
    plain = p.flash_attn_paged_func(d[:, 1].contiguous(), *where, new, 300, **c.scales)
    out = p.flash_attn_paged_func(d[:, 1], *where, new, 300, **c.scales)
    assert torch.equal(out, plain)
    check_attention(packed[:, 1], c, [new, new], True, out)
    cg, pl = cumulative([2]).cuda(), torch.full((4,), 256, dtype=torch.int32, device="cuda")[1:3]
    share_table = table.clone()
    share_table[1, :16] = share_table[0, :16]
    args = (c.dk, c.dv, share_table, cu, c.dlens, new, 300)
    assert torch.equal(p.flash_attn_paged_prefix_func(d[:, 1], *args, cg, pl, 256, **c.scales), p.flash_attn_paged_prefix_func(d[:, 1].contiguous(), *args, cg, pl, 256, **c.scales))
    for k, v in ((d[:, 1, :2], d[:, 2, 2:]), (d[:, 1, :2].contiguous(), d[:, 2, 2:].contiguous())):
        q = p.paged_append_func(d[:, 0], k, v, *where, **c.scales)
        assert torch.equal(q, d[:, 0])
        got = p.paged_read_func(*where[:5], 2 * new, dtype=torch.bfloat16, **c.scales)
        want = [ref_quantise(t.double().cpu(), torch.bfloat16)[0] for t in (k, v)]
        assert same(got[0].cpu().double(), want[0]) and same(got[1].cpu().double(), want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 40])
def test_views_of_8_bit_pools(lib, new):
    from flash_attn import flash_attn_paged_interface as p
    c = Cache8([130, 90, 61], 2, 64, 32, torch.bfloat16, 8).gpu()
    qkv, cu = randn(3 * new, 8, 64, seed=2, dtype=torch.bfloat16).cuda(), cumulative([new] * 3).cuda()
    pools = torch.full((2, c.n_pages + 2, 3, 32, 80), 9, dtype=torch.uint8, device="cuda")
    for i, x in enumerate((c.dk, c.dv)):
        pools[i, 1:-1, :2, :, 16:] = x.view(torch.uint8).transpose(1, 2)
    view = [x[1:-1, :2, :, 16:].transpose(1, 2).view(torch.float8_e4m3fn) for x in pools]
    wide = torch.full((3, c.dtable.shape[1] + 5), 7, dtype=torch.int32, device="cuda")
    wide[:, 2:-3] = c.dtable
    got = []
    for k, v, table, ks, vs in ((c.dk, c.dv, c.dtable, c.dks.clone(), c.dvs.clone()), (*view, wide[:, 2:-3], c.dks.clone(), c.dvs.clone())):
        s = dict(k_scales=ks, v_scales=vs)
        q = p.paged_append_func(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], k, v, table, cu, c.dlens, **s)
        got.append((q, p.flash_attn_paged_func(q, k, v, table, cu, c.dlens, new, 130, **s), ks, vs, k.contiguous().view(torch.uint8), v.contiguous().view(torch.uint8),
                    *p.paged_read_func(k, v, table, cu, c.dlens, 3 * new, dtype=torch.bfloat16, **s)))
    assert all(torch.equal(a, b) for a, b in zip(*got))
    assert (pools[:, :, 2] == 9).all() and (pools[:, 0] == 9).all() and (pools[:, -1] == 9).all() and (pools[..., :16] == 9).all()


# ---- GPU: serving

@pytest.mark.gpu
@pytest.mark.parametrize("store", [None, torch.float8_e4m3fn])
def test_a_serving_loop_with_forks(lib, store):
    """a prompt, four forks of it, single tokens of all of them: attention over what the cache says it holds (read), at each step"""
    from flash_attn.flash_attn_paged_interface import PagedKVCache
    H, HK, D, dtype = 8, 2, 64, torch.bfloat16
    cache = PagedKVCache(2, 200, 32, HK, D, dtype=dtype, store_dtype=store)
    cos, sin = (t.cuda() for t in tables(2000, D, dtype))
    w = torch.ones(D, dtype=dtype, device="cuda")
    seed = 0

    def step(seqs, new):
        nonlocal seed
        s = cache.step(seqs, new)
        for layer in range(2):
            seed += 1
            qkv = randn(sum(new), H + 2 * HK, D, dtype=dtype, seed=seed).cuda()
            q = s.append(layer, qkv[:, :H], qkv[:, H:H + HK], qkv[:, H + HK:], q_weight=w, k_weight=w, cos_half=cos, sin_half=sin)
            out = s.attend(layer, q)
            k, v, cu = (t.cpu() for t in cache.read(layer, seqs))
            c = Cache([cache.length(x) for x in seqs], HK, D, 16, dtype, 0)
            for b, n in enumerate(c.lens):
                page, slot = c.where(b, n)
                c.k[page, slot], c.v[page, slot] = k[cu[b]:cu[b + 1]], v[cu[b]:cu[b + 1]]
            check_attention(q.cpu(), c, new, True, out)
        return s

    with torch.no_grad():
        a = cache.add()
        step([a], [1500])
        forks = [cache.fork(a, n) for n in (None, 1490, 1024, 700)]
        free = cache.free_pages()
        s = step([a] + forks, [1] * 5)
        # (700 tokens fill 21 pages of 32: a run of five would save less than the four that share 1024; those filled their pages)
        assert s.prefix[0].tolist() == [0, 4, 5] and s.prefix[1].tolist() == [1024] * 4 + [0] and cache.free_pages() == free - 1
        step([a] + forks[:2], [3, 1, 2])
        cache.remove(a)
        step(forks, [1, 1, 1, 1])
    for f in forks:
        cache.remove(f)
    assert cache.free_pages() == 200


@pytest.mark.gpu
def test_mha_over_a_cache_in_8_bits(lib):
    """FlashMHA.forward_cached: the block on a cache in 8 bits is the block with attention over what the cache holds"""
    from flash_attn.flash_attention import FlashMHA
    from flash_attn.flash_attn_paged_interface import PagedKVCache
    torch.manual_seed(1)
    m = FlashMHA(256, 4, causal=True, use_rotary_emb="1d", qk_norm=True, device="cuda", dtype=torch.float16).eval()
    x = torch.randn(70, 256, device="cuda", dtype=torch.float16)
    with torch.no_grad():
        c8, c16 = PagedKVCache(1, 12, 16, 4, 64, store_dtype=torch.float8_e4m3fn), PagedKVCache(1, 12, 16, 4, 64)
        a, b = c8.add(), c16.add()
        for at, n in ((0, 50), (50, 1), (51, 19)):
            y8 = m.forward_cached(x[at:at + n], c8.step([a], [n]))
            m.forward_cached(x[at:at + n], c16.step([b], [n]))
            # the same block on a cache in 16 bits that holds what the other one stands for
            k, v, _ = c8.read(0, [a])
            k16, v16 = c16.layer(0)
            t = torch.arange(at + n, device="cuda")
            page = torch.tensor(c16._pages[b], device="cuda")[t // 16]
            k16[page, t % 16], v16[page, t % 16] = k, v
            from flash_attn.flash_attn_paged_interface import flash_attn_paged_func
            q, kk, _ = m.Wqkv(x[at:at + n]).reshape(n, 3, 4, 64).unbind(1)
            from flash_attn.rotary import apply_qk_norm_rotary
            cos, sin = m.rotary_emb.tables_to(at + n, q)
            q, _ = apply_qk_norm_rotary(q, kk, m.q_norm_weight, m.k_norm_weight, cos, sin, positions=torch.arange(at, at + n, dtype=torch.int32, device="cuda"))
            cu, lens = cumulative([n]).cuda(), torch.tensor([at + n], dtype=torch.int32, device="cuda")
            o = flash_attn_paged_func(q, k16, v16, torch.tensor([list(c16._pages[b])], dtype=torch.int32, device="cuda"), cu, lens, n, at + n)
            y16 = m.out_proj(o.reshape(n, 256))
            # probabilities rounded at other places (2 u of the largest value on each side), the result once on each (u of it), through the projection's weights, which rounds
            # once on each side (u); fp32 sums of 256 products
            u = half_step(torch.float16)
            bound = m.out_proj.weight.float().abs().sum(1) * v.float().abs().max() * (6 * u + 1e-4) + 2 * u * y16.float().abs() + 1e-4
            assert ((y8.float() - y16.float()).abs() <= bound).all(), (at, ((y8.float() - y16.float()).abs() / bound).max())
