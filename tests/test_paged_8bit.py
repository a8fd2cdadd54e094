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
        spread = kw.pop("spread", 0.0)
        super().__init__(*a, **kw)
        g = torch.Generator().manual_seed(7)
        dtype, out = self.k.dtype, []
        for name in ("k", "v"):
            x = getattr(self, name).double()
            x = x * torch.exp(spread * torch.randn(x.shape[:-1], generator=g, dtype=torch.float64))[..., None]
            there = ~x.isnan().all(-1)
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
