"""The paged key / value cache and the norm of queries and keys in front of it: what the entry points refuse and the index arithmetic (CPU), and the
kernels against the definitions in 64 bits (GPU).

Tolerances are counted, not measured.  u: half a step of the element type (2^-11 fp16, 2^-8 bf16).  e = 2^-24: a rounding in fp32."""
import ctypes
import math
import os
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
E32 = 2.0 ** -24
DTYPES = [torch.float16, torch.bfloat16]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ---- the definitions, in 64 bits on the CPU

def ref_norm_rotary(x, w, cos, sin, t, eps):
    """x: (rows, heads, D) float64; t: (rows,) table rows"""
    y = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w
    if cos is None:
        return y
    c, s = cos[t][:, None], sin[t][:, None]
    a, b = y[..., 0::2], y[..., 1::2]
    return torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)


def tables(rows, D, dtype):
    angle = torch.outer(torch.arange(rows, dtype=torch.float64), 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D))
    return torch.cos(angle).to(dtype), torch.sin(angle).to(dtype)


class Cache:
    """A pool with sequences of the given lengths in it, pages in no order, NaN wherever nothing was stored."""

    def __init__(self, lens, HK, D, PS, dtype, seed, head_major=True, spare=3, cols=None):
        g = torch.Generator().manual_seed(seed)
        pages = [-(-n // PS) for n in lens]
        self.n_pages, self.PS, self.lens = sum(pages) + spare, PS, list(lens)
        order = torch.randperm(self.n_pages, generator=g).to(torch.int32)
        self.table = torch.full((len(lens), cols or max(max(pages), 1)), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(pages):
            self.table[b, :n] = order[at:at + n]
            at += n
        shape = (self.n_pages, HK, PS, D) if head_major else (self.n_pages, PS, HK, D)
        self.k = torch.full(shape, math.nan, dtype=dtype)
        self.v = torch.full(shape, math.nan, dtype=dtype)
        if head_major:
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        for b, n in enumerate(lens):
            for j in range(n):
                p = self.table[b, j // PS]
                self.k[p, j % PS] = torch.randn(HK, D, generator=g).to(dtype)
                self.v[p, j % PS] = torch.randn(HK, D, generator=g).to(dtype)
        self.weights = torch.zeros(self.n_pages, HK, PS)
        self.positions = torch.zeros(self.n_pages, HK, PS, dtype=torch.int32)

    def where(self, b, n):
        j = torch.arange(n)
        return self.table[b][j // self.PS].long(), j % self.PS

    def gpu(self):
        # (a copy that keeps the strides)
        self.dk, self.dv = (t.transpose(1, 2).contiguous().cuda().transpose(1, 2) if t.stride(1) < t.stride(2) else t.contiguous().cuda() for t in (self.k, self.v))
        self.dtable, self.dlens = self.table.cuda(), torch.tensor(self.lens, dtype=torch.int32).cuda()
        self.dweights, self.dpositions = self.weights.cuda(), self.positions.cuda()
        return self


def cumulative(n):
    return torch.tensor([0] + list(torch.tensor(n).cumsum(0)), dtype=torch.int32)


def ref_attention(q, cache, new, causal, scale):
    """out (total, H, D), lse {(b, h): (Lq,)}, received (n_pages, HK, PS), and the bounds of the errors of scores and of values"""
    H, HK, D = q.shape[1], cache.k.shape[2], q.shape[2]
    G = H // HK
    out, lse = torch.zeros(q.shape, dtype=torch.float64), {}
    got = torch.zeros(cache.n_pages, HK, cache.PS, dtype=torch.float64)
    tol = torch.zeros(q.shape, dtype=torch.float64)
    ds = 0.0
    at = 0
    for b, n in enumerate(new):
        Lk = cache.lens[b]
        page, slot = cache.where(b, Lk)
        for h in range(H):
            qh = q[at:at + n, h].double()
            k, v = cache.k[page, slot, h // G].double(), cache.v[page, slot, h // G].double()
            s = qh @ k.t() * scale
            if causal:
                s = s.masked_fill(torch.arange(Lk)[None] >= (Lk - n + 1 + torch.arange(n))[:, None], -math.inf)
            top = torch.logsumexp(s, 1) if Lk else torch.full((n,), -math.inf, dtype=torch.float64)
            p = torch.exp(s - torch.where(top.isinf(), 0.0, top)[:, None])
            o = p @ v if Lk else torch.zeros(n, D, dtype=torch.float64)
            out[at:at + n, h], lse[b, h] = o, top
            if Lk:
                got[page, h // G, slot] += p.sum(0)
                # a score: D products summed in fp32, scaled: (D + 4) roundings of at most the sum of magnitudes; the argument of the exponential 4 more
                mag = (qh.abs() @ k.abs().t()).max().item() * scale if n else 0.0
                ds = max(ds, (D + 4) * E32 * mag + 4 * E32 * 2 * mag)
                # probabilities rounded by u each, numerator and denominator alike: 2 u of the largest value; the scores' errors likewise; the sums of Lk
                # terms in fp32; the result's rounding
                u = half_step(q.dtype)
                tol[at:at + n, h] = (2 * u + 2 * ds + 2 * (Lk + 8) * E32) * v.abs().max() + u * o.abs()
        at += n
    return out, lse, got, tol, ds


# ---- CPU

def test_index_arithmetic_stays_in_bounds(tmp_path):
    """what is read from device memory and becomes an address, at the ends of its range"""
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(r'''
#include <cassert>
#include <climits>
#include <initializer_list>
#include "fa_paged_index.h"
using namespace fa;
int main() {
  const int v[] = {INT_MIN, INT_MIN + 1, -65536, -2, -1, 0, 1, 2, 6, 7, 8, 15, 16, 100, 65536, INT_MAX - 1, INT_MAX};
  for (int a : v)
    for (int n : {1, 2, 7, 8, 1 << 30, INT_MAX}) {
      assert(page_in_pool(a, n) >= 0 && page_in_pool(a, n) < n);
      assert(table_row(a, n) >= 0 && table_row(a, n) < n);
      assert(keys_in_reach(a, n) >= 0 && keys_in_reach(a, n) <= n);
      if (page_is_one(a, n)) assert(page_in_pool(a, n) == a);
      if (a >= 0 && a < n) assert(page_in_pool(a, n) == a && table_row(a, n) == a && keys_in_reach(a, n) == a && page_is_one(a, n));
      for (int begin : v)
        for (int end : v)
          for (int row : {0, 1, 5, 100}) {
            const bool sane = begin >= 0 && end >= begin && row >= begin && row < end;

            const int s = append_slot(a, begin, end, row, 50, n);
            assert(s >= -1 && s < n);
            if (!sane || end - begin > 50 || a < end - row) assert(s == -1);
            else if (a - (end - row) < n) assert(s == a - (end - row));
          }
    }
  assert(append_slot(10, 3, 7, 3, 4, 100) == 6 && append_slot(10, 3, 7, 6, 4, 100) == 9 && append_slot(10, 3, 7, 7, 4, 100) == -1);
  assert(append_slot(3, 3, 7, 3, 4, 100) == -1 && append_slot(10, 3, 7, 6, 4, 9) == -1);
}
''')
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", os.path.join(ROOT, "flash-attention_amd", "csrc"), str(src), "-o", str(exe)], check=True)
    subprocess.run([str(exe)], check=True)


def _cache_args(be, c):
    c.k_cache = c.v_cache = 1 << 20
    c.k_page_stride = c.v_page_stride = 2 * 16 * 64
    c.k_slot_stride = c.v_slot_stride = 64
    c.k_head_stride = c.v_head_stride = 16 * 64
    c.page_table = c.seqlens_k = c.cu_seqlens_q = c.key_weights = c.key_positions = 1 << 20
    c.table_row_stride = c.table_cols = 4
    c.n_pages, c.page_size = 8, 16
    c.batch, c.nheads_q, c.nheads_k, c.head_dim = 2, 4, 2, 64
    c.total_q, c.max_seqlen_q, c.max_seqlen_k = 0, 4, 64  # (no rows: a call that passes every check enqueues nothing)


def _args(be, kind):
    a = {"norm": be.QkNormArgs, "append": be.PagedAppendArgs, "fwd": be.PagedFwdArgs, "weights": be.PagedFwdArgs, "evict": be.PagedEvictArgs}[kind]()
    a.struct_bytes = ctypes.sizeof(a)
    if kind != "norm":
        _cache_args(be, a.cache)
    if kind == "norm":
        a.q = a.k = a.q_out = a.k_out = a.q_weight = a.k_weight = 1 << 20
        a.nheads_q, a.nheads_k, a.head_dim = 4, 2, 64
    elif kind == "evict":
        a.budget, a.recent = 8, 2
        a.next_positions, a.new_seqlens_k, a.workspace, a.workspace_bytes = 1 << 20, 1 << 21, 1 << 20, 0
    elif kind in ("fwd", "weights"):
        a.softmax_scale = 0.125
    return a


ENTRY = {"norm": "fa_qk_norm_rotary", "append": "fa_paged_append", "fwd": "fa_paged_fwd", "weights": "fa_paged_key_weights", "evict": "fa_paged_evict"}


@pytest.mark.parametrize("kind, change, says", [
    (k, *r) for k in ENTRY for r in [({"struct_bytes": 8}, "struct size")]
] + [
    (k, *r) for k in ("norm", "append", "fwd", "weights") for r in [({"dtype": 2}, "dtype"), ({"dtype": -1}, "dtype")]
] + [
    (k, *r) for k in ("append", "fwd", "weights", "evict") for r in [
        ({"cache.head_dim": 48}, "head_dim"), ({"cache.page_size": 8}, "page_size"), ({"cache.page_size": 48}, "page_size"), ({"cache.page_size": 2048}, "page_size"),
        ({"cache.batch": 0}, "positive"), ({"cache.nheads_k": 0}, "positive"), ({"cache.n_pages": 0}, "positive"), ({"cache.table_cols": 0}, "positive"),
        ({"cache.max_seqlen_k": 0}, "positive"), ({"cache.page_table": None}, "null"), ({"cache.seqlens_k": None}, "null"), ({"cache.table_row_stride": 3}, "overlap"),
        ({"cache.seqlens_k": (1 << 20) + 2}, "4-byte"), ({"cache.k_cache": None}, "k_cache"), ({"cache.k_cache": (1 << 20) + 8}, "16-byte"),
        ({"cache.k_slot_stride": 60}, "multiples of 8"), ({"cache.k_slot_stride": 1 << 24}, "multiples of 8"), ({"cache.k_head_stride": -64}, "multiples of 8"),
        ({"cache.k_page_stride": 4}, "multiples of 8"),
        ({"cache.page_size": 1024, "cache.table_cols": 1 << 21, "cache.table_row_stride": 1 << 21, "cache.max_seqlen_k": 2 ** 31 - 1}, "2^30 keys")]
] + [
    (k, *r) for k in ("append", "fwd", "weights") for r in [
        ({"cache.nheads_q": 3}, "multiple of nheads_k"), ({"cache.nheads_q": 4096}, "multiple of nheads_k"), ({"cache.cu_seqlens_q": None}, "cu_seqlens_q"),
        ({"cache.max_seqlen_q": 0}, "new tokens"), ({"cache.total_q": -1}, "new tokens")]
] + [
    (k, {"cache.v_cache": None}, "v_cache") for k in ("append", "fwd", "evict")
] + [
    (k, {"softmax_scale": s}, "softmax_scale") for k in ("fwd", "weights") for s in (0.0, -1.0, math.inf, math.nan)
] + [
    ("append", {"cache.k_slot_stride": 8}, "overlap"), ("append", {"cache.v_head_stride": 0}, "overlap"), ("append", {"cache.k_page_stride": 0}, "overlap"),
    ("append", {"cache.total_q": 1}, "k and v"), ("append", {"cache.total_q": 1, "k": 1 << 20, "v": 1 << 20, "q": 1 << 20}, "q and q_out"),
    ("append", {"cache.total_q": 1, "k": 1 << 20, "v": 1 << 20, "k_weight": 1 << 20, "weight_dtype": 1}, "weights must be"),
    ("append", {"cache.total_q": 1, "k": 1 << 20, "v": 1 << 20, "cos_table": 1 << 20}, "come together"),
    ("append", {"cache.total_q": 1, "k": 1 << 20, "v": 1 << 20, "eps": -1.0}, "eps"),
    ("fwd", {"cache.total_q": 1}, "q must be"), ("fwd", {"cache.total_q": 1, "q": 1 << 20}, "o must be"),
    ("weights", {"cache.total_q": 1, "q": 1 << 20}, "softmax_lse"),
    ("evict", {"budget": 0}, "budget"), ("evict", {"recent": -1}, "recent"), ("evict", {"new_seqlens_k": 1 << 20, "cache.seqlens_k": 1 << 20}, "may not be"),
    ("evict", {"cache.key_weights": None}, "needed"), ("evict", {"next_positions": None}, "needed"), ("evict", {"cache.key_weights": (1 << 20) + 4}, "16-byte"), ("evict", {"cache.batch": 40000}, "65535"), ("evict", {}, "workspace"),
    ("norm", {"head_dim": 24}, "head_dim"), ("norm", {"weight_dtype": 1}, "weights must be"), ("norm", {"n_rows": -1}, "n_rows"), ("norm", {"n_rows": 1 << 30}, "n_rows"),
    ("norm", {"nheads_q": -1}, "heads"), ("norm", {"eps": -1.0}, "eps"), ("norm", {"eps": math.nan}, "eps"),
    ("norm", {"n_rows": 1, "cos_table": 1 << 20}, "come together"), ("norm", {"n_rows": 1, "cos_table": 1 << 20, "sin_table": 1 << 20}, "empty table"),
    ("norm", {"n_rows": 1, "cos_table": 1 << 20, "sin_table": 1 << 20, "table_rows": 4, "seqlen": 5}, "4 rows"),
    ("norm", {"n_rows": 1, "q": None}, "null"), ("norm", {"n_rows": 1, "q": (1 << 20) + 2}, "16-byte"), ("norm", {"n_rows": 1, "q_row_stride": 4}, "multiples of 8"),
    ("norm", {"n_rows": 2}, "overlap"),
])
def test_entry_points_refuse(lib, kind, change, says):
    from flash_attn import flash_attn_gfx950 as be
    a = _args(be, kind)
    for name, value in change.items():
        at = a
        for part in name.split(".")[:-1]:
            at = getattr(at, part)
        setattr(at, name.split(".")[-1], value)
    assert getattr(lib, ENTRY[kind])(ctypes.byref(a)) < 0
    assert says in lib.fa_last_error().decode(), lib.fa_last_error()


@pytest.mark.parametrize("kind", ["norm", "append", "fwd", "weights"])
def test_calls_without_rows_do_nothing(lib, kind):
    from flash_attn import flash_attn_gfx950 as be
    assert getattr(lib, ENTRY[kind])(ctypes.byref(_args(be, kind))) == 0, lib.fa_last_error()


def test_struct_sizes_match_the_header(tmp_path):
    from flash_attn import flash_attn_gfx950 as be
    names = ("fa_qk_norm_args", "fa_paged_cache", "fa_paged_append_args", "fa_paged_fwd_args", "fa_paged_evict_args")
    src, exe = tmp_path / "s.c", tmp_path / "s"
    src.write_text('#include "flash_attn_gfx950.h"\n#include <stdio.h>\nint main(void) { printf("%s", %s); return 0; }\n' % (
        " ".join(["%zu"] * len(names)), ", ".join("sizeof(%s)" % n for n in names)))
    subprocess.run(["gcc", "-std=c99", "-pedantic", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    sizes = [int(x) for x in subprocess.run([str(exe)], check=True, stdout=subprocess.PIPE).stdout.split()]
    assert sizes == [ctypes.sizeof(c) for c in (be.QkNormArgs, be.PagedCacheArgs, be.PagedAppendArgs, be.PagedFwdArgs, be.PagedEvictArgs)]


def test_workspace_sizes_depend_on_the_integers_alone(lib):
    from flash_attn import flash_attn_gfx950 as be
    a = _args(be, "fwd")
    a.cache.max_seqlen_q, a.cache.max_seqlen_k, a.cache.table_cols, a.cache.table_row_stride = 1, 100000, 7000, 7000
    n = lib.fa_paged_fwd_workspace_bytes(ctypes.byref(a))
    assert n > 0
    a.cache.k_cache = a.cache.v_cache = None
    assert lib.fa_paged_fwd_workspace_bytes(ctypes.byref(a)) == n
    a.cache.max_seqlen_k = 100
    assert lib.fa_paged_fwd_workspace_bytes(ctypes.byref(a)) == 0
    a.cache.head_dim = 20
    assert lib.fa_paged_fwd_workspace_bytes(ctypes.byref(a)) == 0


@pytest.mark.parametrize("turn", [False, True])
def test_norm_rotary_gradient_formula_against_differences(turn):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(3, 2, 16, generator=g, dtype=torch.float64, requires_grad=True)
    w = torch.randn(16, generator=g, dtype=torch.float64, requires_grad=True)
    cos, sin = tables(9, 16, torch.float64) if turn else (None, None)
    assert torch.autograd.gradcheck(lambda x, w: ref_norm_rotary(x, w, cos, sin, torch.tensor([0, 8, 3]), 1e-3), (x, w))


# ---- GPU: norm and rotation

def _norm_case(rows, H, HK, D, dtype, wdtype, seed, packed):
    g = torch.Generator().manual_seed(seed)
    if packed:  # q and k as strided views of one tensor, as a fused projection leaves them
        qkv = torch.randn(rows, H + 2 * HK, D, generator=g).to(dtype).cuda()
        q, k = qkv[:, :H], qkv[:, H:H + HK]
    else:
        q, k = (torch.randn(rows, n, D, generator=g).to(dtype).cuda() for n in (H, HK))
    w = [(1 + 0.3 * torch.randn(D, generator=g)).to(wdtype).cuda() for _ in range(2)]
    pos = torch.randint(0, 50, (rows,), generator=g, dtype=torch.int32)
    return q, k, w, pos


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, H, HK, D, fp32, packed, turn", [
    (1, 1, 1, 16, False, False, True), (61, 12, 12, 64, False, False, True), (7, 3, 1, 32, True, True, True), (130, 8, 2, 128, False, True, True),
    (5, 40, 40, 128, True, False, True),  # rows wider than a workgroup
    (33, 33, 1, 128, False, False, True),  # ... beside one that is not
    (2500, 4, 4, 64, False, True, True), (300, 1, 5, 16, True, False, False), (17, 6, 6, 128, False, False, False),
    (6000, 20, 3, 128, False, True, True), (12000, 8, 8, 64, True, True, True)])  # more rows than the launch has workgroups for
def test_norm_rotary_forward_and_backward(dtype, rows, H, HK, D, fp32, packed, turn):
    from flash_attn.rotary import apply_qk_norm_rotary
    eps = 1e-5
    wdtype = torch.float32 if fp32 else dtype
    q, k, w, pos = _norm_case(rows, H, HK, D, dtype, wdtype, rows + D, packed)
    cos, sin = tables(50, D, dtype)
    for t in (q, k, *w):
        t.requires_grad_()
    args = (cos.cuda(), sin.cuda(), pos.cuda()) if turn else (None, None, None)
    q2, k2 = apply_qk_norm_rotary(q, k, w[0], w[1], *args, eps=eps)
    g = torch.Generator().manual_seed(7)
    dq, dk = (torch.randn(t.shape, generator=g).to(dtype).cuda() for t in (q, k))
    grads = torch.autograd.grad((q2, k2), (q, k, *w), (dq, dk))
    u, uw = half_step(dtype), half_step(wdtype)
    c64, s64 = (cos.double(), sin.double()) if turn else (None, None)
    for x, y, ww, dy, dx, dw in ((q, q2, w[0], dq, grads[0], grads[2]), (k, k2, w[1], dk, grads[1], grads[3])):
        x64, w64 = x.detach().cpu().double().requires_grad_(), ww.detach().cpu().double().requires_grad_()
        want = ref_norm_rotary(x64, w64, c64, s64, pos.long(), eps)
        gx, gw = torch.autograd.grad(want, (x64, w64), dy.cpu().double())
        want = want.detach()
        # fp32 along the way: D + 16 roundings of magnitudes that the two products of a pair have (at most the pair's length each)
        pair = (want[..., 0::2].pow(2) + want[..., 1::2].pow(2)).sqrt().repeat_interleave(2, -1)
        assert ((y.detach().cpu().double() - want).abs() <= u * want.abs() + (D + 16) * E32 * 2 * pair + 1e-7).all()
        # dx: the difference of two terms, the second with a sum over D
        r = 1 / torch.sqrt(x64.detach().pow(2).mean(-1, keepdim=True) + eps)
        gt = dy.cpu().double()
        if turn:
            c, s = c64[pos.long()][:, None], s64[pos.long()][:, None]
            a, b = gt[..., 0::2], gt[..., 1::2]
            gt = torch.stack((a * c + b * s, b * c - a * s), -1).flatten(-2)
        size = dy.cpu().double().reshape(rows, -1, D // 2, 2).norm(dim=-1).repeat_interleave(2, -1)
        xh, ga = x64.detach() * r, size * w64.detach().abs()
        mag = r * (ga + xh.abs() * (ga * xh.abs()).mean(-1, keepdim=True))
        assert ((dx.cpu().double() - gx).abs() <= u * gx.abs() + (2 * D + 40) * E32 * mag + 1e-7).all()
        n = rows * x.shape[1]
        assert ((dw.cpu().double() - gw).abs() <= uw * gw.abs() + (n + D + 40) * E32 * (size * xh.abs()).sum((0, 1)) + 1e-7).all()
        assert dw.dtype == wdtype and dx.shape == x.shape


@pytest.mark.gpu
def test_norm_rotary_of_a_batch_takes_places_in_the_sequence_and_repeats_bit_for_bit():
    from flash_attn.rotary import apply_qk_norm_rotary
    g = torch.Generator().manual_seed(3)
    q, k = torch.randn(3, 37, 4, 64, generator=g).half().cuda().requires_grad_(), torch.randn(3, 37, 2, 64, generator=g).half().cuda()
    w = torch.ones(64, dtype=torch.float16, device="cuda").requires_grad_()
    cos, sin = (t.cuda() for t in tables(40, 64, torch.float16))
    pos = torch.arange(37, dtype=torch.int32).repeat(3).cuda()
    a = apply_qk_norm_rotary(q, k, w, w, cos, sin)
    b = apply_qk_norm_rotary(q.reshape(111, 4, 64), k.reshape(111, 2, 64), w, w, cos, sin, positions=pos)
    assert torch.equal(a[0].reshape(111, 4, 64), b[0]) and torch.equal(a[1].reshape(111, 2, 64), b[1])
    # positions outside the tables stand for their ends
    far = torch.where(pos == 36, 1000, torch.where(pos == 0, -5, pos))
    near = torch.where(pos == 36, 39, pos)
    x, y = (apply_qk_norm_rotary(q.reshape(111, 4, 64), k.reshape(111, 2, 64), w, w, cos, sin, positions=p)[0] for p in (far, near))
    assert torch.equal(x, y)
    grads = [torch.autograd.grad(apply_qk_norm_rotary(q, k, w, w, cos, sin)[0].float().square().sum(), (q, w)) for _ in range(3)]
    assert all(torch.equal(g0, g1) for other in grads[1:] for g0, g1 in zip(grads[0], other))


@pytest.mark.gpu
def test_norm_rotary_keeps_special_values_apart():
    """a vector of zeros, of infinities, with a NaN: what the formula gives, in that vector alone"""
    from flash_attn.rotary import apply_qk_norm_rotary
    q = torch.randn(4, 2, 32, generator=torch.Generator().manual_seed(0)).bfloat16()
    q[0, 0], q[1, 1, 3], q[2, 0, 5] = 0, math.inf, math.nan
    w = torch.ones(32, dtype=torch.bfloat16).cuda()
    y, _ = apply_qk_norm_rotary(q.cuda(), q.cuda(), w, w, eps=1e-6)
    y = y.cpu()
    assert (y[0, 0] == 0).all() and y[2, 0].isnan().all()
    assert y[1, 1, 3].isnan() and (torch.cat((y[1, 1, :3], y[1, 1, 4:])) == 0).all()
    rest = torch.ones(4, 2, dtype=torch.bool)
    rest[1, 1] = rest[2, 0] = False
    assert y[rest].isfinite().all()


# ---- GPU: the cache

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens, new, H, HK, D, PS, head_major, norm, turn, fp32", [
    ([5], [5], 1, 1, 16, 16, True, False, False, False),
    ([40, 17, 1], [1, 1, 1], 8, 2, 64, 16, True, True, True, False),
    ([33, 64, 100, 16], [33, 0, 7, 16], 6, 3, 128, 32, False, True, True, True),
    ([700] + list(range(1, 80)), [650] + [1] * 79, 4, 4, 32, 64, True, True, True, False),  # more sequences than a wave has lanes; several rows a workgroup
    ([300, 90], [290, 61], 20, 20, 128, 16, False, False, True, False),
    ([900, 3, 710], [880, 1, 700], 20, 20, 128, 16, True, True, True, False)])  # more rows than the launch has workgroups for
def test_append(dtype, lens, new, H, HK, D, PS, head_major, norm, turn, fp32):
    from flash_attn.flash_attn_paged_interface import paged_append_func
    c = Cache(lens, HK, D, PS, dtype, 1, head_major).gpu()
    g = torch.Generator().manual_seed(2)
    total, spare = sum(new), 2  # two rows behind the last sequence
    rows = torch.randn(total + spare, H + 2 * HK, D, generator=g).to(dtype)
    q, k, v = rows[:, :H], rows[:, H:H + HK], rows[:, H + HK:]
    drows = rows.cuda()
    dq, dk, dv = drows[:, :H], drows[:, H:H + HK], drows[:, H + HK:]
    wdtype = torch.float32 if fp32 else dtype
    w = [(1 + 0.3 * torch.randn(D, generator=g)).to(wdtype) for _ in range(2)]
    cos, sin = tables(max(lens), D, dtype)
    before = [t.clone() for t in (c.dk, c.dv, c.dweights, c.dpositions)]
    c.dweights.fill_(3.0)
    c.dpositions.fill_(-7)
    opt = {}
    if norm:
        opt.update(q_weight=w[0].cuda(), k_weight=w[1].cuda(), eps=1e-5)
    if turn:
        opt.update(cos_half=cos.cuda(), sin_half=sin.cuda())
    out = paged_append_func(dq, dk, dv, c.dk, c.dv, c.dtable, cumulative(new).cuda(), c.dlens, key_weights=c.dweights, key_positions=c.dpositions, **opt)
    u = half_step(dtype)
    kc, vc, wc, pc = c.k.clone(), c.v.clone(), torch.full_like(c.weights, 3.0), torch.full_like(c.positions, -7)
    stored = torch.zeros(c.n_pages, PS, dtype=torch.bool)
    at = 0
    for b, n in enumerate(new):
        t = torch.arange(lens[b] - n, lens[b])
        page, slot = c.table[b][t // PS].long(), t % PS
        for x, y, ww in ((q, out[:, :].cpu(), w[0]), (k, None, w[1])):
            x64 = x[at:at + n].double()
            if norm:
                want = ref_norm_rotary(x64, ww.double(), *((cos.double(), sin.double()) if turn else (None, None)), t, 1e-5)
            elif turn:
                a, bb = x64[..., 0::2], x64[..., 1::2]
                cc, ss = cos.double()[t][:, None], sin.double()[t][:, None]
                want = torch.stack((a * cc - bb * ss, bb * cc + a * ss), -1).flatten(-2)
            else:
                want = x64
            have = (y[at:at + n] if y is not None else c.dk.cpu()[page, slot]).double()
            pair = (want[..., 0::2].pow(2) + want[..., 1::2].pow(2)).sqrt().repeat_interleave(2, -1)
            assert ((have - want).abs() <= u * want.abs() + (D + 16) * E32 * 2 * pair + 1e-7).all()
        stored[page, slot] = True
        vc[page, slot] = v[at:at + n]
        wc[page, :, slot], pc[page, :, slot] = 0.0, t.to(torch.int32)[:, None]
        at += n
    same = lambda a, b: torch.equal(torch.nan_to_num(a.float(), 123.0), torch.nan_to_num(b.float(), 123.0))  # noqa: E731
    assert same(c.dv.cpu(), vc) and torch.equal(c.dweights.cpu(), wc) and torch.equal(c.dpositions.cpu(), pc)
    assert same(c.dk.cpu()[~stored], before[0].cpu()[~stored])  # nothing else was touched


@pytest.mark.gpu
def test_append_drops_what_has_no_slot_and_takes_given_positions():
    """entries of the table that are no pages, tokens before the first slot or behind the last: dropped; the pool's other pages stay as they are"""
    from flash_attn.flash_attn_paged_interface import paged_append_func
    c = Cache([40, 40, 40], 2, 64, 16, torch.float16, 1).gpu()
    table = c.table.clone()
    table[0, 1], table[0, 2] = -3, c.n_pages  # sequence 0: only its first page is one
    lens = torch.tensor([40, 2, 49], dtype=torch.int32)  # sequence 1: four new tokens of two; sequence 2: its last token is behind the table
    new = [20, 4, 3]
    rows = torch.randn(27, 2, 64, generator=torch.Generator().manual_seed(5)).half()
    kc = c.k.clone()
    for row, (b, j) in enumerate([(0, 20 + i) for i in range(20)] + [(1, i - 2) for i in range(4)] + [(2, 46 + i) for i in range(3)]):
        if b == 1 and j >= 0 or b == 2 and j < 48:
            kc[table[b, j // 16], j % 16] = rows[row]
    pos = torch.arange(100, 127, dtype=torch.int32)
    assert paged_append_func(None, rows.cuda(), rows.cuda(), c.dk, c.dv, table.cuda(), cumulative(new).cuda(), lens.cuda(), positions=pos.cuda(),
                             key_positions=c.dpositions) is None
    assert torch.equal(torch.nan_to_num(c.dk.cpu(), 99.0), torch.nan_to_num(kc, 99.0))
    assert c.dpositions.cpu()[table[1, 0], 0, :2].tolist() == [122, 123] and c.dpositions.cpu()[table[2, 2], 1, 14:].tolist() == [124, 125]


ATTEND = [
    # lens, new, H, HK, D, PS, head_major: few rows a key head
    ([1], [1], 1, 1, 16, 16, True), ([31, 32, 33], [1, 1, 1], 4, 4, 64, 16, True), ([500], [1], 12, 12, 64, 16, True),
    ([129, 1000, 16, 255], [1, 1, 1, 1], 8, 2, 128, 64, True), ([700, 90], [5, 3], 12, 2, 32, 32, False), ([2000, 3, 1301], [4, 3, 2], 8, 1, 128, 128, True),
    ([300, 0, 77], [1, 1, 1], 6, 2, 64, 16, False), ([90, 20], [0, 1], 2, 2, 128, 16, True), ([3000], [32], 2, 2, 16, 256, True),
    ([400 - i for i in range(70)], [1] * 70, 4, 2, 32, 32, True),  # more sequences than a wave has lanes
    # many rows
    ([64], [64], 2, 2, 64, 16, True), ([200, 333], [130, 33], 4, 4, 64, 16, True), ([517, 100, 129], [257, 100, 1], 8, 2, 128, 32, False),
    ([150, 40], [150, 40], 6, 2, 32, 64, True), ([1500], [40], 4, 4, 128, 128, True), ([100, 300], [90, 70], 3, 1, 16, 16, True),
    ([1100], [17], 24, 1, 64, 1024, True), ([30, 200], [60, 100], 2, 1, 128, 16, True),  # more new tokens than keys: the first see none
    ([20, 0], [50, 40], 2, 1, 64, 16, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens, new, H, HK, D, PS, head_major", ATTEND)
def test_attention_and_weights(dtype, causal, lens, new, H, HK, D, PS, head_major):
    from flash_attn.flash_attn_paged_interface import flash_attn_paged_func, paged_key_weights_func
    c = Cache(lens, HK, D, PS, dtype, 11, head_major).gpu()
    q = torch.randn(sum(new), H, D, generator=torch.Generator().manual_seed(12)).to(dtype)
    cu, mq, mk = cumulative(new).cuda(), max(new), max(max(lens), 1)
    want, lse64, got64, tol, ds = ref_attention(q, c, new, causal, D ** -0.5)
    out, lse = flash_attn_paged_func(q.cuda(), c.dk, c.dv, c.dtable, cu, c.dlens, mq, mk, causal=causal, return_softmax_lse=True)
    assert ((out.cpu().double() - want).abs() <= tol + 1e-7).all(), (out.cpu().double() - want).abs().max()
    alone = flash_attn_paged_func(q.cuda(), c.dk, c.dv, c.dtable, cu, c.dlens, mq, mk, causal=causal)
    assert ((alone.cpu().double() - want).abs() <= tol + 1e-7).all()
    lse_in = torch.full((len(lens), H, (mq + 15) // 16 * 16), math.nan)
    for (b, h), x in lse64.items():
        have = lse[b, h, :new[b]].cpu().double()
        dead = x == -math.inf
        assert torch.equal(have == -math.inf, dead)
        # a sum of Lk exponentials in fp32, its logarithm and the scaled maximum
        assert ((have - x)[~dead].abs() <= ds + (lens[b] + 16) * E32 + 8 * E32 * (x[~dead].abs() + 8)).all()
        lse_in[b, h, :new[b]] = x.float()
    c.dweights.fill_(0.5)
    w = paged_key_weights_func(q.cuda(), lse_in.cuda(), c.dk, c.dweights, c.dtable, cu, c.dlens, mq, mk, causal=causal)
    assert w is c.dweights
    # a term exp(s - lse): the score's error, lse rounded to fp32, the exponential; sums of all rows in fp32
    top = max([x[x > -math.inf].abs().max().item() for x in lse64.values() if (x > -math.inf).any()] or [0.0])
    rel = ds + 8 * E32 * (top + 8) + (max(new) * (H // HK) + 64) * E32
    assert ((w.cpu().double() - 0.5 - got64).abs() <= rel * got64 + 2 * E32).all()


@pytest.mark.gpu
@pytest.mark.parametrize("mk", [640, 1300, 5000, 9000])  # the bound chooses the launch: a workgroup a pair, or shares of the line of all keys
@pytest.mark.parametrize("lens, HK, D", [
    ([1, 200, 127, 0, 640] * 7, 4, 64), ([600, 3] * 33, 4, 32), ([129, 128, 300, 5, 640, 1, 1] * 10, 5, 16), ([513, 70] * 33, 5, 128)])
def test_few_rows_however_the_pairs_are_dealt_out(lens, HK, D, mk):
    from flash_attn.flash_attn_paged_interface import flash_attn_paged_func
    c = Cache(lens, HK, D, 16, torch.float16, 21, cols=600).gpu()
    new = [0 if i % 9 == 8 else 1 + (i % 4 == 1) for i in range(len(lens))]
    q = torch.randn(sum(new), 2 * HK, D, generator=torch.Generator().manual_seed(22)).half()
    want, lse64, _, tol, ds = ref_attention(q, c, new, True, D ** -0.5)
    call = lambda: flash_attn_paged_func(q.cuda(), c.dk, c.dv, c.dtable, cumulative(new).cuda(), c.dlens, 2, mk, return_softmax_lse=True)  # noqa: E731
    out, lse = call()
    assert ((out.cpu().double() - want).abs() <= tol + 1e-7).all()
    for (b, h), x in lse64.items():
        have = lse[b, h, :new[b]].cpu().double()
        dead = x == -math.inf
        assert torch.equal(have == -math.inf, dead)
        assert ((have - x)[~dead].abs() <= ds + (lens[b] + 16) * E32 + 8 * E32 * (x[~dead].abs() + 8)).all()
    for _ in range(3):
        assert torch.equal(call()[0], out)  # the same bits each time


@pytest.mark.gpu
@pytest.mark.parametrize("new, mk", [([1, 1], 5000), ([40, 70], 400)])
def test_attention_ignores_what_lies_behind(new, mk):
    """strided queries and outputs, rows behind the last sequence, a longer table and bound than needed: the same bits, nothing else written"""
    from flash_attn import flash_attn_gfx950 as be
    c = Cache([300, 140], 2, 64, 16, torch.float16, 3, cols=400).gpu()
    total = sum(new)
    wide = torch.randn(total + 3, 9, 64, generator=torch.Generator().manual_seed(4)).half().cuda()
    q, cu = wide[:, 3:7], cumulative(new).cuda()
    out = torch.full((total + 3, 6, 64), 7.0, dtype=torch.float16, device="cuda")
    be.paged_fwd(q, c.dk, c.dv, c.dtable, cu, c.dlens, max(new), mk, 0.125, True, out=out[:, 1:5])
    plain = be.paged_fwd(q[:total].contiguous(), c.dk, c.dv, c.dtable, cu, c.dlens, max(new), mk, 0.125, True)[0]
    assert torch.equal(out[:total, 1:5], plain)
    assert (out[total:] == 7).all() and (out[:, 0] == 7).all() and (out[:, 5] == 7).all()


@pytest.mark.gpu
def test_attention_reads_no_page_outside_the_pool():
    """table entries that are no pages stand for the pool's first or last one"""
    from flash_attn.flash_attn_paged_interface import flash_attn_paged_func
    c = Cache([100, 100], 1, 64, 16, torch.float16, 3, spare=0).gpu()
    q = torch.randn(2, 1, 64, generator=torch.Generator().manual_seed(4)).half().cuda()
    bad, good = c.table.clone(), c.table.clone()
    bad[0, 2], bad[1, 3] = -2 ** 31, 2 ** 31 - 1
    good[0, 2], good[1, 3] = 0, c.n_pages - 1
    c.dk.nan_to_num_(0.25)
    c.dv.nan_to_num_(0.25)
    cu = cumulative([1, 1]).cuda()
    a, b = (flash_attn_paged_func(q, c.dk, c.dv, t.cuda(), cu, c.dlens, 1, 100) for t in (bad, good))
    assert torch.equal(a, b)
    # lengths beyond the table: as far as it goes
    a, b = (flash_attn_paged_func(q, c.dk, c.dv, good.cuda(), cu, torch.tensor(n, dtype=torch.int32).cuda(), 1, 100000) for n in ([2 ** 31 - 1, -5], [112, 0]))
    assert torch.equal(a, b) and (b[1] == 0).all()


def ref_evict(c, lens, weights, positions, nxt, budget, recent):
    """(moves {(b, h): [(to, from)]}, new lengths)"""
    moves = {}
    for b, n in enumerate(lens):
        page, slot = c.where(b, n)
        for h in range(weights.shape[1]):
            if n <= budget:
                continue
            w, p = weights[page, h, slot].tolist(), positions[page, h, slot].tolist()
            rank = lambda j: (0, 0.0, j) if p[j] >= nxt[b] - recent else (1, math.inf if w[j] != w[j] else -w[j], j)  # noqa: E731
            stay = set(sorted(range(n), key=rank)[:budget])
            moves[b, h] = list(zip([j for j in range(budget) if j not in stay], [j for j in range(budget, n) if j in stay]))
    return moves, [min(n, budget) for n in lens]


@pytest.mark.gpu
@pytest.mark.parametrize("lens, HK, D, PS, budget, recent, kind", [
    ([17], 1, 16, 16, 16, 4, "random"), ([100, 40, 64], 3, 64, 16, 40, 8, "random"), ([100, 100], 2, 128, 32, 99, 0, "random"), ([300, 7], 2, 32, 64, 1, 0, "random"),
    ([257, 300], 2, 64, 16, 200, 200, "random"), ([200], 2, 64, 16, 100, 300, "random"), ([500, 129], 2, 64, 128, 128, 16, "ties"), ([400], 3, 32, 16, 150, 10, "special"),
    ([5000, 4097], 1, 16, 64, 2500, 100, "ties"), ([17000], 1, 16, 256, 9000, 1000, "random"), ([33000, 20], 1, 16, 1024, 20000, 50, "ties")])
def test_evict(lens, HK, D, PS, budget, recent, kind):
    from flash_attn.flash_attn_paged_interface import paged_evict_func
    g = torch.Generator().manual_seed(len(lens) + budget)
    c = Cache([1] * len(lens), HK, D, PS, torch.bfloat16, 2)  # (made by hand below: long sequences)
    pages = [-(-n // PS) for n in lens]
    c.n_pages, c.lens = sum(pages) + 2, list(lens)
    c.table = torch.full((len(lens), max(pages)), -1, dtype=torch.int32)
    order, at = torch.randperm(c.n_pages, generator=g).to(torch.int32), 0
    for b, n in enumerate(pages):
        c.table[b, :n] = order[at:at + n]
        at += n
    c.k, c.v = (torch.randn(c.n_pages, HK, PS, D, generator=g).bfloat16().transpose(1, 2) for _ in range(2))
    c.weights = torch.rand(c.n_pages, HK, PS, generator=g) * torch.tensor([1.0, 1e-30, 1e30])[torch.randint(0, 3, (c.n_pages, HK, PS), generator=g)]
    if kind == "ties":
        c.weights = torch.randint(0, 3, c.weights.shape, generator=g).float() * 0.5 * torch.where(torch.rand(c.weights.shape, generator=g) < 0.5, 1.0, -0.0)
    if kind == "special":
        pick = torch.randint(0, 8, c.weights.shape, generator=g)
        for i, x in enumerate((math.nan, math.inf, -math.inf, -1.0, -0.0)):
            c.weights[pick == i] = x
    c.positions = torch.zeros(c.n_pages, HK, PS, dtype=torch.int32)
    for b, n in enumerate(lens):
        page, slot = c.where(b, n)
        for h in range(HK):
            c.positions[page, h, slot] = torch.randperm(n, generator=g).to(torch.int32)
    c.gpu()
    c.dweights, c.dpositions = c.weights.cuda(), c.positions.cuda()
    moves, lens2 = ref_evict(c, lens, c.weights, c.positions, lens, budget, recent)
    k, v, w, p = c.k.clone(), c.v.clone(), c.weights.clone(), c.positions.clone()
    for (b, h), pairs in moves.items():
        for to, frm in pairs:
            tp, ts, fp, fs = c.table[b, to // PS], to % PS, c.table[b, frm // PS], frm % PS
            k[tp, ts, h], v[tp, ts, h] = c.k[fp, fs, h], c.v[fp, fs, h]
            w[tp, h, ts], p[tp, h, ts] = c.weights[fp, h, fs], c.positions[fp, h, fs]
    out = paged_evict_func(c.dk, c.dv, c.dweights, c.dpositions, c.dtable, c.dlens, c.dlens, budget, recent, max(lens))
    assert out.tolist() == lens2
    assert torch.equal(c.dpositions.cpu(), p)
    assert torch.equal(torch.nan_to_num(c.dweights.cpu(), 55.0), torch.nan_to_num(w, 55.0)) and torch.equal(c.dk.cpu(), k) and torch.equal(c.dv.cpu(), v)
