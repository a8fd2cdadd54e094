"""The operators of a serving process whose cache is kept in 8 bits, and whose sequences share a prefix, as cases to be timed: new tokens quantised as they
are stored into a cache's pages and read back, whole sequences read back, attention of new tokens over pages in 8 bits, and attention of a batch whose
sequences begin with the same keys.

A page in 8 bits holds, for every slot and key head, a row of e4m3 values and one exponent: the row stands for its values times 2^exponent.  The
exponent is the smallest that brings the row's largest finite value to 448 or below.

A case is a dict of plain values:
  path      store     the new tokens' q and k normalised and turned (norm), k and v quantised into the pages of their sequences; then the new tokens' keys and
                      values as the pages hold them (which is how a user sees what was stored)
            read      the keys and values of whole sequences out of their pages
            attend    attention of the new tokens over the pages, causal, grouped heads
            prefix    the same for sequences that come in groups, each of which begins with the same pages
  dtype     fp16 / bf16: of q, and of what is stored or read;   bits: of the cache's values, 8 or 16
  B, H, HK, D: sequences, query heads, key heads, head dim;   PS: slots of a page
  N         keys in the longest sequence's cache, the new tokens among them (prefix: behind what is shared)
  min_frac  the lengths are spread evenly between min_frac * N and N;   new: new tokens of each sequence (store, attend, prefix)
  groups    prefix: groups of B / groups sequences;   P: keys that the sequences of the first group share, min_frac * P those of the last; whole pages of them count
  lse       attend, prefix: the logarithms of the softmax's sums are wanted, too

`own` False: the operators as plain tensor operations in 32 bits.  True: the package's operators.
"""
import functools
import math
import os
import sys

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
# Exponents of a row: from where the dtype still holds every value of a row (2^-9 of the scale is e4m3's last step) to where a row's largest value is
# the dtype's.
_EXPONENTS = {"fp16": (-15, 8), "bf16": (-100, 120)}
_EPS = 1e-6


def listed():
    return [
        # one token of each of 32 conversations goes into the cache
        dict(name="store_step", path="store", dtype="bf16", bits=8, B=32, H=32, HK=8, D=128, PS=16, N=2048, min_frac=0.25, new=1, norm=True),
        # long prompts go into the cache
        dict(name="store_prompts", path="store", dtype="fp16", bits=8, B=8, H=16, HK=16, D=64, PS=64, N=5000, min_frac=0.6, new=2500, norm=True),
        # a short conversation is taken out of the cache, to be kept elsewhere
        dict(name="read_one", path="read", dtype="fp16", bits=8, B=1, H=12, HK=12, D=64, PS=16, N=333, min_frac=1.0),
        # the prompts of a batch are taken out of the cache, for layers that want them packed
        dict(name="read_prompts", path="read", dtype="bf16", bits=8, B=8, H=8, HK=8, D=128, PS=64, N=8001, min_frac=0.3),
        # one token of one interactive user on a short history: latency
        dict(name="attend_one", path="attend", dtype="fp16", bits=8, B=1, H=12, HK=12, D=64, PS=16, N=500, min_frac=1.0, new=1, lse=False),
        # five drafted tokens of each of four conversations are looked at together
        dict(name="attend_draft", path="attend", dtype="fp16", bits=8, B=4, H=16, HK=4, D=64, PS=32, N=7001, min_frac=0.4, new=5, lse=True),
        # one token for each of 32 conversations of a serving process, histories of uneven length
        dict(name="attend_step", path="attend", dtype="bf16", bits=8, B=32, H=32, HK=8, D=128, PS=64, N=16384, min_frac=0.25, new=1, lse=False),
        # a chunk of each of four long prompts behind what is cached of them
        dict(name="attend_chunk", path="attend", dtype="bf16", bits=8, B=4, H=32, HK=8, D=128, PS=128, N=8192, min_frac=0.5, new=1024, lse=False),
        # five answers to one question, just begun
        dict(name="prefix_short", path="prefix", dtype="fp16", bits=16, B=5, H=12, HK=12, D=64, PS=16, N=77, min_frac=0.1, new=1, groups=1, P=1000, lse=False),
        # three assistants with a system prompt each, four conversations of each, three drafted tokens
        dict(name="prefix_groups", path="prefix", dtype="fp16", bits=8, B=12, H=12, HK=4, D=64, PS=32, N=999, min_frac=0.5, new=3, groups=3, P=3333, lse=True),
        # one token for each of 32 conversations behind one long system prompt
        dict(name="prefix_step", path="prefix", dtype="bf16", bits=16, B=32, H=32, HK=8, D=128, PS=64, N=1024, min_frac=0.1, new=1, groups=1, P=8192, lse=False),
        # many samples of answers about one long document
        dict(name="prefix_samples", path="prefix", dtype="bf16", bits=8, B=64, H=32, HK=8, D=128, PS=64, N=1500, min_frac=0.3, new=1, groups=1, P=16384, lse=False),
    ]


def _spread(most, least, n):
    return [most - (most - least) * i // max(1, n - 1) for i in range(n)]


def _own(c):
    """Keys of each sequence that are its own, longest first (prepare() shuffles them); the new tokens at least."""
    return [max(n, c.get("new", 1)) for n in _spread(c["N"], max(1, round(c["min_frac"] * c["N"])), c["B"])]


def _shared(c):
    """Keys that the sequences of each group share: whole pages"""
    if c["path"] != "prefix":
        return [0]
    return [n // c["PS"] * c["PS"] for n in _spread(c["P"], round(c["min_frac"] * c["P"]), c["groups"])]


def work(case):
    """Each input read once and each output written once, what a group shares once; the products of attention, causal."""
    c, lens = case, _own(case)
    row_q, row = c["H"] * c["D"] * 2, 2 * c["HK"] * c["D"] * 2
    held = 2 * c["HK"] * (c["D"] + 1) if c["bits"] == 8 else row
    if c["path"] == "read":
        return {"bytes": float(sum(lens) * (held + row)), "flops": float(sum(lens) * c["HK"] * c["D"])}
    rows = c["B"] * c["new"]
    if c["path"] == "store":
        nbytes = rows * ((2 * row_q + 2 * c["D"] if c["norm"] else 0) + row + held + held + row)
        return {"bytes": float(nbytes), "flops": float(rows * ((c["H"] + c["HK"]) * 10 * c["norm"] + 6 * c["HK"]) * c["D"])}
    shared = _shared(c)
    each = c["B"] // len(shared)
    scores = sum(c["new"] * n - c["new"] * (c["new"] - 1) / 2.0 for n in lens) + sum(float(c["new"]) * each * n for n in shared)
    nbytes = (sum(lens) + sum(shared)) * held + 2 * rows * row_q + (4 * rows * c["H"] if c["lse"] else 0)
    return {"bytes": float(nbytes), "flops": 4.0 * c["H"] * c["D"] * scores}


def draw(rng):
    def log_int(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    path = rng.choice(["store", "store", "read", "attend", "attend", "attend", "prefix", "prefix", "prefix"])
    HK = rng.choice([1, 2, 4, 8, 12])
    c = dict(path=path, dtype=rng.choice(["fp16", "bf16"]), bits=8 if path in ("store", "attend") else rng.choice([8, 8, 16]), H=HK * rng.choice([1, 1, 2, 3, 4, 8]),
             HK=HK, D=rng.choice([32, 64, 64, 128, 128]), PS=rng.choice([16, 32, 64, 128, 256]), min_frac=rng.choice([1.0, round(rng.uniform(0.1, 0.95), 3)]))
    if path == "store":
        c.update(new=rng.choice([1, 1, log_int(2, 12), log_int(16, 2500)]), norm=rng.random() < 0.7)
        c["N"] = max(c["new"], log_int(20, 8000))
        most = 2e8
    elif path == "read":
        c.update(N=log_int(1, 16000))
        most = 3e8
    elif path == "attend":
        c.update(new=rng.choice([1, 1, 1, log_int(2, 12), log_int(16, 1000)]), lse=rng.random() < 0.4)
        c["N"] = max(c["new"], log_int(20, 16000))
        most = 6e8
    else:
        c.update(new=rng.choice([1, 1, 1, log_int(2, 8), log_int(16, 200)]), lse=rng.random() < 0.4, groups=rng.choice([1, 1, 1, 2, 3, 5]), P=log_int(100, 16000))
        c["N"] = max(c["new"], log_int(10, 3000))
        most = 2.8e8
    step = c.get("groups", 1)

    def cost(B):
        d = dict(c, B=B)
        w, pool = work(d), 2.0 * sum(_own(d)) * HK * c["D"]
        scores = 4.0 * c["H"] * c.get("new", 0) * (c["N"] + c.get("P", 0)) * B if path in ("attend", "prefix") else 0.0
        return max(w["bytes"] / most, w["flops"] / 3e11, pool / 6.6e8, scores / 4e9)

    B = step
    while B < 64 and cost(B + step) <= 1.0:
        B += step
    c["B"] = step * log_int(1, B // step)
    return c


# ---- rows in 8 bits

def _exponents(x, dtype):
    """The exponent of each row of x (..., D)"""
    top = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)
    part, e = torch.frexp(top)  # top = part * 2^e, part in [1/2, 1) and 448 = 7/8 * 2^9
    least, most = _EXPONENTS[dtype]
    return torch.where(top > 0, e - 9 + (part > 0.875), least).clamp(least, most)


def _power(e):
    """2^e in 32 bits, for exponents of normal numbers"""
    return ((e + 127) << 23).view(torch.float32)


def _quantise(x, dtype):
    """x (..., D) in 32 bits or more: (e4m3 values, exponents + 127 in bytes)"""
    e = _exponents(x, dtype)
    # (the largest rows of a dtype stop at 240: 256 times the scale would be more than the dtype holds)
    most = torch.where(e == _EXPONENTS[dtype][1], 240.0, 448.0).to(x.dtype)[..., None]
    y = x * _power(-e)[..., None]
    y = torch.where(x.isfinite(), torch.minimum(torch.maximum(y, -most), most), math.nan)
    return y.float().to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def _values(codes, exponents):
    """In 32 bits: what rows of e4m3 values and their exponents' bytes stand for"""
    return codes.view(torch.float8_e4m3fn).float() * _power(exponents.int() - 127)[..., None]


# ---- inputs

def _cumulative(n):
    return torch.cat([n.new_zeros(1), n.cumsum(0, dtype=torch.int32)])


def _tables(rows, D, dtype, dev):
    angle = torch.outer(torch.arange(rows, device=dev, dtype=torch.float64),
                        10000.0 ** (-torch.arange(0, D, 2, device=dev, dtype=torch.float64) / D))
    return torch.cos(angle).to(dtype), torch.sin(angle).to(dtype)


def prepare(case, seed):
    c = case
    dev, dtype = torch.device("cuda", torch.cuda.current_device()), _DTYPES[c["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    path, B, H, HK, D, PS = c["path"], c["B"], c["H"], c["HK"], c["D"], c["PS"]
    mine = torch.tensor(_own(c), dtype=torch.int32)[torch.randperm(B, generator=host)]
    shared = torch.tensor(_shared(c), dtype=torch.int32)
    each = B // len(shared)
    lens = mine + shared.repeat_interleave(each)

    def normal(*shape):
        return torch.randn(shape, device=dev, generator=gen).to(dtype)

    def pool_of(pages):
        """(values, exponents or None) of a cache whose rows differ in size, as keys and values do; a page holds its tokens head by head"""
        out = torch.empty((pages, HK, PS, D), device=dev, dtype=torch.float8_e4m3fn if c["bits"] == 8 else dtype)
        exps = torch.empty((pages, HK, PS), device=dev, dtype=torch.uint8) if c["bits"] == 8 else None
        many = max(1, (1 << 26) // (HK * PS * D))  # (in pieces: a whole cache in 32 bits would be four times its size again)
        for i in range(0, pages, many):
            n = min(many, pages - i)
            x = torch.randn((n, HK, PS, D), device=dev, generator=gen)
            x *= torch.randn((n, HK, PS, 1), device=dev, generator=gen).mul(0.4).exp()
            x = x.to(dtype)
            if c["bits"] == 8:
                out[i:i + n], exps[i:i + n] = _quantise(x.float(), c["dtype"])
            else:
                out[i:i + n] = x
        return out.transpose(1, 2), exps

    # pages in no order, a page in eight of none of the sequences
    s = {"case": c}
    cols = -(-int(lens.max()) // PS)
    n_shared, n_mine = (shared // PS).tolist(), [-(-int(n) // PS) for n in mine]
    used = sum(n_shared) + sum(n_mine)
    pool = used + used // 8 + 1
    order = torch.randperm(pool, generator=host).to(torch.int32)
    table = torch.zeros(B, cols, dtype=torch.int32)
    at = 0
    for g, n in enumerate(n_shared):
        table[g * each:(g + 1) * each, :n] = order[at:at + n]
        at += n
    for b, n in enumerate(n_mine):
        table[b, n_shared[b // each]:n_shared[b // each] + n] = order[at:at + n]
        at += n
    s["table"], s["seqlens"] = table.to(dev), lens.to(dev)
    s["k_cache"], s["k_scales"] = pool_of(pool)
    s["v_cache"], s["v_scales"] = pool_of(pool)
    if path == "read":
        s["cu"], s["total"] = _cumulative(lens).to(dev), int(lens.sum())
        return s
    new = c["new"]
    s["cu"], s["total"] = _cumulative(torch.full((B,), new, dtype=torch.int32)).to(dev), B * new
    if path != "store" or c["norm"]:
        s["q"] = normal(B * new, H, D)
    if path == "store":
        s["k"], s["v"] = normal(B * new, HK, D), normal(B * new, HK, D)
        if c["norm"]:
            s["q_weight"] = (1.0 + 0.2 * torch.randn(D, device=dev, generator=gen)).to(dtype)
            s["k_weight"] = (1.0 + 0.2 * torch.randn(D, device=dev, generator=gen)).to(dtype)
            s["cos"], s["sin"] = _tables(c["N"], D, dtype, dev)
    if path == "prefix":
        s["max_own"], s["max_shared"], s["max_k"] = int(mine.max()), int(shared.max()), int(lens.max())
        s["shared"] = shared.repeat_interleave(each).to(dev)
        s["cu_groups"] = torch.arange(0, B + 1, each, dtype=torch.int32, device=dev)
    return s


# ---- plain forms

def _norm_rotary(x, weight, cos, sin, positions):
    """x: (rows, heads, D) in 32 bits"""
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS) * weight.float()
    c, s = cos.float()[positions][:, None], sin.float()[positions][:, None]
    a, b = y[..., 0::2], y[..., 1::2]
    return torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)


def _places(s):
    """(page, slot in the page, number in the sequence) of every packed row"""
    c, cu = s["case"], s["cu"].long()
    row = torch.arange(s["total"], device=cu.device)
    seq = torch.searchsorted(cu[1:], row, right=True)
    slot = s["seqlens"].long()[seq] - (cu[1:] - cu[:-1])[seq] + row - cu[seq]
    return s["table"].long()[seq, slot // c["PS"]], slot % c["PS"], slot


def _held(s, name, page, at):
    """(places, HK, D) in 32 bits: what the cache holds at slots `at` of the pages"""
    x = s[name + "_cache"]
    if s["case"]["bits"] == 16:
        return x[page, at].float()
    return _values(x.view(torch.uint8)[page, at], s[name + "_scales"][page, :, at])


def _plain_store(s):
    c = s["case"]
    page, at, slot = _places(s)
    q, k = None, s["k"].float()
    if c["norm"]:
        q = _norm_rotary(s["q"].float(), s["q_weight"], s["cos"], s["sin"], slot).to(s["q"].dtype)
        k = _norm_rotary(k, s["k_weight"], s["cos"], s["sin"], slot)
    codes, exps = _quantise(k, c["dtype"])
    s["k_cache"].view(torch.uint8)[page, at], s["k_scales"][page, :, at] = codes.view(torch.uint8), exps
    codes, exps = _quantise(s["v"].float(), c["dtype"])
    s["v_cache"].view(torch.uint8)[page, at], s["v_scales"][page, :, at] = codes.view(torch.uint8), exps
    return (q,) + _plain_read(s)


def _plain_read(s):
    page, at, _ = _places(s)
    return tuple(_held(s, n, page, at).to(_DTYPES[s["case"]["dtype"]]) for n in "kv")


def _keys(s, name, first, most, rows):
    """(rows, HK, most, D) in 32 bits: keys or values first[i] .. of the sequences `rows`; of a page that a sequence lacks, anything"""
    c = s["case"]
    table = s["table"].long()[rows]
    slot = first[:, None] + torch.arange(most, device=table.device)
    page = table.gather(1, (slot // c["PS"]).clamp(max=table.shape[1] - 1))
    at = slot % c["PS"]
    return _held(s, name, page.flatten(), at.flatten()).view(len(rows), most, c["HK"], c["D"]).transpose(1, 2).contiguous()


def _plain_attend(s):
    c = s["case"]
    B, HK, G, new, D = c["B"], c["HK"], c["H"] // c["HK"], c["new"], c["D"]
    dev = s["q"].device
    q = s["q"].float().view(B, new, HK, G, D).permute(0, 2, 1, 3, 4).reshape(B, HK, new * G, D)
    shared = s["shared"].long() if c["path"] == "prefix" else torch.zeros(B, dtype=torch.long, device=dev)
    most = s["max_own"] if c["path"] == "prefix" else c["N"]
    every = torch.arange(B, device=dev)
    seen = (s["seqlens"].long() - shared)[:, None] - new + torch.arange(1, new + 1, device=dev)  # own keys that each new token sees
    x = torch.matmul(q, _keys(s, "k", shared, most, every).transpose(2, 3).contiguous()) * D ** -0.5
    x = x.view(B, HK, new, G, most).masked_fill(torch.arange(most, device=dev) >= seen[:, None, :, None, None], -math.inf).view(B, HK, new * G, most)
    top = x.amax(-1, keepdim=True)
    if c["path"] == "prefix" and s["max_shared"]:  # a group's keys once, for the rows of all its sequences
        groups, P = c["groups"], s["max_shared"]
        firsts = s["cu_groups"][:-1].long()
        lens = shared[firsts]
        qg = q.view(groups, B // groups, HK, new * G, D).transpose(1, 2).reshape(groups, HK, -1, D)
        y = torch.matmul(qg, _keys(s, "k", torch.zeros_like(lens), P, firsts).transpose(2, 3).contiguous()) * D ** -0.5
        y = y.masked_fill(torch.arange(P, device=dev) >= lens[:, None, None, None], -math.inf)

        def by_sequence(t):
            return t.view(groups, HK, B // groups, new * G, -1).transpose(1, 2).reshape(B, HK, new * G, -1)

        def by_group(t):
            return t.view(groups, B // groups, HK, new * G, -1).transpose(1, 2).reshape(groups, HK, -1, t.shape[-1])

        top = torch.maximum(top, by_sequence(y.amax(-1, keepdim=True)))
        y = torch.exp(y - by_group(top))
        sums = by_sequence(y.sum(-1, keepdim=True))
        o = by_sequence(torch.matmul(y, _keys(s, "v", torch.zeros_like(lens), P, firsts)))
        del y
    else:
        sums = o = 0.0
    x = torch.exp(x - top)
    sums = sums + x.sum(-1, keepdim=True)
    o = (o + torch.matmul(x, _keys(s, "v", shared, most, every))) / sums
    o = o.view(B, HK, new, G, D).transpose(1, 2).reshape(B * new, c["H"], D).to(s["q"].dtype)
    if not c["lse"]:
        return o
    lse = (top + torch.log(sums)).view(B, HK, new, G).transpose(2, 3).reshape(B, c["H"], new)
    return o, lse


@functools.lru_cache(None)
def _package():
    sys.path.insert(0, os.path.abspath("flash-attention_amd"))  # the package's folder in the repository this runs in
    from flash_attn import flash_attn_paged_interface
    return flash_attn_paged_interface


@torch.no_grad()
def run(state):
    s, c = state, state["case"]
    path = c["path"]
    if not own:
        return {"store": _plain_store, "read": _plain_read, "attend": _plain_attend, "prefix": _plain_attend}[path](s)
    paged = _package()
    cache = (s["k_cache"], s["v_cache"], s["table"], s["cu"], s["seqlens"])
    scales = dict(k_scales=s["k_scales"], v_scales=s["v_scales"])
    if path == "store":
        norm = dict(q_weight=s["q_weight"], k_weight=s["k_weight"], cos_half=s["cos"], sin_half=s["sin"], eps=_EPS) if c["norm"] else {}
        q = paged.paged_append_func(s.get("q"), s["k"], s["v"], *cache, **norm, **scales)
        return (q,) + tuple(paged.paged_read_func(*cache, s["total"], dtype=s["k"].dtype, **scales))
    if path == "read":
        return paged.paged_read_func(*cache, s["total"], dtype=_DTYPES[c["dtype"]], **scales)
    if path == "attend":
        out = paged.flash_attn_paged_func(s["q"], *cache, c["new"], c["N"], causal=True, return_softmax_lse=c["lse"], **scales)
    else:
        out = paged.flash_attn_paged_prefix_func(s["q"], *cache, c["new"], s["max_k"], s["cu_groups"], s["shared"], s["max_shared"], causal=True,
                                                 return_softmax_lse=c["lse"], **scales)
    return (out[0], out[1][:, :, :c["new"]]) if c["lse"] else out


# ---- the definitions in 64 bits

@functools.lru_cache(None)
def _e4m3(dev):
    """The 256 values of e4m3, from their fields: a sign, four bits of exponent, three of mantissa"""
    def value(code):
        sign, e, m = (-1.0 if code & 128 else 1.0), code >> 3 & 15, code & 7
        return math.nan if e == 15 and m == 7 else sign * (m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10))
    return torch.tensor([value(i) for i in range(256)], dtype=torch.float64, device=dev)


def _rounded(x, dtype):
    """Rows of x (n, D) in 64 bits as a cache in 8 bits holds them"""
    least, most = _EXPONENTS[dtype]
    top = x.abs().amax(1)
    e = torch.ceil(torch.log2(top / 448.0)).clamp(least, most)
    e = torch.where(448.0 * 2.0 ** (e - 1) >= top, e - 1, torch.where(448.0 * 2.0 ** e < top, e + 1, e)).clamp(least, most)  # (the logarithm's last bit)
    y = (x / (2.0 ** e)[:, None]).clamp(-448.0, 448.0)
    step = 2.0 ** (torch.frexp(y.abs().clamp(min=2.0 ** -6)).exponent.double() - 4)
    y = torch.round(y / step) * step
    return torch.where((e == most)[:, None], y.clamp(-240.0, 240.0), y) * (2.0 ** e)[:, None]


def _held_exactly(s, name, page, at, h):
    x = s[name + "_cache"]
    if s["case"]["bits"] == 16:
        return x[page, at, h].double()
    return _e4m3(x.device)[x.view(torch.uint8)[page, at, h].long()] * (2.0 ** (s[name + "_scales"][page, h, at].double() - 127))[:, None]


def _exact_read(s):
    c, lens, out = s["case"], s["seqlens"].tolist(), [[], []]
    for b, n in enumerate(lens):
        t = torch.arange(n, device=s["table"].device)
        page, at = s["table"][b][t // c["PS"]].long(), t % c["PS"]
        for i, name in enumerate("kv"):
            out[i].append(torch.stack([_held_exactly(s, name, page, at, h) for h in range(c["HK"])], 1))
    return tuple(torch.cat(x) for x in out)


def _exact_store(s):
    c, new = s["case"], s["case"]["new"]
    k, v, q = s["k"].double(), s["v"].double(), s["q"].double() if c["norm"] else None
    end = s["seqlens"].tolist()
    for b in range(c["B"]):
        at = slice(b * new, (b + 1) * new)
        t = torch.arange(end[b] - new, end[b], device=k.device)
        if c["norm"]:
            turn = torch.complex(s["cos"].double()[t], s["sin"].double()[t])
            for x, w in ((q, s["q_weight"].double()), (k, s["k_weight"].double())):
                for h in range(x.shape[1]):
                    y = x[at, h] * w / torch.sqrt(x[at, h].square().sum(1, keepdim=True) / c["D"] + _EPS)
                    x[at, h] = torch.view_as_real(torch.view_as_complex(y.reshape(new, -1, 2).contiguous()) * turn).flatten(1)
        for x in (k, v):
            for h in range(c["HK"]):
                x[at, h] = _rounded(x[at, h], c["dtype"])
    return q, k, v


def _exact_attend(s):
    c, new, G = s["case"], s["case"]["new"], s["case"]["H"] // s["case"]["HK"]
    out, lse = s["q"].double(), torch.empty(c["B"], c["H"], new, dtype=torch.float64, device=s["q"].device)
    for b, n in enumerate(s["seqlens"].tolist()):
        t = torch.arange(n, device=out.device)
        page, at = s["table"][b][t // c["PS"]].long(), t % c["PS"]
        hidden = t[None, :] > (n - new + torch.arange(new, device=t.device))[:, None]
        for hk in range(c["HK"]):
            k, v = _held_exactly(s, "k", page, at, hk), _held_exactly(s, "v", page, at, hk)
            for h in range(hk * G, (hk + 1) * G):
                x = (s["q"][b * new:(b + 1) * new, h].double() @ k.t() / math.sqrt(c["D"])).masked_fill(hidden, -math.inf)
                out[b * new:(b + 1) * new, h] = torch.softmax(x, 1) @ v
                lse[b, h] = torch.logsumexp(x, 1)
    return (out, lse) if c["lse"] else out


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    return {"store": _exact_store, "read": _exact_read, "attend": _exact_attend, "prefix": _exact_attend}[case["path"]](s)
