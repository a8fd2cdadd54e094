"""The operators around a paged key/value cache, as cases to be timed: queries and keys normalised and turned by their positions (forward and
backward), new tokens stored into a cache's pages, attention of new tokens over the pages, the attention weight that every cached key has
received, and the eviction of keys that received little.

A case is a dict of plain values:
  path      norm      RMS norm of each head of q and k with the position rotation (train: forward and backward through autograd)
            append    the new tokens' q and k normalised and turned, k and v stored into the pages of their sequences
            attend    attention of the new tokens over the pages, causal, grouped heads
            weights   what each cached key receives of the new tokens' attention, added to what it has received
            evict     per key head the newest and the heaviest keys stay, the others go, the rest closes up
  dtype     fp16 / bf16;   B, H, HK, D: sequences, query heads, key heads, head dim;   PS: slots of a page
  N         norm: tokens of the longest sequence; else: keys in the longest sequence's cache, the new tokens among them
  min_frac  the lengths are spread evenly between min_frac * N and N;   new: new tokens of each sequence (append, attend, weights)
  budget, recent   evict: keys that stay in a head, newest ones that stay in any case

`own` False: the operators as plain tensor operations in 32 bits.  True: the package's operators.
"""
import functools
import math
import os
import sys

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
_EPS = 1e-6


def listed():
    return [
        # one short prompt of an interactive user: nothing but launches
        dict(name="norm_prompt", path="norm", dtype="fp16", B=1, H=12, HK=12, D=64, N=61, min_frac=1.0, train=False),
        # a packed training batch of uneven documents
        dict(name="norm_ragged_train", path="norm", dtype="fp16", B=8, H=12, HK=12, D=64, N=1021, min_frac=0.5, train=True),
        # a training step's layer of a model with 128-wide heads that share keys
        dict(name="norm_train", path="norm", dtype="bf16", B=16, H=16, HK=4, D=128, N=2048, min_frac=1.0, train=True),
        # one token of each of 32 conversations goes into the cache
        dict(name="append_step", path="append", dtype="bf16", B=32, H=32, HK=8, D=128, PS=16, N=4096, min_frac=0.25, new=1),
        # long prompts go into the cache
        dict(name="append_prompts", path="append", dtype="fp16", B=8, H=16, HK=16, D=64, PS=64, N=5000, min_frac=0.6, new=2500),
        # one token of one interactive user on a short history: latency
        dict(name="attend_step_one", path="attend", dtype="fp16", B=1, H=12, HK=12, D=64, PS=16, N=500, min_frac=1.0, new=1),
        # one token for each of 32 conversations of a serving process, histories of uneven length
        dict(name="attend_step", path="attend", dtype="bf16", B=32, H=32, HK=8, D=128, PS=64, N=16384, min_frac=0.25, new=1),
        # a chunk of each of four long prompts behind what is cached of them
        dict(name="attend_chunk", path="attend", dtype="bf16", B=4, H=32, HK=8, D=128, PS=128, N=8192, min_frac=0.5, new=1024),
        # the weights of a decode step's keys
        dict(name="weights_step", path="weights", dtype="bf16", B=8, H=32, HK=8, D=128, PS=64, N=16384, min_frac=0.5, new=1),
        # the weights of a prompt chunk's keys
        dict(name="weights_chunk", path="weights", dtype="fp16", B=4, H=16, HK=8, D=64, PS=32, N=4001, min_frac=0.5, new=509),
        # a decode step has put one key over the budget of each sequence
        dict(name="evict_step", path="evict", dtype="bf16", B=32, H=32, HK=8, D=128, PS=16, N=2049, min_frac=1.0, budget=2048, recent=256),
        # prompts are cut to the budget
        dict(name="evict_prompts", path="evict", dtype="bf16", B=8, H=32, HK=8, D=128, PS=64, N=16384, min_frac=0.3, budget=4096, recent=512),
    ]


def _lens(c):
    """Sequence lengths of a case, longest first (prepare() shuffles them); a cache holds the new tokens at least."""
    lo, hi, B = max(1, round(c["min_frac"] * c["N"])), c["N"], c["B"]
    return [max(hi - (hi - lo) * i // max(1, B - 1), c.get("new", 1)) for i in range(B)]


def work(case):
    """Each input read once and each output written once; the products of attention and of the weights, causal."""
    c, lens = case, _lens(case)
    total, row_q, row_k = sum(lens), c["H"] * c["D"] * 2, c["HK"] * c["D"] * 2
    if c["path"] == "norm":
        nbytes = total * (row_q + row_k) * (4 if c["train"] else 2) + 2 * c["N"] * c["D"] + 4 * total
        return {"bytes": float(nbytes), "flops": float(total * (c["H"] + c["HK"]) * c["D"] * (30 if c["train"] else 10))}
    if c["path"] == "evict":
        moved = sum(min(c["budget"], max(0, n - c["budget"])) for n in lens) / 2  # about: a kept key behind the budget for each hole
        moved = min(moved, sum(c["budget"] * max(0, n - c["budget"]) / n for n in lens)) * c["HK"]
        nbytes = 8 * total * c["HK"] + moved * (4 * c["D"] * 2 + 16)
        return {"bytes": float(nbytes), "flops": 0.0}
    rows = c["B"] * c["new"]
    if c["path"] == "append":
        nbytes = 2 * rows * (row_q + 2 * row_k) + 8 * rows * c["HK"] + 2 * rows * c["D"]
        return {"bytes": float(nbytes), "flops": float(rows * (c["H"] + c["HK"]) * c["D"] * 10)}
    scores = sum(c["new"] * n - c["new"] * (c["new"] - 1) / 2.0 for n in lens)
    if c["path"] == "attend":
        return {"bytes": float(2 * total * row_k + 2 * rows * row_q), "flops": 4.0 * c["H"] * c["D"] * scores}
    return {"bytes": float(total * row_k + rows * row_q + 4 * rows * c["H"] + 8 * total * c["HK"]), "flops": 2.0 * c["H"] * c["D"] * scores}


def draw(rng):
    def log_int(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    path = rng.choice(["norm", "norm", "append", "attend", "attend", "attend", "weights", "weights", "evict"])
    HK = rng.choice([1, 2, 4, 8, 12])
    c = dict(path=path, dtype=rng.choice(["fp16", "bf16"]), H=HK * rng.choice([1, 1, 2, 3, 4, 8]), HK=HK, D=rng.choice([32, 64, 64, 128, 128]),
             min_frac=rng.choice([1.0, round(rng.uniform(0.1, 0.95), 3)]))
    if path == "norm":
        c.update(N=log_int(1, 4096), train=rng.random() < 0.6)
        most = 6e8
    elif path == "evict":
        c.update(PS=rng.choice([16, 32, 64, 128, 256]), N=log_int(30, 16000))
        c["budget"] = max(1, int(c["N"] * rng.uniform(0.2, 0.95)))
        c["recent"] = int(c["budget"] * rng.uniform(0.0, 0.4))
        most = 3e8
    else:
        c.update(PS=rng.choice([16, 32, 64, 128, 256]), new=rng.choice([1, 1, 1, log_int(2, 12), log_int(16, 1200)]))
        c["N"] = max(c["new"], log_int(20, 16000))
        most = {"append": 2e8, "attend": 1.2e9, "weights": 6e8}[path]
    c["B"] = 1

    def cost(B):
        w, pool = work(dict(c, B=B)), 0.0
        if path != "norm":
            pool = 4.0 * sum(_lens(dict(c, B=B))) * c["HK"] * c["D"]  # (a case's cache is at most the largest listed one's)
        return max(w["bytes"] / most, w["flops"] / 3e11, pool / 1.3e9)

    B = 1
    while B < 64 and cost(B + 1) <= 1.0:
        B += 1
    c["B"] = log_int(1, B)
    return c


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
    path, B, H, HK, D = c["path"], c["B"], c["H"], c["HK"], c["D"]
    lens = torch.tensor(_lens(c), dtype=torch.int32)[torch.randperm(B, generator=host)]

    def normal(*shape):
        out = torch.empty(shape, device=dev, dtype=dtype)  # (in pieces: a whole cache in 32 bits would be twice its size again)
        flat = out.view(-1)
        for i in range(0, flat.numel(), 1 << 27):
            piece = flat[i:i + (1 << 27)]
            piece.copy_(torch.randn(piece.numel(), device=dev, dtype=torch.float32, generator=gen))
        return out

    s = {"case": c}
    if path in ("norm", "append"):
        s["q_weight"] = (1.0 + 0.2 * torch.randn(D, device=dev, generator=gen)).to(dtype)
        s["k_weight"] = (1.0 + 0.2 * torch.randn(D, device=dev, generator=gen)).to(dtype)
        s["cos"], s["sin"] = _tables(c["N"], D, dtype, dev)
    if path == "norm":
        cu = _cumulative(lens)
        total = int(cu[-1])
        s["positions"] = (torch.arange(total) - torch.repeat_interleave(cu[:-1], lens)).to(torch.int32).to(dev)
        s["q"], s["k"] = normal(total, H, D), normal(total, HK, D)
        if c["train"]:
            for n in ("q", "k", "q_weight", "k_weight"):
                s[n].requires_grad_()
            s["dq"], s["dk"] = normal(total, H, D), normal(total, HK, D)
        return s

    # the cache: pages in no order, a page in eight of none of the sequences
    PS, N = c["PS"], c["N"]
    n_pages = [-(-int(n) // PS) for n in lens]
    pool = sum(n_pages) + sum(n_pages) // 8 + 1
    order = torch.randperm(pool, generator=host).to(torch.int32)
    table = torch.zeros(B, -(-N // PS), dtype=torch.int32)
    at = 0
    for b, n in enumerate(n_pages):
        table[b, :n] = order[at:at + n]
        at += n
    s["table"], s["seqlens"] = table.to(dev), lens.to(dev)
    s["k_cache"] = normal(pool, HK, PS, D).transpose(1, 2)  # a page holds its keys head by head
    if path != "weights":
        s["v_cache"] = normal(pool, HK, PS, D).transpose(1, 2)
    if path != "attend":
        # weights as attention leaves them: a few keys hold most, many hold nothing at all
        w = torch.rand(pool, HK, PS, device=dev, generator=gen)
        s["weights"] = torch.where(w < 0.1, 0.0, w ** 6 * 8.0)
        s["key_positions"] = torch.zeros(pool, HK, PS, device=dev, dtype=torch.int32)
    if path == "evict":
        # the sequences have been cut before: a head's keys lie in no order, the newest among them
        pages, slots = table.to(dev).long(), torch.arange(N, device=dev)
        where = torch.rand(B, HK, N, device=dev, generator=gen)
        where = where.masked_fill(slots[None, None] >= s["seqlens"][:, None, None], 2.0).argsort(-1).argsort(-1)
        live = (slots[None, None] < s["seqlens"][:, None, None]).expand(B, HK, N)
        bi, hi, ji = live.nonzero(as_tuple=True)
        s["key_positions"][pages[bi, ji // PS], hi, ji % PS] = where[bi, hi, ji].to(torch.int32)
        s["next"] = s["seqlens"].clone()
        return s
    new = c["new"]
    s["cu"] = _cumulative(torch.full((B,), new, dtype=torch.int32)).to(dev)
    s["q"] = normal(B * new, H, D)
    if path == "append":
        s["k"], s["v"] = normal(B * new, HK, D), normal(B * new, HK, D)
    if path == "weights":
        s["lse"] = _lse(s)
    return s


# ---- plain forms

def _norm_rotary(x, weight, cos, sin, positions):
    """x: (rows, heads, D) in 32 bits"""
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS) * weight.float()
    c, s = cos.float()[positions][:, None], sin.float()[positions][:, None]
    a, b = y[..., 0::2], y[..., 1::2]
    return torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)


def _rows(s):
    """(sequence, place in the chunk) of every new token"""
    cu = s["cu"].long()
    row = torch.arange(s["q"].shape[0], device=cu.device)
    seq = torch.searchsorted(cu[1:], row, right=True)
    return seq, row - cu[seq]


def _keys(cache, s):
    """(B, HK, keys, D) in 32 bits, zeros behind a sequence's last key"""
    c = s["case"]
    x = cache[s["table"].long()].flatten(1, 2)[:, :c["N"]].permute(0, 2, 1, 3).float()
    return x.masked_fill(torch.arange(c["N"], device=x.device)[None, None, :, None] >= s["seqlens"][:, None, None, None], 0.0)


def _scores(s):
    """(B, HK, group, new, keys) in 32 bits, -inf where a new token does not see a key"""
    c = s["case"]
    B, HK, G, new, D = c["B"], c["HK"], c["H"] // c["HK"], c["new"], c["D"]
    q = s["q"].float().view(B, new, HK, G, D).permute(0, 2, 3, 1, 4).reshape(B, HK, G * new, D)
    x = (torch.matmul(q, _keys(s["k_cache"], s).transpose(2, 3).contiguous()) * D ** -0.5).view(B, HK, G, new, -1)
    seen = s["seqlens"][:, None] - new + torch.arange(1, new + 1, device=q.device)  # (B, new)
    return x.masked_fill(torch.arange(c["N"], device=q.device) >= seen[:, None, None, :, None], -math.inf)


def _lse(s):
    """(B, H, new rounded up to 16): what the attention over the same keys gives"""
    c = s["case"]
    x = torch.logsumexp(_scores(s).double(), -1).flatten(1, 2)
    out = torch.zeros(c["B"], c["H"], -(-c["new"] // 16) * 16, device=x.device)
    out[:, :, :c["new"]] = x
    return out


def _plain_norm(s):
    q, k = (_norm_rotary(s[n].float(), s[n + "_weight"], s["cos"], s["sin"], s["positions"].long()).to(s[n].dtype) for n in ("q", "k"))
    return q, k


def _plain_append(s):
    c = s["case"]
    seq, i = _rows(s)
    slot = s["seqlens"].long()[seq] - c["new"] + i
    page, at = s["table"].long()[seq, slot // c["PS"]], slot % c["PS"]
    q, k = (_norm_rotary(s[n].float(), s[n + "_weight"], s["cos"], s["sin"], slot).to(s[n].dtype) for n in ("q", "k"))
    s["k_cache"][page, at], s["v_cache"][page, at] = k, s["v"]
    s["weights"][page, :, at] = 0.0
    s["key_positions"][page, :, at] = slot.to(torch.int32)[:, None]
    return q


def _plain_attend(s):
    c = s["case"]
    x = _scores(s)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    o = torch.matmul(x.flatten(2, 3), _keys(s["v_cache"], s).contiguous()).view(*x.shape[:-1], c["D"]) / x.sum(-1, keepdim=True)
    return o.permute(0, 3, 1, 2, 4).reshape(c["B"] * c["new"], c["H"], c["D"]).to(s["q"].dtype)


def _plain_weights(s):
    c = s["case"]
    lse = s["lse"][:, :, :c["new"]].reshape(c["B"], c["HK"], -1, c["new"], 1)
    got = torch.exp(_scores(s) - lse).sum((2, 3))  # (B, HK, keys)
    slots = torch.arange(c["N"], device=got.device)
    b, h, j = (slots < s["seqlens"][:, None, None]).expand_as(got).nonzero(as_tuple=True)
    at = (s["table"].long()[b, j // c["PS"]], h, j % c["PS"])
    s["weights"][at] = s["weights"][at] + got[b, h, j]
    return s["weights"]


def _plain_evict(s, weights, positions):
    c = s["case"]
    B, HK, N, PS, budget = c["B"], c["HK"], c["N"], c["PS"], c["budget"]
    slots = torch.arange(N, device=weights.device)
    page = s["table"].long()[:, slots // PS][:, None].expand(B, HK, N)
    head, at = torch.arange(HK, device=weights.device)[None, :, None].expand(B, HK, N), (slots % PS).expand(B, HK, N)
    live = slots < s["seqlens"][:, None, None]
    key = weights[page, head, at].double()
    key = torch.where(key.isnan(), -math.inf, key.clamp(max=1e300))  # (+inf below the newest, above every number)
    newest = positions[page, head, at] >= (s["next"] - c["recent"])[:, None, None]
    key = torch.where(newest, math.inf, key)
    # heaviest first, ties to the lowest slot; what is no key comes last
    order = torch.where(live, key, -math.inf).sort(dim=-1, descending=True, stable=True).indices
    order = order.gather(-1, (~live.expand(B, HK, N).gather(-1, order)).to(torch.int8).sort(dim=-1, stable=True).indices)
    stays = torch.zeros(B, HK, N, dtype=torch.bool, device=key.device)
    stays.scatter_(-1, order[..., :budget], True)
    stays &= live
    cut = (s["seqlens"] > budget)[:, None, None]
    hole = cut & ~stays & (slots < budget)
    comes = cut & stays & (slots >= budget)
    # the n-th hole takes the n-th key from behind
    to, frm = hole.nonzero(as_tuple=True), comes.nonzero(as_tuple=True)
    dst, src = (page[to], to[1], at[to]), (page[frm], frm[1], at[frm])
    weights[dst], positions[dst] = weights[src], positions[src]
    k, v = s["k_cache"], s["v_cache"]
    k[dst[0], dst[2], dst[1]], v[dst[0], dst[2], dst[1]] = k[src[0], src[2], src[1]], v[src[0], src[2], src[1]]
    return s["seqlens"].clamp(max=budget)


@functools.lru_cache(None)
def _package():
    sys.path.insert(0, os.path.abspath("flash-attention_amd"))  # the package's folder in the repository this runs in
    from flash_attn import flash_attn_paged_interface, rotary
    return flash_attn_paged_interface, rotary


def run(state):
    s, c = state, state["case"]
    path = c["path"]
    if own:
        paged, rotary = _package()
    if path == "norm":
        with torch.set_grad_enabled(c["train"]):
            if own:
                q, k = rotary.apply_qk_norm_rotary(s["q"], s["k"], s["q_weight"], s["k_weight"], s["cos"], s["sin"], positions=s["positions"], eps=_EPS)
            else:
                q, k = _plain_norm(s)
            if not c["train"]:
                return q, k
            return (q, k) + torch.autograd.grad((q, k), (s["q"], s["k"], s["q_weight"], s["k_weight"]), (s["dq"], s["dk"]))
    with torch.no_grad():
        if path == "append":
            if own:
                q = paged.paged_append_func(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["cu"], s["seqlens"],
                                            q_weight=s["q_weight"], k_weight=s["k_weight"], cos_half=s["cos"], sin_half=s["sin"], eps=_EPS,
                                            key_weights=s["weights"], key_positions=s["key_positions"])
            else:
                q = _plain_append(s)
            return q, s["k_cache"], s["v_cache"], s["weights"], s["key_positions"]
        if path == "attend":
            if own:
                return paged.flash_attn_paged_func(s["q"], s["k_cache"], s["v_cache"], s["table"], s["cu"], s["seqlens"], c["new"], c["N"], causal=True)
            return _plain_attend(s)
        if path == "weights":
            if own:
                return paged.paged_key_weights_func(s["q"], s["lse"], s["k_cache"], s["weights"], s["table"], s["cu"], s["seqlens"], c["new"], c["N"],
                                                    causal=True)
            return _plain_weights(s)
        # (the weights and positions change in place: a copy, so that every pass finds the same ones; the keys and values that a pass moves are
        # the same every time)
        w, p = s["weights"].clone(), s["key_positions"].clone()
        if own:
            n = paged.paged_evict_func(s["k_cache"], s["v_cache"], w, p, s["table"], s["seqlens"], s["next"], c["budget"], c["recent"], c["N"])
        else:
            n = _plain_evict(s, w, p)
        return s["k_cache"], s["v_cache"], w, p, n


# ---- the definitions in 64 bits

def _turned(x, weight, cos, sin, t):
    """One head's rows x (n, D), normalised and turned by the angles of table rows t, and the normalised rows and their factors"""
    r = (x.pow(2).sum(1) / x.shape[1] + _EPS).pow(-0.5)
    xh = x * r[:, None]
    z = torch.view_as_complex((xh * weight).view(x.shape[0], -1, 2)) * torch.complex(cos[t], sin[t])
    return torch.view_as_real(z).reshape(x.shape), xh, r


def _exact_norm(s):
    outs, grads, wgrads = [], [], []
    cos, sin, t = s["cos"].double(), s["sin"].double(), s["positions"].long()
    for n in ("q", "k"):
        x, w = s[n].detach().double(), s[n + "_weight"].detach().double()
        out, dx, dw = torch.empty_like(x), torch.empty_like(x), torch.zeros_like(w)
        for h in range(x.shape[1]):
            out[:, h], xh, r = _turned(x[:, h], w, cos, sin, t)
            if s["case"]["train"]:
                dy = s["d" + n][:, h].double()
                g = torch.view_as_complex(dy.reshape(dy.shape[0], -1, 2)) * torch.complex(cos[t], -sin[t])
                g = torch.view_as_real(g).reshape(dy.shape)
                dw += (g * xh).sum(0)
                dx[:, h] = r[:, None] * (g * w - xh * (g * w * xh).mean(1, keepdim=True))
        outs.append(out)
        grads.append(dx)
        wgrads.append(dw)
    return tuple(outs) if not s["case"]["train"] else tuple(outs + grads + wgrads)


def _exact_append(s):
    c = s["case"]
    q, kc, vc = s["q"].double(), s["k_cache"].double(), s["v_cache"].double()
    cos, sin = s["cos"].double(), s["sin"].double()
    lens, table = s["seqlens"].tolist(), s["table"]
    for b in range(c["B"]):
        at = torch.arange(b * c["new"], (b + 1) * c["new"], device=q.device)
        t = torch.arange(lens[b] - c["new"], lens[b], device=q.device)
        page = table[b][t // c["PS"]].long()
        for h in range(c["H"]):
            q[at, h] = _turned(s["q"][at, h].double(), s["q_weight"].double(), cos, sin, t)[0]
        for h in range(c["HK"]):
            kc[page, t % c["PS"], h] = _turned(s["k"][at, h].double(), s["k_weight"].double(), cos, sin, t)[0]
            vc[page, t % c["PS"], h] = s["v"][at, h].double()
            s["weights"][page, h, t % c["PS"]] = 0
    return q, kc, vc, s["weights"].double(), None


def _pairs(s):
    """For each sequence and key head: its place in the pool, its keys in 64 bits and the probabilities and logarithms of sums of its new tokens"""
    c = s["case"]
    G, new = c["H"] // c["HK"], c["new"]
    for b, n in enumerate(s["seqlens"].tolist()):
        t = torch.arange(n, device=s["q"].device)
        page, at = s["table"][b][t // c["PS"]].long(), t % c["PS"]
        hidden = t[None, :] > (n - new + torch.arange(new, device=t.device))[:, None]
        for hk in range(c["HK"]):
            k = s["k_cache"][page, at, hk].double()
            for g in range(G):
                x = s["q"][b * new:(b + 1) * new, hk * G + g].double() @ k.t() / math.sqrt(c["D"])
                yield b, hk, hk * G + g, page, at, x.masked_fill(hidden, -math.inf)


def _exact_attend(s):
    new, out = s["case"]["new"], s["q"].double()
    for b, hk, h, page, at, x in _pairs(s):
        out[b * new:(b + 1) * new, h] = torch.softmax(x, 1) @ s["v_cache"][page, at, hk].double()
    return out


def _exact_weights(s):
    new, w = s["case"]["new"], s["weights"].double()
    for b, hk, h, page, at, x in _pairs(s):
        w[page, hk, at] += torch.exp(x - s["lse"][b, h, :new].double()[:, None]).sum(0)
    return w


def _exact_evict(s):
    c = s["case"]
    kc, vc, w = s["k_cache"].double(), s["v_cache"].double(), s["weights"].double()
    weights, positions = s["weights"].cpu(), s["key_positions"].cpu()
    table, lens, nxt = s["table"].cpu().long(), s["seqlens"].tolist(), s["next"].tolist()
    to, frm = [], []
    for b, n in enumerate(lens):
        if n <= c["budget"]:
            continue
        t = torch.arange(n)
        page, at = table[b][t // c["PS"]], t % c["PS"]
        for h in range(c["HK"]):
            old = (positions[page, h, at] < nxt[b] - c["recent"]).tolist()
            heavy = weights[page, h, at].tolist()
            kept = sorted(range(n), key=lambda j: (old[j], -heavy[j] if old[j] else 0.0, j))[:c["budget"]]
            left = sorted(set(range(c["budget"])) - set(kept))
            for d, f in zip(left, sorted(j for j in kept if j >= c["budget"])):
                to.append((int(page[d]), h, int(at[d])))
                frm.append((int(page[f]), h, int(at[f])))
    if to:
        d, f = (torch.tensor(x, device=w.device).t() for x in (to, frm))
        w[d[0], d[1], d[2]] = w[f[0], f[1], f[2]]
        for cache in (kc, vc):
            cache[d[0], d[2], d[1]] = cache[f[0], f[2], f[1]]
    return kc, vc, w, None, None


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "append": _exact_append, "attend": _exact_attend, "weights": _exact_weights, "evict": _exact_evict}[case["path"]](s)
