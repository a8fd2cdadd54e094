"""The paged cache as a serving loop uses it, the norm of queries and keys inside attention and FlashMHA, graphs, streams, caches beyond 32-bit offsets; and
what the Python entry points refuse."""
import math

import pytest
import torch

from test_paged import DTYPES, Cache, cumulative, half_step, ref_attention, ref_evict, ref_norm_rotary, tables


def randn(*shape, seed, dtype=torch.float16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


# ---- CPU: the book of pages, refusals

def test_the_book_of_pages():
    from flash_attn.flash_attn_paged_interface import PagedKVCache
    c = PagedKVCache(2, 10, 16, 2, 64, device="cpu", key_weights=True)
    a, b = c.add(), c.add()
    s = c.step([a, b], [20, 3])
    assert s.page_table.tolist() == [[0, 1], [2, -1]] and s.seqlens_k.tolist() == [20, 3] and s.cu_seqlens.tolist() == [0, 20, 23]
    assert s.positions.tolist() == list(range(20)) + [0, 1, 2] and (s.max_seqlen_q, s.max_seqlen_k, s.max_position, s.total) == (20, 20, 20, 23)
    s = c.step([b], [14])
    assert s.page_table.tolist() == [[2, 3]] and s.seqlens_k.tolist() == [17] and s.positions.tolist() == list(range(3, 17)) and c.free_pages() == 6
    with pytest.raises(RuntimeError, match="6 free pages, the step needs 7"):
        c.step([a, b], [100, 16])
    assert c.free_pages() == 6 and c.length(a) == 20 and c.length(b) == 17  # nothing has changed
    c.remove(a)
    assert c.free_pages() == 8
    d = c.add()
    assert c.step([d, b], [33, 0]).page_table.tolist() == [[0, 1, 4], [2, 3, -1]]
    assert c.layer(1)[0].shape == (10, 16, 2, 64)
    for bad in (lambda: c.step([d, d], [1, 1]), lambda: c.step([a], [1]), lambda: c.step([], []), lambda: c.step([d], [0]), lambda: c.step([d], [-1]),
                lambda: c.step([d], [1, 2]), lambda: c.evict([d], 0, 0), lambda: c.evict([d], 4, -1), lambda: c.evict([b, b], 4, 0)):
        with pytest.raises(RuntimeError):
            bad()
    with pytest.raises(RuntimeError, match="key_weights=True"):
        e = PagedKVCache(1, 4, 16, 1, 64, device="cpu")
        e.evict([e.add()], 4, 0)
    for args in ((1, 4, 24, 1, 64), (1, 4, 8, 1, 64), (1, 4, 2048, 1, 64), (0, 4, 16, 1, 64), (1, 0, 16, 1, 64), (1, 4, 16, 1, 80)):
        with pytest.raises(RuntimeError):
            PagedKVCache(*args, device="cpu")
    with pytest.raises(RuntimeError):
        PagedKVCache(1, 4, 16, 1, 64, dtype=torch.float32, device="cpu")


def test_tensors_on_the_host_are_refused(lib):
    from flash_attn import flash_attn_paged_interface as p
    from flash_attn.rotary import apply_qk_norm_rotary
    q, c = torch.zeros(3, 2, 64).half(), torch.zeros(4, 16, 2, 64).half()
    w, i32 = torch.ones(64).half(), torch.zeros(2, dtype=torch.int32)
    meta = torch.zeros(4, 2, 16)
    calls = (lambda: apply_qk_norm_rotary(q, q, w, w), lambda: p.paged_append_func(q, q, q, c, c, i32[:1, None], i32, i32[:1]),
             lambda: p.flash_attn_paged_func(q, c, c, i32[:1, None], i32, i32[:1], 3, 3),
             lambda: p.paged_key_weights_func(q, torch.zeros(1, 2, 16), c, meta, i32[:1, None], i32, i32[:1], 3, 3),
             lambda: p.paged_evict_func(c, c, meta, meta.int(), i32[:1, None], i32[:1], i32[:1], 2, 1, 3))
    for call in calls:
        with pytest.raises(RuntimeError, match="GPU"):
            call()


# ---- GPU

@pytest.mark.gpu
def test_python_entry_points_refuse(lib):
    from flash_attn import flash_attn_paged_interface as p
    from flash_attn.rotary import apply_qk_norm_rotary
    c = Cache([20, 9], 2, 64, 16, torch.float16, 1).gpu()
    q, cu = randn(3, 4, 64, seed=0).cuda(), cumulative([2, 1]).cuda()
    kv = q[:, :2]
    w = torch.ones(64, dtype=torch.float16, device="cuda")
    cos, sin = (t.cuda() for t in tables(30, 64, torch.float16))
    lse = torch.zeros(2, 4, 16, device="cuda")
    attend = lambda **o: p.flash_attn_paged_func(**{**dict(q=q, k_cache=c.dk, v_cache=c.dv, page_table=c.dtable, cu_seqlens_q=cu, seqlens_k=c.dlens,  # noqa: E731
                                                         max_seqlen_q=2, max_seqlen_k=20), **o})
    append = lambda **o: p.paged_append_func(**{**dict(q=q, k=kv, v=kv, k_cache=c.dk, v_cache=c.dv, page_table=c.dtable, cu_seqlens=cu, seqlens_k=c.dlens,  # noqa: E731
                                                       q_weight=w, k_weight=w, cos_half=cos, sin_half=sin), **o})
    weigh = lambda **o: p.paged_key_weights_func(**{**dict(q=q, softmax_lse=lse, k_cache=c.dk, key_weights=c.dweights, page_table=c.dtable, cu_seqlens_q=cu,  # noqa: E731
                                                           seqlens_k=c.dlens, max_seqlen_q=2, max_seqlen_k=20), **o})
    evict = lambda **o: p.paged_evict_func(**{**dict(k_cache=c.dk, v_cache=c.dv, key_weights=c.dweights, key_positions=c.dpositions, page_table=c.dtable,  # noqa: E731
                                                     seqlens_k=c.dlens, next_positions=c.dlens, budget=30, recent=2, max_seqlen_k=20), **o})
    norm = lambda **o: apply_qk_norm_rotary(**{**dict(q=q, k=kv, q_weight=w, k_weight=w, cos_half=cos, sin_half=sin), **o})  # noqa: E731
    for call in (attend, append, weigh, evict, norm):
        call()
    # rows that 16-byte loads cannot reach: copied by the differentiable function, refused by the cache's
    odd = torch.zeros(3, 4, 65, dtype=torch.float16, device="cuda")[..., 1:]
    odd.copy_(q)
    assert torch.equal(norm(q=odd)[0], norm()[0])
    bad = [
        (attend, dict(q=q.bfloat16())), (attend, dict(q=q[:, :3])), (attend, dict(q=q[..., :32])), (attend, dict(q=odd)), (attend, dict(v_cache=c.dv[:3])),
        (attend, dict(k_cache=c.dk.float(), v_cache=c.dv.float())), (attend, dict(page_table=c.dtable.long())), (attend, dict(page_table=c.dtable[0])),
        (attend, dict(seqlens_k=c.dlens[:1])), (attend, dict(seqlens_k=c.dlens.long())), (attend, dict(cu_seqlens_q=cu[:2])), (attend, dict(max_seqlen_q=0)),
        (attend, dict(max_seqlen_k=0)), (attend, dict(softmax_scale=-1.0)), (attend, dict(softmax_scale=math.inf)), (attend, dict(k_cache=c.dk[..., :48], v_cache=c.dv[..., :48])),
        (attend, dict(q=q.clone().requires_grad_())),
        (append, dict(k=q)), (append, dict(v=kv[:2])), (append, dict(q=q[:2])), (append, dict(q_weight=None)), (append, dict(k_weight=w.bfloat16())),
        (append, dict(q_weight=w[:32])), (append, dict(sin_half=None)), (append, dict(cos_half=cos[:, :16])), (append, dict(positions=cu[:2])),
        (append, dict(positions=torch.zeros(3, device="cuda"))), (append, dict(key_weights=c.dweights[:2])), (append, dict(key_positions=c.dweights)),
        (append, dict(eps=-1.0)), (append, dict(k_cache=c.dk[:1].expand(c.n_pages, -1, -1, -1))),
        (weigh, dict(softmax_lse=lse[..., :15])), (weigh, dict(softmax_lse=lse.half())), (weigh, dict(key_weights=c.dweights.half())), (weigh, dict(key_weights=None)),
        (evict, dict(budget=0)), (evict, dict(recent=-1)), (evict, dict(next_positions=c.dlens[:1])), (evict, dict(key_positions=c.dweights)), (evict, dict(v_cache=None)),
        (norm, dict(k=kv[:2])), (norm, dict(q=q[..., :48], k=kv[..., :48], q_weight=w[:48], k_weight=w[:48], cos_half=None, sin_half=None)), (norm, dict(q=q.float())),
        (norm, dict(positions=cu[:2])), (norm, dict(cos_half=cos[:2], sin_half=sin[:2])), (norm, dict(eps=math.nan)), (norm, dict(q_weight=w.cpu())),
    ]
    for i, (call, change) in enumerate(bad):
        print(i, sorted(change))  # (shown with a failure)
        with pytest.raises(RuntimeError):
            call(**change)
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_native_calls_are_taken(lib):
    """the calls of a serving loop do not go by way of the Python binding"""
    from flash_attn import flash_attn_gfx950 as be
    c = Cache([20, 9], 2, 64, 16, torch.float16, 1).gpu()
    q, cu = randn(2, 4, 64, seed=0).cuda(), cumulative([1, 1]).cuda()
    w = torch.ones(64, dtype=torch.float16, device="cuda")
    n = be.passes()
    with torch.no_grad():
        assert n.qk_norm_rotary(q, q, w, w, None, None, None, 1e-6) is not None
        assert n.paged_append(q, q[:, :2], q[:, 2:], c.dk, c.dv, c.dtable, cu, c.dlens, w, w, None, None, None, 1e-6, None, None) is not None
        out, lse = n.paged_fwd(q, c.dk, c.dv, c.dtable, cu, c.dlens, 1, 20, None, True, True)
        assert n.paged_key_weights(q, lse, c.dk, c.dweights, c.dtable, cu, c.dlens, 1, 20, None, True) is True
        assert n.paged_evict(c.dk, c.dv, c.dweights, c.dpositions, c.dtable, c.dlens, c.dlens, 8, 2, 20) is not None


@pytest.mark.gpu
def test_native_and_python_calls_agree(lib):
    from flash_attn import flash_attn_gfx950 as be
    from flash_attn import flash_attn_paged_interface as p
    c = Cache([200, 90], 2, 64, 16, torch.bfloat16, 1).gpu()
    q, cu = randn(5, 4, 64, seed=0, dtype=torch.bfloat16).cuda(), cumulative([2, 3]).cuda()
    a, lse = p.flash_attn_paged_func(q, c.dk, c.dv, c.dtable, cu, c.dlens, 3, 200, return_softmax_lse=True)
    b, lse2 = be.paged_fwd(q, c.dk, c.dv, c.dtable, cu, c.dlens, 3, 200, 0.125, True, return_lse=True)
    assert torch.equal(a, b) and torch.equal(lse[0, :, :2], lse2[0, :, :2]) and torch.equal(lse[1, :, :3], lse2[1, :, :3])
    w1, w2 = c.dweights.clone(), c.dweights.clone()
    p.paged_key_weights_func(q, lse, c.dk, w1, c.dtable, cu, c.dlens, 3, 200)
    be.paged_key_weights(q, lse, c.dk, w2, c.dtable, cu, c.dlens, 3, 200, 0.125, True)
    assert torch.equal(w1, w2) and w1.sum() > 0
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    x, y = (torch.empty_like(q) for _ in range(2))
    be.qk_norm_rotary(q, q, x, y, w, w, None, None)
    assert torch.equal(be.passes().qk_norm_rotary(q, q, w, w, None, None, None, 1e-6)[0], x)
    got = []
    for f in (lambda *t: p.paged_evict_func(*t, c.dtable, c.dlens, c.dlens, 50, 10, 200), lambda *t: be.paged_evict(*t, c.dtable, c.dlens, c.dlens, 50, 10, 200)):
        t = [x.clone() for x in (c.dk, c.dv, w1, c.dpositions)]
        got.append([*t, f(*t)])
    assert all(torch.equal(torch.nan_to_num(x), torch.nan_to_num(y)) for x, y in zip(*got))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H, HK, D, PS, turn", [(4, 2, 64, 16, True), (8, 1, 128, 32, True), (3, 3, 32, 16, False)])
def test_a_serving_loop(dtype, H, HK, D, PS, turn):
    """prompts, a chunk behind a prompt, single tokens, an eviction, further tokens, a sequence removed and another in its pages: every call against the
    definitions on what the cache held before it"""
    from flash_attn.flash_attn_paged_interface import PagedKVCache
    cache = PagedKVCache(2, 40, PS, HK, D, dtype=dtype, key_weights=True)
    g = torch.Generator().manual_seed(H)
    w = [(1 + 0.2 * torch.randn(D, generator=g)).to(dtype) for _ in range(2)]
    cos, sin = tables(200, D, dtype)
    opt = dict(q_weight=w[0].cuda(), k_weight=w[1].cuda())
    if turn:
        opt.update(cos_half=cos.cuda(), sin_half=sin.cuda())
    u = half_step(dtype)
    a, b, c = cache.add(), cache.add(), cache.add()
    seen = {a: 0, b: 0, c: 0}

    def state(step, layer, seqs):
        """the cache as the definitions read it"""
        s = Cache.__new__(Cache)
        s.k, s.v = (t.cpu() for t in cache.layer(layer))
        s.table, s.lens, s.PS, s.n_pages = step.page_table.cpu(), step.seqlens_k.tolist(), PS, s.k.shape[0]
        s.weights, s.positions = cache.key_weights[layer].cpu(), cache.key_positions[layer].cpu()
        return s

    def one(seqs, new):
        step = cache.step(seqs, new)
        for layer in range(2):
            x = torch.randn(sum(new), H + 2 * HK, D, generator=g).to(dtype)
            dx = x.cuda()
            q = step.append(layer, dx[:, :H], dx[:, H:H + HK], dx[:, H + HK:], **opt)
            s = state(step, layer, seqs)
            at = 0
            for i, (seq, n) in enumerate(zip(seqs, new)):  # what was stored
                t = torch.arange(seen[seq], seen[seq] + n)
                for src, have, ww in ((x[at:at + n, :H], q[at:at + n].cpu(), w[0]), (x[at:at + n, H:H + HK], None, w[1])):
                    page, slot = s.where(i, s.lens[i])
                    have = s.k[page, slot][s.lens[i] - n:] if have is None else have
                    want = ref_norm_rotary(src.double(), ww.double(), cos.double() if turn else None, sin.double() if turn else None, t, 1e-6)
                    pair = (want[..., 0::2].pow(2) + want[..., 1::2].pow(2)).sqrt().repeat_interleave(2, -1)
                    assert ((have.double() - want).abs() <= u * want.abs() + (D + 16) * 2.0 ** -24 * 2 * pair + 1e-7).all()
                page, slot = s.where(i, s.lens[i])
                assert torch.equal(s.v[page, slot][s.lens[i] - n:], x[at:at + n, H + HK:])
                assert torch.equal(s.positions[page, :, slot][s.lens[i] - n:], t.to(torch.int32)[:, None].expand(n, HK))
                at += n
            out = step.attend(layer, q)
            want, lse, got, tol, ds = ref_attention(q.cpu(), s, new, True, D ** -0.5)
            assert ((out.cpu().double() - want).abs() <= tol + 1e-7).all()
            # (the probabilities are formed with the forward's lse, off by what test_paged counts for it: twice the score's error and the sums)
            rel = 2 * ds + 2 * (max(s.lens) + max(new) * H + 128) * 2.0 ** -24 + 64 * 2.0 ** -24
            assert ((cache.key_weights[layer].cpu().double() - s.weights.double() - got).abs() <= rel * got + 2.0 ** -22 * (s.weights.double() + got)).all()
        for seq, n in zip(seqs, new):
            seen[seq] += n

    one([a, b, c], [37, 1, 70])
    one([b, a], [20, 1])
    one([a, b, c], [1, 1, 1])
    table = cache.step([a, c], [0, 1])  # (one more token of c whose keys are still to come: stored below)
    for layer in range(2):
        x = torch.randn(1, H + 2 * HK, D, generator=g).to(dtype).cuda()
        table.attend(layer, table.append(layer, x[:, :H], x[:, H:H + HK], x[:, H + HK:], **opt))
    seen[c] += 1
    before = [state(table, layer, [a, c]) for layer in range(2)]
    free = cache.free_pages()
    cache.evict([a, c], 24, 6)
    assert cache.length(a) == cache.length(c) == 24 and cache.length(b) == 22 and cache.free_pages() > free
    for layer, s in enumerate(before):
        moves, lens = ref_evict(s, s.lens, s.weights, s.positions, [seen[a], seen[c]], 24, 6)
        for (i, h), pairs in moves.items():
            for to, frm in pairs:
                tp, fp = s.table[i, to // PS], s.table[i, frm // PS]
                for t in (s.k, s.v):
                    t[tp, to % PS, h] = t[fp, frm % PS, h]
                for t in (s.weights, s.positions):
                    t[tp, h, to % PS] = t[fp, h, frm % PS]
        k, v = (t.cpu() for t in cache.layer(layer))
        for i in range(2):
            page, slot = s.where(i, 24)
            assert torch.equal(k[page, slot], s.k[page, slot]) and torch.equal(v[page, slot], s.v[page, slot])
            assert torch.equal(cache.key_weights[layer].cpu()[page, :, slot], s.weights[page, :, slot])
    one([c, a, b], [1, 3, 1])
    cache.remove(a)
    d = cache.add()
    seen[d] = 0
    one([d, b], [50, 2])
    one([b, d, c], [1, 1, 1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens, H, D, causal, p, turn, fp32", [([61], 3, 64, True, 0.0, True, False), ([40, 128, 7], 2, 32, False, 0.0, True, True),
                                                                ([100, 100], 4, 128, True, 0.0, False, False), ([90, 33], 2, 64, True, 0.1, True, False)])
def test_attention_with_norm_and_rotation(dtype, lens, H, D, causal, p, turn, fp32):
    """flash_attn_unpadded_qkvpacked_norm_rotary_func is the norm and the attention one after the other: the same bits, and the same gradients where
    those take the same kernels"""
    from flash_attn.flash_attn_interface import flash_attn_unpadded_func, flash_attn_unpadded_qkvpacked_norm_rotary_func
    from flash_attn.rotary import apply_qk_norm_rotary
    total, cu = sum(lens), cumulative(lens).cuda()
    qkv = randn(total, 3, H, D, seed=1, dtype=dtype).cuda().requires_grad_()
    w = [(1 + 0.2 * randn(D, seed=s, dtype=torch.float32)).to(torch.float32 if fp32 else dtype).cuda().requires_grad_() for s in (2, 3)]
    cos, sin = (t.cuda() for t in tables(max(lens), D, dtype)) if turn else (None, None)
    pos = torch.cat([torch.arange(n) for n in lens]).to(torch.int32).cuda()
    dout = randn(total, H, D, seed=4, dtype=dtype).cuda()
    gen = torch.cuda.default_generators[0]
    gen.manual_seed(11)
    out = flash_attn_unpadded_qkvpacked_norm_rotary_func(qkv, *w, cos, sin, cu, max(lens), p, causal=causal)
    grads = torch.autograd.grad(out, (qkv, *w), dout)
    gen.manual_seed(11)
    q, k = apply_qk_norm_rotary(qkv[:, 0], qkv[:, 1], *w, cos, sin, positions=pos)
    ref = flash_attn_unpadded_func(q, k, qkv[:, 2], cu, cu, max(lens), max(lens), p, causal=causal)
    want = torch.autograd.grad(ref, (qkv, *w), dout)
    assert torch.equal(out, ref) and all(torch.equal(x, y) for x, y in zip(grads, want))


@pytest.mark.gpu
def test_rows_behind_the_last_sequence_have_no_part_in_attention_with_norm():
    """as many rows as sequences of the longest length would have, and only some of them in sequences"""
    from flash_attn.flash_attn_interface import flash_attn_unpadded_qkvpacked_norm_rotary_func
    cu, w = cumulative([5, 10]).cuda(), torch.ones(64, dtype=torch.float16, device="cuda").requires_grad_()
    cos, sin = (t.cuda() for t in tables(10, 64, torch.float16))
    full = randn(20, 3, 2, 64, seed=1).cuda()
    full[15:] = math.nan
    dout = randn(20, 2, 64, seed=2).cuda()
    got = []
    for rows in (15, 20):
        torch.empty(4096, dtype=torch.float16, device="cuda").fill_(math.nan)  # (what fresh tensors may hold)
        qkv = full[:rows].clone().requires_grad_()
        out = flash_attn_unpadded_qkvpacked_norm_rotary_func(qkv, w, w, cos, sin, cu, 10, 0.0, causal=True)
        dqkv, dw = torch.autograd.grad(out, (qkv, w), dout[:rows])
        got.append((out[:15], dqkv[:15], dw))
    assert all(torch.equal(a, b) for a, b in zip(*got)) and got[0][2].isfinite().all()


@pytest.mark.gpu
def test_sizes_that_no_field_holds_are_refused():
    """no head, no slot, and numbers beyond 32 bits: errors, not other numbers"""
    from flash_attn import flash_attn_paged_interface as p
    c = Cache([20, 9], 2, 64, 16, torch.float16, 1).gpu()
    q, cu = randn(3, 4, 64, seed=0).cuda(), cumulative([2, 1]).cuda()
    where = (c.dtable, cu, c.dlens)
    evict = lambda k, v, *n: p.paged_evict_func(k, v, c.dweights, c.dpositions, c.dtable, c.dlens, c.dlens, *n)  # noqa: E731
    none, empty = c.dk[:, :, :0], q[:, :0]
    calls = (lambda: p.flash_attn_paged_func(q, none, none, *where, 2, 20), lambda: p.paged_append_func(q, empty, empty, none, none, *where),
             lambda: p.paged_append_func(None, empty, empty, none, none, *where), lambda: p.flash_attn_paged_func(q, c.dk[:0], c.dv[:0], *where, 2, 20),
             lambda: p.paged_key_weights_func(q, torch.zeros(2, 4, 16, device="cuda"), none, c.dweights[:, :0].contiguous(), *where, 2, 20),
             lambda: p.flash_attn_paged_func(q, c.dk, c.dv, *where, 2 ** 32 + 2, 20), lambda: p.flash_attn_paged_func(q, c.dk, c.dv, *where, 2, 2 ** 32 + 20),
             lambda: evict(c.dk, c.dv, 2 ** 32 + 5, 2, 20), lambda: evict(c.dk, c.dv, 5, 2 ** 32, 20), lambda: evict(c.dk, c.dv, 5, 2, 2 ** 32 + 20),
             lambda: evict(none, none, 5, 2, 20))
    for i, call in enumerate(calls):
        print(i, flush=True)  # (shown with a failure)
        with pytest.raises(RuntimeError):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("rotary", [None, "1d", "2d"])
@pytest.mark.parametrize("padded", [False, True])
def test_mha_with_norm(rotary, padded):
    """FlashMHA(qk_norm=True) is its projections, the norm with the rotation and the attention one after the other, and gives every parameter a gradient"""
    from flash_attn.flash_attention import FlashMHA
    from flash_attn.rotary import apply_qk_norm_rotary
    torch.manual_seed(0)
    m = FlashMHA(128, 4, causal=rotary != "2d", use_rotary_emb=rotary, qk_norm=True, device="cuda", dtype=torch.float16)
    torch.nn.init.uniform_(m.q_norm_weight, 0.5, 1.5)
    torch.nn.init.uniform_(m.k_norm_weight, 0.5, 1.5)
    x = torch.randn(2, 49, 128, device="cuda", dtype=torch.float16)
    mask = None
    if padded:
        keep = torch.ones(2, 49, dtype=torch.bool, device="cuda")
        keep[1, 30:] = False
        mask = type("Mask", (), {"bool_matrix": keep})
    y, _ = m(x, None, None, key_padding_mask=mask)
    y.float().square().sum().backward()
    assert y.shape == x.shape and all(p.grad is not None and p.grad.isfinite().all() and p.grad.abs().sum() > 0 for p in m.parameters())
    with torch.no_grad():
        qkv = m.Wqkv(x).reshape(2, 49, 3, 4, 32)
        q, k = apply_qk_norm_rotary(qkv[:, :, 0], qkv[:, :, 1], m.q_norm_weight, m.k_norm_weight, *(m.rotary_emb.half_tables(qkv) if rotary == "1d" else (None, None)))
        qkv = torch.stack([q, k, qkv[:, :, 2]], dim=2).requires_grad_()
        if rotary == "2d":
            qkv = m.rotary_emb.rotate_qkv_(qkv.detach())
        with torch.enable_grad():  # (padded batches without a gradient take another kernel)
            z = m.inner_attn(qkv.detach().requires_grad_(), key_padding_mask=mask, causal=m.causal)[0]
        assert torch.equal(m.out_proj(z.detach().reshape(2, 49, 128)), y.detach())


@pytest.mark.gpu
@pytest.mark.parametrize("norm, rotary", [(True, "1d"), (False, "1d"), (True, None), (False, None)])
def test_mha_from_the_cache_is_mha_on_the_whole(norm, rotary):
    """prompt, chunk and single tokens through FlashMHA.forward_cached against forward on the whole sequences"""
    from flash_attn.flash_attention import FlashMHA
    from flash_attn.flash_attn_paged_interface import PagedKVCache
    torch.manual_seed(1)
    m = FlashMHA(128, 4, causal=True, use_rotary_emb=rotary, qk_norm=norm, device="cuda", dtype=torch.float16).eval()
    if norm:
        torch.nn.init.uniform_(m.q_norm_weight, 0.5, 1.5)
        torch.nn.init.uniform_(m.k_norm_weight, 0.5, 1.5)
    xs = [torch.randn(n, 128, device="cuda", dtype=torch.float16) for n in (50, 31)]
    with torch.no_grad():
        whole = [m(x[None], None, None)[0][0] for x in xs]
        cache = PagedKVCache(1, 12, 16, 4, 32)
        ids = [cache.add(), cache.add()]
        parts, at = [[], []], [0, 0]
        for new in ([33, 5], [9, 20], [1, 1], [1, 0], [1, 1], [5, 4]):
            x = torch.cat([xs[i][at[i]:at[i] + n] for i, n in enumerate(new)])
            y = m.forward_cached(x, cache.step(ids, new))
            for i, (n, piece) in enumerate(zip(new, y.split(new))):
                parts[i].append(piece)
                at[i] += n
    assert at == [50, 31]
    # What differs: attention rounds probabilities at other reference points (2 u of the largest value on each side) and the result once on each side
    # (u of it); the projection multiplies that by its weights' magnitudes, and sums 128 products in fp32 and rounds (u of the result on each side).
    # |v| is at most the largest entry of x W^T + b.
    with torch.no_grad():
        u = half_step(torch.float16)
        vmax = max((x.float() @ m.Wqkv.weight[256:].float().t() + m.Wqkv.bias[256:].float()).abs().max().item() for x in xs)
        row = m.out_proj.weight.float().abs().sum(1)
        for w, p in zip(whole, parts):
            bound = row * vmax * (6 * u + 1e-4) + 2 * u * w.float().abs() + 1e-4
            assert ((torch.cat(p).float() - w.float()).abs() <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 40])
def test_a_captured_step_follows_its_tensors(new):
    """store, attend, weigh and evict in one graph: replayed with other tokens, lengths and tables in the same tensors, with eager calls in between, it gives
    what eager calls give"""
    from flash_attn import flash_attn_paged_interface as p
    lens = [[200, 77], [90, 300], [41, 40], [299, 301], [200, 77]]
    caches = [Cache(n, 2, 64, 16, torch.float16, i, cols=20, spare=60 - sum(-(-x // 16) for x in n)).gpu() for i, n in enumerate(lens)]
    qkvs = [randn(2 * new, 8, 64, seed=i).cuda() for i in range(len(lens))]
    cu = cumulative([new, new]).cuda()
    w = torch.ones(64, dtype=torch.float16, device="cuda")
    cos, sin = (t.cuda() for t in tables(400, 64, torch.float16))

    def step(c, qkv):
        q = p.paged_append_func(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], c["k"], c["v"], c["table"], cu, c["lens"], q_weight=w, k_weight=w, cos_half=cos, sin_half=sin,
                                key_weights=c["w"], key_positions=c["p"])
        out, lse = p.flash_attn_paged_func(q, c["k"], c["v"], c["table"], cu, c["lens"], new, 310, return_softmax_lse=True)
        p.paged_key_weights_func(q, lse, c["k"], c["w"], c["table"], cu, c["lens"], new, 310)
        n = p.paged_evict_func(c["k"], c["v"], c["w"], c["p"], c["table"], c["lens"], c["lens"], 64, 16, 310)
        return out, n

    def fresh(c):
        return dict(k=c.dk.nan_to_num(0.5), v=c.dv.nan_to_num(0.5), table=c.dtable.clone(), lens=c.dlens.clone(), w=c.dweights.clone(), p=c.dpositions.clone())

    with torch.no_grad():
        static, qkv = fresh(caches[0]), qkvs[0].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(static, qkv)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, n = step(static, qkv)
        for i, c in enumerate(caches):
            eager = fresh(c)
            want = step(eager, qkvs[i])
            for k, v in fresh(c).items():
                static[k].copy_(v)
            qkv.copy_(qkvs[i])
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want[0]) and torch.equal(n, want[1]), i
            assert all(torch.equal(static[k], eager[k]) for k in static), i


@pytest.mark.gpu
def test_norm_captured_with_its_backward():
    from flash_attn.rotary import apply_qk_norm_rotary
    q, k = (randn(130, 4, 64, seed=i).cuda().requires_grad_() for i in (0, 1))
    w = torch.ones(64, device="cuda").requires_grad_()
    cos, sin = (t.cuda() for t in tables(130, 64, torch.float16))
    dq, dk = (randn(130, 4, 64, seed=i).cuda() for i in (2, 3))

    def step(q, k, w):
        y = apply_qk_norm_rotary(q, k, w, w, cos, sin)
        return y + torch.autograd.grad(y, (q, k, w), (dq, dk))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(q, k, w)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(q, k, w)
    for i in range(3):
        with torch.no_grad():
            q.copy_(randn(130, 4, 64, seed=10 + i))
            w.copy_(1 + 0.1 * randn(64, seed=20 + i, dtype=torch.float32))
        want = step(*(t.detach().clone().requires_grad_() for t in (q, k, w)))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


@pytest.mark.gpu
def test_calls_on_another_stream():
    from flash_attn import flash_attn_paged_interface as p
    from flash_attn.rotary import apply_qk_norm_rotary
    c = Cache([3000, 2100], 2, 64, 16, torch.float16, 3).gpu()
    q = randn(2, 4, 64, seed=1).cuda()
    cu = cumulative([1, 1]).cuda()
    want = p.flash_attn_paged_func(q, c.dk, c.dv, c.dtable, cu, c.dlens, 1, 3000)
    side = torch.cuda.Stream()
    x = torch.randn(2048, 2048, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):
            x = x @ x * 1e-3  # (work in front, so that a call on the default stream would read too early)
        late = q * 0 + x[:2, :4, None].to(q.dtype).nan_to_num(0.0, 0.0, 0.0) * 0 + q
        got = p.flash_attn_paged_func(late, c.dk, c.dv, c.dtable, cu, c.dlens, 1, 3000)
        w = torch.ones(64, dtype=torch.float16, device="cuda")
        a = apply_qk_norm_rotary(late, late, w, w)[0]
    side.synchronize()
    assert torch.equal(got, want)
    assert torch.equal(a, apply_qk_norm_rotary(q, q, w, w)[0])


@pytest.mark.gpu
def test_calls_of_two_threads_on_their_own_streams():
    """scratch belongs to a call: two threads' calls overlap and give what each gives alone"""
    import threading
    from flash_attn import flash_attn_paged_interface as p
    jobs = []
    for i, (lens, new) in enumerate((([9000, 5000, 100], 1), ([3000, 2500], 20))):
        c = Cache(lens, 2, 64, 64, torch.float16, 30 + i).gpu()
        q, cu = randn(len(lens) * new, 8, 64, seed=i).cuda(), cumulative([new] * len(lens)).cuda()
        jobs.append(lambda q=q, c=c, cu=cu, new=new, n=max(lens): p.flash_attn_paged_func(q, c.dk, c.dv, c.dtable, cu, c.dlens, new, n))
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
@pytest.mark.parametrize("new", [1, 30])
def test_views_give_what_copies_give(new):
    """queries, keys and values of a packed tensor, a page table inside a wider one, lengths and offsets inside longer tensors, pools inside larger ones"""
    from flash_attn import flash_attn_paged_interface as p
    got = []
    for views in (False, True):
        c = Cache([130, 90, 61], 2, 64, 32, torch.bfloat16, 8).gpu()
        k, v, w, pos = c.dk.nan_to_num(0.5), c.dv.nan_to_num(0.25), c.dweights, c.dpositions
        qkv = randn(3 * new, 8, 64, seed=2, dtype=torch.bfloat16).cuda()
        q, kn, vn = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
        cu, table, lens = cumulative([new] * 3).cuda(), c.dtable, c.dlens
        if views:
            pools = torch.full((2, c.n_pages + 2, 3, 32, 64), 9.0, dtype=torch.bfloat16, device="cuda")
            pools[0, 1:-1, :2], pools[1, 1:-1, :2] = k.transpose(1, 2), v.transpose(1, 2)
            k, v = (x[1:-1, :2].transpose(1, 2) for x in pools)
            wide = torch.full((3, table.shape[1] + 5), 7, dtype=torch.int32, device="cuda")
            wide[:, 2:-3] = table
            table = wide[:, 2:-3]
            lens, cu = torch.cat([lens[:1], lens, lens])[1:4], torch.cat([cu[:1], cu, cu])[1:5]
        else:
            q, kn, vn = q.contiguous(), kn.contiguous(), vn.contiguous()
        q = p.paged_append_func(q, kn, vn, k, v, table, cu, lens, key_weights=w, key_positions=pos)
        out, lse = p.flash_attn_paged_func(q, k, v, table, cu, lens, new, 130, return_softmax_lse=True)
        p.paged_key_weights_func(q, lse, k, w, table, cu, lens, new, 130)
        n = p.paged_evict_func(k, v, w, pos, table, lens, lens, 70, 8, 130)
        got.append((q, out, lse[..., :new], k, v, w, pos, n))
        if views:
            assert (pools[:, :, 2] == 9).all() and (pools[:, 0] == 9).all() and (pools[:, -1] == 9).all()
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 50])
def test_a_cache_beyond_32_bit_offsets(new):
    """pages whose offsets pass 2^32 bytes (and 2^31 elements) give what pages at the front give"""
    from flash_attn import flash_attn_paged_interface as p
    PS, HK, D, lens = 64, 2, 128, [500, 211]
    pages = -(-(5 << 30) // (PS * HK * D * 2))
    big = [torch.empty(pages, HK, PS, D, dtype=torch.float16, device="cuda").transpose(1, 2) for _ in range(2)]
    meta = [torch.zeros(pages, HK, PS, device="cuda"), torch.zeros(pages, HK, PS, dtype=torch.int32, device="cuda")]
    small = Cache(lens, HK, D, PS, torch.float16, 5).gpu()
    small.dk.nan_to_num_(0.0)
    small.dv.nan_to_num_(0.0)
    far = pages - small.n_pages
    for b, s in zip(big, (small.dk, small.dv)):
        b[far:] = s
    table = torch.where(small.dtable >= 0, small.dtable + far, -1).to(torch.int32)
    qkv, cu = randn(2 * new, 8, D, seed=6).cuda(), cumulative([new, new]).cuda()
    got = []
    for k, v, t, w, pos in ((*big, table, *meta), (small.dk, small.dv, small.dtable, small.dweights, small.dpositions)):
        q = p.paged_append_func(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], k, v, t, cu, small.dlens, key_weights=w, key_positions=pos)
        out, lse = p.flash_attn_paged_func(q, k, v, t, cu, small.dlens, new, 500, return_softmax_lse=True)
        p.paged_key_weights_func(q, lse, k, w, t, cu, small.dlens, new, 500)
        n = p.paged_evict_func(k, v, w, pos, t, small.dlens, small.dlens, 100, 20, 500)
        got.append((out, lse[..., :new], k[-small.n_pages:], v[-small.n_pages:], w[-small.n_pages:], pos[-small.n_pages:], n))
    assert all(torch.equal(a, b) for a, b in zip(*got))
