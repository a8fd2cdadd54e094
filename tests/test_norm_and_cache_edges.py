"""Calls at the edges of the norm of queries and keys and of the paged cache: no key heads, forward-mode tangents, rotation tables that are too short, modules in 16
bits, tensors at odd addresses, tables and steps under capture.

Tolerances are counted: u is half a step of the element type, 2^-24 a rounding in fp32."""
import math
import pickle

import pytest
import torch
from torch.autograd import forward_ad

from test_paged import DTYPES, Cache, cumulative, half_step, tables


def randn(*shape, seed, dtype=torch.float16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


# ---- a norm of queries alone

@pytest.mark.gpu
@pytest.mark.parametrize("fp32", [False, True])
def test_keys_without_heads_leave_their_weight_a_gradient_of_zeros(fp32):
    from flash_attn.rotary import apply_qk_norm_rotary
    q = randn(5, 2, 64, seed=0).cuda().requires_grad_()
    w = [torch.ones(64, dtype=torch.float32 if fp32 else torch.float16, device="cuda").requires_grad_() for _ in range(2)]
    dq = randn(5, 2, 64, seed=1).cuda()
    want = torch.autograd.grad(apply_qk_norm_rotary(q, q.detach(), *w)[0], (q, w[0]), dq)
    k = torch.zeros(5, 0, 64, dtype=torch.float16, device="cuda").requires_grad_()
    q2, k2 = apply_qk_norm_rotary(q, k, *w)
    assert k2.shape == k.shape
    fresh = [torch.full((n,), math.nan, device="cuda") for n in [64, 128, 256, 1024, 4096] * 8]  # (what new tensors hold)
    del fresh
    got = torch.autograd.grad((q2, k2), (q, k, *w), (dq, torch.zeros_like(k2)))
    assert torch.equal(got[0], want[0]) and got[1].shape == k.shape and torch.equal(got[2], want[1])
    assert torch.equal(got[3], torch.zeros_like(got[3]))


# ---- forward-mode tangents: nothing here has a rule for them

def test_forward_tangents_are_refused_by_the_cache(lib):
    """also under no_grad, which forward mode does not heed; a tensor whose tangents are switched off is a plain one (and refused for its device here)"""
    from flash_attn import flash_attn_paged_interface as p
    q, c = torch.zeros(3, 2, 64).half(), torch.zeros(4, 16, 2, 64).half()
    i32, meta, lse = torch.zeros(2, dtype=torch.int32), torch.zeros(4, 2, 16), torch.zeros(1, 2, 16)
    w = torch.ones(64).half()
    with forward_ad.dual_level(), torch.no_grad():
        d = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        calls = [lambda q=q, k=q, v=q, w=w: p.paged_append_func(q, k, v, c, c, i32[:1, None], i32, i32[:1], w, w),
                 lambda q=q, k=c, v=c: p.flash_attn_paged_func(q, k, v, i32[:1, None], i32, i32[:1], 3, 3),
                 lambda q=q, l=lse, k=c: p.paged_key_weights_func(q, l, k, meta, i32[:1, None], i32, i32[:1], 3, 3),
                 lambda k=c, v=c: p.paged_evict_func(k, v, meta, meta.int(), i32[:1, None], i32[:1], i32[:1], 2, 1, 3)]
        for call in calls:
            for i, t in enumerate(call.__defaults__):
                with pytest.raises(RuntimeError, match="forward mode"):
                    call(*call.__defaults__[:i], d(t))
            with pytest.raises(RuntimeError, match="GPU"):
                call()
        with forward_ad._set_fwd_grad_enabled(False), pytest.raises(RuntimeError, match="GPU"):
            calls[1](d(q))


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [False, True])
def test_forward_tangents_do_not_pass_the_native_calls(lib, grad):
    from flash_attn import flash_attn_paged_interface as p
    from flash_attn.rotary import apply_qk_norm_rotary
    c = Cache([20, 9], 2, 64, 16, torch.float16, 1).gpu()
    q, cu = randn(3, 4, 64, seed=0).cuda(), cumulative([2, 1]).cuda()
    w = torch.ones(64, dtype=torch.float16, device="cuda")
    before = [t.clone() for t in (c.dk, c.dv, c.dweights, c.dpositions)]
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        d = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        where = (c.dtable, cu, c.dlens)
        out, lse = p.flash_attn_paged_func(q, c.dk, c.dv, *where, 2, 20, return_softmax_lse=True)
        for args in ((d(q), q, w, w), (q, d(q), w, w), (q, q, d(w), w), (q, q, w, d(w)), (d(q)[:, :2], q, w, w)):
            with pytest.raises(NotImplementedError):
                apply_qk_norm_rotary(*args)
        for call in (lambda: p.paged_append_func(d(q), q[:, :2], q[:, 2:], c.dk, c.dv, *where), lambda: p.paged_append_func(None, q[:, :2], d(q)[:, 2:], c.dk, c.dv, *where),
                     lambda: p.paged_append_func(q, q[:, :2], q[:, 2:], c.dk, c.dv, *where, w, d(w)), lambda: p.flash_attn_paged_func(d(q), c.dk, c.dv, *where, 2, 20),
                     lambda: p.flash_attn_paged_func(q, d(c.dk), c.dv, *where, 2, 20), lambda: p.paged_key_weights_func(d(q), lse, c.dk, c.dweights, *where, 2, 20),
                     lambda: p.paged_evict_func(c.dk, d(c.dv), c.dweights, c.dpositions, c.dtable, c.dlens, c.dlens, 8, 2, 20)):
            with pytest.raises(RuntimeError, match="forward mode"):
                call()
        with forward_ad._set_fwd_grad_enabled(False):
            assert torch.equal(p.flash_attn_paged_func(d(q), c.dk, c.dv, *where, 2, 20), out)
    same = [torch.equal(torch.nan_to_num(a), torch.nan_to_num(b)) for a, b in zip(before, (c.dk, c.dv, c.dweights, c.dpositions))]
    assert all(same)  # (nothing was stored)


# ---- rotation tables that end before the positions do

@pytest.mark.gpu
def test_attention_with_norm_refuses_tables_shorter_than_its_sequences():
    from flash_attn.flash_attn_interface import flash_attn_unpadded_qkvpacked_norm_rotary_func as f
    qkv, cu = randn(50, 3, 2, 64, seed=1).cuda(), cumulative([20, 30]).cuda()
    w = torch.ones(64, dtype=torch.float16, device="cuda")
    cos, sin = (t.cuda() for t in tables(30, 64, torch.float16))
    want = f(qkv, w, w, cos, sin, cu, 30, 0.0, causal=True)
    for rows, longest in ((29, 30), (1, 30), (30, 31)):
        with pytest.raises(RuntimeError, match="rows"):
            f(qkv, w, w, cos[:rows], sin[:rows], cu, longest, 0.0, causal=True)
    longer = (t.cuda() for t in tables(64, 64, torch.float16))
    assert torch.equal(f(qkv, w, w, *longer, cu, 30, 0.0, causal=True), want)


def test_a_step_refuses_tables_that_its_positions_outgrow(lib):
    """before anything is stored; sequences of the step without a new token do not count"""
    from flash_attn.flash_attn_paged_interface import PagedKVCache
    c = PagedKVCache(1, 8, 16, 2, 64, device="cpu")
    a, b = c.add(), c.add()
    c.step([a], [40])
    s = c.step([a, b], [0, 5])
    assert s.max_position == 5
    q = torch.zeros(5, 2, 64).half()
    for rows in (1, 4):
        with pytest.raises(RuntimeError, match="rows"):
            s.append(0, q, q, q, **dict(zip(("cos_half", "sin_half"), tables(rows, 64, torch.float16))))
    for rows in (5, 41):  # (long enough: what is refused is the host's tensors)
        with pytest.raises(RuntimeError, match="GPU"):
            s.append(0, q, q, q, **dict(zip(("cos_half", "sin_half"), tables(rows, 64, torch.float16))))
    s = c.step([a, b], [1, 0])
    assert s.max_position == 41
    with pytest.raises(RuntimeError, match="rows"):
        s.append(0, q[:1], q[:1], q[:1], **dict(zip(("cos_half", "sin_half"), tables(40, 64, torch.float16))))


# ---- modules in 16 bits

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [16, 64, 128])
def test_tables_of_a_module_in_16_bits_are_formed_in_32(dtype, dim):
    """.half() and .bfloat16() round the buffer of frequencies too.  An angle is a position times a frequency: three roundings in fp32 (power, reciprocal, product) of at
    most two steps each, so off by 6 * 2^-23 of itself; cosines by that, their own few steps, and one rounding."""
    from flash_attn.rotary import RotaryEmbedding
    N = 5000
    plain = RotaryEmbedding(dim)
    like = torch.zeros(1, N, 3, 1, dim, dtype=dtype)
    emb = RotaryEmbedding(dim).to(dtype)
    angle = torch.outer(torch.arange(N, dtype=torch.float64), 10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim))
    for got, same, exact in zip(emb.tables_to(N, like), emb.half_tables(like), (torch.cos(angle), torch.sin(angle))):
        assert got.dtype == dtype and got.shape[0] >= N and torch.equal(got[:N], same)
        assert ((got[:N].double() - exact).abs() <= half_step(dtype) + 6 * 2.0 ** -23 * angle + 2.0 ** -21).all()
    # a module in 32 bits: what its buffer says, as before
    want = torch.outer(torch.arange(N, dtype=torch.float32), plain.inv_freq)
    assert torch.equal(plain.tables_to(N, like)[0][:N], torch.cos(want).to(dtype)) and torch.equal(plain.half_tables(like)[1], torch.sin(want).to(dtype))
    other = {"inv_freq": plain.inv_freq / 2}
    plain.load_state_dict(other)
    assert torch.equal(plain.half_tables(like)[0], torch.cos(want / 2).to(dtype))
    back = RotaryEmbedding(dim).to(dtype).float()
    plain = RotaryEmbedding(dim)
    assert torch.equal(back.inv_freq, plain.inv_freq) and back.inv_freq.dtype == torch.float32


@pytest.mark.parametrize("dtype", DTYPES)
def test_other_frequencies_stay_through_16_bits(dtype):
    """loaded before a cast: not rounded at all; loaded into a module in 16 bits: as they were loaded"""
    from flash_attn.rotary import RotaryEmbedding
    like, other = torch.zeros(1, 9, 3, 1, 64), RotaryEmbedding(64).inv_freq * 0.3
    emb = RotaryEmbedding(64)
    emb.half_tables(like), emb(like[:, :, 0], like[:, :, 0], seq_dimension=-3)
    emb.load_state_dict({"inv_freq": other})
    want = torch.cos(torch.outer(torch.arange(9.0), other))
    assert torch.equal(emb._update_cos_sin_tables(like[:, :, 0], seq_dimension=-3)[0][:, ::2], want)
    assert torch.equal(emb.to(dtype).half_tables(like)[0], want) and torch.equal(emb.to(dtype).cpu().half_tables(like)[0], want)
    assert torch.equal(emb.float().inv_freq, other) and torch.equal(emb.half_tables(like)[0], want)
    emb = RotaryEmbedding(64).to(dtype)
    emb.half_tables(like)
    emb.load_state_dict({"inv_freq": other})
    want = torch.cos(torch.outer(torch.arange(9.0), other.to(dtype).float()))
    assert torch.equal(emb.half_tables(like)[0], want) and torch.equal(emb.float().inv_freq, other.to(dtype).float())
    emb.inv_freq = RotaryEmbedding(64).inv_freq
    assert torch.equal(emb.half_tables(like)[0], RotaryEmbedding(64).half_tables(like)[0])
    copy = pickle.loads(pickle.dumps(RotaryEmbedding(64).to(dtype)))
    assert torch.equal(copy.half_tables(like)[0], RotaryEmbedding(64).half_tables(like)[0])
    with torch.device("meta"):
        emb = RotaryEmbedding(64).to(dtype)
    emb = emb.to_empty(device="cpu")
    emb.load_state_dict(RotaryEmbedding(64).to(dtype).state_dict())
    assert torch.equal(emb.half_tables(like)[0], RotaryEmbedding(64).half_tables(like)[0])


@pytest.mark.gpu
def test_a_module_in_16_bits_serves_far_positions_as_one_in_32_bits_does():
    """the same projections: a module made in fp16 (frequencies in fp32) and one turned to fp16, at positions beyond 2048"""
    from flash_attn.flash_attention import FlashMHA
    from flash_attn.flash_attn_paged_interface import PagedKVCache
    torch.manual_seed(2)
    made = FlashMHA(128, 2, causal=True, use_rotary_emb="1d", device="cuda", dtype=torch.float16).eval()
    turned = FlashMHA(128, 2, causal=True, use_rotary_emb="1d", device="cuda").half().eval()
    turned.load_state_dict(made.state_dict())
    x = torch.randn(2101, 128, device="cuda", dtype=torch.float16)
    outs = []
    with torch.no_grad():
        for m in (made, turned):
            cache = PagedKVCache(1, 140, 16, 2, 64)
            seq = cache.add()
            outs.append([m.forward_cached(x[a:b], cache.step([seq], [b - a])) for a, b in ((0, 2100), (2100, 2101))])
        tables = [m.rotary_emb.tables_to(2101, x) for m in (made, turned)]
        whole = [m(x[None], None, None)[0] for m in (made, turned)]
    # the frequencies of both are fp32 numbers, at most two steps apart: angles by 2 * 2^-23 of themselves, and a rounding to 16 bits on each side
    gap = 2 * half_step(torch.float16) + 2 * 2.0 ** -23 * 4096 + 2.0 ** -21
    assert all((a.float() - b.float()).abs().max() <= gap for a, b in zip(*tables))
    # a vector turned by tables off by g is off by at most 2 g of its length, a score by 4 g |q| |k| / 8, and an output by that (twice) of the largest value
    with torch.no_grad():
        qkv = (x.float() @ made.Wqkv.weight.float().t() + made.Wqkv.bias.float()).view(-1, 3, 2, 64)
        size = qkv.norm(dim=-1).amax(0)  # (3, heads)
        step = 2 * 4 * gap * (size[0] * size[1]).max().item() / 8 * qkv[:, 2].abs().max().item() + 6 * half_step(torch.float16) * qkv[:, 2].abs().max().item()
        bound = made.out_proj.weight.float().abs().sum(1) * step + 1e-3
    for a, b in zip(outs[0] + whole[:1], outs[1] + whole[1:]):
        assert ((a.float() - b.float()).abs() <= bound).all()


def test_tables_of_two_threads():
    """threads that ask one module for tables of different lengths get theirs"""
    import threading
    from flash_attn.rotary import RotaryEmbedding
    emb, wrong = RotaryEmbedding(16), []

    def ask(lengths):
        x = {n: torch.zeros(1, n, 1, 1, 16) for n in lengths}
        for _ in range(300):
            for n in lengths:
                if emb.half_tables(x[n])[0].shape[0] != n or emb.tables_to(n, x[n])[0].shape[0] < n:
                    wrong.append(n)

    threads = [threading.Thread(target=ask, args=(n,)) for n in ((3, 300, 5000), (7, 900), (2000, 20000))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


# ---- tensors at odd addresses

def odd_address(t):
    """the same values, contiguous, one element behind an aligned address"""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    flat[1:] = t.reshape(-1)
    got = flat[1:].view(t.shape)
    assert got.is_contiguous() and got.data_ptr() % 16
    return got


def test_rows_at_an_odd_address_are_copied_to_an_even_one():
    from flash_attn.rotary import _kernel_rows
    t = odd_address(randn(3, 2, 64, seed=0))
    got = _kernel_rows(t)
    assert got.data_ptr() % 16 == 0 and got.is_contiguous() and torch.equal(got, t)
    view = randn(3, 4, 64, seed=1)[:, :2]
    assert _kernel_rows(view) is view


@pytest.mark.gpu
@pytest.mark.parametrize("four", [False, True])
def test_norm_of_tensors_at_odd_addresses(four):
    """as input (the Python function) and as incoming gradient (the native one, and Python's)"""
    from flash_attn.rotary import apply_qk_norm_rotary
    q, k = randn(6, 4, 64, seed=0).cuda(), randn(6, 2, 64, seed=1).cuda()
    dq, dk = randn(6, 4, 64, seed=2).cuda(), randn(6, 2, 64, seed=3).cuda()
    if four:
        q, k, dq, dk = (t.view(2, 3, *t.shape[1:]) for t in (q, k, dq, dk))
    w = torch.ones(64, dtype=torch.float16, device="cuda").requires_grad_()
    cos, sin = (t.cuda() for t in tables(6, 64, torch.float16))

    def step(q, k, dq, dk):
        q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
        y = apply_qk_norm_rotary(q, k, w, w, cos, sin)
        return y + torch.autograd.grad(y, (q, k, w), (dq, dk))

    want = step(q, k, dq, dk)
    for odd in ((0,), (1,), (2,), (3,), (0, 3), (2, 3)):
        got = step(*(odd_address(t) if i in odd else t for i, t in enumerate((q, k, dq, dk))))
        assert all(torch.equal(a, b) for a, b in zip(got, want)), odd
    # a gradient as autograd makes it: a piece of a longer one
    x, y = q.detach().requires_grad_(), k.detach().requires_grad_()
    out = apply_qk_norm_rotary(x, y, w, w, cos, sin)
    joined = torch.cat([torch.zeros(1, dtype=torch.float16, device="cuda"), out[0].flatten()])
    up = torch.cat([torch.zeros(1, dtype=torch.float16, device="cuda"), dq.flatten()])
    got = torch.autograd.grad((joined, out[1]), (x, y, w), (up, dk))
    assert all(torch.equal(a, b) for a, b in zip(got, want[2:]))


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["plain", "rotary", "norm", "blocks"])
def test_attention_takes_a_gradient_at_an_odd_address(which):
    from flash_attn import flash_attn_interface as f
    from flash_attn.flash_blocksparse_attn_interface import flash_blocksparse_attn_func
    qkv, cu = randn(50, 3, 2, 64, seed=1).cuda().requires_grad_(), cumulative([20, 30]).cuda()
    w = torch.ones(64, dtype=torch.float16, device="cuda")
    cos, sin = (t.cuda() for t in tables(30, 64, torch.float16))
    dout = randn(50, 2, 64, seed=2).cuda()
    call = {"plain": lambda: f.flash_attn_unpadded_qkvpacked_func(qkv, cu, 30, 0.0, causal=True),
            "blocks": lambda: flash_blocksparse_attn_func(qkv, cu, torch.ones(2, 1, device="cuda"), 0.0, 32),
            "rotary": lambda: f.flash_attn_unpadded_qkvpacked_rotary_func(qkv, cos, sin, cu, 30, 0.0, causal=True),
            "norm": lambda: f.flash_attn_unpadded_qkvpacked_norm_rotary_func(qkv, w, w, cos, sin, cu, 30, 0.0, causal=True)}[which]
    want, = torch.autograd.grad(call(), qkv, dout)
    got, = torch.autograd.grad(call(), qkv, odd_address(dout))
    assert torch.equal(got, want)


# ---- the tables that a module keeps, and graphs

@pytest.mark.gpu
def test_tables_made_under_capture_are_the_graphs_own():
    """a graph's memory holds nothing before its first replay: tables that a capture made are not handed to other calls"""
    from flash_attn.rotary import RotaryEmbedding
    like = torch.zeros(1, device="cuda", dtype=torch.float16)
    want = RotaryEmbedding(64).cuda().tables_to(300, like)
    emb = RotaryEmbedding(64).cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cos, sin = emb.tables_to(300, like)
        out = cos + 0
    got = emb.tables_to(300, like)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0])
        assert torch.equal(emb.tables_to(300, like)[0], want[0])


@pytest.mark.gpu
def test_tables_that_a_graph_reads_outlive_their_growth():
    from flash_attn.rotary import RotaryEmbedding
    like = torch.zeros(1, device="cuda", dtype=torch.float16)
    emb = RotaryEmbedding(64).cuda()
    want = [t.clone() for t in emb.tables_to(300, like)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cos, sin = emb.tables_to(300, like)
        out = cos + sin
    for n in (600, 5000):
        assert emb.tables_to(n, like)[0].shape[0] >= n
        emb.tables_to(n, like.bfloat16())
        fresh = [torch.full_like(want[0], math.nan) for _ in range(64)]  # (the memory of tensors that are gone)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0] + want[1])
        del fresh
    assert emb.tables_to(300, like)[0] is emb.tables_to(4000, like)[0]


@pytest.mark.gpu
def test_half_tables_that_a_graph_reads_outlive_those_of_other_lengths():
    from flash_attn.rotary import RotaryEmbedding
    emb = RotaryEmbedding(64).cuda()
    x = [torch.zeros(1, n, 3, 1, 64, device="cuda", dtype=torch.float16) for n in (300, 301, 40, 5000)]
    want = [t.clone() for t in emb.half_tables(x[0])]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cos, sin = emb.half_tables(x[0])
        out = cos + sin
    for y in x[1:]:
        assert [t.shape[0] for t in emb.half_tables(y)] == [y.shape[1]] * 2
        fresh = [torch.full_like(want[0], math.nan) for _ in range(64)]  # (the memory of tensors that are gone)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0] + want[1])
        del fresh
    # the values of forward()'s tables
    cos, sin = emb._update_cos_sin_tables(x[3][:, :, 0], seq_dimension=-3)
    assert all(torch.equal(a, b[:, ::2]) for a, b in zip(emb.half_tables(x[3]), (cos, sin)))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["2d", "1d", "elementwise"])
@pytest.mark.parametrize("warm", [False, True])
def test_rotations_in_a_graph_and_beside_it(kind, warm):
    """captured before or after the module has tables, replayed behind eager calls of other lengths: the graph and the eager calls give what a new module gives"""
    from flash_attn.rotary import RotaryEmbedding, RotaryEmbedding2D
    make = lambda: (RotaryEmbedding2D if kind == "2d" else RotaryEmbedding)(64).cuda()  # noqa: E731

    def turn(emb, x):
        if kind == "elementwise":
            return torch.stack([*emb(x[:, :, 0], x[:, :, 1], seq_dimension=-3), x[:, :, 2]], 2)
        return emb.rotate_qkv_(x.clone())

    x = {n: randn(2, n, 3, 2, 64, seed=n).cuda() for n in (49, 64, 2025)}
    want = {n: turn(make(), t) for n, t in x.items()}
    emb, still = make(), x[49].clone()
    if warm:
        turn(emb, x[49])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = turn(emb, still)
    assert torch.equal(turn(emb, x[49]), want[49])
    for n in (64, 2025, 49):
        assert torch.equal(turn(emb, x[n]), want[n])
        fresh = [torch.full((m,), math.nan, device="cuda", dtype=torch.float16) for m in (64, 98, 1568, 3136, 6272) * 16]  # (the memory of tensors that are gone)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[49])
        del fresh


@pytest.mark.gpu
def test_tables_made_on_one_stream_are_whole_on_another():
    from flash_attn.rotary import RotaryEmbedding
    like = torch.zeros(1, device="cuda", dtype=torch.float16)
    want = RotaryEmbedding(128).cuda().tables_to(1 << 16, like)
    emb = RotaryEmbedding(128).cuda()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    x = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(a):
        for _ in range(20):
            x = x @ x * 1e-3  # (work in front of the tables)
        emb.tables_to(1 << 16, like)
    with torch.cuda.stream(b):
        got = [t.clone() for t in emb.tables_to(1 << 16, like)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.gpu
def test_steps_and_evictions_are_not_made_under_capture():
    """their numbers are the host's: a replay would find those of another step"""
    from flash_attn.flash_attn_paged_interface import PagedKVCache
    cache = PagedKVCache(1, 8, 16, 2, 64, key_weights=True)
    seq = cache.add()
    cache.step([seq], [40])
    graph, y = torch.cuda.CUDAGraph(), torch.zeros(1, device="cuda")
    with torch.cuda.graph(graph):
        for call in (lambda: cache.step([seq], [1]), lambda: cache.evict([seq], 20, 2)):
            with pytest.raises(RuntimeError, match="captur"):
                call()
        y += 1
    assert cache.length(seq) == 40 and cache.free_pages() == 5
    assert cache.step([seq], [1]).seqlens_k.tolist() == [41]


# ---- the book

def test_eviction_keeps_no_more_recent_keys_than_its_budget():
    """the newest could not all stay, and the budget would go to the lowest slots: refused, whatever the lengths"""
    from flash_attn.flash_attn_paged_interface import PagedKVCache
    c = PagedKVCache(1, 10, 16, 2, 64, device="cpu", key_weights=True)
    a = c.add()
    for _ in range(2):
        with pytest.raises(RuntimeError, match="recent"):
            c.evict([a], 30, 31)
        c.evict([a], 41, 41)  # (nothing to cut)
        c.step([a], [20])
    assert c.length(a) == 40


def test_a_step_attends_with_its_own_number_of_tokens(lib):
    from flash_attn.flash_attn_paged_interface import PagedKVCache
    c = PagedKVCache(1, 10, 16, 2, 64, device="cpu")
    s = c.step([c.add()], [5])
    for n in (4, 6, 0):
        with pytest.raises(RuntimeError, match="5 tokens"):
            s.attend(0, torch.zeros(n, 2, 64).half())
    with pytest.raises(RuntimeError, match="GPU"):
        s.attend(0, torch.zeros(5, 2, 64).half())


# ---- the module in bf16

@pytest.mark.gpu
@pytest.mark.parametrize("rotary", [None, "1d", "2d"])
@pytest.mark.parametrize("padded", [False, True])
def test_mha_with_norm_in_bf16(rotary, padded):
    """what forward_cached() serves, forward() runs and trains: against the definition in 64 bits from the module's own projections"""
    from flash_attn.flash_attention import FlashMHA
    torch.manual_seed(0)
    m = FlashMHA(128, 4, causal=rotary != "2d", use_rotary_emb=rotary, qk_norm=True, device="cuda", dtype=torch.bfloat16)
    x = torch.randn(2, 49, 128, device="cuda", dtype=torch.bfloat16)
    keep = torch.ones(2, 49, dtype=torch.bool, device="cuda")
    mask = None
    if padded:
        keep[1, 30:] = False
        mask = type("Mask", (), {"bool_matrix": keep})
    y, _ = m(x, None, None, key_padding_mask=mask)
    y.float().square().sum().backward()
    assert y.dtype == torch.bfloat16 and all(p.grad is not None and p.grad.isfinite().all() and p.grad.abs().sum() > 0 for p in m.parameters())
    with torch.no_grad():
        qkv = m.Wqkv(x).reshape(2, 49, 3, 4, 32)
        q, k = (t / (t.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() for t in (qkv[:, :, 0].double(), qkv[:, :, 1].double()))
        if rotary:
            q, k = m.rotary_emb(q, k, seq_dimension=-3)
        s = (q.transpose(1, 2) @ k.permute(0, 2, 3, 1).contiguous()) * 32 ** -0.5
        s = s.masked_fill(~keep[:, None, None, :], -math.inf)
        if m.causal:
            s = s.masked_fill(torch.ones(49, 49, dtype=torch.bool, device="cuda").triu(1), -math.inf)
        v = qkv[:, :, 2].double().transpose(1, 2).contiguous()
        ctx = (torch.softmax(s, -1) @ v).transpose(1, 2).reshape(2, 49, 128)
        want = ctx @ m.out_proj.weight.double().t() + m.out_proj.bias.double()
        # q and k: one rounding of the norm (2d: and one of each turn), tables rounded (2 u of a vector): 6 u of |q| |k| = 32 in a score, times the scale; attention
        # rounds probabilities and its result; the projection rounds once
        u = half_step(torch.bfloat16)
        vmax = v.abs().max().item()
        bound = m.out_proj.weight.double().abs().sum(1) * vmax * (2 * 2 * 6 * u * 32 * 32 ** -0.5 + 4 * u) + u * want.abs() + 1e-3
        assert ((y.double() - want).abs() <= bound)[keep].all()
