"""The one-kernel backward (launch policy 0x20) in processes of several streams: a hardware queue's launches begin at an XCD of their own."""
import pytest
import torch


def setup(lens_q, lens_k, H, dtype=torch.float16, seed=1):
    """q, k, v, dout, the forward's output and lse, and the call of a backward into NaN"""
    from flash_attn import flash_attn_gfx950 as be
    g = torch.Generator().manual_seed(seed)
    q, dout = (torch.randn(sum(lens_q), H, 64, generator=g).to(dtype).cuda() for _ in range(2))
    k, v = (torch.randn(sum(lens_k), H, 64, generator=g).to(dtype).cuda() for _ in range(2))
    cu_q, cu_k = (torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda() for lens in (lens_q, lens_k))
    o, lse = be.fwd(q, k, v, cu_q, cu_k, max(lens_q), max(lens_k), 0.0, 0.125, False, False, False, None)

    def run():
        grads = [torch.full_like(t, float("nan")) for t in (q, k, v)]
        be.bwd(dout, q, k, v, o, lse, *grads, cu_q, cu_k, max(lens_q), max(lens_k), 0.0, 0.125, False, False, None)
        return grads
    return run


@pytest.fixture
def one_kernel():
    from flash_attn import flash_attn_gfx950 as be
    be.set_launch_policy(0x20)
    yield be
    be.set_launch_policy(0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens_q, lens_k, H", [([300, 77], [300, 77], 3), ([200, 31, 512], [640, 129, 96], 3), ([1024, 2048], [2048, 1500], 8)])
def test_one_kernel_backward_on_every_stream(dtype, lens_q, lens_k, H, one_kernel):
    """the same bits on each of more streams than there are hardware queues, and on the first one behind them; the two kernels' within the rounding of the results"""
    be = one_kernel
    run = setup(lens_q, lens_k, H, dtype)
    want = run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(9)]
    for i, s in enumerate(streams + [torch.cuda.current_stream()]):
        with torch.cuda.stream(s):
            got = run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
    be.set_launch_policy(0x10)
    u = torch.finfo(dtype).eps / 2
    for a, b in zip(want, run()):
        assert (a.float() - b.float()).abs().max() <= 4 * u * b.float().abs().max()  # (a few fp32 sums in another order, and a rounding on each side)


@pytest.mark.gpu
def test_one_kernel_backwards_of_several_streams_take_turns(one_kernel):
    """a launch's workgroups wait for each other and need places side by side: launches of more streams at once, 32 key tiles each, give what each gives alone"""
    runs = [setup([256, 700], [4096, 3000], 8, seed=i) for i in range(5)]
    want = [run() for run in runs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in runs], []
    for _ in range(6):
        for run, s in zip(runs, streams):
            with torch.cuda.stream(s):
                got.append(run())
    torch.cuda.synchronize()
    for i, grads in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(grads, want[i % len(runs)])), i


@pytest.mark.gpu
def test_the_one_kernel_backward_is_not_captured(one_kernel):
    """a graph's replays could not take their turn: it holds the two kernels"""
    be = one_kernel
    run = setup([300, 77], [300, 77], 3)
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    be.set_launch_policy(0x10)
    want = run()
    for _ in range(3):
        for t in got:
            t.fill_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
