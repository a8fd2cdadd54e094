"""Calls at the edges of the norm of queries and keys and of the paged cache: no key heads, forward-mode tangents, rotation tables that are too short, modules in 16
bits, tensors at odd addresses, tables and steps under capture.

Tolerances are counted: u is half a step of the element type, 2^-24 a rounding in fp32."""
import math

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
