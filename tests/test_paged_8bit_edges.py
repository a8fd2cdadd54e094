"""The paged cache in 8 bits and shared prefixes: bits of scores.

Tolerances are counted, not measured: u half a step of the element type, e = 2^-24 a rounding in fp32 (see test_paged.py)."""
import math

import pytest
import torch

from test_paged import E32, cumulative
from test_paged_8bit import DTYPES, Cache8, ref_quantise


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
