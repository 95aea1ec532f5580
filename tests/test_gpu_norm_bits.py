"""rms_norm_fp8's values are y over its scale, rounded once (gpu).

Rows of ones normed without an eps are ones, so y is the weight; blocks whose largest
value is 448 s, s of eight bits, have the scale s exactly, and values t s the quotient t
exactly: those halfway between two E4M3 values go to the even one.  No tolerance.
"""
import numpy as np
import pytest
import torch

import gateddeltanet_amd as g

pytestmark = pytest.mark.gpu


def weights(n, block):
    """(weight, quotients, scales) of n values in blocks: all ties of E4M3 and its
    values, times the block's scale."""
    odd = torch.arange(129, 256, 2).double() / 128
    scale = (odd.repeat(n // block // 64 + 1)[:n // block] * 2.0**-3)[:, None]
    ties = torch.cat([(1 + torch.arange(1, 16) / 16) * 2.0**e for e in range(-6, 9)] + [torch.arange(1, 16) * 2.0**-10])
    ties = torch.cat([ties, -ties]).double()
    t = ties.repeat(n // len(ties) + 1)[:n].reshape(-1, block).clamp(-448, 448)
    t[:, 0] = 448
    return (t * scale).float().reshape(-1).cuda(), t.float().reshape(-1).cuda(), scale.float().reshape(-1).cuda()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("heads,dim,block", [(1, 2048, 32), (1, 2048, 128), (8, 256, 64), (1, 12288, 64), (1, 20480, 128), (1, 256, 0),
                                             (1, 4096, 0), (1, 16384, 0), (1, 20480, 0), (40, 64, 0), (5, 1024, 0)])
def test_ties_go_to_the_even_value(dtype, heads, dim, block):
    n = heads * dim
    for shift in (range(0, 64, 9) if block == 0 else (0,)):  # (a row's one scale: other ones in turn)
        w, t, scale = weights(n, block or n)
        if block == 0:
            other = (129 + 2 * shift) / 128
            w, scale = w / scale * other, torch.full_like(scale, other)
            assert torch.equal(w, t * other)
        x = torch.ones((3, heads, dim), dtype=dtype, device="cuda")
        q, s = g.rms_norm_fp8(x, w.reshape(heads, dim), block=block, eps=0.0)
        assert torch.equal(s, scale.expand(3, -1))
        want = t.to(torch.float8_e4m3fn).float()
        got = q.reshape(3, -1).float()
        assert torch.equal(got, want.expand(3, -1)), int((got != want).sum())


@pytest.mark.parametrize("block", [0, 32, 128])
@pytest.mark.parametrize("size", [1.0, 1e-20, 1e-28, 1e30, 3e36])
def test_values_are_the_quotients(size, block):
    """Of weights of all bits and sizes, against divisions and conversions on the CPU."""
    gen = torch.Generator(device="cuda").manual_seed(block)
    for dim in (128, 2048, 16384, 20480):  # (weights beyond FP32 are infinities: NaN and 0 on both sides)
        w = torch.randn(dim, generator=gen, device="cuda") * torch.exp(3 * torch.randn(dim, generator=gen, device="cuda")) * size
        q, s = g.rms_norm_fp8(torch.ones((2, dim), device="cuda"), w, block=block, eps=0.0)
        blocks = w.cpu().numpy().reshape(-1, block or dim)
        # (numpy's FP32 division: torch's on the GPU by a number is a product with its reciprocal)
        with np.errstate(invalid="ignore"):
            scale = np.abs(blocks).max(1) / np.float32(448)
            quotients = blocks / scale[:, None]
        assert torch.equal(s.cpu(), torch.from_numpy(scale).expand(2, -1))
        want = torch.from_numpy(quotients).to(torch.float8_e4m3fn).reshape(-1).view(torch.uint8)
        assert torch.equal(q.view(torch.uint8).cpu(), want.expand(2, -1)), dim


def test_an_infinite_value_in_a_block():
    w = torch.arange(1, 65, device="cuda").float()
    w[40] = float("inf")
    q, s = g.rms_norm_fp8(torch.ones((1, 64), device="cuda"), w, block=32, eps=0.0)
    assert s[0, 0] == 32 / 448 and s[0, 1] == float("inf") and torch.isnan(q.float()[0, 40])
    assert (q.float()[0, :32] != 0).all() and (q.float()[0, 32:40] == 0).all() and (q.float()[0, 41:] == 0).all()
