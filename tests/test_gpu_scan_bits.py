"""What gdn_scan_prefill forms y from is held to FP32, whatever y's type (gpu): sums
that cancel, where an operand cut short would show above y's one rounding.

Tolerance.  y is the sum of two or three values below 2 in size, each the sum of three
BF16 terms: nine additions at most, each off by 2^-24 of a partial sum below 4, so
9 * 2^-22 < 2^-18; and half a step of y's type.
"""
import pytest
import torch

import gateddeltanet_amd as g

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
TYPES = pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
DIMS = pytest.mark.parametrize("N,P", [(64, 64), (128, 64), (256, 64), (64, 128), (128, 128), (256, 256)])
TOL = 2.0**-18


def near(gen, *shape):
    """Values in 1 .. 2 and others within 2^-12 of them, of all 24 bits."""
    u = 1 + torch.rand(shape, generator=gen, device="cuda")
    return u, u + (torch.rand(shape, generator=gen, device="cuda") - 0.5) * 2.0**-11


def close(got, want, what):
    half = 0.0 if got.dtype == FP32 else torch.finfo(got.dtype).eps / 2
    diff = (got.double() - want).abs()
    assert (diff <= half * want.abs() + TOL).all(), (what, float((diff - half * want.abs()).max()))


@TYPES
@DIMS
def test_the_state_in_y(dtype, N, P):
    """Two rows of a state that nearly cancel, read by a C of two ones."""
    lens, heads = [1, 40, 0, 70], 3
    n, gen = sum(lens), torch.Generator(device="cuda").manual_seed(N + P)
    pool = torch.zeros((len(lens), heads, N, P), device="cuda")
    u, v = near(gen, len(lens), heads, P)
    pool[:, :, 5], pool[:, :, N - 3] = u, -v
    x, B = torch.zeros((n, heads, P), dtype=dtype, device="cuda"), torch.zeros((n, 1, N), dtype=dtype, device="cuda")
    C = B.clone()
    C[:, 0, 5] = C[:, 0, N - 3] = 1
    out = g.scan_prefill(x, torch.zeros((n, heads), device="cuda"), -torch.ones(heads, device="cuda"), B, C,
                         torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda(), state_in=pool)
    want = (u.double() - v.double()).repeat_interleave(torch.tensor(lens, device="cuda"), 0)
    close(out, want, "C S")


@TYPES
@DIMS
def test_the_tokens_in_y(dtype, N, P):
    """Two tokens of a sequence that nearly cancel at the second, in one tile, in two, and
    in two chunks, and what D adds there."""
    pairs, heads = [(0, 1), (3, 37), (1, 69), (14, 16), (30, 31)] * 3, 4
    lens = [b + 1 for _, b in pairs]
    ends = torch.tensor([0] + lens).cumsum(0)
    n, gen = int(ends[-1]), torch.Generator(device="cuda").manual_seed(N + P)
    first, second = ends[:-1].cuda() + torch.tensor([a for a, _ in pairs], device="cuda"), ends[1:].cuda() - 1
    h, x = torch.zeros((n, heads), device="cuda"), torch.zeros((n, heads, P), dtype=dtype, device="cuda")
    h[first], h[second] = near(gen, len(pairs), heads)
    x[first], x[second] = 1, -1
    D = 2.0**-12 * torch.rand(heads, generator=gen, device="cuda")
    B = torch.zeros((n, 1, N), dtype=dtype, device="cuda")
    B[:, 0, 9] = 1
    out = g.scan_prefill(x, h, torch.zeros(heads, device="cuda"), B, B, ends.to(torch.int32).cuda(), D=D)
    want = h[first].double() - h[second].double() - D.double()
    close(out[second], want[..., None].expand(-1, -1, P), "M x")
