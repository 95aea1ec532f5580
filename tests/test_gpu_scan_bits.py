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


def test_products_of_fp32_values():
    """B x^T and C S, each (a - 1) b from a b - b, for which six of nine products of three
    terms are formed.  In 2^-24 of a b: left out is at most 2 (a and b of 24 bits that come
    next to that).  A matrix instruction cuts what it adds 2^-24 below its largest operand:
    1 in the one whose operands are b's first term, 2^-7 and less in the other five (their
    operands are a's or b's later terms), and rounds six sums of 2^-7 and less: 3 + 11 2^-7
    in all.  Of C S's two rows it adds one before the other: their sum in between, between
    1 and 2, is cut and rounded once more, 2."""
    step = 2.0**-23
    k = torch.arange(64, device="cuda").double()
    a = (1 + step * (0x7FBF - 0x11 * k)).float()
    b = (1 + step * (0xFFFF - 0x105 * k)).float()
    want = (a.double() - 1)[:, None] * b.double()
    size = 2.0**-24 * a.double()[:, None] * b.double()
    bound = (3 + 11 / 128) * size
    N, P = 64, 64
    x, B = b.expand(2, 1, P).contiguous(), torch.stack([a, -torch.ones_like(a)])[:, None]
    cu, pool = torch.tensor([0, 2], dtype=torch.int32).cuda(), torch.zeros((1, 1, N, P), device="cuda")
    h, A = torch.ones((2, 1), device="cuda"), torch.zeros(1, device="cuda")
    g.scan_prefill(x, h, A, B, torch.zeros_like(B), cu, state_out=pool)
    assert ((pool[0, 0].double() - want).abs() <= bound).all(), float(((pool[0, 0].double() - want) / bound).abs().max())
    S, C = torch.zeros((1, 1, N, P), device="cuda"), torch.zeros((64, 1, N), device="cuda")
    S[0, 0, 3] = S[0, 0, 9] = b
    C[:, 0, 3], C[:, 0, 9] = a, -1
    none = torch.zeros((64, 1, P), device="cuda")
    y = g.scan_prefill(none, torch.zeros((64, 1), device="cuda"), A, torch.zeros_like(C), C, cu * 32, state_in=S)
    assert ((y[:, 0].double() - want).abs() <= bound + 2 * size).all(), float(((y[:, 0].double() - want) / bound).abs().max())
