"""gdn_rms_norm against the norm in 64 bits (gpu).

Tolerances.  h is one rounding of 2^-24 of itself (three with a gate in front, and the
gate's own 8, see SiLU's in test_gpu_conv).  A square goes through five roundings in
its lane's eight values, one for each further vector of the lane (10 at 20000 values) and
eight in a tree: 23 of all its sum, with h's twice 45, so the root is off by 23 2^-24 and
three of its own; h, weight, gate and their products add 22.  REL = 64 2^-24 of the value
covers them.  16 bits add half a step of the type; E4M3 half of a step, 2^-4 of the
value or 2^-10 below its normals, beside the scale's REL.
"""
import pytest
import torch

import gateddeltanet_amd as g

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
TYPES = pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
REL = 64 * 2.0**-24


def reference(x, w, eps=1e-6, residual=None, gate=None, gate_first=False):
    h = x.double() if residual is None else x.double() + residual.double()
    u = h
    if gate is not None:
        s = gate.double() * torch.sigmoid(gate.double())
        u = h * s if gate_first else h
    y = u / (u.square().mean(-1, keepdim=True) + eps).sqrt()
    if w is not None:
        y = y * w.double()
    return (y * s if gate is not None and not gate_first else y), h


def close(got, want, what, rel=REL):
    half = 0.0 if got.dtype == FP32 else torch.finfo(got.dtype).eps / 2
    least = {FP16: 2.0**-25, BF16: 2.0**-130, FP32: 2.0**-130}[got.dtype]
    diff = (got.double() - want).abs()
    assert (diff <= (half + rel) * want.abs() * (1 + 2.0**-20) + least).all(), (
        what, float((diff / want.abs().clamp_min(1e-30)).max()))


def close_fp8(q, scales, want, block, what):
    """Values and scales against y in 64 bits, rows of blocks."""
    rows = want.shape[0]
    y = want.reshape(rows, -1)
    blocks = y.reshape(rows, -1, block or y.shape[1])
    top = blocks.abs().amax(-1)
    s = torch.where(top >= 2.0**-100, top / 448, 1.0)
    assert scales.shape == s.shape and scales.dtype == FP32
    assert ((scales.double() - s).abs() <= (REL + 2.0**-23) * s).all(), what
    v = blocks / s[..., None]
    got = q.float().double().reshape(v.shape)
    assert ((got - v).abs() <= (2.0**-4 + 3 * REL) * v.abs() + 2.0**-10).all(), (what, float((got - v).abs().max()))
    assert got.abs().max() <= 448


def inputs(shape, dtype, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = [torch.randn(shape, generator=gen, device="cuda") for _ in range(3)]
    w = 1 + 0.3 * torch.randn(shape[1:], generator=gen, device="cuda")
    return (1.5 * normal[0]).to(dtype), (4 * normal[1]).to(dtype), (2 * normal[2]).to(dtype), w


DIMS = [1, 2, 7, 8, 9, 63, 64, 65, 128, 200, 256, 257, 512, 513, 1000, 1024, 1500, 2048, 2049, 4096, 5000, 8192, 8193, 12000, 16384, 16385, 20000]


@TYPES
@pytest.mark.parametrize("dim", DIMS)
def test_dims(dtype, dim):
    x, r, gate, w = inputs((5, dim), dtype, dim)
    for gate_first in (False, True):
        out, total = g.rms_norm(x, w, residual=r, gate=gate, gate_first=gate_first, eps=1e-5)
        y, h = reference(x, w, 1e-5, r, gate, gate_first)
        close(out, y, dim)
        close(total, h, dim, 2.0**-24)
        q, s, total = g.rms_norm_fp8(x, w, residual=r, gate=gate, gate_first=gate_first, eps=1e-5)
        close_fp8(q, s, y, 0, dim)
        close(total, h, dim, 2.0**-24)
    close(g.rms_norm(x), reference(x, None)[0], dim)


@pytest.mark.parametrize("rows", [1, 3, 1023, 1024, 1025, 2500])
@pytest.mark.parametrize("dim", [64, 700, 1024, 2048])
def test_rows_either_side_of_a_change_of_layout(rows, dim):
    x, r, _, w = inputs((rows, dim), BF16, rows)
    out, total = g.rms_norm(x, w, residual=r)
    y, h = reference(x, w, residual=r)
    close(out, y, rows)
    close(total, h, rows, 2.0**-24)
    q, s = g.rms_norm_fp8(x, w)
    close_fp8(q, s, reference(x, w)[0], 0, rows)


@TYPES
@pytest.mark.parametrize("heads,dim", [(8, 256), (3, 64), (5, 128), (2, 512), (4, 100), (16, 512), (32, 512), (7, 33), (2, 9000),
                                       (1, 128), (3, 96), (48, 100), (40, 48), (2000, 1), (300, 33), (9, 1000), (3, 2048),
                                       (2, 2049), (64, 200)])
def test_heads(dtype, heads, dim):
    x, r, gate, w = inputs((6, heads, dim), dtype, heads * dim)
    for weight in (w, w[0].contiguous()):
        for gate_first in (False, True):
            out = g.rms_norm(x, weight, gate=gate, gate_first=gate_first)
            y, _ = reference(x, weight, gate=gate, gate_first=gate_first)
            close(out, y, (heads, dim))
            q, s, total = g.rms_norm_fp8(x, weight, gate=gate, gate_first=gate_first, residual=r)
            y, h = reference(x, weight, gate=gate, gate_first=gate_first, residual=r)
            close_fp8(q, s, y, 0, (heads, dim))
            close(total, h, (heads, dim), 2.0**-24)


@pytest.mark.parametrize("heads,dim", [(3, 64), (5, 128), (3, 256), (9, 512), (4, 100)])
def test_rows_of_heads_without_an_eps(heads, dim):
    """Heads that do not fill a layout's lanes: nothing of what is not there."""
    x, r, gate, w = inputs((6, heads, dim), FP32, heads * dim)
    q, s = g.rms_norm_fp8(x, w, gate=gate, eps=0.0)
    y, _ = reference(x, w, gate=gate, eps=0.0)
    close_fp8(q, s, y, 0, (heads, dim))


@TYPES
@pytest.mark.parametrize("block", [32, 64, 128])
@pytest.mark.parametrize("shape", [(3, 128), (70, 2048), (4, 384), (5, 8, 256), (2, 3, 8320), (1100, 1024), (9, 6400)])
def test_blocks(dtype, block, shape):
    x, r, gate, w = inputs(shape, dtype, block)
    q, s, total = g.rms_norm_fp8(x, w, block=block, residual=r, gate=gate)
    y, h = reference(x, w, residual=r, gate=gate)
    close_fp8(q, s, y, block, shape)
    close(total, h, shape, 2.0**-24)


@TYPES
def test_strided_and_misaligned_rows(dtype):
    wide = [torch.randn((40, 1031), device="cuda").to(dtype) for _ in range(3)]
    x, r, gate = wide[0][:, 3:703], wide[1][:, 11:711], wide[2][:, 300:1000]
    w = torch.rand(701, device="cuda")[1:]
    room, sums = torch.full((40, 900), 5.0, dtype=dtype, device="cuda"), torch.full((40, 701), 5.0, dtype=dtype, device="cuda")
    g.rms_norm(x, w, residual=r, gate=gate, out=room[:, 100:800], sum_out=sums[:, 1:])
    y, h = reference(x, w, residual=r, gate=gate)
    close(room[:, 100:800], y, "out")
    close(sums[:, 1:], h, "sum", 2.0**-24)
    assert (room[:, :100] == 5).all() and (room[:, 800:] == 5).all() and (sums[:, 0] == 5).all()
    bytes_ = torch.zeros((40, 900), dtype=torch.float8_e4m3fn, device="cuda")
    q, s = g.rms_norm_fp8(x, w, gate=gate, out=bytes_[:, 7:707])
    close_fp8(bytes_[:, 7:707].contiguous(), s, reference(x, w, gate=gate)[0], 0, "fp8")
    assert (bytes_[:, :7].float() == 0).all() and (bytes_[:, 707:].float() == 0).all()


@TYPES
@pytest.mark.parametrize("dim", [100, 2048, 9000])
def test_in_place(dtype, dim):
    x, r, gate, w = inputs((7, dim), dtype, dim)
    want, total = g.rms_norm(x, w, residual=r, gate=gate)
    for out_at, sum_at in (("x", "r"), ("r", "x"), ("gate", "r"), ("x", None), (None, "r"), ("gate", "x")):
        y = {"x": x.clone(), "r": r.clone(), "gate": gate.clone(), None: None}
        a, b = g.rms_norm(y["x"], w, residual=y["r"], gate=y["gate"], out=y[out_at], sum_out=y[sum_at])
        assert torch.equal(a, want) and torch.equal(b, total), (out_at, sum_at)
    q, s, _ = g.rms_norm_fp8(x, w, residual=r)
    y = r.clone()
    q2, s2, t2 = g.rms_norm_fp8(x, w, residual=y, sum_out=y)
    assert t2 is y and torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s, s2)


def test_overlaps_are_refused():
    x, r, gate, w = inputs((4, 64), BF16)
    for kw in (dict(out=x, sum_out=x), dict(sum_out=gate, gate=gate), dict(out=r, sum_out=r)):
        with pytest.raises(g.GDNError):
            g.rms_norm(x, w, residual=r, **kw)
    room = torch.zeros((5, 64), dtype=BF16, device="cuda")
    with pytest.raises(g.GDNError):
        g.rms_norm(room[:4], w, out=room[1:])
    with pytest.raises(g.GDNError):
        g.rms_norm_fp8(room[:4], w, out=room.view(torch.float8_e4m3fn)[:4, :64])


def test_extremes():
    """Rows of zeros, of a type's largest and smallest values, tiny ones."""
    x = torch.zeros((6, 300), device="cuda")
    x[1] = 3e38
    x[2] = 1e-30
    x[3, 5] = 1e-38
    x[4] = 1e18
    x[5, 0] = 1.0
    out = g.rms_norm(x)
    assert (out[0] == 0).all() and (out[1] == 0).all()  # (squares beyond FP32's range)
    close(out[2:], reference(x[2:], None)[0], "small, large")
    q, s = g.rms_norm_fp8(x)
    assert s[0] == 1 and (q[0].float() == 0).all()
    close_fp8(q[2:], s[2:], reference(x[2:], None)[0], 0, "small, large")
    y = x.clone()
    y[2, 3], y[4, 7] = float("nan"), float("inf")
    out = g.rms_norm(y)
    assert torch.isnan(out[2]).all() and torch.equal(out[[0, 1, 3, 5]], g.rms_norm(x)[[0, 1, 3, 5]])
    q, s = g.rms_norm_fp8(y)
    assert torch.isnan(s[2]) and torch.isnan(q[2].float()).all()
    assert torch.isnan(q[4, 7].float()) and not torch.isfinite(s[4]).any()
    q2, s2 = g.rms_norm_fp8(x)
    keep = [0, 1, 3, 5]
    assert torch.equal(q[keep].view(torch.uint8), q2[keep].view(torch.uint8)) and torch.equal(s[keep], s2[keep])


def test_scale_takes_the_largest_value_to_448():
    x = torch.randn((50, 256), device="cuda")
    q, s = g.rms_norm_fp8(x, block=64)
    assert (q.float().abs().reshape(50, 4, 64).amax(-1) == 448).all()


@pytest.mark.parametrize("dim", [256, 2048, 10000])
def test_captured_and_replayed(dim):
    x, r, gate, w = inputs((30, dim), BF16)
    out, total = torch.empty_like(x), torch.empty_like(x)
    q, s = torch.empty_like(x, dtype=torch.float8_e4m3fn), torch.empty((30, 1), device="cuda")

    def work():
        g.rms_norm(x, w, residual=r, gate=gate, out=out, sum_out=total)
        g.rms_norm_fp8(total, w, out=q, scales=s)

    work()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        work()
    for seed in range(3):
        y, _, _, _ = inputs((30, dim), BF16, 9 + seed)
        x.copy_(y)
        work()
        want = [t.clone() for t in (out, total, q.view(torch.uint8), s)]
        for t in (out, total, s):
            t.fill_(9.0)
        q.view(torch.uint8).fill_(1)
        torch.cuda.synchronize()
        graph.replay()
        for t, u in zip((out, total, q.view(torch.uint8), s), want):
            assert torch.equal(t, u)


def test_two_streams_at_once():
    x, r, gate, w = inputs((500, 2048), BF16)
    want = g.rms_norm(x, w, gate=gate)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for st in streams:
            with torch.cuda.stream(st):
                got.append(g.rms_norm(x, w, gate=gate))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in got)


def test_offsets_beyond_32_bits():
    x = torch.zeros((300_000, 8192), dtype=BF16, device="cuda")
    x[-3:] = torch.randn((3, 8192), device="cuda").to(BF16)
    out = g.rms_norm(x)
    close(out[-3:], reference(x[-3:], None)[0], "last rows")
    q, s = g.rms_norm_fp8(x, block=128)
    close_fp8(q[-3:], s[-3:], reference(x[-3:], None)[0], 128, "last rows")


def test_many_short_heads():
    x, _, gate, w = inputs((1_200_000, 16, 8), BF16)
    out = g.rms_norm(x, w[0].contiguous(), gate=gate)
    for s in (slice(0, 3), slice(599_999, 600_002), slice(1_199_997, 1_200_000)):
        close(out[s], reference(x[s], w[0], gate=gate[s])[0], s)


def test_refusals_of_tensors():
    x, r, gate, w = inputs((4, 2, 64), BF16)
    for bad in (dict(x=x.double()), dict(x=x.cpu()), dict(x=x[0, 0]), dict(x=x[:, :, ::2]), dict(x=x.transpose(0, 1)),
                dict(weight=w.to(BF16)), dict(weight=w[:, :3]), dict(weight=w[0, :5]), dict(residual=r.float()),
                dict(gate=gate[:3]), dict(gate_first=True), dict(sum_out=r), dict(out=r.float()), dict(eps=-1.0),
                dict(eps=float("nan")), dict(residual=r, sum_out=r[:, :1])):
        call = {"x": x, "weight": w, **bad}
        with pytest.raises(g.GDNError):
            g.rms_norm(call.pop("x"), call.pop("weight"), **call)
    for bad in (dict(block=16), dict(block=128), dict(block=-1), dict(scales=torch.empty((4, 2), device="cuda")),
                dict(out=torch.empty_like(x)), dict(x=torch.zeros((), device="cuda"))):
        call = {"x": x, **bad}
        with pytest.raises(g.GDNError):
            g.rms_norm_fp8(call.pop("x"), **call)
    with pytest.raises(g.GDNError):
        g.rms_norm(x, w.clone().requires_grad_())
    with torch.no_grad():
        g.rms_norm(x, w.clone().requires_grad_())


def test_writes_count_as_modifications():
    x, r, _, w = inputs((4, 64), BF16)
    out, before = torch.empty_like(x), r._version
    version = out._version
    g.rms_norm(x, w, residual=r, out=out, sum_out=r)
    assert out._version > version and r._version > before


def test_nothing_to_do():
    none = torch.zeros((0, 64), dtype=BF16, device="cuda")
    assert g.rms_norm(none).shape == (0, 64)
    q, s = g.rms_norm_fp8(none, block=32)
    assert q.shape == (0, 64) and s.shape[0] == 0


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("dim", [100, 2048, 20000])
def test_tiny_heads_with_and_without_an_eps(dtype, dim):
    """As the header says: FP32's squares hold heads of 2^-63 and more, or any with an eps
    of 2^-126; with less, infinities and NaN."""
    x, _, _, w = inputs((4, dim), FP32, dim)
    x = x.sign() * x.abs().clamp(0.25, 4)
    y = (x * 2.0**-61).to(dtype)
    close(g.rms_norm(y, w, eps=0.0), reference(y, w, 0.0)[0], "2^-63 and more")
    for size in (2.0**-64, 2.0**-70, 2.0**-90):
        y = (x * size).to(dtype)
        close(g.rms_norm(y, w, eps=2.0**-126), reference(y, w, 2.0**-126)[0], size)
    y[:, 3] = 0
    out = g.rms_norm(y, w, eps=0.0)
    assert torch.isnan(out[:, 3]).all() and torch.isinf(out[:, 4:]).all()
    q, s = g.rms_norm_fp8(y, w, eps=0.0)
    assert not torch.isfinite(s).any()


def test_scales_of_tiny_blocks():
    """1 for a block whose largest value is below 2^-100, the value over 448 from there up."""
    w = torch.ones(96, device="cuda")
    w[:32] *= 2.0**-100
    w[32:64] *= torch.nextafter(torch.tensor(2.0**-100), torch.tensor(0.0)).item()
    q, s = g.rms_norm_fp8(torch.ones((1, 96), device="cuda"), w, block=32, eps=0.0)
    assert s[0].tolist() == [torch.tensor(2.0**-100).div(torch.tensor(448.0)).item(), 1.0, torch.tensor(1.0).div(torch.tensor(448.0)).item()]
    assert (q[0, :32].float() == 448).all() and (q[0, 32:64].float() == 0).all() and (q[0, 64:].float() == 448).all()
