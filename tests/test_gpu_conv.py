"""gdn_conv_prefill and gdn_conv_step against the convolution in 64 bits (gpu).

Tolerances.  A window's sum has at most width products and the bias, width + 1
roundings of 2^-24 of what has been added up, so (width + 2) 2^-24 of the sum of
magnitudes; SiLU's slope is at most 1.1.  SiLU itself: the exponential to 2^-23 and
2^-26, its reciprocal to 2^-23, two more roundings, 6.6 2^-24 in all, taken as 8; below
-88 it is 0 for less than 2^-118.  An output of 16 bits adds half a step of its type.
Tails are copies.
"""
import pytest
import torch

import gateddeltanet_amd as g

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
TYPES = pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])


def inputs(n, channels, width, dtype, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*s):
        return torch.randn(s, generator=gen, device="cuda")

    return (2 * normal(n, channels)).to(dtype), normal(channels, width), normal(channels)


def reference(x, w, bias, tail, silu):
    """(y, its tolerance but the rounding, tail') of one sequence, in 64 bits."""
    width = w.shape[1]
    z = torch.cat([tail, x]).double()
    n = x.shape[0]
    y = sum(z[j:j + n] * w[:, j].double() for j in range(width))
    size = sum((z[j:j + n] * w[:, j].double()).abs() for j in range(width))
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    tol = (width + 2) * 2.0**-24 * size
    if silu:
        y = y * torch.sigmoid(y)
        tol = 1.1 * tol + 8 * 2.0**-24 * y.abs() + 2.0**-118
    return y, tol, torch.cat([tail, x])[n:]


def close(got, want, tol, what):
    half = 0.0 if got.dtype == FP32 else torch.finfo(got.dtype).eps / 2
    least = 2.0**-25 if got.dtype == FP16 else 0.0  # half a step of its subnormals
    diff = (got.double() - want).abs()
    assert (diff <= half * want.abs() + least + 1.01 * tol).all(), (what, float((diff - half * want.abs() - tol).max()))


def cumulative(lens, start=0):
    return torch.tensor([start] + lens).cumsum(0).to(torch.int32).cuda()


def check_packed(lens, channels, width, dtype, start=True, silu=True, bias=True, first=0, behind=0, seed=0, shuffle=True,
                 in_place=True, x=None):
    n = first + sum(lens) + behind
    made, w, b = inputs(n, channels, width, dtype, seed)
    x = made if x is None else x
    b = b if bias else None
    cu = cumulative(lens, first)
    n_slots = len(lens) + 2
    where = torch.randperm(n_slots, generator=torch.Generator().manual_seed(seed))[:len(lens)].tolist() if shuffle else list(
        range(len(lens)))
    tails = torch.randn((n_slots, width - 1, channels), device="cuda").to(dtype)
    pool = tails.clone()
    into = pool if in_place else torch.full_like(pool, 7.0)
    before = into.clone()
    out = torch.full((n, channels), 5.0, dtype=dtype, device="cuda")
    got = g.conv_prefill(x, w, cu, bias=b, silu=silu, state_in=pool if start else None, state_out=into,
                         slots=torch.tensor(where, dtype=torch.int32).cuda() if shuffle else None, out=out)
    assert got is out
    at = first
    for i, m in enumerate(lens):
        tail = tails[where[i]] if start else torch.zeros_like(tails[0])
        y, tol, end = reference(x[at:at + m], w, b, tail, silu)
        close(out[at:at + m], y, tol, f"sequence {i} of {m} tokens")
        assert torch.equal(into[where[i]], end), f"tail of sequence {i}, {m} tokens"
        at += m
    assert (out[:first] == 5).all() and (out[at:] == 5).all()
    rest = [i for i in range(n_slots) if i not in where]
    assert torch.equal(into[rest], before[rest])
    return out, into


LENS = [0, 1, 2, 3, 4, 5, 0, 31, 32, 33, 70, 1, 1, 0]


@TYPES
@pytest.mark.parametrize("width", [2, 3, 4])
@pytest.mark.parametrize("channels", [1, 7, 8, 64, 2048, 2051])
def test_prefill(dtype, width, channels):
    check_packed(LENS, channels, width, dtype, seed=channels + width)


@TYPES
@pytest.mark.parametrize("start,silu,bias,in_place", [(False, True, False, True), (True, False, True, False),
                                                      (False, False, False, False), (True, True, False, False)])
def test_prefill_options(dtype, start, silu, bias, in_place):
    check_packed(LENS, 96, 4, dtype, start, silu, bias, in_place=in_place, seed=3)


@pytest.mark.parametrize("lens", [[1], [3], [4], [1000], [0], [0, 0], [1] * 200, [2] * 33 + [400] + [0] * 70, []])
def test_prefill_lengths(lens):
    check_packed(lens, 264, 4, BF16, shuffle=False, seed=len(lens))


def test_rows_before_and_behind_the_sequences_are_left():
    check_packed([40, 0, 3], 128, 4, BF16, first=37, behind=50, seed=8)
    check_packed([1, 300], 128, 3, FP32, first=200, behind=200, seed=9)


@TYPES
def test_strided_and_misaligned_rows(dtype):
    """Columns of a fused projection, at an odd element."""
    n, channels = sum(LENS), 77
    wide = torch.randn((n, 301), device="cuda").to(dtype)
    check_packed(LENS, channels, 4, dtype, seed=4, x=wide[:, 13:13 + channels])


def test_sequences_without_a_slot_are_left_out():
    x, w, b = inputs(30, 64, 4, BF16)
    pool = torch.randn((2, 3, 64), device="cuda").to(BF16)
    before = pool.clone()
    out = torch.full_like(x, 5.0)
    g.conv_prefill(x, w, cumulative([10, 10, 10]), bias=b, state_in=pool, state_out=pool, out=out,
                   slots=torch.tensor([-1, 1, 2], dtype=torch.int32).cuda())
    assert (out[:10] == 5).all() and (out[20:] == 5).all() and torch.equal(pool[0], before[0])
    y, tol, end = reference(x[10:20], w, b, before[1], True)
    close(out[10:20], y, tol, "the one with a slot")
    assert torch.equal(pool[1], end)


@TYPES
@pytest.mark.parametrize("channels", [1, 8, 100, 6144])
def test_step(dtype, channels):
    n, slots = 9, 12
    x, w, b = inputs(n, channels, 4, dtype, channels)
    tails = torch.randn((slots, 3, channels), device="cuda").to(dtype)
    where = [3, -1, 0, 11, 12, 5, 7, -5, 1]
    for in_place in (True, False):
        pool, out = tails.clone(), torch.full_like(x, 5.0)
        into = pool if in_place else tails.clone()
        g.conv_step(x, w, pool, bias=b, slots=torch.tensor(where, dtype=torch.int32).cuda(), out=out,
                    state_out=None if in_place else into)
        for i, s in enumerate(where):
            if 0 <= s < slots:
                y, tol, end = reference(x[i:i + 1], w, b, tails[s], True)
                close(out[i:i + 1], y, tol, i)
                assert torch.equal(into[s], end)
            else:
                assert (out[i] == 5).all()
        rest = [s for s in range(slots) if s not in where]
        assert torch.equal(into[rest], tails[rest])


@pytest.mark.parametrize("width", [2, 3, 4])
def test_steps_follow_a_prefill(width):
    """A prompt at once, in two parts and token by token: the same bits."""
    x, w, b = inputs(40, 136, width, FP32, width)
    tail = torch.zeros((1, width - 1, 136), device="cuda")
    whole = g.conv_prefill(x, w, cumulative([40]), bias=b, state_out=tail)
    pool = torch.zeros_like(tail)
    one = g.conv_prefill(x[:17], w, cumulative([17]), bias=b, state_out=pool)
    two = g.conv_prefill(x[17:38], w, cumulative([21]), bias=b, state_in=pool, state_out=pool)
    rest = [g.conv_step(x[i:i + 1], w, pool, bias=b) for i in (38, 39)]
    assert torch.equal(torch.cat([one, two] + rest), whole) and torch.equal(pool, tail)


def test_step_over_its_input():
    x, w, b = inputs(5, 200, 4, BF16)
    tails = torch.randn((5, 3, 200), device="cuda").to(BF16)
    a, c = tails.clone(), tails.clone()
    want = g.conv_step(x, w, a, bias=b)
    y = x.clone()
    assert g.conv_step(y, w, c, bias=b, out=y) is y
    assert torch.equal(y, want) and torch.equal(a, c)
    with pytest.raises(g.GDNError):
        g.conv_step(y, w, c, bias=b, out=y[:, :].as_strided((5, 200), (199, 1)))


def test_values_that_are_not_finite_stay_with_their_window():
    x, w, b = inputs(60, 32, 4, FP32)
    clean = g.conv_prefill(x, w, cumulative([30, 30]), bias=b)
    y = x.clone()
    y[29, 3], y[5, 7], y[40, 9] = float("nan"), float("inf"), -float("inf")
    out = g.conv_prefill(y, w, cumulative([30, 30]), bias=b)
    touched = torch.zeros_like(x, dtype=torch.bool)
    touched[29, 3] = touched[5:9, 7] = touched[40:44, 9] = True
    assert torch.equal(out[~touched], clean[~touched])
    assert torch.isnan(out[29, 3])
    big = torch.full((4, 8), 200.0, device="cuda")
    ones = torch.tensor([0.0, 0.0, 0.0, 1.0], device="cuda").repeat(8, 1)
    assert torch.equal(g.conv_prefill(big, ones, cumulative([4])), big)
    assert (g.conv_prefill(-big, ones, cumulative([4])).abs() == 0).all()


@pytest.mark.parametrize("ends", [[0, 30, 10, 50], [20, 10, 5, 0], [-5, 10, 200, 300], [50, 50, 0, 50], [60, 70, 80, 90]])
def test_ends_that_fall_or_pass_the_rows_write_nothing_else(ends):
    room = torch.full((50 + 64, 72), 5.0, device="cuda")
    x, w, b = inputs(50, 72, 4, FP32)
    pool = torch.full((5 + 4, 3, 72), 3.0, device="cuda")
    g.conv_prefill(x, w, torch.tensor(ends, dtype=torch.int32).cuda(), bias=b, state_in=pool[2:7], state_out=pool[2:7],
                   slots=torch.tensor([0, 2, 4], dtype=torch.int32).cuda(), out=room[32:82])
    assert (room[:32] == 5).all() and (room[82:] == 5).all()
    assert (pool[[0, 1, 3, 5, 7, 8]] == 3).all()


def test_captured_and_replayed():
    x, w, b = inputs(90, 512, 4, BF16)
    cu, pool = cumulative([50, 0, 40]), torch.zeros((3, 3, 512), dtype=BF16, device="cuda")
    token, out = torch.zeros((3, 512), dtype=BF16, device="cuda"), torch.zeros((90, 512), dtype=BF16, device="cuda")
    after = torch.zeros_like(token)

    def work():
        g.conv_prefill(x, w, cu, bias=b, state_out=pool, out=out)
        g.conv_step(token, w, pool, bias=b, out=after)

    work()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        work()
    for seed in range(4):
        y, _, _ = inputs(93, 512, 4, BF16, 50 + seed)
        x.copy_(y[:90])
        token.copy_(y[90:])
        work()
        want = [t.clone() for t in (out, pool, after)]
        for t in (out, pool, after):
            t.fill_(9.0)
        torch.cuda.synchronize()
        graph.replay()
        for t, u in zip((out, pool, after), want):
            assert torch.equal(t, u)


def test_replayed_with_other_sequences():
    """A graph of the most rows and sequences, replayed with other ends and slots: padded
    sequences are empty or have a slot of -1, rows behind the last are left."""
    n, channels, width = 150, 264, 4
    x, w, b = inputs(n, channels, width, FP32)
    cu, slots = torch.zeros(6, dtype=torch.int32, device="cuda"), torch.zeros(5, dtype=torch.int32, device="cuda")
    pool, out = torch.zeros((7, width - 1, channels), device="cuda"), torch.zeros_like(x)
    g.conv_prefill(x, w, cu, bias=b, state_in=pool, state_out=pool, slots=slots, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g.conv_prefill(x, w, cu, bias=b, state_in=pool, state_out=pool, slots=slots, out=out)
    first = torch.randn(pool.shape, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    for lens, where in [([150, 0, 0, 0, 0], [3, -1, -1, -1, -1]), ([1, 70, 0, 30, 2], [0, 6, 1, 2, 5]),
                        ([0, 0, 0, 0, 0], [4, 3, 2, 1, 0]), ([17, 15, 60, 16, 3], [6, 5, 4, 3, 7])]:
        cu.copy_(cumulative(lens))
        slots.copy_(torch.tensor(where, dtype=torch.int32))
        pool.copy_(first)
        out.fill_(5.0)
        torch.cuda.synchronize()
        graph.replay()
        at, used = 0, []
        for m, slot in zip(lens, where):
            part = slice(at, at + m)
            at += m
            if not 0 <= slot < 7:
                assert (out[part] == 5).all()
                continue
            used.append(slot)
            y, tol, end = reference(x[part], w, b, first[slot], True)
            close(out[part], y, tol, f"{m} tokens")
            assert torch.equal(pool[slot], end), m
        rest = [i for i in range(7) if i not in used]
        assert (out[at:] == 5).all() and torch.equal(pool[rest], first[rest])


def test_on_a_stream_of_its_own():
    x, w, b = inputs(64, 2048, 4, BF16)
    want = g.conv_prefill(x, w, cumulative([64]), bias=b)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        y = x * 1.0
        torch.cuda._sleep(5_000_000)
        y.copy_(x)
        out = g.conv_prefill(y, w, cumulative([64]), bias=b)
    stream.synchronize()
    assert torch.equal(out, want)


def test_offsets_beyond_32_bits():
    """Rows and tails that start past 2^32 bytes."""
    channels, n = 8192, 300_000
    x = torch.empty((n, channels), dtype=BF16, device="cuda")
    x[-2000:] = torch.randn((2000, channels), device="cuda").to(BF16)
    _, w, b = inputs(1, channels, 4, BF16)
    out = torch.empty_like(x)
    pool = torch.zeros((100_000, 3, channels), dtype=BF16, device="cuda")
    cu, slots = torch.tensor([n - 1500, n - 700, n], dtype=torch.int32).cuda(), torch.tensor([99_999, 99_000], dtype=torch.int32).cuda()
    g.conv_prefill(x, w, cu, bias=b, state_in=pool, state_out=pool, slots=slots, out=out)
    zero = torch.zeros((3, channels), dtype=BF16, device="cuda")
    for a, e, s in ((n - 1500, n - 700, 99_999), (n - 700, n, 99_000)):
        y, tol, end = reference(x[a:e], w, b, zero, True)
        close(out[a:e], y, tol, s)
        assert torch.equal(pool[s], end)


def test_refusals_of_tensors():
    x, w, b = inputs(8, 16, 4, BF16)
    cu, pool = cumulative([8]), torch.zeros((1, 3, 16), dtype=BF16, device="cuda")
    good = dict(bias=b, state_in=pool, state_out=pool)
    g.conv_prefill(x, w, cu, **good)
    for bad in (dict(weight=w.to(BF16)), dict(weight=w[:, :3].contiguous()), dict(weight=w[:8]), dict(x=x.double()),
                dict(x=x[:, ::2]), dict(x=x.cpu()), dict(cu=cu.long()), dict(cu=cu.cpu()), dict(bias=b[:3]),
                dict(state_in=pool.float()), dict(state_out=pool[:, :2]), dict(out=x), dict(out=x[:, :8]),
                dict(slots=cu[:1].long()), dict(x=x[0]), dict(cu=torch.zeros((0,), dtype=torch.int32, device="cuda")),
                dict(cu=cumulative([4, 4]))):
        call = {"x": x, "weight": w, "cu": cu, **good, **bad}
        with pytest.raises(g.GDNError):
            g.conv_prefill(call.pop("x"), call.pop("weight"), call.pop("cu"), **call)
    with pytest.raises(g.GDNError):
        g.conv_step(x[:1], w.clone().requires_grad_(), pool)
    with pytest.raises(g.GDNError):
        g.conv_step(x, w, pool)  # eight tokens, one tail
    with torch.no_grad():
        g.conv_step(x[:1], w.clone().requires_grad_(), pool)


def test_writes_count_as_modifications():
    x, w, b = inputs(8, 16, 4, BF16)
    pool, out = torch.zeros((8, 3, 16), dtype=BF16, device="cuda"), torch.empty_like(x)
    versions = out._version, pool._version
    g.conv_step(x, w, pool, out=out)
    assert out._version > versions[0] and pool._version > versions[1]
    versions = out._version, pool._version
    g.conv_prefill(x, w, cumulative([8]), state_out=pool, out=out)
    assert out._version > versions[0] and pool._version > versions[1]


def test_nothing_to_do():
    _, w, b = inputs(1, 16, 4, BF16)
    none = torch.zeros((0, 16), dtype=BF16, device="cuda")
    assert g.conv_prefill(none, w, cumulative([])).shape == (0, 16)
    assert g.conv_step(none, w, torch.zeros((3, 3, 16), dtype=BF16, device="cuda")).shape == (0, 16)
    pool = torch.randn((2, 3, 16), device="cuda").to(BF16)
    into = torch.zeros_like(pool)
    g.conv_prefill(none, w, cumulative([0, 0]), state_in=pool, state_out=into)
    assert torch.equal(into, pool)


def test_one_row_over_its_input_whatever_its_strides():
    """A single row's stride is not looked at, in place neither."""
    x, w, b = inputs(1, 200, 4, BF16)
    pool = torch.randn((1, 3, 200), device="cuda").to(BF16)
    a, c = pool.clone(), pool.clone()
    want = g.conv_step(x, w, a, bias=b)
    y = x.clone()
    g.conv_step(y.as_strided((1, 200), (999, 1)), w, c, bias=b, out=y)
    assert torch.equal(y, want) and torch.equal(a, c)
    y = x.clone()
    with pytest.raises(g.GDNError):  # a row of its own, but not the same one
        g.conv_step(y[:, 1:], w[1:].contiguous(), torch.zeros((1, 3, 199), dtype=BF16, device="cuda"), out=y[:, :199])


@TYPES
@pytest.mark.parametrize("width", [2, 3])
@pytest.mark.parametrize("channels", [5, 136, 2051])
def test_step_of_every_width(dtype, width, channels):
    n, slots, where = 5, 6, [4, 0, -1, 5, 2]
    x, w, b = inputs(n, channels, width, dtype, channels + width)
    tails = torch.randn((slots, width - 1, channels), device="cuda").to(dtype)
    for bias, silu, start in ((b, True, True), (None, False, True), (b, True, False)):
        pool, out = tails.clone(), torch.full_like(x, 5.0)
        into = pool if start else None
        g.conv_step(x, w, into, bias=bias, silu=silu, slots=torch.tensor(where, dtype=torch.int32).cuda(), out=out)
        for i, s in enumerate(where):
            if s < 0 or (not start and s >= n):  # (without tails there are as many slots as sequences)
                assert (out[i] == 5).all()
                continue
            y, tol, end = reference(x[i:i + 1], w, bias, tails[s] if start else torch.zeros_like(tails[s]), silu)
            close(out[i:i + 1], y, tol, i)
            assert torch.equal(pool[s], end if start else tails[s])
        rest = [s for s in range(slots) if s not in where]
        assert torch.equal(pool[rest], tails[rest])
