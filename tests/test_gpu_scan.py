"""gdn_scan_prefill and gdn_scan_step against the scan token by token in 64 bits (gpu).

Tolerances.  A token's y is two chained sums (S^T C, the chunk's products), a state's
update one, each of at most state_dim + 64 products rounded to FP32; n roundings of
2^-24 in no order add up to sqrt(n) 2^-24 of a sum's size.  A step carries four
roundings of its own, and with them a decay exp(G) |G| exp(G) 4 2^-24, at most 1.5 2^-24 of
what it decays.  Relative to the norm of a sequence's whole result that is
TOL = 4 sqrt(state_dim + 64) 2^-24 (4.3e-6 at 256).  A y of 16 bits is formed from
operands of two BF16 terms, off by 2^-16 at most and by 2^-16 / sqrt(12) in the mean, one in
each of its two sums: taken as 2^-16 of the root mean square; and half a step of the
type, eps / 2 of the value.  LEAST: what FP32
has no normal number for, below 2^-126 a product, of up to 2^16 products of factors
below 2^6 (a step of 200 below zero is e^-200).
"""
import math

import pytest
import torch

import gateddeltanet_amd as g

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
TYPES = pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])


LEAST = 2.0**-126 * 2**16 * 2**6


def tol(N):
    return 4 * math.sqrt(N + 64) * 2.0**-24


def inputs(n, heads, groups, N, P, dtype, seed=0, dt_dtype=None):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*s):
        return torch.randn(s, generator=gen, device="cuda")

    def uniform(lo, hi, *s):
        return lo + (hi - lo) * torch.rand(s, generator=gen, device="cuda")

    x, B, C = normal(n, heads, P), normal(n, groups, N) / 4, normal(n, groups, N) / 4
    return {"x": x.to(dtype), "dt": (2 * normal(n, heads)).to(dt_dtype or dtype), "A": -uniform(0.2, 16, heads),
            "B": B.to(dtype), "C": C.to(dtype), "D": normal(heads), "dt_bias": uniform(-6, -2, heads)}


def rows(a, s):
    return {k: v[s] if k in ("x", "dt", "B", "C") else v for k, v in a.items()}


def call(op, a, *rest, **kw):
    """op with the arguments of inputs() (those not there: not given)."""
    more = {k: a[k] for k in ("D", "dt_bias") if k in a}
    return op(a["x"], a["dt"], a["A"], a["B"], a["C"], *rest, **{"softplus": True, **more, **kw})


def reference(a, S, softplus=True):
    """(y, S') of one sequence, in 64 bits."""
    x = a["x"].double()
    n, heads, _ = x.shape
    group = heads // a["B"].shape[1]
    B, C = (a[k].double().repeat_interleave(group, 1) for k in ("B", "C"))
    h = a["dt"].double() + (a["dt_bias"].double() if "dt_bias" in a else 0.0)
    if softplus:
        h = torch.where(h > 500, h, torch.log1p(torch.exp(h)))
    decay = torch.exp(h * a["A"].double())
    y = a["D"].double()[:, None] * x if "D" in a else torch.zeros_like(x)
    S = S.double().clone()
    for t in range(n):
        S = S * decay[t, :, None, None] + (h[t, :, None] * B[t])[..., None] * x[t, :, None, :]
        y[t] += (S * C[t, :, :, None]).sum(1)
    return y, S


def close(got, want, t, what):
    """Elementwise, and for FP32 by the norm too (per value: of the root mean
    square, times 8 for the largest of many)."""
    assert torch.isfinite(got).all(), what
    if want.numel() == 0:
        return
    diff, rms = (got.double() - want).abs(), want.square().mean().sqrt()
    half = 0.0
    if got.dtype != FP32:
        half, t = torch.finfo(got.dtype).eps / 2, t + 2.0**-16
    assert (diff <= half * want.abs() + 8 * t * torch.maximum(want.abs(), rms.expand_as(want)) + LEAST).all(), (
        what, float((diff - half * want.abs()).max()), float(rms))
    if half == 0.0:
        assert diff.square().mean().sqrt() <= t * rms + LEAST, (what, float(diff.square().mean().sqrt() / rms))


def cumulative(lens, start=0):
    return torch.tensor([start] + lens).cumsum(0).to(torch.int32).cuda()


def check_packed(lens, heads, groups, N, P, dtype, start=True, seed=0, shuffle=False, first=0, behind=0, a=None, **kw):
    n = first + sum(lens) + behind
    a = inputs(n, heads, groups, N, P, dtype, seed) if a is None else a
    n_slots = len(lens) + (3 if shuffle else 0)
    where = list(range(len(lens)))
    slots = None
    if shuffle:
        where = torch.randperm(n_slots, generator=torch.Generator().manual_seed(seed))[:len(lens)].tolist()
        slots = torch.tensor(where, dtype=torch.int32).cuda()
    gen = torch.Generator(device="cuda").manual_seed(seed + 1)
    S0 = 0.3 * torch.randn((n_slots, heads, N, P), generator=gen, device="cuda")
    pool = S0.clone()
    out = torch.full((n, heads, P), 5.0, dtype=dtype, device="cuda")
    call(g.scan_prefill, a, cumulative(lens, first), state_in=pool if start else None, state_out=pool, slots=slots, out=out, **kw)
    at = first
    for i, m in enumerate(lens):
        init = S0[where[i]] if start else torch.zeros_like(S0[0])
        y, S = reference(rows(a, slice(at, at + m)), init, kw.get("softplus", True))
        close(out[at:at + m], y, tol(N), f"y of sequence {i}, {m} tokens")
        close(pool[where[i]], S, tol(N), f"state of sequence {i}, {m} tokens")
        at += m
    rest = [i for i in range(n_slots) if i not in where]
    assert torch.equal(pool[rest], S0[rest])
    assert (out[:first] == 5).all() and (out[at:] == 5).all()
    return a, out, pool


LENS = [0, 1, 31, 32, 33, 63, 64, 65, 0, 130, 16, 17]


@TYPES
@pytest.mark.parametrize("N,P,heads,groups", [(128, 64, 4, 1), (64, 64, 2, 2), (128, 128, 3, 3), (64, 128, 4, 2),
                                              (256, 64, 2, 1), (256, 256, 1, 1), (64, 256, 2, 2), (128, 256, 1, 1)])
def test_prefill(dtype, N, P, heads, groups):
    check_packed(LENS, heads, groups, N, P, dtype, shuffle=True, seed=N + P)


@pytest.mark.parametrize("lens", [[1], [2], [15], [64], [65], [128], [129], [1] * 9, [0], [0, 0, 7, 0], []])
def test_prefill_lengths_from_zero_state(lens):
    check_packed(lens, 2, 1, 128, 64, BF16, start=False, seed=len(lens) + sum(lens))


@TYPES
@pytest.mark.parametrize("N,P,lens", [(64, 64, [1500]), (128, 64, [700, 0, 257, 256, 1, 255, 513, 3]), (256, 128, [1100, 600])])
def test_prefill_of_sequences_in_segments(dtype, N, P, lens):
    """Sequences of one to a dozen segments, in and out of the same slots."""
    check_packed(lens, 2, 1, N, P, dtype, shuffle=True, seed=N)


@TYPES
@pytest.mark.parametrize("N,P,heads,n", [(64, 64, 4, 257), (128, 128, 8, 1409), (128, 128, 8, 1407), (256, 256, 3, 2600),
                                         (64, 128, 2, 256)])
def test_prefill_either_side_of_a_change_of_segments(dtype, N, P, heads, n):
    check_packed([n // 2 + 11, 0, n - n // 2 - 11], heads, 1, N, P, dtype, shuffle=True, seed=n)


@pytest.mark.parametrize("kept", ["same", "apart", "read", "written", "neither"])
@pytest.mark.parametrize("P", [64, 256])
def test_pools_of_sequences_in_segments(kept, P):
    """One pool read and written, two, one that is only read or written, none; a padded
    sequence (slot -1) among the sequences."""
    lens, N = [300, 520, 0, 129, 128], 64
    a = inputs(sum(lens), 2, 1, N, P, FP32, seed=21)
    gen = torch.Generator(device="cuda").manual_seed(22)
    first = 0.3 * torch.randn((6, 2, N, P), generator=gen, device="cuda")
    source, sink = first.clone(), 0.3 * torch.randn(first.shape, generator=gen, device="cuda")
    before = sink.clone()
    where = [5, 0, 3, -1, 1]
    state_in = source if kept in ("same", "apart", "read") else None
    state_out = source if kept == "same" else sink if kept in ("apart", "written") else None
    slots = torch.tensor(where, dtype=torch.int32).cuda()
    if kept == "neither":  # (as many slots as sequences: the numbers are held to them)
        where = [4, 0, 3, -1, 1]
        slots = torch.tensor(where, dtype=torch.int32).cuda()
    out = torch.full_like(a["x"], 5.0)
    call(g.scan_prefill, a, cumulative(lens), state_in=state_in, state_out=state_out, slots=slots, out=out)
    at = 0
    for i, m in enumerate(lens):
        part, slot = slice(at, at + m), where[i]
        at += m
        if slot < 0:
            assert (out[part] == 5).all()
            continue
        y, S = reference(rows(a, part), torch.zeros_like(first[0]) if state_in is None else first[slot])
        close(out[part], y, tol(N), f"y of sequence {i}")
        if state_out is not None:
            close(state_out[slot], S, tol(N), f"state of sequence {i}")
    if kept != "same":
        assert torch.equal(source, first)
    rest = [i for i in range(6) if i not in where] if state_out is sink else list(range(6))
    assert torch.equal(sink[rest], before[rest])


@pytest.mark.parametrize("lens", [[0] * 30 + [700] + [1] * 32 + [600], [0] * 30 + [700] + [1] * 33 + [600], [600] * 20],
                         ids=["64", "65", "20"])
def test_prefill_of_long_sequences_among_many(lens):
    """Sequences of several segments, up to 64 of all lengths and more."""
    check_packed(lens, 2, 1, 64, 64, FP32, shuffle=True, seed=3)


@pytest.mark.parametrize("lens", [[5000], [2500, 1, 2600, 1024, 1025]])
def test_prefill_long(lens):
    check_packed(lens, 1, 1, 64, 64, FP32, seed=9)
    check_packed(lens, 8, 2, 128, 64, BF16, seed=10)


def test_prefill_of_a_batch_that_fills_the_gpu():
    """A sequence's results are its own alone, whichever kernels' shapes."""
    lens = [0, 1, 33, 100, 64, 7, 32, 65] + [5 + i for i in range(24)]
    a, out, pool = check_packed(lens, 16, 2, 64, 64, FP32, seed=5)
    cu = cumulative(lens).tolist()
    gen = torch.Generator(device="cuda").manual_seed(6)
    S0 = 0.3 * torch.randn(pool.shape, generator=gen, device="cuda")
    for i in range(0, len(lens), 5):
        s, S = slice(cu[i], cu[i + 1]), S0[i:i + 1].clone()
        y = call(g.scan_prefill, rows(a, s), cumulative([lens[i]]), state_in=S, state_out=S)
        assert torch.equal(y, out[s]) and torch.equal(S[0], pool[i]), i


def test_rows_before_and_behind_the_sequences_are_left():
    check_packed([40, 0, 3], 2, 1, 64, 64, BF16, first=37, behind=50, seed=8)
    check_packed([1, 900, 2], 2, 2, 64, 64, FP32, first=400, behind=700, seed=9)


@TYPES
def test_strided_rows_and_steps_of_both_types(dtype):
    """Slices of one fused projection, its steps in the rows' type or FP32, at
    an odd element."""
    n, heads, groups, N, P = 150, 4, 2, 64, 64
    wide = torch.randn((n, 8 + heads * P + 2 * groups * N + 24), device="cuda").to(dtype)
    x = wide[:, 8:8 + heads * P].unflatten(1, (heads, P))
    B = wide[:, 264:392].unflatten(1, (groups, N))
    C = wide[:, 392:520].unflatten(1, (groups, N))
    for dt in (wide[:, 521:525], torch.randn((n, 9), device="cuda")[:, 3:7]):
        a = {**inputs(n, heads, groups, N, P, dtype), "x": x, "B": B, "C": C, "dt": dt}
        check_packed([70, 80], heads, groups, N, P, dtype, a=a)
        pool = torch.zeros((n, heads, N, P), device="cuda")
        y = call(g.scan_step, a, pool)
        for i in (0, 77, 149):
            want, S = reference(rows(a, slice(i, i + 1)), torch.zeros((heads, N, P), device="cuda"))
            close(y[i:i + 1], want, tol(N), i)
            close(pool[i], S, tol(N), i)


@TYPES
def test_without_softplus_bias_and_skip(dtype):
    n, heads, N, P = 100, 2, 128, 64
    a = inputs(n, heads, 1, N, P, dtype, 3)
    a["dt"] = torch.rand((n, heads), device="cuda").to(dtype) * 0.1
    del a["D"], a["dt_bias"]
    check_packed([60, 40], heads, 1, N, P, dtype, a=a, softplus=False)
    S0 = torch.randn((n, heads, N, P), device="cuda")
    pool = S0.clone()
    y = call(g.scan_step, a, pool, softplus=False)
    for i in (0, 99):
        want, S = reference(rows(a, slice(i, i + 1)), S0[i], False)
        close(y[i:i + 1], want, tol(N), i)
        close(pool[i], S, tol(N), i)


def test_decays_from_none_to_all():
    """Steps of zero keep the state as it is; large ones clear it; growth too."""
    n, heads, N, P = 130, 4, 64, 64
    a = inputs(n, heads, 1, N, P, FP32, 4)
    a["dt"] = torch.zeros((n, heads), device="cuda")
    a["dt"][::7, 1] = 40.0
    a["dt"][:, 2] = 0.01
    a["dt"][64, 3] = 3e4
    a["A"] = torch.tensor([-1.0, -8.0, 1.5, -16.0], device="cuda")
    del a["dt_bias"]
    check_packed([n], heads, 1, N, P, FP32, a=a, softplus=False)
    a["A"][2] = 0.1
    check_packed([50, 80], heads, 1, N, P, FP32, a=a, softplus=True)


def test_softplus_of_far_values():
    n, N, P = 9, 64, 64
    a = inputs(n, 1, 1, N, P, FP32, 5)
    a["dt"] = torch.tensor([-200.0, -80.0, -20.0, -1.0, 0.0, 1.0, 20.0, 80.0, 600.0], device="cuda")[:, None].contiguous()
    del a["dt_bias"]
    check_packed([n], 1, 1, N, P, FP32, a=a)
    pool = torch.zeros((n, 1, N, P), device="cuda")
    y = call(g.scan_step, a, pool)
    for i in range(n):
        want, S = reference(rows(a, slice(i, i + 1)), torch.zeros((1, N, P), device="cuda"))
        close(y[i:i + 1], want, tol(N), i)
        close(pool[i], S, tol(N), i)


@TYPES
@pytest.mark.parametrize("N,P,heads,groups", [(128, 64, 4, 1), (64, 64, 2, 2), (256, 256, 2, 1), (128, 128, 3, 3), (64, 256, 2, 1)])
def test_step(dtype, N, P, heads, groups):
    n, n_slots = 9, 12
    a = inputs(n, heads, groups, N, P, dtype, N)
    S0 = 0.3 * torch.randn((n_slots, heads, N, P), device="cuda")
    where = [3, -1, 0, 11, 12, 5, 7, -5, 1]
    for in_place in (True, False):
        pool, out = S0.clone(), torch.full_like(a["x"], 5.0)
        into = pool if in_place else S0.clone()
        call(g.scan_step, a, pool, slots=torch.tensor(where, dtype=torch.int32).cuda(), out=out,
             state_out=None if in_place else into)
        for i, s in enumerate(where):
            if 0 <= s < n_slots:
                y, S = reference(rows(a, slice(i, i + 1)), S0[s])
                close(out[i:i + 1], y, tol(N), i)
                close(into[s], S, tol(N), i)
            else:
                assert (out[i] == 5).all()
        rest = [s for s in range(n_slots) if s not in where]
        assert torch.equal(into[rest], S0[rest])


def test_steps_follow_a_prefill():
    n, heads, N, P = 90, 2, 128, 64
    a = inputs(n, heads, 1, N, P, FP32, 12)
    y, S = reference(a, torch.zeros((heads, N, P), device="cuda"))
    pool = torch.zeros((1, heads, N, P), device="cuda")
    got = [call(g.scan_prefill, rows(a, slice(0, 60)), cumulative([60]), state_out=pool),
           call(g.scan_prefill, rows(a, slice(60, 80)), cumulative([20]), state_in=pool, state_out=pool)]
    got += [call(g.scan_step, rows(a, slice(i, i + 1)), pool) for i in range(80, 90)]
    close(torch.cat(got), y, tol(N), "y")
    close(pool[0], S, tol(N), "state")


def test_values_that_are_not_finite_stay_with_their_head():
    """In a prefill with the tokens up to 63 before them, in the sequence."""
    heads, N, P = 3, 64, 64
    a = inputs(200, heads, 3, N, P, FP32, 2)
    lens = [100, 100]
    clean, S0 = torch.empty_like(a["x"]), torch.empty((2, heads, N, P), device="cuda")
    call(g.scan_prefill, a, cumulative(lens), state_out=S0, out=clean)
    for name, at in (("x", (150, 1, 5)), ("B", (150, 1, 5)), ("C", (150, 1, 5)), ("dt", (150, 1))):
        b = {**a, name: a[name].clone()}
        b[name][at] = float("nan")
        S = torch.empty_like(S0)
        out = call(g.scan_prefill, b, cumulative(lens), state_out=S)
        touched = torch.zeros_like(out, dtype=torch.bool)
        touched[100:, 1] = True
        assert torch.equal(out[~touched], clean[~touched]), name
        assert torch.equal(S[[0, 0, 1, 1], [0, 1, 0, 2]], S0[[0, 0, 1, 1], [0, 1, 0, 2]]) and torch.equal(S[0], S0[0]), name
        assert torch.isnan(out[150, 1]).any()


@pytest.mark.parametrize("ends", [[0, 300, 10, 500], [200, 100, 50, 0], [-5, 10, 2000, 3000], [500, 500, 0, 500], [600, 700, 800, 900],
                                  [0, 500, 0, 500]])
def test_ends_that_fall_or_pass_the_rows_write_nothing_else(ends):
    n, heads, N, P = 500, 2, 64, 64
    a = inputs(n, heads, 1, N, P, FP32, 2)
    room = torch.full((n + 128, heads, P), 5.0, device="cuda")
    pool = torch.full((9, heads, N, P), 3.0, device="cuda")
    call(g.scan_prefill, a, torch.tensor(ends, dtype=torch.int32).cuda(), state_in=pool[2:7], state_out=pool[2:7],
         slots=torch.tensor([0, 2, 4], dtype=torch.int32).cuda(), out=room[64:64 + n])
    assert (room[:64] == 5).all() and (room[64 + n:] == 5).all()
    assert (pool[[0, 1, 3, 5, 7, 8]] == 3).all()


def test_captured_and_replayed():
    heads, N, P = 4, 128, 64
    a, step = inputs(900, heads, 1, N, P, BF16, 1), inputs(3, heads, 1, N, P, BF16, 2)
    cu = cumulative([700, 0, 200])
    pool, out = torch.zeros((3, heads, N, P), device="cuda"), torch.zeros_like(a["x"])
    after = torch.zeros_like(step["x"])

    def work():
        call(g.scan_prefill, a, cu, state_out=pool, out=out)
        call(g.scan_step, step, pool, out=after)

    work()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        work()
    for seed in range(4):
        for k, v in inputs(900, heads, 1, N, P, BF16, 30 + seed).items():
            a[k].copy_(v)
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
    n, heads, N, P = 1500, 2, 64, 64
    a = inputs(n, heads, 1, N, P, FP32, 1)
    cu, slots = torch.zeros(6, dtype=torch.int32, device="cuda"), torch.zeros(5, dtype=torch.int32, device="cuda")
    pool, out = torch.zeros((7, heads, N, P), device="cuda"), torch.zeros_like(a["x"])
    call(g.scan_prefill, a, cu, state_in=pool, state_out=pool, slots=slots, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(g.scan_prefill, a, cu, state_in=pool, state_out=pool, slots=slots, out=out)
    first = 0.3 * torch.randn(pool.shape, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    for lens, where in [([1500, 0, 0, 0, 0], [3, -1, -1, -1, -1]), ([1, 700, 0, 300, 2], [0, 6, 1, 2, 5]),
                        ([0, 0, 0, 0, 0], [4, 3, 2, 1, 0]), ([129, 128, 600, 257, 300], [6, 5, 4, 3, 7])]:
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
            y, S = reference(rows(a, part), first[slot])
            close(out[part], y, tol(N), f"y of {m} tokens")
            close(pool[slot], S, tol(N), f"state of {m} tokens")
        rest = [i for i in range(7) if i not in used]
        assert (out[at:] == 5).all() and torch.equal(pool[rest], first[rest])


def test_two_streams_at_once():
    heads, N, P = 4, 64, 64
    jobs = []
    for i in range(2):
        a = inputs(1500, heads, 1, N, P, BF16, i)
        jobs.append((a, torch.cuda.Stream(), call(g.scan_prefill, a, cumulative([1500]))))
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (a, stream, _) in enumerate(jobs):
            with torch.cuda.stream(stream):
                got[i].append(call(g.scan_prefill, a, cumulative([1500])))
    torch.cuda.synchronize()
    for i, (_, _, want) in enumerate(jobs):
        assert all(torch.equal(y, want) for y in got[i])


def test_offsets_beyond_32_bits():
    """Rows and slots that start past 2^32 bytes."""
    n, heads, N, P = 600_000, 64, 64, 64
    a = inputs(1200, heads, 1, N, P, BF16, 1)
    x = torch.zeros((n, heads, P), dtype=BF16, device="cuda")
    small = {"dt": torch.zeros((n, heads), dtype=BF16, device="cuda"), "B": torch.zeros((n, 1, N), dtype=BF16, device="cuda"),
             "C": torch.zeros((n, 1, N), dtype=BF16, device="cuda")}
    x[-1200:] = a["x"]
    for k in small:
        small[k][-1200:] = a[k]
    pool = torch.zeros((5000, heads, N, P), device="cuda")
    cu, slots = torch.tensor([n - 1200, n - 100, n], dtype=torch.int32).cuda(), torch.tensor([4999, 4000], dtype=torch.int32).cuda()
    out = call(g.scan_prefill, {**a, "x": x, **small}, cu, state_in=pool, state_out=pool, slots=slots)
    zero = torch.zeros((heads, N, P), device="cuda")
    for lo, hi, s in ((0, 1100, 4999), (1100, 1200, 4000)):
        y, S = reference(rows(a, slice(lo, hi)), zero)
        close(out[n - 1200 + lo:n - 1200 + hi], y, tol(N), s)
        close(pool[s], S, tol(N), s)


@TYPES
def test_rows_nearly_16_mb_apart(dtype):
    """Rows' offsets in a chunk and the clamped last row's fit their 32 bits."""
    n, heads, N, P = 150, 2, 64, 64
    a = inputs(n, heads, 1, N, P, dtype, 7)
    apart = (1 << 24) // a["x"].element_size() - 8
    room = torch.zeros(n * apart, dtype=dtype, device="cuda")
    far = dict(a)
    for k, at in (("x", 0), ("B", 128), ("C", 192)):
        far[k] = room[at:].as_strided(a[k].shape, (apart, a[k].shape[2], 1))
        far[k].copy_(a[k])
    out = room[512:].as_strided(a["x"].shape, (apart, P, 1))
    cu = cumulative([100, 1, 49])
    pool = torch.zeros((3, heads, N, P), device="cuda")
    call(g.scan_prefill, far, cu, state_out=pool, out=out)
    want = torch.zeros_like(pool)
    y = call(g.scan_prefill, a, cu, state_out=want)
    assert torch.equal(out, y) and torch.equal(pool, want)


def test_many_sequences():
    lens = [(i * 7) % 5 for i in range(5000)]
    n = sum(lens)
    a = inputs(n, 1, 1, 64, 64, BF16, 1)
    pool = torch.zeros((5000, 1, 64, 64), device="cuda")
    out = call(g.scan_prefill, a, cumulative(lens), state_out=pool)
    cu = cumulative(lens).tolist()
    for i in (0, 1, 2499, 4998, 4999):
        y, S = reference(rows(a, slice(cu[i], cu[i + 1])), torch.zeros((1, 64, 64), device="cuda"))
        close(out[cu[i]:cu[i + 1]], y, tol(64), i)
        close(pool[i], S, tol(64), i)


def test_workspaces():
    a = inputs(900, 2, 1, 64, 64, BF16, 1)
    want = call(g.scan_prefill, a, cumulative([900]))
    room = torch.empty(1 << 22, dtype=torch.uint8, device="cuda")
    assert torch.equal(call(g.scan_prefill, a, cumulative([900]), workspace=room), want)
    for bad in (room[:64], room[8:], room.float(), room[::2]):
        with pytest.raises(g.GDNError):
            call(g.scan_prefill, a, cumulative([900]), workspace=bad)


def test_refusals_of_tensors():
    a = inputs(8, 4, 2, 64, 64, BF16)
    cu, pool = cumulative([8]), torch.zeros((1, 4, 64, 64), device="cuda")
    call(g.scan_prefill, a, cu, state_in=pool, state_out=pool)
    for bad in ({"x": a["x"].double()}, {"x": a["x"].float()}, {"x": a["x"][:, :3]}, {"B": a["B"].float()}, {"B": a["B"][:7]},
                {"C": a["C"][:, :1]}, {"dt": a["dt"].double()}, {"dt": a["dt"][:, :2]}, {"A": a["A"].to(BF16)}, {"A": a["A"][:2]},
                {"D": a["D"][:3]}, {"dt_bias": a["dt_bias"].double()}, {"x": a["x"].cpu()}, {"x": a["x"][:, :, :32]},
                {"B": torch.zeros((8, 3, 64), dtype=BF16, device="cuda"), "C": torch.zeros((8, 3, 64), dtype=BF16, device="cuda")},
                {"B": torch.zeros((8, 2, 96), dtype=BF16, device="cuda"), "C": torch.zeros((8, 2, 96), dtype=BF16, device="cuda")}):
        with pytest.raises(g.GDNError):
            call(g.scan_prefill, {**a, **bad}, cu)
    for bad in (dict(state_in=pool[:, :2]), dict(state_out=pool.to(BF16)), dict(out=a["x"]), dict(slots=cu.long())):
        with pytest.raises(g.GDNError):
            call(g.scan_prefill, a, cu, **bad)
    with pytest.raises(g.GDNError):
        call(g.scan_prefill, a, cumulative([4, 4]), state_out=pool)
    with pytest.raises(g.GDNError):
        call(g.scan_step, a, pool)
    with pytest.raises(g.GDNError):
        call(g.scan_prefill, {**a, "A": a["A"].clone().requires_grad_()}, cu)


def test_writes_count_as_modifications():
    a = inputs(8, 4, 2, 64, 64, BF16)
    pool, out = torch.zeros((8, 4, 64, 64), device="cuda"), torch.empty_like(a["x"])
    versions = out._version, pool._version
    call(g.scan_step, a, pool, out=out)
    assert out._version > versions[0] and pool._version > versions[1]
    versions = out._version, pool._version
    call(g.scan_prefill, a, cumulative([8]), state_out=pool, out=out)
    assert out._version > versions[0] and pool._version > versions[1]


@TYPES
@pytest.mark.parametrize("N,P", [(64, 64), (128, 64), (256, 64), (64, 128), (256, 256)])
def test_tokens_before_a_value_that_is_not_finite(dtype, N, P):
    """They are as if it were not there, in its 16 tokens, chunk and segment too; its own
    and, of the state, those behind it are not finite."""
    heads, lens, at = 2, [150, 700], 150
    n = sum(lens)
    a = inputs(n, heads, 2, N, P, dtype, seed=N + P)
    clean, S0 = torch.empty_like(a["x"]), torch.empty((2, heads, N, P), device="cuda")
    call(g.scan_prefill, a, cumulative(lens), state_out=S0, out=clean)
    for k, (name, value) in enumerate([(name, v) for name in ("x", "B", "C", "dt") for v in ("nan", "inf", "-inf")]):
        if name == "dt" and value == "-inf":
            continue  # (its softplus is 0)
        for t in (k % 3, 15 + k % 2, 31 + k % 3, 63 + k % 2, 90 + k, 470 + 17 * k):
            b = {**a, name: a[name].clone()}
            b[name][(at + t, 1, 5) if name in ("x", "B", "C") else (at + t, 1)] = float(value)
            S = torch.empty_like(S0)
            out = call(g.scan_prefill, b, cumulative(lens), state_out=S)
            assert torch.equal(out[:at + t], clean[:at + t]), (name, value, t)
            assert torch.equal(out[:, 0], clean[:, 0]) and torch.equal(S[:, 0], S0[:, 0]) and torch.equal(S[0], S0[0])
            own = out[at + t:, 1, 5] if name == "x" else out[at + t:at + t + 1, 1] if name == "C" else out[at + t:, 1]
            assert not torch.isfinite(own[0]).any(), (name, value, t)
            if name == "C":
                assert torch.equal(out[at + t + 1:], clean[at + t + 1:]) and torch.equal(S, S0)
            else:
                assert not torch.isfinite(S[1, 1]).all(), (name, value, t)
