"""gdn_delta_prefill and gdn_delta_step against the recurrence token by token
in 64 bits (gpu).

Tolerances.  A token's update is four chained sums (S^T k, the chunk's
triangular system, the update, S^T q), each of at most key_dim + 64 products
rounded to FP32; n roundings of 2^-24 in no order add up to sqrt(n) 2^-24 of a
sum's size.  Relative to the norm of a sequence's whole result that is
TOL = 4 sqrt(key_dim + 64) 2^-24 (4.3e-6 at 256).  A BF16 or FP16 output adds
half a step of its type, eps / 2 of the value.
"""
import math

import pytest
import torch

import gateddeltanet_amd as g

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def tol(dk):
    return 4 * math.sqrt(dk + 64) * 2.0**-24


def inputs(n, hq, hv, dk, dv, dtype, seed=0, l2norm=True):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*s):
        return torch.randn(s, generator=gen, device="cuda")

    q, k, v = (normal(n, h, d) for h, d in ((hq, dk), (hq, dk), (hv, dv)))
    if not l2norm:
        q, k = q * dk**-0.5, k * dk**-0.5
    gate = -0.3 * torch.rand((n, hv), generator=gen, device="cuda") ** 4
    beta = torch.sigmoid(normal(n, hv))
    return q.to(dtype), k.to(dtype), v.to(dtype), gate, beta


def reference(q, k, v, gate, beta, S, l2norm=True, scale=None):
    """(o, S') of one sequence, in 64 bits."""
    group = v.shape[1] // q.shape[1]
    scale = q.shape[2] ** -0.5 if scale is None else scale
    q, k = (x.double().repeat_interleave(group, 1) for x in (q, k))
    if l2norm:
        q, k = (x / (x.square().sum(-1, keepdim=True) + 1e-6).sqrt() for x in (q, k))
    v, a, beta = v.double(), gate.double().exp(), beta.double()
    S, o = S.double().clone(), torch.zeros(v.shape, dtype=torch.float64, device=v.device)
    for t in range(q.shape[0]):
        S = S * a[t, :, None, None]
        d = beta[t, :, None] * (v[t] - (S * k[t, :, :, None]).sum(1))
        S = S + k[t, :, :, None] * d[:, None, :]
        o[t] = scale * (S * q[t, :, :, None]).sum(1)
    return o, S


def close(got, want, t, what):
    """Elementwise half a step of the type, and t of the norm (per value: of
    the root mean square, times 8 for the largest of many)."""
    assert torch.isfinite(got).all(), what
    if want.numel() == 0:
        return
    diff = (got.double() - want).abs()
    rms = want.square().mean().sqrt()
    half = 0.0 if got.dtype == FP32 else torch.finfo(got.dtype).eps / 2
    assert (diff <= half * want.abs() + 8 * t * torch.maximum(want.abs(), rms.expand_as(want))).all(), (
        what, float((diff - half * want.abs()).max()), float(rms))
    if half == 0.0:
        assert diff.square().mean().sqrt() <= t * rms, (what, float(diff.square().mean().sqrt() / rms))


def check_packed(lens, hq, hv, dk, dv, dtype, start, l2norm=True, scale=None, seed=0, shuffle=False):
    n = sum(lens)
    q, k, v, gate, beta = inputs(n, hq, hv, dk, dv, dtype, seed, l2norm)
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    slots = None
    n_slots = len(lens) + (3 if shuffle else 0)
    where = list(range(len(lens)))
    if shuffle:
        where = torch.randperm(n_slots, generator=torch.Generator().manual_seed(seed))[:len(lens)].tolist()
        slots = torch.tensor(where, dtype=torch.int32).cuda()
    gen = torch.Generator(device="cuda").manual_seed(seed + 1)
    S0 = 0.3 * torch.randn((n_slots, hv, dk, dv), generator=gen, device="cuda")
    pool = S0.clone()
    out = g.delta_prefill(q, k, v, gate, beta, cu, state_in=pool if start else None, state_out=pool, slots=slots,
                          l2norm=l2norm, scale=scale)
    at = 0
    for i, m in enumerate(lens):
        s = slice(at, at + m)
        init = S0[where[i]] if start else torch.zeros_like(S0[0])
        o, S = reference(q[s], k[s], v[s], gate[s], beta[s], init, l2norm, scale)
        close(out[s], o, tol(dk), f"o of sequence {i}, {m} tokens")
        close(pool[where[i]], S, tol(dk), f"state of sequence {i}, {m} tokens")
        at += m
    rest = [i for i in range(n_slots) if i not in where]
    assert torch.equal(pool[rest], S0[rest])
    return out, pool


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("dk,dv,hq,hv", [(256, 256, 2, 2), (128, 128, 1, 3), (64, 64, 2, 4), (128, 256, 1, 1),
                                         (256, 64, 1, 2), (64, 128, 3, 3)])
def test_prefill(dtype, dk, dv, hq, hv):
    check_packed([0, 1, 31, 32, 33, 63, 64, 65, 0, 130, 16, 17], hq, hv, dk, dv, dtype, True, shuffle=True, seed=dk + dv)


@pytest.mark.parametrize("dtype,dk,dv,hq,hv,n", [(FP32, 128, 128, 8, 16, 8), (FP32, 256, 256, 4, 8, 6), (FP16, 128, 128, 16, 16, 9),
                                                 (FP16, 64, 256, 4, 16, 5), (BF16, 64, 64, 4, 16, 17), (FP32, 64, 64, 2, 16, 16),
                                                 (BF16, 256, 256, 2, 8, 9)])
def test_prefill_of_batches_that_fill_the_gpu(dtype, dk, dv, hq, hv, n):
    """A sequence's results are its own alone, bit for bit."""
    lens = [0, 1, 33, 100, 64, 7, 32, 65][: n] + [5 + i for i in range(n - 8)]
    q, k, v, gate, beta = inputs(sum(lens), hq, hv, dk, dv, dtype, n + dk)
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    out, pool = check_packed(lens, hq, hv, dk, dv, dtype, True, seed=n + dk)
    gen = torch.Generator(device="cuda").manual_seed(n + dk + 1)
    S0 = 0.3 * torch.randn((n, hv, dk, dv), generator=gen, device="cuda")
    for i in range(0, n, 3):
        s = slice(int(cu[i]), int(cu[i + 1]))
        S = S0[i:i + 1].clone()
        o = g.delta_prefill(q[s], k[s], v[s], gate[s], beta[s], torch.tensor([0, lens[i]], dtype=torch.int32).cuda(),
                            state_in=S, state_out=S)
        assert torch.equal(o, out[s]) and torch.equal(S[0], pool[i]), i


@pytest.mark.parametrize("lens", [[1], [2], [15], [64], [128], [129], [1, 1, 1, 1, 1, 1, 1, 1, 1], [0], [0, 0, 7, 0]])
def test_prefill_lengths_from_zero_state(lens):
    check_packed(lens, 1, 2, 256, 256, BF16, False, seed=len(lens) + sum(lens))


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
def test_prefill_long(dtype):
    check_packed([1500], 1, 1, 256, 64, dtype, True, seed=9)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
def test_prefill_without_l2norm_and_with_a_scale(dtype):
    check_packed([70, 40], 1, 2, 128, 64, dtype, True, l2norm=False, scale=0.25, seed=4)


def test_prefill_many_sequences_of_one_token():
    check_packed([1] * 300, 1, 1, 64, 64, BF16, True, seed=5, shuffle=True)


def test_prefill_repeated_keys():
    """Equal keys: the triangular system is as far from the identity as it
    gets (every entry beta exp(G_m - G_s))."""
    n, dk = 100, 128
    q, k, v, gate, beta = inputs(n, 1, 1, dk, 64, FP32, 3)
    k = k[:1].expand(n, -1, -1).contiguous()
    beta.fill_(1.0)
    gate.zero_()
    cu = torch.tensor([0, n], dtype=torch.int32).cuda()
    S = torch.zeros((1, 1, dk, 64), device="cuda")
    out = g.delta_prefill(q, k, v, gate, beta, cu, state_out=S)
    o, want = reference(q, k, v, gate, beta, torch.zeros_like(S[0]))
    # each step replaces what the key holds, so a token's rounding stays in
    # the next ones' differences: 64 of them in a chunk's system
    close(out, o, 8 * tol(dk), "o")
    close(S[0], want, 8 * tol(dk), "state")


def test_prefill_in_two_calls():
    q, k, v, gate, beta = inputs(200, 2, 4, 128, 128, FP32, 6)
    S = torch.zeros((1, 4, 128, 128), device="cuda")
    T = torch.zeros_like(S)
    cu = [torch.tensor([0, n], dtype=torch.int32).cuda() for n in (200, 90, 110)]
    whole = g.delta_prefill(q, k, v, gate, beta, cu[0], state_out=S)
    parts = [g.delta_prefill(q[s], k[s], v[s], gate[s], beta[s], c, state_in=T, state_out=T)
             for s, c in ((slice(0, 90), cu[1]), (slice(90, 200), cu[2]))]
    close(torch.cat(parts), whole.double(), 2 * tol(128), "o")
    close(T, S.double(), 2 * tol(128), "state")


def test_prefill_rows_of_no_sequence_and_left_out_sequences():
    """Rows before the first and behind the last sequence, and those of
    sequences with slots outside the pool: o as it was, nothing read (NaN)."""
    n, hv = 300, 2
    q, k, v, gate, beta = inputs(n, 1, hv, 64, 64, BF16, 7)
    for x in (q, k, v, gate, beta):
        x[:20], x[100:130], x[280:] = float("nan"), float("nan"), float("nan")
    cu = torch.tensor([20, 100, 130, 280], dtype=torch.int32).cuda()
    for bad in (-1, 2, 2**31 - 1, -2**31):
        S0 = torch.randn((2, hv, 64, 64), device="cuda")
        pool, out = S0.clone(), torch.full_like(v, 7.0)
        slots = torch.tensor([1, bad, 0], dtype=torch.int32).cuda()
        g.delta_prefill(q, k, v, gate, beta, cu, state_in=pool, state_out=pool, slots=slots, out=out)
        for i, s in ((1, slice(20, 100)), (0, slice(130, 280))):
            o, S = reference(q[s], k[s], v[s], gate[s], beta[s], S0[i])
            close(out[s], o, tol(64), "o")
            close(pool[i], S, tol(64), "state")
        assert (out[:20] == 7).all() and (out[100:130] == 7).all() and (out[280:] == 7).all()


def test_prefill_ends_are_held_to_the_rows():
    """cu_seqlens that pass the rows, fall or start below zero: held to the
    rows; the sequences that are whole are right."""
    q, k, v, gate, beta = inputs(90, 1, 1, 64, 64, FP32, 8)
    cu = torch.tensor([-5, 40, 90, 1000, 60, 2**31 - 1], dtype=torch.int32).cuda()
    S = torch.zeros((5, 1, 64, 64), device="cuda")
    out = torch.zeros_like(v)
    g.delta_prefill(q, k, v, gate, beta, cu, state_out=S, out=out)
    o, want = reference(q[:40], k[:40], v[:40], gate[:40], beta[:40], torch.zeros_like(S[0]))
    close(S[0], want, tol(64), "state")
    close(out[:40], o, tol(64), "o")
    assert (S[2] == 0).all() and (S[3] == 0).all()  # nothing left past row 90, and an end before its start


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
def test_strided_rows(dtype):
    """q, k, v and o as slices of wider rows, g and beta of one."""
    n, hq, hv, dk, dv = 75, 2, 4, 64, 128
    q, k, v, gate, beta = inputs(n, hq, hv, dk, dv, dtype, 10)
    wide = torch.full((n, 2 * hq * dk + 2 * hv * dv + 64), float("nan"), dtype=dtype, device="cuda")
    at = [0, hq * dk, 2 * hq * dk, 2 * hq * dk + hv * dv]
    qs, ks, vs, os_ = (wide[:, a:a + h * d].unflatten(1, (h, d))
                       for a, h, d in zip(at, (hq, hq, hv, hv), (dk, dk, dv, dv)))
    gb = torch.full((n, 2 * hv + 1), float("nan"), device="cuda")
    gs, bs = gb[:, :hv], gb[:, hv:2 * hv]
    for dst, src in ((qs, q), (ks, k), (vs, v), (gs, gate), (bs, beta)):
        dst.copy_(src)
    cu = torch.tensor([0, 5, n], dtype=torch.int32).cuda()
    want = g.delta_prefill(q, k, v, gate, beta, cu)
    g.delta_prefill(qs, ks, vs, gs, bs, cu, out=os_)
    assert torch.equal(os_, want) and torch.isnan(wide[:, -64:]).all()
    S, T = (torch.ones((n, hv, dk, dv), device="cuda") for _ in range(2))
    want = g.delta_step(q, k, v, gate, beta, S)
    g.delta_step(qs, ks, vs, gs, bs, T, out=os_)
    assert torch.equal(os_, want) and torch.equal(S, T) and torch.isnan(wide[:, -64:]).all()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("dk,dv,hq,hv,n", [(256, 256, 2, 2, 1), (256, 256, 8, 8, 9), (128, 128, 1, 3, 5),
                                           (64, 64, 2, 4, 33), (128, 256, 1, 1, 70), (256, 64, 1, 2, 3),
                                           (64, 128, 3, 3, 2), (64, 64, 1, 1, 300)])
def test_step(dtype, dk, dv, hq, hv, n):
    q, k, v, gate, beta = inputs(n, hq, hv, dk, dv, dtype, n + dk)
    gen = torch.Generator(device="cuda").manual_seed(n)
    S0 = 0.3 * torch.randn((n + 5, hv, dk, dv), generator=gen, device="cuda")
    slots = torch.randperm(n + 5, generator=gen, device="cuda")[:n].to(torch.int32)
    left_out = n > 2
    if left_out:
        slots[1] = -1
        slots[n - 1] = n + 5
    pool, out = S0.clone(), torch.full_like(v, 7.0)
    g.delta_step(q, k, v, gate, beta, pool, slots=slots, out=out)
    used = []
    for i, s in enumerate(slots.tolist()):
        if not 0 <= s < n + 5:
            assert (out[i] == 7).all()
            continue
        used.append(s)
        if i % 7 and n > 40:
            continue
        o, S = reference(q[i:i + 1], k[i:i + 1], v[i:i + 1], gate[i:i + 1], beta[i:i + 1], S0[s])
        close(out[i], o[0], tol(dk), f"o {i}")
        close(pool[s], S, tol(dk), f"state {i}")
    rest = [i for i in range(n + 5) if i not in used]
    assert torch.equal(pool[rest], S0[rest])


def test_step_into_another_pool_and_without_one():
    q, k, v, gate, beta = inputs(3, 1, 2, 64, 64, BF16, 2)
    S = torch.randn((3, 2, 64, 64), device="cuda")
    S0, T = S.clone(), torch.zeros_like(S)
    o1 = g.delta_step(q, k, v, gate, beta, S, state_out=T)
    assert torch.equal(S, S0)
    o2 = g.delta_step(q, k, v, gate, beta, S)
    assert torch.equal(o1, o2) and torch.equal(S, T)


def test_prefill_of_single_tokens_is_the_step():
    q, k, v, gate, beta = inputs(6, 2, 2, 256, 256, FP32, 12)
    S0 = torch.randn((6, 2, 256, 256), device="cuda")
    S, T = S0.clone(), S0.clone()
    cu = torch.arange(7, dtype=torch.int32).cuda()
    a = g.delta_prefill(q, k, v, gate, beta, cu, state_in=S, state_out=S)
    b = g.delta_step(q, k, v, gate, beta, T)
    close(a, b.double(), 2 * tol(256), "o")
    close(S, T.double(), 2 * tol(256), "state")


def test_nothing_to_do():
    """No sequences: nothing is touched.  No tokens: the states go through."""
    q, k, v, gate, beta = inputs(5, 1, 2, 64, 64, BF16, 1)
    out = torch.full_like(v, 7.0)
    S = torch.ones((3, 2, 64, 64), device="cuda")
    g.delta_prefill(q, k, v, gate, beta, torch.zeros(1, dtype=torch.int32).cuda(), state_in=S, state_out=S, out=out)
    assert (out == 7).all() and (S == 1).all()
    none = [x[:0] for x in (q, k, v, gate, beta)]
    T = torch.zeros_like(S)
    o = g.delta_prefill(*none, torch.zeros(4, dtype=torch.int32).cuda(), state_in=S, state_out=T)
    assert o.shape == (0, 2, 64) and torch.equal(S, T)
    assert g.delta_step(*none, S).shape == (0, 2, 64) and (S == 1).all()


def test_many_sequences_of_all_lengths():
    """More sequences than the order's steps tell apart, some longer than its
    last step."""
    lens = [(7 * i) % 90 for i in range(400)]
    q, k, v, gate, beta = inputs(sum(lens), 1, 1, 64, 64, BF16, 22)
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    S = torch.zeros((400, 1, 64, 64), device="cuda")
    out = g.delta_prefill(q, k, v, gate, beta, cu, state_out=S)
    for i in range(0, 400, 29):
        s = slice(int(cu[i]), int(cu[i + 1]))
        o, want = reference(q[s], k[s], v[s], gate[s], beta[s], torch.zeros_like(S[i]))
        close(out[s], o, tol(64), f"o {i}")
        close(S[i], want, tol(64), f"state {i}")
    q, k, v, gate, beta = inputs(17000, 1, 1, 64, 64, BF16, 23)
    cu = torch.tensor([0, 100, 17000], dtype=torch.int32).cuda()  # 265 chunks
    S = torch.zeros((2, 1, 64, 64), device="cuda")
    g.delta_prefill(q, k, v, gate, beta, cu, state_out=S)
    T = torch.zeros_like(S[:1])
    for a in range(100, 17000, 4225):
        s = slice(a, a + 4225)
        g.delta_prefill(q[s], k[s], v[s], gate[s], beta[s], torch.tensor([0, 4225], dtype=torch.int32).cuda(),
                        state_in=T, state_out=T)
    close(S[1], T[0].double(), 2 * tol(64), "state of 16900 tokens")


def test_decays_at_their_ends():
    """g = -inf and a decay below FP32 clear the state, also in the middle of
    a chunk; g = 0 and beta = 0 leave it."""
    n = 80
    q, k, v, gate, beta = inputs(n, 1, 3, 64, 64, FP32, 13)
    gate[37, 0], gate[70, 0], gate[5, 1] = -math.inf, -200.0, -1e30
    gate[:, 2] = 0.0
    beta[:, 2] = 0.0
    S0 = torch.randn((1, 3, 64, 64), device="cuda")
    S, cu = S0.clone(), torch.tensor([0, n], dtype=torch.int32).cuda()
    out = g.delta_prefill(q, k, v, gate, beta, cu, state_in=S, state_out=S)
    o, want = reference(q, k, v, gate, beta, S0[0])
    close(out, o, tol(64), "o")
    close(S[0], want, tol(64), "state")
    assert torch.equal(S[0, 2], S0[0, 2])
    S = S0.clone()
    g.delta_step(q[:1], k[:1], v[:1], torch.full_like(gate[:1], -math.inf), beta[:1], S)
    _, want = reference(q[:1], k[:1], v[:1], torch.full_like(gate[:1], -math.inf), beta[:1], S0[0])
    close(S[0], want, tol(64), "state")


def test_a_nan_stays_in_its_sequence_and_head():
    lens = [70, 100, 66]
    q, k, v, gate, beta = inputs(sum(lens), 2, 4, 64, 64, BF16, 14)
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    S, T = (torch.zeros((3, 4, 64, 64), device="cuda") for _ in range(2))
    want = g.delta_prefill(q, k, v, gate, beta, cu, state_out=S)
    v[70 + 80, 1, 3] = float("nan")
    beta[70 + 90, 2] = float("nan")
    got = g.delta_prefill(q, k, v, gate, beta, cu, state_out=T)
    same = torch.ones(sum(lens), 4, dtype=torch.bool)
    same[70 + 64:170, 1:3] = False  # the second chunk of the two heads
    assert torch.equal(got[same], want[same])
    assert torch.isnan(got[169, 1, 3]) and torch.isnan(got[169, 2]).all()
    keep = torch.ones(3, 4, dtype=torch.bool)
    keep[1, 1:3] = False
    assert torch.equal(T[keep], S[keep]) and torch.isnan(T[1, 2]).all()


def test_two_runs_agree_bit_for_bit():
    lens = [300, 1, 77]
    q, k, v, gate, beta = inputs(sum(lens), 8, 8, 256, 256, BF16, 15)
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    S = [torch.zeros((3, 8, 256, 256), device="cuda") for _ in range(2)]
    out = [g.delta_prefill(q, k, v, gate, beta, cu, state_out=s) for s in S]
    assert torch.equal(out[0], out[1]) and torch.equal(S[0], S[1])


def test_captured_and_on_another_stream():
    """A graph of a prefill and two steps, replayed between eager work."""
    lens = [40, 0, 90]
    n = len(lens)
    q, k, v, gate, beta = inputs(sum(lens), 2, 4, 128, 64, BF16, 16)
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    S = torch.zeros((n, 4, 128, 64), device="cuda")

    def work():
        a = g.delta_prefill(q, k, v, gate, beta, cu, state_out=S)
        b = g.delta_step(q[:n], k[:n], v[:n], gate[:n], beta[:n], S)
        c = g.delta_step(q[n:2 * n], k[n:2 * n], v[n:2 * n], gate[n:2 * n], beta[n:2 * n], S)
        return a, b, c

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = work()
    for seed in range(4):
        for x, y in zip((q, k, v, gate, beta), inputs(sum(lens), 2, 4, 128, 64, BF16, 20 + seed)):
            x.copy_(y)
        S.zero_()
        want, Sw = [x.clone() for x in work()], S.clone()
        torch.cuda.synchronize()
        S.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want)) and torch.equal(S, Sw), seed


def test_tensor_refusals():
    q, k, v, gate, beta = inputs(4, 2, 4, 64, 64, BF16, 1)
    cu = torch.tensor([0, 4], dtype=torch.int32).cuda()
    S = torch.zeros((1, 4, 64, 64), device="cuda")
    P = torch.zeros((4, 4, 64, 64), device="cuda")
    ok = dict(state_in=S, state_out=S)
    g.delta_prefill(q, k, v, gate, beta, cu, **ok)
    bad = [
        ((q.double(), k, v, gate, beta, cu), ok), ((q, k.float(), v, gate, beta, cu), ok),
        ((q.cpu(), k, v, gate, beta, cu), ok), ((q, k.cpu(), v, gate, beta, cu), ok),
        ((q, k[:3], v, gate, beta, cu), ok), ((q, k, v[:3], gate, beta, cu), ok),
        ((q, k, v.transpose(1, 2), gate, beta, cu), ok), ((q, k, v, gate.bfloat16(), beta, cu), ok),
        ((q, k, v, gate[:, :3], beta, cu), ok), ((q, k, v, gate, beta[:3], cu), ok),
        ((q, k, v, gate, beta.t().contiguous().t(), cu), ok),
        ((q, k, v, gate, beta, cu.long()), ok), ((q, k, v, gate, beta, cu.cpu()), ok),
        ((q, k, v, gate, beta, cu), dict(state_in=S.double())), ((q, k, v, gate, beta, cu), dict(state_out=S.cpu())),
        ((q, k, v, gate, beta, cu), dict(state_in=S, state_out=P)),
        ((q, k, v, gate, beta, cu), dict(state_in=S.transpose(2, 3))),
        ((q, k, v, gate, beta, cu), dict(**ok, slots=torch.zeros(2, dtype=torch.int32).cuda())),
        ((q, k, v, gate, beta, cu), dict(**ok, slots=torch.zeros(1).cuda())),
        ((q, k, v, gate, beta, cu), dict(out=torch.empty_like(v).float())),
        ((q, k, v, gate, beta, cu), dict(workspace=torch.empty(16, dtype=torch.uint8).cuda())),
        ((q[:, :, :32], k[:, :, :32], v, gate, beta, cu), {}),
        ((q, k, v, gate, beta, torch.tensor([0, 2, 4], dtype=torch.int32).cuda()), ok),  # two sequences, one state
    ]
    for args, kw in bad:
        with pytest.raises(g.GDNError):
            g.delta_prefill(*args, **kw)
    flat = torch.zeros(4 * 2 * 64 + 8, dtype=BF16).cuda()
    odd = flat[1:1 + 4 * 2 * 64].view(4, 2, 64)  # rows at odd addresses
    with pytest.raises(g.GDNError):
        g.delta_prefill(odd, k, v, gate, beta, cu)
    with pytest.raises(g.GDNError):
        g.delta_step(odd, k, v, gate, beta, P)
    with pytest.raises(g.GDNError):
        g.delta_step(q, k, v, gate, beta, S)


def test_one_row_of_any_stride():
    """A single token's rows have no stride to keep to."""
    q, k, v, gate, beta = inputs(1, 1, 2, 64, 128, BF16, 51)
    odd = [torch.as_strided(x, x.shape, (s, *x.stride()[1:])) for x, s in ((q, 3), (k, 1 << 40), (v, 0), (gate, 7))]
    S = torch.ones((1, 2, 64, 128), device="cuda")
    T = S.clone()
    cu = torch.tensor([0, 1], dtype=torch.int32).cuda()
    assert torch.equal(g.delta_step(*odd, beta, S), g.delta_step(q, k, v, gate, beta, T)) and torch.equal(S, T)
    assert torch.equal(g.delta_prefill(*odd, beta, cu, state_out=S), g.delta_prefill(q, k, v, gate, beta, cu, state_out=T))
    assert torch.equal(S, T)


@pytest.mark.parametrize("hv", [1, 3])
def test_single_heads_of_transposed_views(hv):
    """Heads in front, as [heads][tokens][dim] holds them: a single head's rows
    are rows all the same, several heads' are not."""
    n, dk, dv = 40, 64, 128
    q, k, v, gate, beta = inputs(n, 1, hv, dk, dv, BF16, 61)
    cu = torch.tensor([0, 7, n], dtype=torch.int32).cuda()

    def heads_first(x):
        return torch.empty((x.shape[1], n, x.shape[2]), dtype=BF16, device="cuda").copy_(x.transpose(0, 1)).transpose(0, 1)

    fq, fk, fv = heads_first(q), heads_first(k), heads_first(v)
    assert fq.stride(1) == n * dk
    out = torch.empty_like(v)
    S, T = (torch.ones((n, hv, dk, dv), device="cuda") for _ in range(2))
    for f, a, b in ((g.delta_prefill, (cu,), (cu,)), (g.delta_step, (S,), (T,))):
        want = f(q, k, v, gate, beta, *a)
        assert torch.equal(f(fq, fk, v, gate, beta, *b), want)
        if hv == 1:
            into = torch.empty((1, n, dv), dtype=BF16, device="cuda").transpose(0, 1)
            if f is g.delta_step:
                T.fill_(1.0)
            assert f(fq, fk, fv, gate, beta, *b, out=into) is into and torch.equal(into, want)
            values = fv.repeat_interleave(2, 2)[..., ::2]  # values apart from each other
        else:
            values = fv
        for kw in (dict(v=values), dict(out=values)):
            with pytest.raises(g.GDNError, match="contiguous in a row"):
                f(q, k, kw.get("v", v), gate, beta, *b, out=kw.get("out", out))
    assert torch.equal(S, T)


def test_tensors_written_in_place_count_as_modified():
    """A value that autograd keeps for a backward pass and an operator then
    writes over is an error there, as after torch's own in-place operations."""
    n, hv, d = 3, 2, 64
    q, k, v, gate, beta = inputs(n, hv, hv, d, d, FP32, 71)
    cu = torch.tensor([0, n], dtype=torch.int32).cuda()
    S, out = torch.ones((n, hv, d, d), device="cuda"), torch.empty_like(v)
    x, y = torch.ones((n, 70), device="cuda"), torch.empty((n, 70), device="cuda")
    tok, lp = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(n, device="cuda")
    calls = [(lambda: g.delta_step(q, k, v, gate, beta, S), [S]),
             (lambda: g.delta_step(q, k, v, gate, beta, S.clone(), state_out=S, out=out), [S, out]),
             (lambda: g.delta_prefill(q, k, v, gate, beta, cu, state_out=S, out=out), [S, out]),
             (lambda: g.logits_process(x, out=y), [y]), (lambda: g.logits_process(x, out=x), [x]),
             (lambda: g.sample_tokens(x, tokens=tok, logprobs=lp), [tok, lp])]
    for call, written in calls:
        before = [t._version for t in written]
        call()
        assert all(t._version > b for t, b in zip(written, before))
    w = torch.ones((n, hv, d, d), device="cuda", requires_grad=True)
    loss = (w * S).sum()
    g.delta_step(q, k, v, gate, beta, S)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        T = torch.ones((n, hv, d, d), device="cuda")
        g.delta_step(q, k, v, gate, beta, T)
    assert g.delta_step(q, k, v, gate, beta, None).shape == v.shape


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
def test_prefill_ends_that_fall(dtype):
    """Ends that fall or pass the rows, over a workspace that holds NaN: a
    sequence that is whole before the fall, and in any case every one whose
    state is not as it was, has its result."""
    n, hv, fill = 290, 2, 7.0
    q, k, v, gate, beta = inputs(n, 1, hv, 64, 64, dtype, 12)
    gen = torch.Generator().manual_seed(12)
    calls = [[-5, 140, 290, 1000, 200, 2**31 - 1], [0, 140, 10, 290, 290, 290], [290, 0, 290], [100, 90, 80, 70, 60, 290],
             [0, 290, 0, 290, 0, 290]]
    calls += [torch.randint(-20, 320, (m,), generator=gen).tolist() for m in range(2, 14)]
    for ends in calls:
        m = len(ends) - 1
        cu = torch.tensor(ends, dtype=torch.int32).cuda()
        S = torch.full((m, hv, 64, 64), fill, device="cuda")
        ws = torch.full((32 << 20,), 255, dtype=torch.uint8, device="cuda")
        g.delta_prefill(q, k, v, gate, beta, cu, state_out=S, workspace=ws)
        for i in range(m):
            first = min(max(ends[i], 0), n)
            s = slice(first, min(max(ends[i + 1], first), n))
            if (S[i] == fill).all():
                assert first != s.stop and any(b < a for a, b in zip(ends, ends[1:])), (ends, i)
                continue
            _, want = reference(q[s], k[s], v[s], gate[s], beta[s], torch.zeros_like(S[0]))
            close(S[i], want, tol(64), f"state {i} of {ends}")
    cu = torch.tensor(calls[0], dtype=torch.int32).cuda()
    S = torch.full((5, hv, 64, 64), fill, device="cuda")
    out = g.delta_prefill(q, k, v, gate, beta, cu, state_out=S)
    for i, s in ((0, slice(0, 140)), (1, slice(140, 290))):
        o, want = reference(q[s], k[s], v[s], gate[s], beta[s], torch.zeros_like(S[0]))
        close(S[i], want, tol(64), f"state {i}")
        close(out[s][:60], o[:60], tol(64), f"o {i}")  # (rows from 200 on are two sequences')
    assert (S[2] == 0).all() and (S[3] == 0).all()
