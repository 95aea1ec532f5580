"""gdn_logits_process, gdn_sample_tokens and gdn_batch_sample against their
definitions in 64 bits on the host (gpu).

Tolerances: processing rounds at most six times to FP32 (division or product,
frequency times count, two differences, the bias, and what the 64-bit side
keeps of them), each half a step of 2^-23 of the largest intermediate, then
once to the type.  A log-probability is a difference of two FP32-exact numbers
and the logarithm of an FP32 sum of exponentials (2^-22 of it), rounded once.
Tokens are equal: their borders come from sums in 64 bits on both sides.
"""
import math

import numpy as np
import pytest
import torch

import gateddeltanet_amd as g

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def row_logits(rows, vocab, dtype, seed, spread=3.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (spread * torch.randn((rows, vocab), generator=gen, device="cuda")).to(dtype)


# ------------------------------------------------------------- processing

def process_ref(x, history=None, length=None, prompt=None, rep=None, pres=None, freq=None, bias=None, mask=None):
    """(result, largest intermediate) of one row in 64 bits; mask bool."""
    x = x.astype(np.float64).copy()
    big = np.abs(x)
    vocab = x.size
    if history is not None:
        h = history[:max(0, min(length, history.size))].astype(np.int64)
        inside = (h >= 0) & (h < vocab)
        place = np.arange(h.size)
        seen = np.unique(h[inside])
        x[seen] = np.where(x[seen] > 0, x[seen] / rep, x[seen] * rep)
        big = np.fmax(big, np.abs(x))
        said, times = np.unique(h[inside & (place >= prompt)], return_counts=True)
        x[said] -= freq * times + pres
        big[said] = np.fmax(big[said], np.abs(freq * times)) + abs(pres)
        big = np.fmax(big, np.abs(x))
    for t, v in (bias or {}).items():
        if 0 <= t < vocab:
            x[t] += v
            big[t] = max(big[t], abs(v), abs(x[t]))
    if mask is not None:
        x[~mask[:vocab]] = -np.inf
    return x, big


def check_rows(out, refs, dtype):
    half = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps  # a step below the normal numbers
    for r, (want, big) in enumerate(refs):
        got = out[r].double().cpu().numpy()
        fin = np.isfinite(want) & (np.abs(want) < torch.finfo(dtype).max)
        np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
        rest = ~np.isfinite(want) & ~np.isnan(want)
        np.testing.assert_array_equal(got[rest], want[rest])
        err = np.abs(got[fin] - want[fin])
        assert (err <= 6 * 2.0**-24 * big[fin] + half * np.abs(want[fin]) * (1 + 2.0**-10) + tiny).all(), (r, err.max())


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 7), (2, 33), (1, 8192), (2, 8193), (5, 32000), (2, 40001)])
def test_process(kind, rows, vocab):
    dtype = TYPES[kind]
    rng = np.random.default_rng(vocab)
    x = row_logits(rows, vocab, dtype, vocab)
    width = 300
    # ids outside the vocabulary among them; few distinct ones, so they repeat
    hist = rng.integers(-3, min(vocab, 90) + 3, (rows, width)).astype(np.int32)
    hist[:, ::5] = vocab - 1 - hist[:, ::5]
    length = rng.integers(0, width + 1, rows).astype(np.int32)
    length[0] = width
    prompt = (length // 2).astype(np.int32)
    rep, pres, freq = (rng.uniform(a, b, rows).astype(np.float32) for a, b in ((0.7, 1.5), (-0.5, 1), (-0.2, 0.5)))
    bias = [{int(t): float(np.float32(rng.normal())) for t in rng.integers(0, vocab, r % 4)} for r in range(rows)]
    offsets = np.cumsum([0] + [len(b) for b in bias])
    mask = rng.random((rows, (vocab + 31) // 32 * 32)) < 0.7
    words = np.packbits(mask, axis=1, bitorder="little").view(np.int32)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    out = g.logits_process(
        x, history=dev(hist), history_len=dev(length), prompt_len=dev(prompt), repetition=dev(rep), presence=dev(pres),
        frequency=dev(freq), mask=dev(words),
        bias=(dev(offsets.astype(np.int32)), dev(np.array([t for b in bias for t in b], np.int32)),
              dev(np.array([v for b in bias for v in b.values()], np.float32))))
    xs = x.float().cpu().numpy()
    check_rows(out, [process_ref(xs[r], hist[r], length[r], prompt[r], rep[r], pres[r], freq[r], bias[r], mask[r])
                     for r in range(rows)], dtype)


def test_process_parts_off_and_in_place():
    x = row_logits(3, 5000, torch.float32, 1)
    assert torch.equal(g.logits_process(x), x)
    hist = torch.tensor([[5, 5, 9], [1, 2, 3], [7, 7, 7]], dtype=torch.int32).cuda()
    n = torch.tensor([3, 0, 2], dtype=torch.int32).cuda()
    f = torch.tensor([0.5, 0.5, 0.25]).cuda()
    want = x.clone()
    want[0, 5] -= 1.0
    want[0, 9] -= 0.5
    want[2, 7] -= 0.5
    assert torch.equal(g.logits_process(x, history=hist, history_len=n, frequency=f), want)
    y = x.clone()
    assert g.logits_process(y, history=hist, history_len=n, frequency=f, out=y) is y
    assert torch.equal(y, want)
    assert torch.equal(g.logits_process(x, history=hist, history_len=n), x)


def test_process_lengths_are_held_to_the_width():
    x = row_logits(3, 100, torch.float32, 2)
    hist = torch.tensor([[3, 4], [3, 4], [3, 4]], dtype=torch.int32).cuda()
    n = torch.tensor([2**31 - 1, -5, 2], dtype=torch.int32).cuda()
    prompt = torch.tensor([1, 0, 2**31 - 1], dtype=torch.int32).cuda()
    p = torch.ones(3).cuda()
    want = x.clone()
    want[0, 4] -= 1.0
    assert torch.equal(g.logits_process(x, history=hist, history_len=n, prompt_len=prompt, presence=p), want)


def test_process_bias_repeats_and_bad_entries():
    """Of equal ids the last entry holds; ids outside the vocabulary and
    offsets past the entries are skipped."""
    x = torch.zeros((3, 64)).cuda()
    ids = torch.tensor([5, 5, 5, -1, 64, 2**31 - 1, 6], dtype=torch.int32).cuda()
    val = torch.tensor([1.0, 2.0, 3.0, 9.0, 9.0, 9.0, 4.0]).cuda()
    off = torch.tensor([0, 6, 100, 3], dtype=torch.int32).cuda()
    out = g.logits_process(x, bias=(off, ids, val))
    want = torch.zeros((3, 64)).cuda()
    want[0, 5], want[1, 6] = 3.0, 4.0
    assert torch.equal(out, want)
    none = torch.zeros(0, dtype=torch.int32).cuda()
    assert torch.equal(g.logits_process(x, bias=(torch.zeros(4, dtype=torch.int32).cuda(), none, none.float())), x)


def test_process_masks():
    """Shared masks, rows without one, rows with nothing allowed, and masked
    places that hold NaN, infinities and the type's lowest value."""
    vocab = 70
    x = row_logits(5, vocab, torch.float32, 3)
    x[:, 0], x[:, 1], x[:, 2], x[:, 3] = math.nan, math.inf, -math.inf, torch.finfo(torch.float32).min
    masks = torch.zeros((2, 3), dtype=torch.int32)
    masks[1, 0], masks[1, 2] = 0x7ffffff0, -1  # bits past the vocabulary do not matter
    index = torch.tensor([1, 0, -1, 2, 1], dtype=torch.int32).cuda()
    out = g.logits_process(x, mask=masks.cuda(), mask_index=index)
    allowed = torch.zeros(vocab, dtype=torch.bool)
    allowed[4:31] = allowed[64:] = True
    assert (out[1] == -math.inf).all()
    for r in (0, 4):
        assert torch.equal(out[r][allowed], x[r][allowed]) and (out[r][~allowed] == -math.inf).all()
    for r in (2, 3):
        assert torch.equal(out[r][1:], x[r][1:]) and torch.isnan(out[r][0])


@pytest.mark.parametrize("kind", list(TYPES))
def test_process_strided_rows_at_any_address(kind):
    dtype = TYPES[kind]
    wide = row_logits(4, 1030, dtype, 5)
    into = torch.full((4, 1111), 7.0, dtype=dtype).cuda()
    x, out = wide[:, 3:1004], into[:, 1:1002]
    hist = torch.arange(4000, dtype=torch.int32).view(4, 1000).remainder(1001).cuda()
    n = torch.full((4,), 900, dtype=torch.int32).cuda()
    rep = torch.full((4,), 1.3).cuda()
    want = g.logits_process(x.contiguous(), history=hist[:, :900].contiguous(), history_len=n, repetition=rep)
    g.logits_process(x, history=hist[:, :900], history_len=n, repetition=rep, out=out)
    assert torch.equal(out, want)
    assert (into[:, 0] == 7).all() and (into[:, 1002:] == 7).all()


def test_process_long_history():
    x = row_logits(2, 3000, torch.float32, 6)
    rng = np.random.default_rng(6)
    hist = rng.integers(0, 2, (2, 150000)).astype(np.int32)
    n = np.array([150000, 70001], np.int32)
    f = np.array([2.0**-10, 2.0**-9], np.float32)
    out = g.logits_process(x, history=torch.from_numpy(hist).cuda(), history_len=torch.from_numpy(n).cuda(),
                           frequency=torch.from_numpy(f).cuda())
    xs = x.cpu().numpy()
    check_rows(out, [process_ref(xs[r], hist[r], n[r], 0, 1.0, 0.0, f[r]) for r in range(2)], torch.float32)


# --------------------------------------------------------------- the draw

def sample_ref(x, u, temp, k, p, mp):
    """Token and log-probability of one row in 64 bits."""
    x = x.astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    if top == -np.inf:
        return -1, -math.inf
    with np.errstate(invalid="ignore"):
        d = np.where(x == top, 0.0, top - x)
    lse = math.log(np.exp(-d).sum())
    order = np.argsort(d, kind="stable")
    if not temp > 0:
        return int(order[0]), -lse
    with np.errstate(over="ignore", invalid="ignore"):
        w = np.exp(-d / np.float64(np.float32(temp)))
    w = np.where(np.isinf(d), 0.0, w)
    ranked = w[order]
    keep = np.ones(x.size, bool)
    if k > 0:
        keep[k:] = False
    p = np.float64(np.float32(p))
    if p < 1:
        m = np.where(keep, ranked, 0.0)
        before = np.concatenate([[0.0], np.cumsum(m)[:-1]])
        keep &= before < p * m.sum()
        keep[0] = True
    keep &= ranked >= min(np.float64(np.float32(mp)), 1.0)
    weight = np.zeros(x.size)
    weight[order[keep]] = ranked[keep]
    run = np.cumsum(weight)
    t = int(np.searchsorted(run, np.float64(np.float32(u)) * run[-1], side="right"))
    t = min(t, int(np.nonzero(weight)[0][-1]))
    return t, -float(d[t]) - lse


def check_sample(x, u, temp, k=None, p=None, mp=None):
    rows = x.shape[0]
    f = lambda a: None if a is None else torch.tensor(a, dtype=torch.float32).cuda()  # noqa: E731
    tok, lp = g.sample_tokens(x, f(u), temperature=f(temp), top_p=f(p), min_p=f(mp),
                              top_k=None if k is None else torch.tensor(k, dtype=torch.int32).cuda())
    xs = x.float().cpu().numpy()
    for r in range(rows):
        want = sample_ref(xs[r], u[r], temp[r], k[r] if k else 0, p[r] if p else 1.0, mp[r] if mp else 0.0)
        assert int(tok[r]) == want[0], (r, int(tok[r]), want, temp[r], k and k[r], p and p[r], mp and mp[r], u[r])
        if want[0] >= 0:
            assert abs(float(lp[r]) - want[1]) <= 2.0**-22 + 2.0**-23 * abs(want[1]), (r, float(lp[r]), want[1])
        else:
            assert float(lp[r]) == -math.inf
    return tok


def settings(rows, seed):
    rng = np.random.default_rng(seed)
    u = rng.random(rows).astype(np.float32).tolist()
    temp = rng.uniform(0.3, 2.0, rows).astype(np.float32).tolist()
    k = rng.choice([0, 1, 2, 5, 50, 1000, 10**6], rows).tolist()
    p = rng.choice([0.0, 0.1, 0.5, 0.9, 0.99, 1.0, 2.0], rows).astype(np.float32).tolist()
    mp = rng.choice([0.0, 0.001, 0.05, 0.5, 1.0, 3.0], rows).astype(np.float32).tolist()
    return u, temp, k, p, mp


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("vocab", [1, 2, 5, 63, 256, 257, 1000, 8192, 8193, 32000, 32768, 32769, 50001])
def test_sample(kind, vocab):
    rows = 24
    x = row_logits(rows, vocab, TYPES[kind], vocab)
    u, temp, k, p, mp = settings(rows, vocab)
    check_sample(x, u, temp)
    check_sample(x, u, temp, k=k)
    check_sample(x, u, temp, p=p)
    check_sample(x, u, temp, mp=mp)
    check_sample(x, u, temp, k, p, mp)


@pytest.mark.parametrize("vocab", [131072, 300007, 1 << 20])
def test_sample_wide(vocab):
    x = row_logits(6, vocab, torch.bfloat16, vocab)
    u, temp, k, p, mp = settings(6, vocab)
    check_sample(x, u, temp, p=[0.9, 0.99, 0.5, 0.999, 1.0, 0.1])
    check_sample(x, u, temp, k, p, mp)


def test_sample_flat_rows():
    """Equal logits: the border is one key's, drawn by index."""
    rows, vocab = 8, 33000
    x = torch.full((rows, vocab), -3.5).cuda()
    x[4:, ::2] = -4.0
    u = [0.0, 0.25, 0.5, 0.999, 0.1, 0.6, 0.75, 0.9]
    temp = [1.0, 0.5, 2.0, 1.0, 1.0, 0.7, 1.0, 3.0]
    # powers of two, so that the shares of equal weights are exact on both sides
    check_sample(x, u, temp, p=[0.5, 0.25, 0.125, 0.75, 0.5, 0.5, 0.25, 0.5])
    check_sample(x, u, temp, k=[1, 7, 20000, 32999, 16500, 16501, 16499, 3])
    check_sample(x, u, temp, k=[1, 7, 20000, 32999, 16500, 16501, 16499, 3], mp=[0.5] * 8)


def test_sample_narrow_steps():
    """Logits that share one step of the first histogram and differ in the
    last bits."""
    rng = np.random.default_rng(1)
    base = np.float32(5.0).view(np.uint32)
    x = torch.from_numpy((base + rng.integers(0, 4000, (4, 20000)).astype(np.uint32)).view(np.float32)).cuda()
    u = [0.2, 0.4, 0.6, 0.8]
    check_sample(x, u, [1.0] * 4, k=[5, 500, 10000, 19999])
    check_sample(x, u, [1.0] * 4, k=[0, 500, 0, 19999], p=[0.3, 0.5, 0.9, 0.01])


def test_sample_negative_and_mixed_signs():
    x = row_logits(8, 3000, torch.float32, 8, spread=0.01)  # around zero, both zeros among them
    x[:, 10], x[:, 20] = 0.0, -0.0
    u, temp, k, p, mp = settings(8, 8)
    check_sample(x, u, [0.01] * 8, k, p, mp)
    check_sample(x - 1000.0, u, temp, k, p, mp)


def test_sample_ends():
    """Rows with nothing to choose, infinities, NaN, the type's lowest value;
    temperatures and draws at and past their ends."""
    inf, nan, low = math.inf, math.nan, torch.finfo(torch.float32).min
    x = torch.tensor([[-inf] * 6, [nan] * 6, [nan, -inf, nan, -inf, nan, -inf], [nan, 1, nan, 0, 1, -inf],
                      [1, inf, 0, inf, nan, -inf], [low] * 6, [-inf, -inf, low, -inf, low, nan],
                      [3.4e38, -3.4e38, 0, 1, 2, 3]]).cuda()
    for temp in (0.0, -1.0, nan, 1e-30, 1e-6, 1.0, 1e30, inf):
        for u in (0.0, 0.5, 1.0 - 2.0**-24):
            check_sample(x, [u] * 8, [temp] * 8)
            check_sample(x, [u] * 8, [temp] * 8, k=[2] * 8, p=[0.5] * 8, mp=[0.1] * 8)
    one = torch.full((8,), 1.0).cuda()
    last = g.sample_tokens(x, one * 1.0, temperature=one)[0].tolist()  # 1 is past the end: the last that counts
    assert last == [-1, -1, -1, 4, 3, 5, 4, 0]
    assert g.sample_tokens(x, one * nan, temperature=one)[0].tolist() == [-1, -1, -1, 1, 1, 0, 2, 0]
    assert g.sample_tokens(x)[0].tolist() == [-1, -1, -1, 1, 1, 0, 2, 0]


def test_sample_strided_rows_at_any_address():
    wide = row_logits(5, 3000, torch.bfloat16, 11)
    x = wide[:, 1:2990]
    u, temp, k, p, mp = settings(5, 11)
    check_sample(x, u, temp, k, p, mp)


def test_sample_without_logprobs_and_into_the_callers_tensors():
    import ctypes

    from gateddeltanet_amd import _lib

    for vocab, dtype in ((5000, torch.float32), (70000, torch.bfloat16)):
        x = row_logits(4, vocab, dtype, 21)
        u = torch.tensor([0.1, 0.4, 0.7, 0.95]).cuda()
        temp = torch.tensor([0.0, 0.7, 1.0, 1.5]).cuda()
        p = torch.tensor([0.9, 0.5, 0.99, 1.0]).cuda()
        want, lp = g.sample_tokens(x, u, temperature=temp, top_p=p)
        tokens, logprobs = torch.zeros(4, dtype=torch.int32).cuda(), torch.zeros(4).cuda()
        got = g.sample_tokens(x, u, temperature=temp, top_p=p, tokens=tokens, logprobs=logprobs)
        assert got[0] is tokens and got[1] is logprobs and torch.equal(tokens, want) and torch.equal(logprobs, lp)
        tokens.zero_()
        a = _lib.GDNSample({torch.float32: 2, torch.bfloat16: 0}[dtype], 4, vocab, 0, vocab, x.data_ptr(), u.data_ptr(),
                           temp.data_ptr(), 0, p.data_ptr(), 0, tokens.data_ptr(), 0)
        lib = _lib.load()
        ws = torch.empty(lib.gdn_sample_workspace(ctypes.byref(a)) + 16, dtype=torch.uint8).cuda()
        assert lib.gdn_sample_tokens(ctypes.byref(a), ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(tokens, want)


@pytest.mark.parametrize("rows", [1, 20, 300, 600])
def test_sample_wide_batches(rows):
    """Long rows in 32 slices, fewer, and one."""
    x = row_logits(rows, 33000, torch.float32, rows)
    u, temp, k, p, mp = settings(rows, rows)
    check_sample(x, u, temp, k, p, mp)


def test_sample_top_p_alone_on_both_sides_of_its_estimate():
    """Borders among the few highest tokens, in the bulk, and on a border
    between tokens that FP32 cannot tell apart: equal weights of which the
    share is a whole number."""
    x = row_logits(12, 30000, torch.float32, 31, spread=2.0)
    x[:, 100] += 14.0
    u = [i / 12 for i in range(12)]
    for temp in (0.5, 1.0, 2.0):
        check_sample(x, u, [temp] * 12, p=[0.01, 0.1, 0.3, 0.5, 0.6, 0.7, 0.8, 0.9, 0.95, 0.99, 0.999, 0.9999])
    y = torch.full((6, 20000), -30.0).cuda()
    y[:, 7:8 + 63] = 5.0  # 64 equal tokens, the others at e^-35
    check_sample(y, u[:6], [1.0] * 6, p=[0.125, 0.25, 0.5, 0.75, 0.015625, 0.984375])


@pytest.mark.parametrize("kind", TYPES)
def test_sample_keeps_more_and_less_than_it_gathers(kind):
    """Kept tokens by the thousand, on both sides of what LDS lists hold."""
    x = row_logits(10, 20000, TYPES[kind], 61, spread=0.7)
    def f(*a):
        return np.array(a, np.float32).tolist()

    u = f(*(0.05 + i / 11 for i in range(10)))
    k = [1000, 1400, 1500, 1530, 1536, 1540, 1600, 2000, 5000, 0]
    check_sample(x, u, [1.0] * 10, k=k)
    check_sample(x, u, f(*[1.3] * 10), k=k, p=f(0.5, 0.99, 0.9, 1.0, 0.999, 0.7, 0.95, 0.8, 0.3, 0.2))
    check_sample(x, u, [1.0] * 10, p=f(0.1, 0.12, 0.14, 0.16, 0.18, 0.2, 0.22, 0.24, 0.26, 0.3),
                 mp=f(0.0, 0.3) * 5)


def test_two_streams_at_once():
    """Calls of all operators on two streams do not share anything."""
    from test_gpu_delta import inputs

    def work(seed):
        data = inputs(300, 1, 2, 128, 128, torch.float16, seed)
        cu = torch.tensor([0, 100, 300], dtype=torch.int32).cuda()
        S = torch.zeros((2, 2, 128, 128), device="cuda")
        x = row_logits(6, 70000, torch.bfloat16, seed)
        u, t, p = (torch.full((6,), v).cuda() for v in (0.3, 0.9, 0.95))
        h = torch.arange(600, dtype=torch.int32).cuda().view(6, 100)
        n = torch.full((6,), 100, dtype=torch.int32).cuda()
        torch.cuda.synchronize()

        def go():
            o = g.delta_prefill(*data, cu, state_out=S)
            o2 = g.delta_step(*(z[:2] for z in data), S)
            y = g.logits_process(x, history=h, history_len=n, presence=t)
            return [o, o2, S.clone(), y, *g.sample_tokens(y, u, temperature=t, top_p=p)]
        return go

    a, b = work(1), work(2)
    want = [[z.clone() for z in f()] for f in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for f, s in zip((a, b), streams):
            with torch.cuda.stream(s):
                got.append(f())
        torch.cuda.synchronize()
        for w, z in zip(want, got):
            assert all(torch.equal(i, j) for i, j in zip(w, z))


def test_wide_rows_captured():
    x = row_logits(3, 100001, torch.bfloat16, 41)
    u, t, p = (torch.full((3,), v).cuda() for v in (0.3, 1.1, 0.9))
    k = torch.tensor([0, 50, 3], dtype=torch.int32).cuda()

    def work():
        return g.sample_tokens(x, u, temperature=t, top_p=p, top_k=k)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = work()
    for seed in range(4):
        x.copy_(row_logits(3, 100001, torch.bfloat16, 50 + seed))
        u.fill_(0.2 * (seed + 1))
        want = [z.clone() for z in work()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured[0], want[0]) and torch.equal(captured[1], want[1])


def test_sample_follows_the_distribution():
    """Evenly spread draws meet each token as often as its probability."""
    x = torch.tensor([[0.0, 1.0, 2.0, -1.0]]).cuda().expand(4096, 4).contiguous()
    u = (torch.arange(4096) + 0.5).div(4096).float().cuda()
    tok = g.sample_tokens(x, u, temperature=torch.ones(4096).cuda())[0].cpu().numpy()
    want = torch.softmax(x[0].double(), 0).cpu().numpy() * 4096
    assert np.abs(np.bincount(tok, minlength=4) - want).max() <= 1


def test_run_of_all_and_captured():
    """Packed prompts, then two tokens a sequence: recurrence, a projection to
    logits, processing, the draw -- against 64 bits, and captured into a graph
    that is replayed between eager passes."""
    from test_gpu_delta import inputs, reference

    lens, hq, hv, d, vocab, n = [37, 1, 90], 2, 2, 64, 700, 3
    total = sum(lens)
    gen = torch.Generator(device="cuda").manual_seed(5)
    W = torch.randn((hv * d, vocab), generator=gen, device="cuda")
    data = inputs(total, hq, hv, d, d, torch.float32, 30)
    steps = [inputs(n, hq, hv, d, d, torch.float32, 31 + i) for i in range(2)]
    us = [torch.rand(n, generator=gen, device="cuda") for _ in range(2)]
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    S = torch.zeros((n, hv, d, d), device="cuda")
    history = torch.zeros((n, 8), dtype=torch.int32, device="cuda")
    mask = torch.randint(-2**31, 2**31, (n, (vocab + 31) // 32), generator=gen, device="cuda").to(torch.int32)
    vals = [torch.full((n,), v, device="cuda") for v in (1.2, 0.5, 0.25, 0.8, 0.9)]
    k50 = torch.full((n,), 50, dtype=torch.int32, device="cuda")

    def work():
        g.delta_prefill(*data, cu, state_out=S)
        got = []
        for i in range(2):
            o = g.delta_step(*steps[i], S)
            x = 4.0 * (o.reshape(n, -1) @ W)
            length = torch.full((n,), i, dtype=torch.int32, device="cuda")
            y = g.logits_process(x, history=history, history_len=length, repetition=vals[0], presence=vals[1],
                                 frequency=vals[2], mask=mask)
            tok, lp = g.sample_tokens(y, us[i], temperature=vals[3], top_k=k50, top_p=vals[4])
            history[:, i] = tok
            got += [o, x, y, tok, lp]
        return got

    got = work()
    at = 0
    states = []
    for m in lens:
        s = slice(at, at + m)
        states.append(reference(*(x[s] for x in data), torch.zeros_like(S[0]))[1])
        at += m
    bits = np.unpackbits(mask.cpu().numpy().view(np.uint8), axis=1, bitorder="little").astype(bool)
    said = [[] for _ in range(n)]
    for i in range(2):
        for r in range(n):
            o, states[r] = reference(*(x[r:r + 1] for x in steps[i]), states[r])
            assert (got[5 * i][r].double() - o[0]).abs().max() <= 1e-5 * o.abs().max()
            x = got[5 * i + 1][r].cpu().numpy()
            y, _ = process_ref(x, np.array(said[r], np.int64), i, 0, np.float32(1.2), 0.5, 0.25, mask=bits[r])
            t, lp = sample_ref(y, float(us[i][r]), 0.8, 50, 0.9, 0.0)
            assert int(got[5 * i + 3][r]) == t and abs(float(got[5 * i + 4][r]) - lp) < 1e-5
            said[r].append(t)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = work()
    for seed in range(3):
        for u in us:
            u.copy_(torch.rand(n, generator=gen, device="cuda"))
        want = [x.clone() for x in work()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        # the library product may choose another order in a graph; what the
        # operators make of its logits has to be theirs
        assert torch.equal(captured[0], want[0]) and torch.equal(captured[5], want[5])
        if torch.equal(captured[1], want[1]):
            assert all(torch.equal(a, b) for a, b in zip(captured[:5], want[:5]))


def test_tensor_refusals():
    x = row_logits(2, 100, torch.float32, 1)
    i2, f2 = torch.zeros(2, dtype=torch.int32).cuda(), torch.zeros(2).cuda()
    h = torch.zeros((2, 4), dtype=torch.int32).cuda()
    m = torch.zeros((2, 4), dtype=torch.int32).cuda()
    o3 = torch.zeros(3, dtype=torch.int32).cuda()
    for kw in (dict(history=h), dict(history_len=i2), dict(repetition=f2), dict(history=h, history_len=f2),
               dict(history=h.long(), history_len=i2), dict(history=h[:1], history_len=i2),
               dict(history=h, history_len=i2, presence=f2[:1]), dict(history=h, history_len=i2, frequency=f2.double()),
               dict(bias=(i2, i2, f2)), dict(bias=(o3, i2, f2[:1])), dict(bias=(o3, i2.cpu(), f2)),
               dict(mask=m[:, :3]), dict(mask=m[:1]), dict(mask=m.long()), dict(mask_index=i2),
               dict(mask=m, mask_index=o3), dict(out=x.half()), dict(out=x[:1]), dict(out=x.cpu())):
        with pytest.raises(g.GDNError):
            g.logits_process(x, **kw)
    for bad in (x.double(), x[0], x.t(), x.cpu()):
        with pytest.raises(g.GDNError):
            g.logits_process(bad)
        with pytest.raises(g.GDNError):
            g.sample_tokens(bad)
    for kw in (dict(temperature=f2), dict(temperature=f2[:1]), dict(top_k=f2), dict(top_p=i2), dict(tokens=o3),
               dict(logprobs=f2.half()), dict(uniform=f2.cpu())):
        with pytest.raises(g.GDNError):
            g.sample_tokens(x, **kw)


# ----------------------------------------------------------- the engine's path

def test_batch_sample():
    """BatchState.sample over the streams' own logits."""
    m = g.Model.synth(num_layers=1, seed=3)
    n = 5
    bs = g.BatchState(m, n)
    try:
        rng = np.random.default_rng(2)
        greedy = bs.step(rng.integers(0, 32000, n))
        logits = np.stack([bs.logits(s) for s in range(n)])
        tok, lp = bs.sample()
        np.testing.assert_array_equal(tok, greedy)
        u, temp, k, p, mp = settings(n, 1)
        histories = [rng.integers(0, 40, c).tolist() for c in (0, 1, 30, 200, 7)]
        histories[3][:5] = np.argsort(logits[3])[-5:].tolist()
        prompt = [0, 1, 10, 0, 9]
        biases = [{}, {5: 2.5}, {}, {int(greedy[3]): -30.0, 77: 1.0}, {}]
        mask = rng.random((n, 32000)) < 0.5
        mask[4] = False
        tok, lp = bs.sample(u, temperature=temp, top_k=k, top_p=p, min_p=mp, repetition=1.3, presence=0.2,
                            frequency=[0.1] * n, histories=histories, prompt_len=prompt, biases=biases, mask=mask)
        for s in range(n):
            y, _ = process_ref(logits[s], np.array(histories[s], np.int64), len(histories[s]), prompt[s],
                               np.float32(1.3), np.float32(0.2), np.float32(0.1), biases[s], mask[s])
            t, want = sample_ref(y.astype(np.float32), u[s], temp[s], k[s], p[s], mp[s])
            assert tok[s] == t and (t < 0 or abs(lp[s] - want) < 1e-5), (s, tok[s], t, lp[s], want)
        assert tok[4] == -1 and lp[4] == -math.inf
        for s in range(n):
            np.testing.assert_array_equal(bs.logits(s), logits[s])  # as they were
        again, _ = bs.sample(u, temperature=1.0, histories=[[]] * n, repetition=1.1)
        plain, _ = bs.sample(u, temperature=1.0)
        np.testing.assert_array_equal(again, plain)
        for kw in (dict(temperature=1.0), dict(repetition=1.1), dict(prompt_len=0)):
            with pytest.raises(g.GDNError):
                bs.sample(**kw)
        with pytest.raises(g.GDNError):
            bs.sample(histories=[[1]])
    finally:
        bs.free()
        m.free()


def test_batch_sample_after_a_prefill_and_its_refusals():
    m = g.Model.synth(num_layers=1, seed=3)
    bs = g.BatchState(m, 3)
    try:
        bs.step([1, 2, 3])
        seed = bs.prefill(1, [5, 6, 7, 8])
        tok, lp = bs.sample()
        assert tok[1] == seed
        for s in range(3):
            x = bs.logits(s).astype(np.float64)
            assert tok[s] == x.argmax() and abs(lp[s] + np.log(np.exp(x - x.max()).sum())) < 1e-5
        one = np.ones(32000, bool)
        one[tok[0]] = False
        again, _ = bs.sample(mask=one)  # one mask for all
        assert again[0] != tok[0] and (bs.sample(mask=one[None])[0] == again).all()
        for kw in (dict(mask=True), dict(mask=np.ones((2, 32000), bool)), dict(mask=one[:-1]), dict(top_k=[1, 2]),
                   dict(temperature=[0.0] * 4, uniform=0.0), dict(histories=[[1 << 40], [], []]),
                   dict(biases=[{}, {}]), dict(histories=[[], []])):
            with pytest.raises(g.GDNError):
                bs.sample(**kw)
    finally:
        bs.free()
        m.free()


def test_process_refuses_fewer_masks_than_rows():
    x = torch.zeros((2, 64)).cuda()
    for n in (0, 1):
        with pytest.raises(g.GDNError, match="masks for 2 rows"):
            g.logits_process(x, mask=torch.zeros((n, 2), dtype=torch.int32).cuda())


def test_batch_sample_of_a_large_vocabulary():
    """Rows of logits longer than LDS: a workspace behind the call's arrays."""
    from gateddeltanet_amd.engine import default_config

    cfg = default_config(1)
    cfg.vocab_size = 40000
    m = g.Model.synth(config=cfg, seed=4)
    n = 3
    bs = g.BatchState(m, n)
    try:
        greedy = bs.step([1, 2, 39999])
        logits = np.stack([bs.logits(s) for s in range(n)])
        for _ in range(2):
            tok, lp = bs.sample()
            np.testing.assert_array_equal(tok, greedy)
            u, temp, k, p, mp = settings(n, 7)
            mask = np.random.default_rng(5).random((n, 40000)) < 0.7
            tok, lp = bs.sample(u, temperature=temp, top_k=k, top_p=p, min_p=mp, histories=[[39999] * 5, [], [7]],
                                frequency=0.5, mask=mask)
            for s in range(n):
                hist = [[39999] * 5, [], [7]][s]
                y, _ = process_ref(logits[s], np.array(hist, np.int64), len(hist), 0, np.float32(1), np.float32(0),
                                   np.float32(0.5), {}, mask[s])
                t, want = sample_ref(y.astype(np.float32), u[s], temp[s], k[s], p[s], mp[s])
                assert tok[s] == t and abs(lp[s] - want) < 1e-5, (s, tok[s], t, lp[s], want)
    finally:
        bs.free()
        m.free()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("vocab", [32768, 261999, 2**18, 2**18 + 1, 2**20 - 1, 2**20])
def test_sample_of_a_flat_row_reaches_every_token(kind, vocab):
    """Equal weights, of equal logits or of an infinite temperature: their sum
    is the largest there is, 2^63 at 2^18 and at 2^20 tokens."""
    us = [0.0, 0.5, 0.998, 0.999, float(np.float32(1 - 2.0**-24))]
    n = len(us)
    flat = torch.full((n, vocab), 0.75, dtype=TYPES[kind], device="cuda")
    spread = row_logits(n, vocab, TYPES[kind], vocab)
    want = [int(np.float64(np.float32(u)) * vocab) for u in us]
    assert want[-1] == vocab - 1
    assert check_sample(flat, us, [1.0] * n).tolist() == want
    assert check_sample(spread, us, [math.inf] * n).tolist() == want
    # a border among equals: the tokens before ceil(p vocab)
    kept = math.ceil(np.float64(np.float32(0.999)) * vocab)
    want = [int(np.float64(np.float32(u)) * kept) for u in us]
    assert check_sample(flat, us, [1.0] * n, p=[0.999] * n).tolist() == want


@pytest.mark.parametrize("kind,vocab", [("fp32", 1000), ("fp32", 32768), ("bf16", 65536), ("fp16", 65536), ("fp32", 40000)])
@pytest.mark.parametrize("temperature", [0.4, 1.0])
def test_sample_top_p_next_to_a_border(kind, vocab, temperature):
    """The FP32 numbers just below and above the share of the tokens before
    one, and others up to 3e-5 away: with the last token of the ranking at the
    end of the row, a number near 1 draws it exactly if it is kept."""
    ranks = [1, 2, 5, 13, 40, 100]
    off = [0.0, 3e-7, 1e-6, 3e-6, 8e-6, 1.2e-5, 3e-5]
    base = row_logits(len(ranks), vocab, TYPES[kind], vocab + 1, spread=2.0)
    xs, ps, keeps = [], [], []
    for x, j in zip(base, ranks):
        d = x.double().cpu().numpy()
        order = np.argsort(-d, kind="stable")
        # the border's token has no equal
        j = next((i for i in range(j, 0, -1) if d[order[i - 1]] > d[order[i]] > d[order[i + 1]]), None)
        if j is None:
            continue
        w = np.exp((d - d.max()) / np.float64(np.float32(temperature)))
        share = w[order[:j]].sum() / w.sum()
        x[[int(order[j]), vocab - 1]] = x[[vocab - 1, int(order[j])]]
        for e in off:
            below = np.nextafter(np.float32(share * (1 - e)), np.float32(0))
            above = np.nextafter(np.float32(share * (1 + e)), np.float32(1))
            for p, kept in ((below, False), (above, True)):
                assert abs(float(p) - share) > 1e-9 * share and (float(p) > share) == kept
                xs.append(x), ps.append(float(p)), keeps.append(kept)
    n = len(xs)
    assert n >= 2 * 3 * len(off)
    tok = check_sample(torch.stack(xs), [1 - 2.0**-24] * n, [temperature] * n, p=ps)
    assert [t == vocab - 1 for t in tok.tolist()] == keeps


@pytest.mark.parametrize("op", ["delta_prefill", "delta_step", "logits_process", "sample_tokens"])
def test_an_error_of_an_earlier_call_is_not_reported_as_a_launchs(op):
    """A HIP call of the program's own that failed (no device of that number)
    and was not asked about: the operators run, and leave its error to it."""
    from test_gpu_delta import inputs

    from gateddeltanet_amd import _lib

    hip = _lib.load()  # (resolves the runtime's symbols too)
    q = inputs(4, 1, 1, 64, 64, torch.float32, 3)
    S, out = torch.zeros((4, 1, 64, 64), device="cuda"), torch.empty((4, 1, 64), device="cuda")
    x = row_logits(4, 1000, torch.float32, 3)
    cu = torch.tensor([0, 4], dtype=torch.int32).cuda()
    ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    y, tok, lp = torch.empty_like(x), torch.empty(4, dtype=torch.int32, device="cuda"), torch.empty(4, device="cuda")
    call = {"delta_prefill": lambda: g.delta_prefill(*q, cu, out=out, workspace=ws),
            "delta_step": lambda: g.delta_step(*q, S, out=out), "logits_process": lambda: g.logits_process(x, out=y),
            "sample_tokens": lambda: g.sample_tokens(x, tokens=tok, logprobs=lp)}[op]
    call()
    torch.cuda.synchronize()
    hip.hipGetLastError()
    try:
        wrong = hip.hipSetDevice(1 << 20)
        assert wrong != 0
        call()
        assert hip.hipGetLastError() == wrong
    finally:
        hip.hipGetLastError()
    torch.cuda.synchronize()


def test_process_into_columns_beside_the_logits():
    """One buffer's columns, logits and output in turn: nothing is shared, so
    it is taken; shifted by a column or a row it would be, and is not."""
    both = row_logits(5, 2000, torch.float32, 8)
    x, out = both[:, :1000], both[:, 1000:]
    p = torch.ones(5).cuda()
    hist, n = torch.arange(5, dtype=torch.int32).view(5, 1).cuda(), torch.ones(5, dtype=torch.int32).cuda()
    want = x.clone()
    want[range(5), range(5)] -= 1.0
    g.logits_process(x, history=hist, history_len=n, presence=p, out=out)
    assert torch.equal(out, want)
    g.logits_process(x[1:], history=hist[1:], history_len=n[1:], presence=p[1:], out=out[:4])
    assert torch.equal(out[:4], want[1:])
    before = both.clone()
    for bad in (both[:, 1:1001], both[:, 999:1999]):
        with pytest.raises(g.GDNError):
            g.logits_process(x, out=bad)
    with pytest.raises(g.GDNError):
        g.logits_process(x[:4], out=x[1:])
    assert torch.equal(both, before)


def test_run_of_all_captured_is_the_eager_run_of_its_logits():
    """Two steps of recurrence, projection, processing and draw in a graph: of
    the logits that it formed, processed rows, tokens and log-probabilities are
    the eager calls', whatever order its library product took."""
    from test_gpu_delta import inputs

    n, hv, d, vocab = 3, 2, 64, 900
    gen = torch.Generator(device="cuda").manual_seed(15)
    W = torch.randn((hv * d, vocab), generator=gen, device="cuda")
    prompt = inputs(90, hv, hv, d, d, torch.float32, 40)
    steps = [inputs(n, hv, hv, d, d, torch.float32, 41 + i) for i in range(2)]
    us = [torch.rand(n, generator=gen, device="cuda") for _ in range(2)]
    cu = torch.tensor([0, 37, 37, 90], dtype=torch.int32).cuda()
    S = torch.zeros((n, hv, d, d), device="cuda")
    history = torch.zeros((n, 8), dtype=torch.int32, device="cuda")
    mask = torch.randint(-2**31, 2**31, (n, (vocab + 31) // 32), generator=gen, device="cuda").to(torch.int32)
    rep, pres, freq, temp, share = (torch.full((n,), v, device="cuda") for v in (1.2, 0.5, 0.25, 0.8, 0.9))
    lengths = [torch.full((n,), i, dtype=torch.int32, device="cuda") for i in range(2)]

    def token(i, x, ids):
        y = g.logits_process(x, history=ids, history_len=lengths[i], repetition=rep, presence=pres, frequency=freq, mask=mask)
        return [y, *g.sample_tokens(y, us[i], temperature=temp, top_p=share)]

    def work():
        g.delta_prefill(*prompt, cu, state_out=S)
        got = []
        for i in range(2):
            o = g.delta_step(*steps[i], S)
            x = 4.0 * (o.reshape(n, -1) @ W)
            got.append([o, x, *token(i, x, history)])
            history[:, i] = got[i][3]
        return got

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = work()
    for _ in range(4):
        for u in us:
            u.copy_(torch.rand(n, generator=gen, device="cuda"))
        eager = [o.clone() for o, *_ in work()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        ids = torch.zeros_like(history)
        for i, (o, x, y, tok, lp) in enumerate(captured):
            assert torch.equal(o, eager[i])
            want = token(i, x, ids)
            assert all(torch.equal(a, b) for a, b in zip((y, tok, lp), want)), i
            ids[:, i] = tok
        assert torch.equal(history, ids)
