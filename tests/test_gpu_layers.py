"""Whole layers from the operators, as a serving program runs them (gpu): a prompt,
then tokens one at a time, against the layer in 64 bits over all tokens at once.

Tolerance.  FP32 throughout: the projections' sums have up to 512 products, the
operators' tolerances (test_gpu_delta, test_gpu_scan, test_gpu_norm, test_gpu_conv)
are 3e-6 of a result at most, and norms pass errors on at their size; ten stages of
4 sqrt(512) 2^-24 = 5.4e-6 add up to 5.4e-5 of the largest value's order, taken as TOL
times the root mean square, times 8 for the largest of many.
"""
import pytest
import torch

import gateddeltanet_amd as g

pytestmark = pytest.mark.gpu

TOL = 5.4e-5
FP32 = torch.float32


def normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def close(got, want, what):
    rms = want.square().mean().sqrt()
    diff = (got.double() - want).abs()
    assert diff.max() <= 8 * TOL * rms and diff.square().mean().sqrt() <= TOL * rms, (what, float(diff.max() / rms))


def silu(x):
    return x * torch.sigmoid(x)


def normed(x, w=None, eps=1e-6):
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    return y if w is None else y * w


def conv64(x, w):
    z = torch.cat([torch.zeros_like(x[:w.shape[1] - 1]), x])
    return silu(sum(z[j:j + x.shape[0]] * w[:, j] for j in range(w.shape[1])))


def cumulative(lens):
    return torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()


HIDDEN, HEADS, DK, DV = 256, 2, 64, 128


def gdn_weights():
    gen = torch.Generator(device="cuda").manual_seed(1)
    wide = HEADS * (2 * DK + DV)
    return {"norm": 1 + 0.1 * normal(gen, HIDDEN), "proj": normal(gen, HIDDEN, wide + HEADS * DV + 2 * HEADS) / 16,
            "conv": 0.5 * normal(gen, wide, 4), "onorm": 1 + 0.1 * normal(gen, DV), "out": normal(gen, HEADS * DV, HIDDEN) / 16}


def gdn_parts(y):
    """q, k and v together, the gate, log decays, betas of a projection."""
    wide = HEADS * (2 * DK + DV)
    gate = y[:, wide:wide + HEADS * DV].unflatten(1, (HEADS, DV))
    a, b = y[:, -2 * HEADS:-HEADS], y[:, -HEADS:]
    return y[:, :wide], gate, -torch.nn.functional.softplus(a) * 0.3, torch.sigmoid(b)


def split_qkv(c):
    q, k, v = c.split([HEADS * DK, HEADS * DK, HEADS * DV], 1)
    return q.unflatten(1, (HEADS, DK)), k.unflatten(1, (HEADS, DK)), v.unflatten(1, (HEADS, DV))


def gdn_layer(w, x, residual, conv_state, state, cu, slots):
    """(out, residual stream) of packed prompts, or (cu None) a token a sequence."""
    h, residual = g.rms_norm(x, w["norm"], residual=residual)
    qkv, gate, decay, beta = gdn_parts(h @ w["proj"])
    if cu is None:
        c = g.conv_step(qkv, w["conv"], conv_state, slots=slots)
        q, k, v = split_qkv(c)
        o = g.delta_step(q, k, v, decay.contiguous(), beta.contiguous(), state, slots=slots)
    else:
        c = g.conv_prefill(qkv, w["conv"], cu, state_in=conv_state, state_out=conv_state, slots=slots)
        q, k, v = split_qkv(c)
        o = g.delta_prefill(q, k, v, decay.contiguous(), beta.contiguous(), cu, state_in=state, state_out=state, slots=slots)
    o = g.rms_norm(o, w["onorm"], gate=gate)
    return o.flatten(1) @ w["out"], residual


def gdn_layer64(w, x, residual):
    w = {k: v.double() for k, v in w.items()}
    residual = x.double() + residual.double()
    qkv, gate, decay, beta = gdn_parts(normed(residual, w["norm"]) @ w["proj"])
    q, k, v = split_qkv(conv64(qkv, w["conv"]))
    q, k = (t / (t.square().sum(-1, keepdim=True) + 1e-6).sqrt() for t in (q, k))
    S, o = torch.zeros((HEADS, DK, DV), dtype=torch.float64, device="cuda"), torch.zeros_like(v)
    for t in range(x.shape[0]):
        S = S * decay[t].exp()[:, None, None]
        d = beta[t, :, None] * (v[t] - (S * k[t][..., None]).sum(1))
        S = S + k[t][..., None] * d[:, None]
        o[t] = DK**-0.5 * (S * q[t][..., None]).sum(1)
    o = normed(o, w["onorm"]) * silu(gate)
    return o.flatten(1) @ w["out"], residual


STATE, DIM, SHEADS = 64, 64, 4


def scan_weights():
    gen = torch.Generator(device="cuda").manual_seed(2)
    inner, wide = SHEADS * DIM, SHEADS * DIM + 2 * STATE
    return {"norm": 1 + 0.1 * normal(gen, HIDDEN), "proj": normal(gen, HIDDEN, wide + inner + SHEADS) / 16,
            "conv": 0.5 * normal(gen, wide, 4), "A": -1 - 7 * torch.rand(SHEADS, generator=gen, device="cuda"),
            "D": normal(gen, SHEADS), "dt_bias": -3 + normal(gen, SHEADS), "onorm": 1 + 0.1 * normal(gen, inner),
            "out": normal(gen, inner, HIDDEN) / 16}


def scan_parts(y):
    wide = SHEADS * DIM + 2 * STATE
    return y[:, :wide], y[:, wide:wide + SHEADS * DIM], y[:, -SHEADS:]


def split_xbc(c):
    x, B, C = c.split([SHEADS * DIM, STATE, STATE], 1)
    return x.unflatten(1, (SHEADS, DIM)), B[:, None], C[:, None]


def scan_layer(w, x, residual, conv_state, state, cu, slots):
    h, residual = g.rms_norm(x, w["norm"], residual=residual)
    xbc, z, dt = scan_parts(h @ w["proj"])
    if cu is None:
        u, B, C = split_xbc(g.conv_step(xbc, w["conv"], conv_state, slots=slots))
        y = g.scan_step(u, dt, w["A"], B, C, state, D=w["D"], dt_bias=w["dt_bias"], softplus=True, slots=slots)
    else:
        u, B, C = split_xbc(g.conv_prefill(xbc, w["conv"], cu, state_in=conv_state, state_out=conv_state, slots=slots))
        y = g.scan_prefill(u, dt, w["A"], B, C, cu, D=w["D"], dt_bias=w["dt_bias"], softplus=True, state_in=state,
                           state_out=state, slots=slots)
    y = g.rms_norm(y.flatten(1), w["onorm"], gate=z, gate_first=True)
    return y @ w["out"], residual


def scan_layer64(w, x, residual):
    w = {k: v.double() for k, v in w.items()}
    residual = x.double() + residual.double()
    xbc, z, dt = scan_parts(normed(residual, w["norm"]) @ w["proj"])
    u, B, C = split_xbc(conv64(xbc, w["conv"]))
    h = torch.log1p(torch.exp(dt + w["dt_bias"]))
    S, y = torch.zeros((SHEADS, STATE, DIM), dtype=torch.float64, device="cuda"), torch.zeros_like(u)
    for t in range(x.shape[0]):
        S = S * torch.exp(h[t] * w["A"])[:, None, None] + (h[t][:, None] * B[t])[..., None] * u[t][:, None]
        y[t] = (S * C[t][..., None]).sum(1) + w["D"][:, None] * u[t]
    return normed(y.flatten(1) * silu(z), w["onorm"]) @ w["out"], residual


LAYERS = {"delta": (gdn_weights, gdn_layer, gdn_layer64, (HEADS, DK, DV), HEADS * (2 * DK + DV)),
          "scan": (scan_weights, scan_layer, scan_layer64, (SHEADS, STATE, DIM), SHEADS * DIM + 2 * STATE)}


@pytest.mark.parametrize("kind", LAYERS)
def test_prompts_in_two_parts_then_tokens(kind):
    weights, layer, layer64, state_shape, wide = LAYERS[kind]
    w, gen = weights(), torch.Generator(device="cuda").manual_seed(3)
    lens, first, steps = [100, 40, 7], [70, 3, 7], 3  # the second part is empty for one of them
    where = [4, 0, 2]
    total = [n + steps for n in lens]
    x = [normal(gen, n, HIDDEN) for n in total]
    r = [normal(gen, n, HIDDEN) for n in total]
    conv_state = torch.zeros((5, 3, wide), device="cuda")
    state = torch.zeros((5, *state_shape), device="cuda")
    slots = torch.tensor(where, dtype=torch.int32).cuda()
    got = [[], [], []]

    def take(pieces, cu):
        out, stream = layer(w, torch.cat([x[i][s] for i, s in enumerate(pieces)]),
                            torch.cat([r[i][s] for i, s in enumerate(pieces)]), conv_state, state, cu, slots)
        at = 0
        for i, s in enumerate(pieces):
            n = s.stop - s.start
            got[i].append((out[at:at + n], stream[at:at + n]))
            at += n

    take([slice(0, n) for n in first], cumulative(first))
    take([slice(a, n) for a, n in zip(first, lens)], cumulative([n - a for a, n in zip(first, lens)]))
    for t in range(steps):
        take([slice(n + t, n + t + 1) for n in lens], None)
    for i in range(3):
        want, stream = layer64(w, x[i], r[i])
        close(torch.cat([a for a, _ in got[i]]), want, (kind, i))
        close(torch.cat([b for _, b in got[i]]), stream, (kind, i))


@pytest.mark.parametrize("kind", LAYERS)
def test_a_step_of_a_layer_captured_and_replayed(kind):
    weights, layer, _, state_shape, wide = LAYERS[kind]
    w, gen = weights(), torch.Generator(device="cuda").manual_seed(4)
    n = 6
    x, r = normal(gen, n, HIDDEN), normal(gen, n, HIDDEN)
    conv_state, state = torch.zeros((n, 3, wide), device="cuda"), torch.zeros((n, *state_shape), device="cuda")
    slots = torch.tensor([0, 1, 2, 3, 4, -1], dtype=torch.int32).cuda()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        layer(w, x, r, conv_state, state, None, slots)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, stream = layer(w, x, r, conv_state, state, None, slots)
    for t in range(4):
        x.copy_(normal(gen, n, HIDDEN))
        before = conv_state.clone(), state.clone()
        want = [y.clone() for y in layer(w, x, r, conv_state, state, None, slots)]
        after = conv_state.clone(), state.clone()
        conv_state.copy_(before[0])
        state.copy_(before[1])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[:5], want[0][:5]) and torch.equal(stream, want[1])
        assert torch.equal(conv_state, after[0]) and torch.equal(state, after[1])


def test_eight_bits_in_front_of_a_projection():
    """rms_norm_fp8's values over its scales, through a product: off by what E4M3's half
    steps add up to, a third of 2^-4 of the product's root mean square and less."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    x, w, m = normal(gen, 64, 2048), 1 + 0.1 * normal(gen, 2048), normal(gen, 2048, 256)
    want = normed(x.double(), w.double()) @ m.double()
    for block in (0, 32, 128):
        q, s = g.rms_norm_fp8(x, w, block=block)
        y = (q.float().reshape(64, s.shape[1], -1) * s[..., None]).reshape(64, 2048) @ m
        err = (y.double() - want).square().mean().sqrt() / want.square().mean().sqrt()
        assert err <= 2.0**-4 / 3**0.5, (block, float(err))
