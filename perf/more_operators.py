"""The operators around a recurrence, and the state space scan, as measurable cases.

A layer of a serving program's own batch: the residual is added and normed
(``rms_norm``, ``rms_norm_fp8``), the projected rows go through the short causal
convolution (``conv_prefill`` over packed prompts, ``conv_step`` a token of every
sequence), then through a recurrence, here the selective state space scan
(``scan_prefill``, ``scan_step``), and the result is normed with a gate.

``run`` computes them in plain torch operations, or through the package where
``own`` is set.  Shapes: the model's (hidden 2048, 8 heads of 256, a convolution of 4
over q, k and v) and generic ones.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CHUNK = 64  # tokens of a chunk in the scan's plain form


def listed():
    return [
        # A chat turn's short prompt, q, k and v of one layer: latency.
        {"name": "conv_70", "op": "conv", "dtype": "bf16", "seqs": 1, "tokens": 70, "channels": 6144, "width": 4,
         "bias": False, "silu": True, "start": False},
        # A batch of prompts and continued turns of all lengths, one empty, one a single token.
        {"name": "conv_ragged_24", "op": "conv", "dtype": "bf16", "seqs": 24, "tokens": 8111, "channels": 6144,
         "width": 4, "bias": False, "silu": True, "start": True},
        # One conversation's next token: latency.
        {"name": "conv_step_1", "op": "conv_step", "dtype": "bf16", "seqs": 1, "slots": 1, "padded": 0,
         "channels": 6144, "width": 4, "bias": False, "silu": True},
        # A large batch in a captured size, some of its rows unused, FP32 activations.
        {"name": "conv_step_201", "op": "conv_step", "dtype": "fp32", "seqs": 201, "slots": 256, "padded": 9,
         "channels": 4352, "width": 4, "bias": True, "silu": True},
        # A short prompt through one scan layer: latency.
        {"name": "scan_70", "op": "scan", "dtype": "bf16", "seqs": 1, "tokens": 70, "heads": 32, "groups": 1,
         "state": 128, "dim": 64, "start": False},
        # A long prompt alone.
        {"name": "scan_4096", "op": "scan", "dtype": "bf16", "seqs": 1, "tokens": 4096, "heads": 32, "groups": 1,
         "state": 128, "dim": 64, "start": False},
        # The busy server's ragged batch, states kept, heads as the delta rule's.
        {"name": "scan_ragged_24", "op": "scan", "dtype": "bf16", "seqs": 24, "tokens": 8111, "heads": 8, "groups": 8,
         "state": 256, "dim": 256, "start": True},
        # FP32 activations, grouped heads.
        {"name": "scan_fp32_grouped", "op": "scan", "dtype": "fp32", "seqs": 5, "tokens": 2005, "heads": 16,
         "groups": 2, "state": 64, "dim": 128, "start": True},
        # A token of the engine's full batch of streams.
        {"name": "scan_step_64", "op": "scan_step", "dtype": "bf16", "seqs": 64, "slots": 80, "padded": 0,
         "heads": 32, "groups": 1, "state": 128, "dim": 64},
        # One conversation's token, FP16: latency.
        {"name": "scan_step_1", "op": "scan_step", "dtype": "fp16", "seqs": 1, "slots": 1, "padded": 0, "heads": 16,
         "groups": 2, "state": 128, "dim": 128},
        # The long prompt's residual stream in front of an 8-bit projection.
        {"name": "norm_4096_fp8", "op": "norm", "dtype": "bf16", "rows": 4096, "heads": 1, "dim": 2048,
         "residual": True, "gate": "", "fp8": True, "block": 0},
        # A batch's tokens, each head's output normed and gated.
        {"name": "norm_gated_64", "op": "norm", "dtype": "bf16", "rows": 64, "heads": 8, "dim": 256,
         "residual": False, "gate": "after", "fp8": False, "block": 0},
    ]


def _log_int(rng, lo, hi):
    return min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    op = rng.choice(["conv", "conv_step", "scan", "scan", "scan_step", "norm", "norm"])
    case = {"op": op, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    seqs = _log_int(rng, 1, 24 if op in ("conv", "scan") else 96)
    packed = {"seqs": seqs, "tokens": _log_int(rng, seqs, 4096), "start": rng.random() < 0.5}
    rows = {"seqs": seqs, "slots": seqs + rng.randint(0, 16), "padded": rng.randint(0, seqs // 8)}
    if op in ("conv", "conv_step"):
        channels = _log_int(rng, 64, 8192)
        if rng.random() < 0.7:  # most layers' are round, some are not
            channels = max(64, channels // 64 * 64)
        return {**case, **(packed if op == "conv" else rows), "channels": channels, "width": rng.choice([4, 4, 4, 3, 2]),
                "bias": rng.random() < 0.5, "silu": rng.random() < 0.8}
    if op in ("scan", "scan_step"):
        state, dim = rng.choice([(128, 64), (128, 64), (64, 64), (128, 128), (64, 128), (256, 64), (256, 256)])
        heads, groups = rng.choice([(32, 1), (16, 2), (8, 8), (24, 4), (6, 1), (7, 7), (1, 1)])
        return {**case, **(packed if op == "scan" else rows), "heads": heads, "groups": groups, "state": state,
                "dim": dim}
    heads = rng.choice([1, 1, 1, 4, 8])
    dim = _log_int(rng, 64, 8192) if heads == 1 else rng.choice([64, 128, 256])
    if heads == 1 and rng.random() < 0.7:
        dim = max(128, dim // 128 * 128)
    return {**case, "rows": _log_int(rng, 1, 4096), "heads": heads, "dim": dim, "residual": rng.random() < 0.5,
            "gate": rng.choice(["", "", "after", "before"]), "fp8": rng.random() < 0.5,
            "block": rng.choice([0, 32, 64, 128]) if dim % 128 == 0 else 0}


# ---------------------------------------------------------------- the inputs

def _lengths(case, seed):
    """`seqs` lengths that add up to `tokens`: uneven, one empty and one of a
    single token where there are four or more."""
    n, total = case["seqs"], case["tokens"]
    rng = random.Random(1000 * total + n + 7919 * seed)
    lens = [0, 1] if n >= 4 else []
    parts = [math.exp(rng.gauss(0, 0.7)) for _ in range(n - len(lens))]
    left = total - sum(lens)
    cuts = [int(left * sum(parts[:i]) / sum(parts)) for i in range(len(parts))] + [left]
    lens += [b - a for a, b in zip(cuts, cuts[1:])]
    rng.shuffle(lens)
    return lens


def prepare(case, seed):
    op, dt = case["op"], DTYPES[case["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    def uniform(lo, hi, *shape):
        return lo + (hi - lo) * torch.rand(shape, generator=gen, device="cuda")

    s = {"case": case}
    if op == "norm":
        shape = (case["rows"], case["heads"], case["dim"])
        s |= {"x": (1.5 * normal(*shape)).to(dt), "weight": 1 + 0.2 * normal(case["dim"]),
              "residual": (4 * normal(*shape)).to(dt) if case["residual"] else None,
              "gate": normal(*shape).to(dt) if case["gate"] else None}
        return s
    n = case["tokens"] if op in ("conv", "scan") else case["seqs"]
    if op in ("conv", "scan"):
        lens = _lengths(case, seed)
        s |= {"longest": max(lens), "cu": torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()}
        slots = case["seqs"]
    else:
        slots = case["slots"]
        s["slots"] = torch.randperm(slots, generator=gen, device="cuda")[:n].to(torch.int32)
        if case["padded"]:
            s["slots"][-case["padded"]:] = -1
    if op in ("conv", "conv_step"):
        ch, width = case["channels"], case["width"]
        s |= {"x": normal(n, ch).to(dt), "weight": uniform(-0.5, 0.5, ch, width),
              "bias": 0.2 * normal(ch) if case["bias"] else None}
        state = normal(slots, width - 1, ch).to(dt)
    else:
        heads, groups, N, P = case["heads"], case["groups"], case["state"], case["dim"]
        # x, B and C as the convolution and SiLU leave them, steps of 1e-3 .. 0.1 behind a softplus
        x, B, C = (torch.nn.functional.silu(normal(n, h, d)).to(dt) for h, d in ((heads, P), (groups, N), (groups, N)))
        step = torch.exp(math.log(1e-3) + math.log(100.0) * uniform(0, 1, heads))
        s |= {"x": x, "B": B, "C": C, "dt": normal(n, heads).to(dt), "A": -uniform(1, 16, heads),
              "D": 1 + 0.2 * normal(heads), "dt_bias": step + torch.log(-torch.expm1(-step))}
        state = 0.5 * normal(slots, heads, N, P)
    if op in ("conv", "scan"):
        s |= {"start": state if case["start"] else None, "end": torch.zeros_like(state)}
    else:
        s |= {"state": state, "out": torch.zeros_like(s["x"])}
    return s


# ------------------------------------------------------------- plain forms

def _activated(y, s):
    if s["bias"] is not None:
        y = y + s["bias"]
    return y * torch.sigmoid(y) if s["case"]["silu"] else y


def _plain_conv(s):
    """Every token's window gathered from the tails and the rows."""
    case = s["case"]
    n, ch, T, W = case["seqs"], case["channels"], case["tokens"], case["width"]
    first, last = s["cu"][:-1].long(), s["cu"][1:].long()
    tails = torch.zeros((n, W - 1, ch), device="cuda") if s["start"] is None else s["start"].float()
    rows = torch.cat([tails.reshape(-1, ch), s["x"].float()])
    back = torch.arange(W - 1, -1, -1, device="cuda")

    def windows(seq, pos, back):  # where the inputs `back` before position pos of the sequence stand
        at = pos[:, None] - back
        return torch.where(at >= 0, n * (W - 1) + first[seq][:, None] + at, (seq[:, None] + 1) * (W - 1) + at)

    token = torch.arange(T, device="cuda")
    seq = torch.searchsorted(last, token, right=True)
    y = (rows[windows(seq, token - first[seq], back)] * s["weight"].t()).sum(1)
    each = torch.arange(n, device="cuda")
    s["end"].copy_(rows[windows(each, last - first - 1, back[1:])])
    return {"out": _activated(y, s).to(s["x"].dtype), "state": s["end"]}


def _plain_conv_step(s):
    live = s["slots"] >= 0
    at = torch.where(live, s["slots"], 0).long()
    z = torch.cat([s["state"][at].float(), s["x"].float()[:, None]], 1)
    y = _activated((z * s["weight"].t()).sum(1), s)
    s["out"].copy_(torch.where(live[:, None], y.to(s["out"].dtype), s["out"]))
    n = s["case"]["seqs"] - s["case"]["padded"]  # the unused rows are the last
    s["state"].index_copy_(0, at[:n], z[:n, 1:].to(s["state"].dtype))
    return {"out": s["out"], "state": s["state"]}


def _step_size(s):
    x = s["dt"].double() + s["dt_bias"]
    return torch.nn.functional.softplus(x, threshold=700.0)


def _plain_scan(s):
    """Chunks of every sequence at once, their states joined by one product;
    running decays in 64 bits."""
    case = s["case"]
    n, heads, N, P = case["seqs"], case["heads"], case["state"], case["dim"]
    group = heads // case["groups"]
    chunks = max(1, -(-s["longest"] // CHUNK))
    first, last = s["cu"][:-1].long(), s["cu"][1:].long()
    at = first[:, None] + torch.arange(chunks * CHUNK, device="cuda")
    there = at < last[:, None]
    at = torch.where(there, at, 0)

    def chunked(x):  # [tokens][heads][...] -> [seq][chunk][head][CHUNK][...], zero where no token is
        y = torch.where(there.reshape(n, -1, *[1] * (x.dim() - 1)), x[at], torch.zeros((), device="cuda", dtype=x.dtype))
        return y.reshape(n, chunks, CHUNK, *x.shape[1:]).transpose(2, 3).contiguous()

    x, B, C = chunked(s["x"].float()), chunked(s["B"].float()), chunked(s["C"].float())
    step = _step_size(s)
    G = chunked(step * s["A"]).cumsum(-1)
    step = chunked(step).float()
    weight = (G[..., :, None] - G[..., None, :]).tril().exp().float().tril() * step[..., None, :]
    products = C @ B.transpose(-1, -2).contiguous()
    B, C, products = (y.repeat_interleave(group, 2) for y in (B, C, products))
    y = (weight * products) @ x
    rest = (G[..., -1:] - G).exp().float() * step
    U = (rest[..., None] * B).transpose(-1, -2).contiguous() @ x
    # the state in front of chunk c (c = chunks: the last) from the chunks before it
    total = torch.nn.functional.pad(G[..., -1].transpose(1, 2).cumsum(-1), (1, 0))
    between = total[..., :, None] - total[..., None, 1:]
    join = torch.where(torch.ones_like(between).tril(-1) > 0, between, -math.inf).exp().float()
    states = (join @ U.transpose(1, 2).reshape(n, heads, chunks, N * P)).reshape(n, heads, chunks + 1, N, P)
    if s["start"] is not None:
        states = states + total.exp().float()[..., None, None] * s["start"][:, :, None]
    y = y + G.exp().float()[..., None] * (C @ states[:, :, :-1].transpose(1, 2))
    y = y.transpose(2, 3).reshape(n, chunks * CHUNK, heads, P)[there] + s["D"][:, None] * s["x"].float()
    s["end"].copy_(states[:, :, -1])
    return {"out": y.to(s["x"].dtype), "state": s["end"]}


def _plain_scan_step(s):
    case = s["case"]
    group = case["heads"] // case["groups"]
    live = s["slots"] >= 0
    at = torch.where(live, s["slots"], 0).long()
    step = _step_size(s)
    a, step, x = (step * s["A"]).exp().float(), step.float(), s["x"].float()
    B, C = (y.float().repeat_interleave(group, 1) for y in (s["B"], s["C"]))
    S = a[..., None, None] * s["state"][at] + (step[..., None] * B)[..., None] * x[..., None, :]
    y = (S * C[..., None]).sum(-2) + s["D"][:, None] * x
    s["out"].copy_(torch.where(live[:, None, None], y.to(s["out"].dtype), s["out"]))
    n = case["seqs"] - case["padded"]  # the unused rows are the last
    s["state"].index_copy_(0, at[:n], S[:n])
    return {"out": s["out"], "state": s["state"]}


def _norm(s, number):
    """(normed rows, the residual's sum) in `number`."""
    case, h = s["case"], s["x"].to(number)
    if case["residual"]:
        h = h + s["residual"].to(number)
    y, gate = h, None
    if case["gate"]:
        gate = s["gate"].to(number)
        gate = gate * torch.sigmoid(gate)
    if case["gate"] == "before":
        y = y * gate
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * s["weight"].to(number)
    return (y * gate if case["gate"] == "after" else y), h


def _scaled(y, block):
    """(values over their scales, scales) of rows in blocks (0: a row's all)."""
    rows = y.shape[0]
    y = y.reshape(rows, -1)
    blocks = y.reshape(rows, -1, block or y.shape[1])
    scale = blocks.abs().amax(-1) / 448
    scale = torch.where(scale > 0, scale, 1.0)
    return blocks / scale[..., None], scale


def _plain_norm(s):
    case = s["case"]
    y, h = _norm(s, torch.float32)
    got = {"sum": h.to(s["x"].dtype)} if case["residual"] else {}
    if not case["fp8"]:
        return {**got, "out": y.to(s["x"].dtype)}
    values, scales = _scaled(y, case["block"])
    return {**got, "out": values.to(torch.float8_e4m3fn).reshape(y.shape), "scales": scales}


# ------------------------------------------------------------------ one pass

def run(state):
    s, case = state, state["case"]
    op = case["op"]
    if not own:
        return {"conv": _plain_conv, "conv_step": _plain_conv_step, "scan": _plain_scan, "scan_step": _plain_scan_step,
                "norm": _plain_norm}[op](s)
    import gateddeltanet_amd as g

    if op == "conv":
        out = g.conv_prefill(s["x"], s["weight"], s["cu"], bias=s["bias"], silu=case["silu"], state_in=s["start"],
                             state_out=s["end"])
        return {"out": out, "state": s["end"]}
    if op == "conv_step":
        g.conv_step(s["x"], s["weight"], s["state"], bias=s["bias"], silu=case["silu"], slots=s["slots"], out=s["out"])
        return {"out": s["out"], "state": s["state"]}
    if op == "scan":
        out = g.scan_prefill(s["x"], s["dt"], s["A"], s["B"], s["C"], s["cu"], D=s["D"], dt_bias=s["dt_bias"],
                             softplus=True, state_in=s["start"], state_out=s["end"])
        return {"out": out, "state": s["end"]}
    if op == "scan_step":
        g.scan_step(s["x"], s["dt"], s["A"], s["B"], s["C"], s["state"], D=s["D"], dt_bias=s["dt_bias"], softplus=True,
                    slots=s["slots"], out=s["out"])
        return {"out": s["out"], "state": s["state"]}
    options = {"eps": 1e-6, "residual": s["residual"], "gate": s["gate"], "gate_first": case["gate"] == "before"}
    if case["fp8"]:
        out, scales, *total = g.rms_norm_fp8(s["x"], s["weight"], block=case["block"], **options)
        got = {"out": out, "scales": scales}
    else:
        out = g.rms_norm(s["x"], s["weight"], **options)
        out, *total = out if case["residual"] else (out,)
        got = {"out": out}
    return {**got, "sum": total[0]} if case["residual"] else got


# --------------------------------------------------------- the definitions

def _exact_conv(s, lens, tails):
    w, outs, ends, at = s["weight"].double(), [], [], 0
    for i, n in enumerate(lens):
        z = torch.cat([tails[i].double(), s["x"][at:at + n].double()])
        outs.append(sum(z[j:j + n] * w[:, j] for j in range(w.shape[1])))
        ends.append(z[n:])
        at += n
    y = torch.cat(outs)
    if s["bias"] is not None:
        y = y + s["bias"].double()
    return y / (1 + torch.exp(-y)) if s["case"]["silu"] else y, torch.stack(ends)


def _exact_scan(s, first, last, S):
    """The recurrence token by token, every sequence at once, in 64 bits."""
    group = s["case"]["heads"] // s["case"]["groups"]
    B, C = (y.double().repeat_interleave(group, 1) for y in (s["B"], s["C"]))
    x, step = s["x"].double(), torch.log1p(torch.exp(s["dt"].double() + s["dt_bias"].double()))
    a = torch.exp(step * s["A"].double())
    y = s["D"].double()[:, None] * x
    steps = [b - a_ for a_, b in zip(first, last)]
    for t in range(max(steps)):
        who = [i for i, n in enumerate(steps) if n > t]
        at = torch.tensor([first[i] + t for i in who], device="cuda")
        who = torch.tensor(who, device="cuda")
        X = S[who] * a[at, :, None, None] + (step[at].unsqueeze(-1) * B[at]).unsqueeze(-1) * x[at].unsqueeze(-2)
        S[who] = X
        y[at] += (C[at].unsqueeze(-2) @ X).squeeze(-2)
    return y, S


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        y, h = _norm(s, torch.float64)
        got = {"sum": h} if case["residual"] else {}
        if not case["fp8"]:
            return {**got, "out": y}
        values, scales = _scaled(y, case["block"])
        return {**got, "out": values.reshape(y.shape), "scales": scales}
    if op in ("conv", "scan"):
        cu = s["cu"].tolist()
        S = torch.zeros_like(s["end"]) if s["start"] is None else s["start"]
        if op == "conv":
            y, S = _exact_conv(s, [b - a for a, b in zip(cu, cu[1:])], S)
        else:
            y, S = _exact_scan(s, cu[:-1], cu[1:], S.double())
        return {"out": y, "state": S}
    n = case["seqs"] - case["padded"]
    used = s["slots"][:n].long()
    S, out = s["state"].double(), torch.zeros(s["x"].shape, dtype=torch.float64, device="cuda")
    if op == "conv_step":
        y, X = _exact_conv({**s, "x": s["x"][:n]}, [1] * n, S[used])
    else:
        y, X = _exact_scan(s, list(range(n)), list(range(1, n + 1)), S[used])
    S[used] = X
    out[:n] = y[:n]
    return {"out": out, "state": S}


# ------------------------------------------------------- what it cannot avoid

def work(case):
    op = case["op"]
    size = 4 if case["dtype"] == "fp32" else 2
    if op == "norm":
        n = case["rows"] * case["heads"] * case["dim"]
        ins = 1 + case["residual"] + bool(case["gate"])
        blocks = case["rows"] * case["heads"] * case["dim"] // case["block"] if case["block"] else case["rows"]
        outs = (n + 4 * blocks if case["fp8"] else n * size) + n * size * case["residual"]
        return {"bytes": n * size * ins + outs + 4 * case["dim"], "flops": 5 * n}
    n = case["tokens"] if op in ("conv", "scan") else case["seqs"] - case["padded"]
    pools = case["seqs"] * (1 + case["start"]) if op in ("conv", "scan") else 2 * n
    if op in ("conv", "conv_step"):
        ch, W = case["channels"], case["width"]
        return {"bytes": (2 * n + pools * (W - 1)) * ch * size + 4 * ch * (W + case["bias"]), "flops": n * ch * (2 * W + 4)}
    heads, S = case["heads"], case["heads"] * case["state"] * case["dim"]
    per = 2 * heads * case["dim"] + 2 * case["groups"] * case["state"] + heads
    return {"bytes": n * per * size + 4 * S * pools + 12 * heads, "flops": 5 * n * S}
