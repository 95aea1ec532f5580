"""The operators on the caller's device tensors, as measurable cases.

A serving program that keeps its own buffers runs a Gated DeltaNet layer's
recurrence over a packed batch of prompts (``delta_prefill``), then a token
for every sequence at a time (``delta_step``), and turns the logits of each
step into tokens: penalties, biases and grammar masks (``logits_process``),
then the draw (``sample_tokens``).

``run`` computes them in plain torch operations, or through the package where
``own`` is set.  Shapes: the model's (8 heads of 256 x 256, vocabulary 32000)
and generic ones (grouped heads, dimensions of 64 and 128, other
vocabularies).
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
C = 64  # tokens of a chunk in the plain form


def listed():
    return [
        # A chat turn's short prompt through one layer: latency.
        {"name": "prefill_70", "op": "prefill", "dtype": "bf16", "seqs": 1, "tokens": 70, "hq": 8, "hv": 8, "dk": 256,
         "dv": 256, "start": False},
        # The benchmark's prompt, one sequence alone.
        {"name": "prefill_4096", "op": "prefill", "dtype": "bf16", "seqs": 1, "tokens": 4096, "hq": 8, "hv": 8,
         "dk": 256, "dv": 256, "start": False},
        # A batch of prompts and continued turns of all lengths, one of them
        # empty, one a single token: the ordinary call of a busy server.
        {"name": "prefill_ragged_24", "op": "prefill", "dtype": "bf16", "seqs": 24, "tokens": 8111, "hq": 8, "hv": 8,
         "dk": 256, "dv": 256, "start": True},
        # FP32 activations (the control arm's type), grouped heads of 128.
        {"name": "prefill_fp32_grouped", "op": "prefill", "dtype": "fp32", "seqs": 5, "tokens": 2005, "hq": 4, "hv": 8,
         "dk": 128, "dv": 128, "start": True},
        # One conversation's next token: latency.
        {"name": "step_1", "op": "step", "dtype": "bf16", "seqs": 1, "slots": 1, "hq": 8, "hv": 8, "dk": 256,
         "dv": 256, "padded": 0},
        # The engine's full batch of streams, FP32 activations.
        {"name": "step_64", "op": "step", "dtype": "fp32", "seqs": 64, "slots": 80, "hq": 8, "hv": 8, "dk": 256,
         "dv": 256, "padded": 0},
        # A large batch in a captured size, some of its rows unused.
        {"name": "step_201_grouped", "op": "step", "dtype": "fp16", "seqs": 201, "slots": 256, "hq": 8, "hv": 16,
         "dk": 128, "dv": 128, "padded": 9},
        # One conversation's logits with penalties: latency.
        {"name": "process_1", "op": "process", "dtype": "fp32", "rows": 1, "vocab": 32000, "history": 700, "bias": 0,
         "mask": False},
        # The full batch with everything on.
        {"name": "process_64", "op": "process", "dtype": "fp32", "rows": 64, "vocab": 32000, "history": 2500,
         "bias": 12, "mask": True},
        # A large vocabulary of odd size in BF16.
        {"name": "process_256_bf16", "op": "process", "dtype": "bf16", "rows": 256, "vocab": 99991, "history": 5000,
         "bias": 3, "mask": True},
        # The full batch, each row with its user's settings.
        {"name": "sample_64", "op": "sample", "dtype": "fp32", "rows": 64, "vocab": 32000, "mode": "mixed"},
        # A few conversations over a large vocabulary, nucleus sampling.
        {"name": "sample_8_wide", "op": "sample", "dtype": "bf16", "rows": 8, "vocab": 131072, "mode": "top_p"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    op = rng.choice(["prefill", "prefill", "step", "process", "sample"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op in ("prefill", "step"):
        dk, dv = rng.choice([(256, 256), (128, 128), (64, 64), (128, 256), (256, 128), (64, 128)])
        hq, hv = rng.choice([(8, 8), (4, 8), (2, 6), (1, 4), (3, 3)])
        case = {"op": op, "dtype": dtype, "hq": hq, "hv": hv, "dk": dk, "dv": dv}
        if op == "prefill":
            seqs = _log_int(rng, 1, 24)
            return {**case, "seqs": seqs, "tokens": _log_int(rng, max(1, seqs), 4096), "start": rng.random() < 0.5}
        seqs = _log_int(rng, 1, 96)
        return {**case, "seqs": seqs, "slots": seqs + rng.randint(0, 16), "padded": rng.randint(0, seqs // 8)}
    if op == "process":
        return {"op": op, "dtype": dtype, "rows": _log_int(rng, 1, 96), "vocab": _log_int(rng, 1000, 131072),
                "history": _log_int(rng, 1, 8000), "bias": rng.choice([0, 1, 20]), "mask": rng.random() < 0.6}
    return {"op": op, "dtype": dtype, "rows": _log_int(rng, 1, 64), "vocab": _log_int(rng, 1000, 131072),
            "mode": rng.choice(["mixed", "top_p", "top_k", "plain", "greedy"])}


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


def _delta_inputs(case, seed, n):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    hq, hv, dk, dv = case["hq"], case["hv"], case["dk"], case["dv"]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    # q, k and v as the short convolution and SiLU leave them; decays of a
    # trained model (a in [1, 16), time steps of 1e-3 .. 0.1)
    q, k, v = (torch.nn.functional.silu(normal(n, h, d)).to(dt) for h, d in ((hq, dk), (hq, dk), (hv, dv)))
    a = 1 + 15 * torch.rand(hv, generator=gen, device="cuda")
    step = torch.exp(math.log(1e-3) + math.log(100.0) * torch.rand(hv, generator=gen, device="cuda"))
    bias = step + torch.log(-torch.expm1(-step))
    g = -a * torch.nn.functional.softplus(normal(n, hv) + bias)
    beta = torch.sigmoid(normal(n, hv))
    return gen, q, k, v, g, beta


def prepare(case, seed):
    op = case["op"]
    if op == "prefill":
        lens = _lengths(case, seed)
        gen, q, k, v, g, beta = _delta_inputs(case, seed, case["tokens"])
        cu = torch.tensor([0] + lens, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()
        shape = (case["seqs"], case["hv"], case["dk"], case["dv"])
        start = 0.05 * torch.randn(shape, generator=gen, device="cuda") if case["start"] else None
        return {"case": case, "longest": max(lens), "q": q, "k": k, "v": v, "g": g, "beta": beta, "cu": cu,
                "start": start, "end": torch.zeros(shape, device="cuda")}
    if op == "step":
        n = case["seqs"]
        gen, q, k, v, g, beta = _delta_inputs(case, seed, n)
        state = 0.05 * torch.randn((case["slots"], case["hv"], case["dk"], case["dv"]), generator=gen, device="cuda")
        slots = torch.randperm(case["slots"], generator=gen, device="cuda")[:n].to(torch.int32)
        if case["padded"]:
            slots[-case["padded"]:] = -1
        return {"case": case, "q": q, "k": k, "v": v, "g": g, "beta": beta, "state": state, "slots": slots,
                "out": torch.zeros_like(v)}
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, vocab = case["rows"], case["vocab"]
    dt = DTYPES[case["dtype"]]
    # a flat bulk and a head of likely tokens
    x = 2.0 * torch.randn((rows, vocab), generator=gen, device="cuda")
    lift = torch.rand((rows, vocab), generator=gen, device="cuda")
    x += 12.0 * torch.rand((rows, vocab), generator=gen, device="cuda") * (lift < 40.0 / vocab)
    x = x.to(dt)

    def uniform(lo, hi):
        return lo + (hi - lo) * torch.rand(rows, generator=gen, device="cuda")

    if op == "process":
        width = case["history"]
        # written text repeats its tokens
        words = torch.randint(0, vocab, (rows, max(1, width // 3)), generator=gen, device="cuda")
        pick = torch.randint(0, words.shape[1], (rows, width), generator=gen, device="cuda")
        history = words.gather(1, pick).to(torch.int32)
        length = torch.randint(0, width + 1, (rows,), generator=gen, device="cuda", dtype=torch.int32)
        length[0] = width
        state = {"case": case, "logits": x, "history": history, "history_len": length, "prompt_len": length // 2,
                 "repetition": uniform(1.0, 1.4), "presence": uniform(0.0, 1.0), "frequency": uniform(0.0, 0.5),
                 "bias": None, "mask": None}
        if case["bias"]:
            n = case["bias"]
            ids = torch.rand((rows, vocab), generator=gen, device="cuda").topk(n).indices.to(torch.int32)
            offsets = (torch.arange(rows + 1, device="cuda") * n).to(torch.int32)
            state["bias"] = (offsets, ids.reshape(-1).contiguous(),
                             4.0 * torch.randn(rows * n, generator=gen, device="cuda"))
        if case["mask"]:
            state["mask"] = torch.randint(-2**31, 2**31, (rows, (vocab + 31) // 32), generator=gen, device="cuda",
                                          dtype=torch.int64).to(torch.int32)
        return state
    mode = case["mode"]
    temperature, top_k, top_p, min_p = uniform(0.5, 1.3), None, None, None
    if mode in ("mixed", "top_k"):
        top_k = torch.randint(1, 200, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    if mode in ("mixed", "top_p"):
        top_p = uniform(0.5, 1.0)
    if mode == "mixed":
        min_p = uniform(0.0, 0.05)
        kind = torch.arange(rows, device="cuda") % 4
        top_k[kind == 1] = 0  # off
        top_p[kind == 2] = 1.0  # off
        temperature[kind == 3] = 0.0  # greedy
    if mode == "greedy":
        temperature.zero_()
    return {"case": case, "logits": x, "uniform": uniform(0.0, 1.0), "temperature": temperature, "top_k": top_k,
            "top_p": top_p, "min_p": min_p}


# ------------------------------------------------------------- plain forms

def _unit(x):
    return x * torch.rsqrt(x.square().sum(-1, keepdim=True) + 1e-6)


def _plain_prefill(s):
    """The chunked (WY) form in FP32 over padded sequences; cumulative decays
    and the triangular inverse in 64 bits."""
    case = s["case"]
    n, hv, dk, dv = case["seqs"], case["hv"], case["dk"], case["dv"]
    group = hv // case["hq"]
    chunks = max(1, -(-s["longest"] // C))
    first, last = s["cu"][:-1].long(), s["cu"][1:].long()
    at = first[:, None] + torch.arange(chunks * C, device="cuda")
    there = at < last[:, None]
    at = torch.where(there, at, 0)

    def chunked(x, scale=None):  # [tokens][heads][...] -> [seq][chunk][head][C][...], zero where no token is
        y = torch.where(there.reshape(n, -1, *[1] * (x.dim() - 1)), x[at], torch.zeros((), device="cuda"))
        return y.reshape(n, chunks, C, *x.shape[1:]).transpose(2, 3)

    q = chunked(_unit(s["q"].float()).repeat_interleave(group, 1)) * dk**-0.5
    k = chunked(_unit(s["k"].float()).repeat_interleave(group, 1))
    v, beta = chunked(s["v"].float()), chunked(s["beta"])
    G = chunked(s["g"]).double().cumsum(-1)
    decay = (G[..., :, None] - G[..., None, :]).tril().exp().float().tril()
    eG, rest = G.exp().float(), (G[..., -1:] - G).exp().float()
    kt = k.transpose(-1, -2).contiguous()
    A = -(beta[..., None] * decay * (k @ kt)).tril(-1).double()
    eye = torch.eye(C, device="cuda", dtype=torch.float64)
    T = eye + A
    for _ in range(5):  # (I - A)^-1 = (I + A)(I + A^2)(I + A^4) ...
        A = A @ A
        T = T + T @ A
    T = T.float()
    M = decay * (q @ kt)
    kd = (rest[..., None] * k).transpose(-1, -2).contiguous()
    S = s["start"] if s["start"] is not None else torch.zeros((n, hv, dk, dv), device="cuda")
    outs = []
    for c in range(chunks):
        d = T[:, c] @ (beta[:, c, ..., None] * (v[:, c] - eG[:, c, ..., None] * (k[:, c] @ S)))
        outs.append(eG[:, c, ..., None] * (q[:, c] @ S) + M[:, c] @ d)
        S = eG[:, c, :, -1, None, None] * S + kd[:, c] @ d
    o = torch.stack(outs, 1).transpose(2, 3).reshape(n, chunks * C, hv, dv)
    s["end"].copy_(S)
    return {"out": o[there].to(s["v"].dtype), "state": s["end"]}


def _plain_step(s):
    case = s["case"]
    group = case["hv"] // case["hq"]
    live = s["slots"] >= 0
    at = torch.where(live, s["slots"], 0).long()
    q = (_unit(s["q"].float()) * case["dk"]**-0.5).repeat_interleave(group, 1)
    k = _unit(s["k"].float()).repeat_interleave(group, 1)
    S = s["state"][at] * s["g"].exp()[..., None, None]
    d = s["beta"][..., None] * (s["v"].float() - (S * k[..., None]).sum(-2))
    S = S + k[..., None] * d[..., None, :]
    o = (S * q[..., None]).sum(-2)
    s["out"].copy_(torch.where(live[:, None, None], o.to(s["out"].dtype), s["out"]))
    n = case["seqs"] - case["padded"]  # the unused rows are the last
    s["state"].index_copy_(0, at[:n], S[:n])
    return {"out": s["out"], "state": s["state"]}


def _plain_process(s):
    x = s["logits"].float()
    rows, vocab = x.shape
    place = torch.arange(s["history"].shape[1], device="cuda")
    ids = s["history"].long()
    seen = torch.zeros((rows, vocab), device="cuda", dtype=torch.int32)
    said = torch.zeros_like(seen)
    seen.scatter_add_(1, ids, (place < s["history_len"][:, None]).int())
    said.scatter_add_(1, ids, ((place < s["history_len"][:, None]) & (place >= s["prompt_len"][:, None])).int())
    r = s["repetition"][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * said - torch.where(said > 0, s["presence"][:, None], 0.0)
    if s["bias"] is not None:
        offsets, tokens, values = s["bias"]
        row = torch.searchsorted(offsets[1:], torch.arange(tokens.numel(), device="cuda", dtype=torch.int32), right=True)
        x = x.index_put((row, tokens.long()), values, accumulate=True)
    if s["mask"] is not None:
        bits = (s["mask"][:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        x = torch.where(bits.reshape(rows, -1)[:, :vocab] > 0, x, -math.inf)
    return x.to(s["logits"].dtype)


def _plain_sample(s):
    # 64 bits: a draw next to a border between two tokens goes by the last digits
    x = s["logits"].double()
    rows, vocab = x.shape
    top = x.max(-1, keepdim=True).values
    T = s["temperature"].double()[:, None]
    greedy = T <= 0
    w = ((x - top) / torch.where(greedy, 1.0, T)).exp()
    order = s["logits"].float().sort(dim=-1, descending=True, stable=True).indices
    ranked = w.gather(1, order)
    rank = torch.arange(vocab, device="cuda")
    kept = torch.ones_like(ranked, dtype=torch.bool)
    if s["top_k"] is not None:
        kept = torch.where(s["top_k"][:, None] > 0, rank < s["top_k"][:, None], kept)
    ranked = torch.where(kept, ranked, 0.0)
    if s["top_p"] is not None:
        p = s["top_p"].double()[:, None]
        before = ranked.cumsum(-1) - ranked
        kept &= (p >= 1) | (before < p * ranked.sum(-1, keepdim=True)) | (rank == 0)
    if s["min_p"] is not None:
        kept &= ranked >= s["min_p"].double()[:, None]
    kept = torch.where(greedy, rank == 0, kept)
    weight = torch.zeros_like(w).scatter_(1, order, torch.where(kept, ranked, 0.0))
    run_sum = weight.cumsum(-1)
    target = s["uniform"].double()[:, None] * run_sum[:, -1:]
    token = torch.minimum((run_sum <= target).sum(-1), (weight > 0).long().mul(rank).max(-1).values)
    logprob = (x - top).gather(1, token[:, None])[:, 0] - (x - top).exp().sum(-1).log()
    return {"token": token.to(torch.int32), "logprob": logprob.float()}


# ------------------------------------------------------------------ one pass

def run(state):
    s, op = state, state["case"]["op"]
    if not own:
        return {"prefill": _plain_prefill, "step": _plain_step, "process": _plain_process, "sample": _plain_sample}[op](s)
    import gateddeltanet_amd as g

    if op == "prefill":
        out = g.delta_prefill(s["q"], s["k"], s["v"], s["g"], s["beta"], s["cu"], state_in=s["start"],
                              state_out=s["end"], l2norm=True)
        return {"out": out, "state": s["end"]}
    if op == "step":
        g.delta_step(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], slots=s["slots"], l2norm=True, out=s["out"])
        return {"out": s["out"], "state": s["state"]}
    if op == "process":
        return g.logits_process(s["logits"], history=s["history"], history_len=s["history_len"],
                                prompt_len=s["prompt_len"], repetition=s["repetition"], presence=s["presence"],
                                frequency=s["frequency"], bias=s["bias"], mask=s["mask"])
    token, logprob = g.sample_tokens(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"],
                                     top_p=s["top_p"], min_p=s["min_p"])
    return {"token": token, "logprob": logprob}


# --------------------------------------------------------- the definitions

def _exact_delta(s, first, last, S):
    """The recurrence token by token, every sequence at once, in 64 bits."""
    group = s["case"]["hv"] // s["case"]["hq"]
    q, k = (x.double().repeat_interleave(group, 1) for x in (s["q"], s["k"]))
    q = q / (q.square().sum(-1, keepdim=True) + 1e-6).sqrt() / math.sqrt(s["case"]["dk"])
    k = k / (k.square().sum(-1, keepdim=True) + 1e-6).sqrt()
    v, alpha, beta = s["v"].double(), s["g"].double().exp(), s["beta"].double()
    o = torch.zeros_like(v)
    steps = [b - a for a, b in zip(first, last)]
    for t in range(max(steps)):
        who = [i for i, n in enumerate(steps) if n > t]
        at = torch.tensor([first[i] + t for i in who], device="cuda")
        who = torch.tensor(who, device="cuda")
        X = S[who] * alpha[at, :, None, None]
        d = beta[at, :, None] * (v[at] - (k[at].unsqueeze(-2) @ X).squeeze(-2))
        X += k[at].unsqueeze(-1) * d.unsqueeze(-2)
        S[who] = X
        o[at] = (q[at].unsqueeze(-2) @ X).squeeze(-2)
    return o, S


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "prefill":
        cu = s["cu"].tolist()
        S = s["start"].double() if case["start"] else torch.zeros_like(s["end"], dtype=torch.float64)
        o, S = _exact_delta(s, cu[:-1], cu[1:], S)
        return {"out": o, "state": S}
    if op == "step":
        # two passes may stand between the inputs and a comparison: this is one
        n = case["seqs"] - case["padded"]
        used = s["slots"][:n].long()
        S = s["state"].double()
        o, X = _exact_delta(s, list(range(n)), list(range(1, n + 1)), S[used])
        S[used] = X
        return {"out": o, "state": S}
    x = s["logits"].double().cpu().numpy()
    if op == "process":
        history, length, prompt = (s[n].cpu().numpy() for n in ("history", "history_len", "prompt_len"))
        rep, pres, freq = (s[n].double().cpu().numpy() for n in ("repetition", "presence", "frequency"))
        for r in range(case["rows"]):
            seen = np.unique(history[r, :length[r]])
            y = x[r, seen]
            x[r, seen] = np.where(y > 0, y / rep[r], y * rep[r])
            said, times = np.unique(history[r, prompt[r]:length[r]], return_counts=True)
            x[r, said] -= times * freq[r] + pres[r]
            if s["bias"] is not None:
                at = slice(r * case["bias"], (r + 1) * case["bias"])
                x[r, s["bias"][1][at].cpu().numpy()] += s["bias"][2][at].double().cpu().numpy()
            if s["mask"] is not None:
                bits = np.unpackbits(s["mask"][r].cpu().numpy().view(np.uint8), bitorder="little")[:case["vocab"]]
                x[r, bits == 0] = -np.inf
        return torch.from_numpy(x).cuda()
    token = _plain_sample(s)["token"].tolist()  # the log-probability is the drawn token's
    logprob = [float(row[t] - row.max() - math.log(np.exp(row - row.max()).sum())) for row, t in zip(x, token)]
    return {"token": None, "logprob": torch.tensor(logprob, dtype=torch.float64, device="cuda")}


# ------------------------------------------------------- what it cannot avoid

def work(case):
    op = case["op"]
    size = 4 if case["dtype"] == "fp32" else 2
    if op in ("prefill", "step"):
        n = case["tokens"] if op == "prefill" else case["seqs"] - case["padded"]
        S = case["hv"] * case["dk"] * case["dv"]
        states = case["seqs"] * (1 + case["start"]) if op == "prefill" else 2 * n
        per = 2 * (case["hq"] * case["dk"] + case["hv"] * case["dv"]) * size + 8 * case["hv"]
        return {"bytes": n * per + 4 * S * states, "flops": 7 * n * S}
    rows, vocab = case["rows"], case["vocab"]
    if op == "process":
        words = rows * ((vocab + 31) // 32) if case["mask"] else 0
        return {"bytes": 2 * rows * vocab * size + 4 * words + 2 * rows * case["history"] + 8 * rows * case["bias"],
                "flops": 2 * rows * vocab}
    return {"bytes": rows * vocab * size + 28 * rows, "flops": 6 * rows * vocab}
