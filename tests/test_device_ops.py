"""Refusals of the operators on device buffers (gdn_delta_*, gdn_logits_process,
gdn_sample_tokens), without a GPU: what the host can see is refused before
anything touches a device, so the addresses here are never read."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

import gateddeltanet_amd as g
from gateddeltanet_amd import _lib

AT = 1 << 20  # an address, 16-byte aligned, never read


def delta(**change):
    a = _lib.GDNDelta(_lib.DTYPE_BF16, 10, 2, 4, 8, 128, 128, 1, 0.1, 4, 512, 512, 1024, 1024, 8,
                      AT, AT, AT, AT, AT, AT, AT, AT, AT, AT)
    if change.pop("step", False):
        a.n_tokens = a.n_seqs
    for k, v in change.items():
        setattr(a, k, v)
    return a


BAD_DELTA = [dict(dtype=3), dict(dtype=-1), dict(key_dim=96), dict(value_dim=512), dict(value_dim=0),
             dict(n_qk_heads=0), dict(n_v_heads=0), dict(n_qk_heads=3), dict(n_v_heads=65536, n_qk_heads=1),
             dict(n_seqs=65536), dict(n_tokens=1 << 31), dict(n_slots=1 << 31), dict(q=0), dict(k=0), dict(v=0),
             dict(o=0), dict(g=0), dict(beta=0), dict(q=AT + 2), dict(k=AT + 8), dict(v=AT + 4), dict(o=AT + 2),
             dict(state_in=AT + 4), dict(state_out=AT + 8), dict(q_stride=516), dict(v_stride=1028),
             dict(k_stride=504), dict(o_stride=1016), dict(g_stride=7)]


@pytest.mark.parametrize("change", BAD_DELTA, ids=lambda c: "-".join(f"{k}={v}" for k, v in c.items()))
def test_delta_refuses(change, capfd):
    lib = _lib.load()
    a = delta(**change)
    assert lib.gdn_delta_prefill(ctypes.byref(a), AT, 1 << 40, None) == -1
    assert "gdn_delta_prefill: " in capfd.readouterr().err
    a = delta(step=True, **{k: v for k, v in change.items() if k not in ("n_seqs", "n_tokens")})
    for k in ("n_seqs", "n_tokens"):
        if k in change:
            a.n_seqs = a.n_tokens = change[k]
    assert lib.gdn_delta_step(ctypes.byref(a), None) == -1
    assert "gdn_delta_step: " in capfd.readouterr().err


def test_delta_refuses_null_and_workspace():
    lib = _lib.load()
    a = delta()
    ref = ctypes.byref(a)
    need = lib.gdn_delta_prefill_workspace(ref)
    assert need > 0
    assert lib.gdn_delta_prefill(None, AT, need, None) == -1
    assert lib.gdn_delta_step(None, None) == -1
    assert lib.gdn_delta_prefill(ref, None, need, None) == -1
    assert lib.gdn_delta_prefill(ref, AT + 8, need, None) == -1
    assert lib.gdn_delta_prefill(ref, AT, need - 1, None) == -1
    assert lib.gdn_delta_prefill(ctypes.byref(delta(cu_seqlens=0)), AT, need, None) == -1
    assert lib.gdn_delta_step(ref, None) == -1  # 10 tokens of two sequences
    assert lib.gdn_delta_prefill_workspace(None) == 0


def test_delta_nothing_to_do():
    lib = _lib.load()
    assert lib.gdn_delta_prefill(ctypes.byref(delta(n_seqs=0)), None, 0, None) == 0
    assert lib.gdn_delta_step(ctypes.byref(delta(n_seqs=0, n_tokens=0)), None) == 0


@pytest.mark.parametrize("dtype,chunk", [(_lib.DTYPE_BF16, 64), (_lib.DTYPE_FP16, 32), (_lib.DTYPE_FP32, 32)])
def test_delta_places_hold_every_chunk(dtype, chunk):
    """The chunks of a sequence have places first / C + number + chunk: none is
    shared, all lie inside the workspace (the kernels' indexing, restated)."""
    import random

    rng = random.Random(3)
    lib = _lib.load()

    def bytes_for(n_tokens, n_seqs):
        return lib.gdn_delta_prefill_workspace(ctypes.byref(delta(dtype=dtype, n_tokens=n_tokens, n_seqs=n_seqs)))

    one = bytes_for(chunk, 1) - bytes_for(0, 1)
    for _ in range(200):
        lens = [rng.choice([0, 1, chunk - 1, chunk, chunk + 1, rng.randint(0, 5 * chunk)]) for _ in range(rng.randint(1, 9))]
        start = rng.randint(0, chunk)
        total = start + sum(lens) + rng.randint(0, 70)
        places = bytes_for(total, len(lens)) // one  # (the sequences' order is less than a place)
        used, first = [], start
        for i, n in enumerate(lens):
            used += [first // chunk + i + c for c in range(-(-n // chunk))]
            first += n
        assert len(set(used)) == len(used) and all(0 <= p < places for p in used), (lens, start, total)


def logits(**change):
    a = _lib.GDNLogits(_lib.DTYPE_FP32, 4, 1000, 50, 6, 4, 1000, 1000, 64, 32, AT, AT, AT, AT, AT, AT, AT, AT, AT, AT,
                       AT, AT, AT)
    for k, v in change.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change", [
    dict(dtype=5), dict(vocab=(1 << 24) + 1), dict(rows=65536), dict(logits=0), dict(out=0), dict(history_len=0),
    dict(bias_ids=0), dict(bias_values=0), dict(logits=AT + 2), dict(out=AT + 1), dict(logits_stride=999),
    dict(out_stride=10), dict(history_stride=49), dict(history_width=1 << 31), dict(n_bias=1 << 31),
    dict(n_masks=1 << 31), dict(mask_stride=31), dict(mask_index=0, n_masks=3),
], ids=lambda c: "-".join(f"{k}={v}" for k, v in c.items()))
def test_logits_process_refuses(change, capfd):
    assert _lib.load().gdn_logits_process(ctypes.byref(logits(**change)), None) == -1
    assert "gdn_logits_process: " in capfd.readouterr().err


def sample(**change):
    a = _lib.GDNSample(_lib.DTYPE_FP32, 4, 1000, 0, 1000, AT, AT, AT, AT, AT, AT, AT, AT)
    for k, v in change.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change", [
    dict(dtype=-2), dict(vocab=(1 << 20) + 1), dict(vocab=0), dict(rows=65536), dict(logits=0), dict(tokens=0),
    dict(uniform=0), dict(logits=AT + 2), dict(logits_stride=999),
], ids=lambda c: "-".join(f"{k}={v}" for k, v in c.items()))
def test_sample_refuses(change, capfd):
    assert _lib.load().gdn_sample_tokens(ctypes.byref(sample(**change)), None, 0, None) == -1
    assert "gdn_sample_tokens: " in capfd.readouterr().err


def test_sample_workspace():
    lib = _lib.load()
    for dtype, most in ((_lib.DTYPE_BF16, 65536), (_lib.DTYPE_FP16, 65536), (_lib.DTYPE_FP32, 32768)):
        assert lib.gdn_sample_workspace(ctypes.byref(sample(dtype=dtype, vocab=most))) == 0
        a = sample(dtype=dtype, vocab=most + 1, logits_stride=most + 1)
        need = lib.gdn_sample_workspace(ctypes.byref(a))
        assert need > 0
        for at, size in ((None, need), (AT + 8, need), (AT, need - 1)):
            assert lib.gdn_sample_tokens(ctypes.byref(a), at, size, None) == -1
    assert lib.gdn_sample_workspace(None) == 0


def test_nothing_to_do_and_null():
    lib = _lib.load()
    assert lib.gdn_logits_process(None, None) == -1 and lib.gdn_sample_tokens(None, None, 0, None) == -1
    assert lib.gdn_logits_process(ctypes.byref(logits(rows=0)), None) == 0
    assert lib.gdn_logits_process(ctypes.byref(logits(vocab=0)), None) == 0
    assert lib.gdn_sample_tokens(ctypes.byref(sample(rows=0)), None, 0, None) == 0


def test_tensors_must_be_on_a_gpu():
    x = torch.zeros((4, 2, 64))
    s, cu = torch.zeros((4, 2)), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(g.GDNError, match="on a GPU"):
        g.delta_prefill(x, x, x, s, s, cu)
    with pytest.raises(g.GDNError, match="on a GPU"):
        g.delta_step(x, x, x, s, s, torch.zeros((4, 2, 64, 64)))
    with pytest.raises(g.GDNError, match="on a GPU"):
        g.logits_process(torch.zeros((2, 10)))
    with pytest.raises(g.GDNError, match="on a GPU"):
        g.sample_tokens(torch.zeros((2, 10)))


def test_batch_sample_refuses_without_an_engine():
    state, tokens = _lib.GDNBatchState(), (ctypes.c_int32 * 4)()
    assert _lib.load().gdn_batch_sample(ctypes.byref(state), None, tokens, None) == -1


@pytest.mark.parametrize("change", [dict(history_width=(1 << 30) + 1, history_stride=1 << 31),
                                    dict(n_bias=(1 << 30) + 1), dict(n_masks=(1 << 30) + 1)],
                         ids=lambda c: next(iter(c)))
def test_logits_process_refuses_what_32_bits_cannot_step_over(change, capfd):
    assert _lib.load().gdn_logits_process(ctypes.byref(logits(**change)), None) == -1
    assert "2^30" in capfd.readouterr().err


@pytest.mark.parametrize("change", [
    dict(n_tokens=0x7fffffff),                                         # 2^25 chunks of 64
    dict(n_seqs=65535, n_slots=65535, n_v_heads=256, v_stride=32768, o_stride=32768, g_stride=256),
    dict(n_seqs=65535, n_slots=65535, n_v_heads=20, v_stride=5120, o_stride=5120, g_stride=20, value_dim=256),
], ids=["chunks", "heads", "tiles"])
def test_prefill_refuses_what_no_grid_holds(change, capfd):
    a = delta(**change)
    assert _lib.load().gdn_delta_prefill(ctypes.byref(a), AT, 1 << 62, None) == -1
    assert "too many chunks or heads" in capfd.readouterr().err


@pytest.mark.parametrize("change", [dict(q_stride=1 << 23), dict(k_stride=-1024), dict(o_stride=1 << 40)],
                         ids=["16MB", "negative", "large"])
def test_delta_refuses_strides(change, capfd):
    lib = _lib.load()
    assert lib.gdn_delta_prefill(ctypes.byref(delta(**change)), AT, 1 << 62, None) == -1
    assert "row stride" in capfd.readouterr().err
    assert lib.gdn_delta_step(ctypes.byref(delta(step=True, **change)), None) == -1
    assert "row stride" in capfd.readouterr().err


def test_delta_refuses_too_few_slots(capfd):
    """Without slots every sequence has the one of its number: none is left out
    silently, with states or without."""
    lib = _lib.load()
    for change in (dict(n_slots=1), dict(n_slots=0, state_in=0, state_out=0)):
        a = delta(slots=0, **change)
        assert lib.gdn_delta_prefill(ctypes.byref(a), AT, 1 << 62, None) == -1
        assert "n_slots" in capfd.readouterr().err
        assert lib.gdn_delta_step(ctypes.byref(delta(step=True, slots=0, **change)), None) == -1
        assert "n_slots" in capfd.readouterr().err


def test_batch_sample_refuses_integers_that_do_not_fit():
    """A setting is taken as it is given or not at all: none wraps past 32 bits
    or loses its fraction on the way to the engine."""
    import types

    import numpy as np

    state = object.__new__(g.BatchState)
    state.n_streams, state._live, state._s = 2, False, _lib.GDNBatchState()
    state.model = types.SimpleNamespace(config=types.SimpleNamespace(vocab_size=100))
    none = [{}, {}]
    for name, kw in [("top_k", dict(top_k=np.array([2**32 + 1, 1]))), ("top_k", dict(top_k=[50.7, 1])),
                     ("top_k", dict(top_k=1e10)), ("top_k", dict(top_k=float("nan"))), ("top_k", dict(top_k=2**70)),
                     ("top_k", dict(top_k=["many", 1])), ("top_k", dict(top_k=[None, 1])),
                     ("top_k", dict(top_k=np.array([2**63, 1], np.uint64))),
                     ("prompt_len", dict(histories=[[1], [2]], prompt_len=np.array([1, 2**40]))),
                     ("prompt_len", dict(histories=[[1], [2]], prompt_len=0.5)),
                     ("history", dict(histories=[[5.5], [1]])), ("history", dict(histories=[[1], np.array([2**31])])),
                     ("history", dict(histories=[[-2**31 - 1], []])), ("history", dict(histories=[[None], []])),
                     ("bias_ids", dict(biases=[{np.int64(2**32 + 5): 1.0}, {}])),
                     ("bias_ids", dict(biases=[{5.5: 1.0}, {}])), ("bias_values", dict(biases=[{5: "much"}, {}]))]:
        with pytest.raises(g.GDNError, match=f"^{name}: expected"):
            state.sample(**kw)
    # what fits comes as far as the engine, which is missing here
    for kw in (dict(top_k=[50.0, np.int64(2)]), dict(top_k=-1), dict(histories=[[], []], prompt_len=[0, 1]), dict(biases=none),
               dict(histories=[np.array([2**31 - 1]), [-2**31]], biases=[{np.int64(5): 1}, {}])):
        with pytest.raises(g.GDNError, match="^gdn_batch_sample failed"):
            state.sample(**kw)


def apart(**change):
    """A delta call whose buffers are megabytes apart."""
    a = delta(**change)
    for i, name in enumerate(("q", "k", "v", "o", "state_in", "state_out")):
        if name not in change:
            setattr(a, name, AT + (i << 24))
    return a


PART = 4 * 8 * 128 * 128  # bytes of a state
O_AT, STATE_AT = AT + (3 << 24), AT + (4 << 24)


@pytest.mark.parametrize("change", [
    dict(o=AT), dict(o=AT + (1 << 24)), dict(o=AT + (2 << 24)), dict(q=O_AT + 16), dict(k=O_AT - 16),
    dict(v=O_AT + 2048 * 3 + 16, v_stride=1024), dict(v=O_AT + 1024, v_stride=2048, o_stride=2048),
    dict(q=O_AT + 2 * 2048 - 16, q_stride=2048, o_stride=2048),
    dict(q=O_AT - 2 * 4096 + 2048 - 16, q_stride=2048, o_stride=2048),
    dict(state_out=STATE_AT + 16), dict(state_out=STATE_AT + 4 * PART - 16), dict(state_out=STATE_AT - 4 * PART + 16),
], ids=lambda c: "-".join(c))
def test_delta_refuses_an_output_over_an_input(change, capfd):
    lib = _lib.load()
    assert lib.gdn_delta_prefill(ctypes.byref(apart(**change)), AT, 1 << 40, None) == -1
    assert "overlap" in capfd.readouterr().err
    a = apart(step=True, **change)
    a.n_tokens = a.n_seqs = 10
    a.n_slots = 4
    assert lib.gdn_delta_step(ctypes.byref(a), None) == -1
    assert "overlap" in capfd.readouterr().err


@pytest.mark.parametrize("change", [
    dict(out_stride=1024), dict(out=AT + 4), dict(out=AT - 4), dict(out=AT + 4000, rows=3), dict(out=AT - 3 * 4000),
    dict(logits_stride=2500, out_stride=2500, out=AT + 4 * 999), dict(logits_stride=1999, out_stride=1999, out=AT + 4000),
    dict(rows=1, out=AT + 4 * 999),
], ids=lambda c: "-".join(f"{k}={v}" for k, v in c.items()))
def test_logits_process_refuses_other_rows_of_its_input(change, capfd):
    assert _lib.load().gdn_logits_process(ctypes.byref(logits(**change)), None) == -1
    assert "overlaps logits" in capfd.readouterr().err


def test_arguments_that_require_gradients_are_refused():
    """None is formed: an output cut off from its inputs would train a model
    wrongly without a word.  Where torch records none they are taken (and
    refused here for not being on a GPU)."""
    x, s, cu = torch.zeros((4, 2, 64)), torch.zeros((4, 2)), torch.zeros(2, dtype=torch.int32)
    S, y, f = torch.zeros((4, 2, 64, 64)), torch.zeros((2, 10)), torch.zeros(2)

    def learnt(t):
        return t.clone().requires_grad_()

    bias = (torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), learnt(f))
    calls = [lambda: g.sample_tokens(learnt(y)), lambda: g.sample_tokens(y, f, temperature=learnt(f)),
             lambda: g.logits_process(learnt(y)), lambda: g.logits_process(y, bias=bias),
             lambda: g.logits_process(y, out=learnt(y)), lambda: g.delta_prefill(x, x, x, s, s, cu, state_in=learnt(S)),
             lambda: g.delta_prefill(x, x, x, s, s, cu, state_out=learnt(S)), lambda: g.delta_step(x, x, x, s, s, learnt(S))]
    for i in range(5):
        a = [x, x, x, s, s]
        a[i] = learnt(a[i])
        calls += [lambda a=a: g.delta_prefill(*a, cu), lambda a=a: g.delta_step(*a, S)]
    for call in calls:
        with pytest.raises(g.GDNError, match="requires gradients"):
            call()
        for off in (torch.no_grad, torch.inference_mode):
            with off(), pytest.raises(g.GDNError, match="on a GPU"):
                call()


def _calls(f):
    """Every operator on tensors, f applied to one floating-point argument (on the CPU:
    the first thing that is looked at is whether gradients are asked for)."""
    def z(*shape):
        return torch.zeros(shape)

    cu, slots = torch.tensor([0, 4], dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    head, state, gates = z(4, 1, 64), z(4, 1, 64, 64), z(4, 1)
    return {
        "conv_prefill": lambda: g.conv_prefill(z(4, 16), f(z(16, 4)), cu),
        "conv_step": lambda: g.conv_step(z(4, 16), z(16, 4), f(z(4, 3, 16))),
        "delta_prefill": lambda: g.delta_prefill(head, head, f(z(4, 1, 64)), gates, gates, cu),
        "delta_step": lambda: g.delta_step(head, head, head, gates, f(gates), state, slots=slots),
        "logits_process": lambda: g.logits_process(f(z(2, 9))),
        "rms_norm": lambda: g.rms_norm(f(z(2, 9))),
        "rms_norm_fp8": lambda: g.rms_norm_fp8(z(2, 9), residual=f(z(2, 9))),
        "sample_tokens": lambda: g.sample_tokens(z(2, 9), f(z(2))),
        "scan_prefill": lambda: g.scan_prefill(head, gates, f(z(1)), head, head, cu),
        "scan_step": lambda: g.scan_step(head, gates, z(1), head, head, f(state)),
    }


@pytest.mark.parametrize("op", _calls(lambda x: x))
def test_tangents_are_refused(op):
    with forward_ad.dual_level():
        call = _calls(lambda x: forward_ad.make_dual(x, torch.ones_like(x)))[op]
        with pytest.raises(g.GDNError, match="tangent"):
            call()
        with torch.no_grad(), pytest.raises(g.GDNError, match="tangent"):
            call()
        with pytest.raises(g.GDNError, match="GPU"):  # none of them has one
            _calls(lambda x: x)[op]()
