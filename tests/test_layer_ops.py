"""Refusals of the operators around the recurrence and of the scan (gdn_conv_*,
gdn_scan_*, gdn_rms_norm), without a GPU: what the host can see is refused before
anything touches a device, so the addresses here are never read."""
import ctypes
import random

import pytest
import torch

import gateddeltanet_amd as g
from gateddeltanet_amd import _lib

AT = 1 << 20  # an address, 16-byte aligned, never read
FAR = 1 << 40


def struct(cls, values, change):
    a = cls()
    for k, v in {**values, **change}.items():
        setattr(a, k, v)
    return a


def ids(c):
    return "-".join(f"{k}={v}" for k, v in c.items())


CONV = dict(dtype=_lib.DTYPE_BF16, n_tokens=10, n_seqs=2, channels=100, width=4, silu=1, n_slots=4, x_stride=120,
            out_stride=100, x=AT, out=FAR, weight=AT, bias=AT, cu_seqlens=AT, slots=AT, state_in=2 * FAR, state_out=2 * FAR)
BAD_CONV = [dict(dtype=3), dict(dtype=-1), dict(width=1), dict(width=5), dict(channels=0), dict(channels=(1 << 20) + 1),
            dict(n_seqs=65536), dict(n_tokens=0xffffff01), dict(n_slots=1 << 31), dict(x=0), dict(out=0), dict(weight=0),
            dict(x=AT + 1), dict(out=FAR + 1), dict(state_in=2 * FAR + 1), dict(x_stride=99), dict(out_stride=-100),
            dict(x_stride=(1 << 40) + 1), dict(slots=0, n_slots=1), dict(out=AT + 200, out_stride=120), dict(out=AT + 2),
            dict(state_out=2 * FAR + 600)]


@pytest.mark.parametrize("change", BAD_CONV, ids=ids)
def test_conv_refuses(change, capfd):
    lib = _lib.load()
    assert lib.gdn_conv_prefill(ctypes.byref(struct(_lib.GDNConv, CONV, change)), None) == -1
    assert "gdn_conv_prefill: " in capfd.readouterr().err
    n = change.get("n_seqs", change.get("n_tokens", 2))
    step = struct(_lib.GDNConv, CONV, {**change, "n_tokens": n, "n_seqs": n})
    assert lib.gdn_conv_step(ctypes.byref(step), None) == -1
    assert "gdn_conv_step: " in capfd.readouterr().err


def test_conv_null_and_nothing_to_do():
    lib = _lib.load()
    assert lib.gdn_conv_prefill(None, None) == -1 and lib.gdn_conv_step(None, None) == -1
    assert lib.gdn_conv_prefill(ctypes.byref(struct(_lib.GDNConv, CONV, dict(cu_seqlens=0))), None) == -1
    assert lib.gdn_conv_step(ctypes.byref(struct(_lib.GDNConv, CONV, {})), None) == -1  # 10 tokens of two sequences
    assert lib.gdn_conv_prefill(ctypes.byref(struct(_lib.GDNConv, CONV, dict(out=AT, out_stride=120))), None) == -1
    assert lib.gdn_conv_prefill(ctypes.byref(struct(_lib.GDNConv, CONV, dict(n_seqs=0))), None) == 0
    assert lib.gdn_conv_step(ctypes.byref(struct(_lib.GDNConv, CONV, dict(n_seqs=0, n_tokens=0))), None) == 0


SCAN = dict(dtype=_lib.DTYPE_BF16, dt_dtype=_lib.DTYPE_FP32, n_tokens=10, n_seqs=2, n_heads=4, n_groups=2, state_dim=128,
            head_dim=64, softplus=1, n_slots=4, x_stride=256, b_stride=256, c_stride=256, dt_stride=4, y_stride=256, x=AT,
            b=AT, c=AT, dt=AT, y=FAR, A=AT, D=AT, dt_bias=AT, cu_seqlens=AT, slots=AT, state_in=2 * FAR, state_out=2 * FAR)
BAD_SCAN = [dict(dtype=3), dict(dtype=-1), dict(dt_dtype=1), dict(dt_dtype=3), dict(state_dim=96), dict(head_dim=32),
            dict(state_dim=0), dict(head_dim=512), dict(n_heads=0), dict(n_groups=0), dict(n_groups=3),
            dict(n_heads=65536, n_groups=1), dict(n_seqs=65536), dict(n_tokens=0xffffff01), dict(n_slots=1 << 31), dict(x=0),
            dict(b=0), dict(c=0), dict(dt=0), dict(y=0), dict(A=0), dict(x=AT + 2), dict(b=AT + 8), dict(c=AT + 4),
            dict(y=FAR + 2), dict(state_in=2 * FAR + 4), dict(state_out=2 * FAR + 8), dict(x_stride=260), dict(b_stride=248),
            dict(c_stride=250), dict(y_stride=128), dict(x_stride=1 << 23), dict(dt_stride=3), dict(slots=0, n_slots=1),
            dict(y=AT), dict(y=AT + 64), dict(x=0x8000000, b=FAR, y_stride=512, b_stride=512),
            dict(state_out=2 * FAR + 4096)]


@pytest.mark.parametrize("change", BAD_SCAN, ids=ids)
def test_scan_refuses(change, capfd):
    lib = _lib.load()
    assert lib.gdn_scan_prefill(ctypes.byref(struct(_lib.GDNScan, SCAN, change)), AT, 1 << 40, None) == -1
    assert "gdn_scan_prefill: " in capfd.readouterr().err
    n = change.get("n_seqs", change.get("n_tokens", 2))
    step = struct(_lib.GDNScan, SCAN, {**change, "n_tokens": n, "n_seqs": n})
    assert lib.gdn_scan_step(ctypes.byref(step), None) == -1
    assert "gdn_scan_step: " in capfd.readouterr().err


def test_scan_null_workspace_and_nothing_to_do():
    lib = _lib.load()
    assert lib.gdn_scan_prefill(None, AT, 1 << 40, None) == -1 and lib.gdn_scan_step(None, None) == -1
    assert lib.gdn_scan_prefill_workspace(None) == 0
    assert lib.gdn_scan_prefill_workspace(ctypes.byref(struct(_lib.GDNScan, SCAN, {}))) == 0  # few tokens
    a = ctypes.byref(struct(_lib.GDNScan, SCAN, dict(n_tokens=5000)))
    need = lib.gdn_scan_prefill_workspace(a)
    assert need > 0
    for ws, size in ((None, need), (AT + 8, need), (AT, need - 1)):
        assert lib.gdn_scan_prefill(a, ws, size, None) == -1
    assert lib.gdn_scan_prefill(ctypes.byref(struct(_lib.GDNScan, SCAN, dict(cu_seqlens=0))), AT, need, None) == -1
    assert lib.gdn_scan_step(ctypes.byref(struct(_lib.GDNScan, SCAN, {})), None) == -1  # 10 tokens of two sequences
    assert lib.gdn_scan_prefill(ctypes.byref(struct(_lib.GDNScan, SCAN, dict(n_seqs=0))), None, 0, None) == 0
    assert lib.gdn_scan_step(ctypes.byref(struct(_lib.GDNScan, SCAN, dict(n_seqs=0, n_tokens=0))), None) == 0


def test_scan_places_hold_every_segment():
    """Segments of a sequence but the last, and the states behind them, have places
    first / seg + segment, none shared, all inside the workspace (the kernels'
    indexing, restated)."""
    rng = random.Random(5)
    for _ in range(300):
        seg = rng.choice([64, 128, 256, 1024])
        lens = [rng.choice([0, 1, seg - 1, seg, seg + 1, 2 * seg, rng.randint(0, 6 * seg)]) for _ in range(rng.randint(1, 9))]
        start = rng.randint(0, 2 * seg)
        total = start + sum(lens) + rng.randint(0, 70)
        kept, first = [], start
        for n in lens:
            cuts = (n - 1) // seg if n else 0
            kept += [first // seg + c for c in range(cuts)]
            first += n
        assert len(set(kept)) == len(kept) and all(0 <= p < total // seg for p in kept)


NORM = dict(dtype=_lib.DTYPE_BF16, rows=10, heads=2, dim=128, gate_first=0, weight_heads=0, fp8=0, block=0, eps=1e-6,
            x_stride=256, residual_stride=256, gate_stride=256, out_stride=256, sum_stride=256, x=AT, residual=AT + (1 << 16),
            gate=AT + (2 << 16), weight=AT, out=FAR, sum=2 * FAR, scales=3 * FAR)
BAD_NORM = [dict(dtype=3), dict(dtype=-1), dict(heads=0), dict(dim=0), dict(heads=8193), dict(rows=1 << 27),
            dict(fp8=1, block=16), dict(fp8=1, block=64, dim=96), dict(fp8=1, block=256), dict(eps=-1.0), dict(eps=float("nan")),
            dict(eps=float("inf")), dict(x=0), dict(out=0), dict(fp8=1, scales=0), dict(x=AT + 1), dict(residual=AT + 65537),
            dict(gate=AT + 65537), dict(out=FAR + 1), dict(sum=2 * FAR + 1), dict(x_stride=255), dict(residual_stride=0),
            dict(gate_stride=-1), dict(out_stride=128), dict(sum_stride=1 << 41), dict(out=2 * FAR), dict(out=AT + 2),
            dict(out=AT, out_stride=300), dict(sum=AT + (2 << 16)), dict(fp8=1, out=AT), dict(sum=AT + 512)]


@pytest.mark.parametrize("change", BAD_NORM, ids=ids)
def test_norm_refuses(change, capfd):
    assert _lib.load().gdn_rms_norm(ctypes.byref(struct(_lib.GDNNorm, NORM, change)), None) == -1
    assert "gdn_rms_norm: " in capfd.readouterr().err


def test_norm_null_and_nothing_to_do():
    lib = _lib.load()
    assert lib.gdn_rms_norm(None, None) == -1
    assert lib.gdn_rms_norm(ctypes.byref(struct(_lib.GDNNorm, NORM, dict(rows=0))), None) == 0


def test_tensors_on_the_cpu_are_refused():
    x, w = torch.zeros((4, 16)), torch.zeros((16, 4))
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(g.GDNError):
        g.conv_prefill(x, w, cu)
    with pytest.raises(g.GDNError):
        g.conv_step(x, w, torch.zeros((4, 3, 16)))
    with pytest.raises(g.GDNError):
        g.rms_norm(x)
    with pytest.raises(g.GDNError):
        g.rms_norm_fp8(x)
    y, b = torch.zeros((4, 1, 64)), torch.zeros((4, 1, 64))
    with pytest.raises(g.GDNError):
        g.scan_prefill(y, torch.zeros((4, 1)), torch.zeros(1), b, b, cu)
    with pytest.raises(g.GDNError):
        g.scan_step(y, torch.zeros((4, 1)), torch.zeros(1), b, b, torch.zeros((4, 1, 64, 64)))


def test_a_scan_of_up_to_256_tokens_needs_no_workspace():
    """Of every shape, as the header says."""
    lib = _lib.load()
    for n_heads, state_dim, head_dim, n_seqs in ((1, 64, 64, 1), (128, 128, 64, 1), (65535, 256, 256, 65535), (8, 256, 128, 256)):
        for dtype in (_lib.DTYPE_BF16, _lib.DTYPE_FP16, _lib.DTYPE_FP32):
            for n_tokens in (0, 1, 64, 65, 128, 255, 256):
                a = struct(_lib.GDNScan, SCAN, dict(dtype=dtype, n_heads=n_heads, n_groups=1, state_dim=state_dim,
                                                    head_dim=head_dim, n_seqs=n_seqs, n_tokens=n_tokens))
                assert lib.gdn_scan_prefill_workspace(ctypes.byref(a)) == 0
