"""gdn_scan_prefill where it cuts sequences, against the scan token by token in 64 bits
(gpu): many sequences, and segments of every length.  Tolerances: test_gpu_scan's.
"""
import ctypes

import pytest
import torch

import gateddeltanet_amd as g
from gateddeltanet_amd import _lib
from test_gpu_scan import BF16, FP16, FP32, call, close, cumulative, inputs, reference, rows, tol

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens", [[1] * 600 + [700, 0, 513, 130] + [2] * 500 + [900, 257],  # more sequences than places
                                  [0] * 1030 + [400, 1, 0, 700, 3, 300], [1, 200] * 40, [5000] + [0] * 64 + [5000]],
                         ids=["places", "past-1024", "two-cuts", "sequences"])
def test_long_sequences_among_more_than_64(lens):
    """Those of several segments, by number or by place, some past the 1024th."""
    a = inputs(sum(lens), 1, 1, 64, 64, FP32, seed=4)
    gen = torch.Generator(device="cuda").manual_seed(5)
    first = 0.3 * torch.randn((len(lens) + 2, 1, 64, 64), generator=gen, device="cuda")
    where = torch.randperm(len(lens) + 2, generator=torch.Generator().manual_seed(6))[:len(lens)].tolist()
    left_out = [i for i in range(len(lens)) if i % 97 == 3]
    slots = [-1 if i in left_out else s for i, s in enumerate(where)]
    pool, out = first.clone(), torch.full_like(a["x"], 5.0)
    call(g.scan_prefill, a, cumulative(lens), state_in=pool, state_out=pool, out=out,
         slots=torch.tensor(slots, dtype=torch.int32).cuda())
    cu = cumulative(lens).tolist()
    for i, n in enumerate(lens):
        part = slice(cu[i], cu[i + 1])
        if i in left_out:
            assert (out[part] == 5).all() and torch.equal(pool[where[i]], first[where[i]])
        elif n > 2 or i % 50 == 0:
            y, S = reference(rows(a, part), first[where[i]])
            close(out[part], y, tol(64), f"y of sequence {i}, {n} tokens")
            close(pool[where[i]], S, tol(64), f"state of sequence {i}, {n} tokens")


@pytest.mark.parametrize("most", [900, 1100], ids=["places", "sequences"])
def test_more_than_1024_sequences_and_places(most):
    """More than a join's grid has workgroups for, more or fewer sequences than places (of
    1024 tokens)."""
    lens = [most] * 1000 + [2100, 2049, 1] * 40
    n = sum(lens)
    a = inputs(n, 1, 1, 64, 64, BF16, seed=7)
    pool = torch.zeros((len(lens), 1, 64, 64), device="cuda")
    out = call(g.scan_prefill, a, cumulative(lens), state_out=pool)
    cu = cumulative(lens).tolist()
    for i in (0, 999, 1000, 1022, 1023, 1024, 1027, 1117):
        y, S = reference(rows(a, slice(cu[i], cu[i + 1])), torch.zeros((1, 64, 64), device="cuda"))
        close(out[cu[i]:cu[i + 1]], y, tol(64), i)
        close(pool[i], S, tol(64), i)


def places(n, heads, N, P, dtype):
    """Segments of a batch's rows that have a state in the workspace: n // their length."""
    a = _lib.GDNScan(dtype={BF16: _lib.DTYPE_BF16, FP16: _lib.DTYPE_FP16, FP32: _lib.DTYPE_FP32}[dtype], n_tokens=n, n_seqs=1,
                     n_heads=heads, n_groups=1, state_dim=N, head_dim=P, n_slots=1)
    return _lib.load().gdn_scan_prefill_workspace(ctypes.byref(a)) // (heads * N * P * 4)


SEGMENTS = [(128, 64, 32, 1900), (256, 64, 32, 3000), (384, 64, 64, 4000), (768, 64, 64, 8000), (1024, 64, 128, 8000),
            (256, 128, 32, 2000), (384, 128, 32, 3000), (768, 128, 64, 4000), (1024, 128, 64, 6000),
            (256, 256, 16, 2000), (384, 256, 16, 3000), (768, 256, 32, 4000), (1024, 256, 32, 6000)]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("seg,P,heads,n", SEGMENTS)
def test_segments_of_every_length(dtype, seg, P, heads, n):
    """Steps, decays and operands refilled over all of a segment's chunks; a sequence of
    three cuts and more, one that ends with a segment, short ones; three of the heads."""
    N = 64 if seg < 1024 else 128
    assert places(n, heads, N, P, dtype) == n // seg
    lens = [n - 2 * seg // 3 - 70, 0, 1, 2 * seg // 3, 69]
    assert lens[0] > 3 * seg or seg == 1024
    lens = lens if seg < 1024 else [3 * seg + 1, 0, n - 3 * seg - 71, 1, 69]
    a = inputs(n, heads, 1, N, P, dtype, seed=seg + P)
    gen = torch.Generator(device="cuda").manual_seed(seg)
    pool = 0.3 * torch.randn((len(lens), heads, N, P), generator=gen, device="cuda")
    some = torch.tensor([0, heads // 2 + 1, heads - 1], device="cuda")
    few = {k: v if k in "BC" else v[:, some] if k in ("x", "dt") else v[some] for k, v in a.items()}
    first = pool[:, some]
    out = call(g.scan_prefill, a, cumulative(lens), state_in=pool, state_out=pool)
    cu = cumulative(lens).tolist()
    for i, m in enumerate(lens):
        y, S = reference(rows(few, slice(cu[i], cu[i + 1])), first[i])
        close(out[cu[i]:cu[i + 1], some], y, tol(N), f"y of sequence {i}, {m} tokens")
        close(pool[i, some], S, tol(N), f"state of sequence {i}, {m} tokens")


@pytest.mark.parametrize("N,P,heads", [(64, 64, 2), (128, 128, 8), (64, 256, 3)])
def test_a_workspace_of_its_size_between_guards(N, P, heads):
    """Every state and decay lies in it, of batches whose ends lie around those of segments,
    before and behind rows of no sequence; and what was there is not read."""
    edge = [1, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300]
    batches = [([n], 0, 0) for n in (257, 319, 320, 321, 383, 384, 385, 512, 513, 640, 641, 1025)]
    batches += [([n, 0, m, 1], first, 20) for n, m, first in zip(edge, edge[3:] + edge[:3], [250, 0, 63, 1, 64, 129, 0, 37, 65, 3, 128])]
    batches += [([1000, 1, 1], 0, 0), ([1, 1000, 1], 62, 0), ([1, 1, 1000], 0, 0), ([130] * 66, 5, 3)]
    for lens, first, behind in batches:
        n = max(first + sum(lens) + behind, 300)
        a = inputs(n, heads, 1, N, P, BF16, seed=n)
        cu = cumulative(lens, first)
        for start in (False, True):  # (slots that are read and written have their starts in it)
            pool = [0.3 * torch.ones((len(lens), heads, N, P), device="cuda") for _ in range(2)]
            args = _lib.GDNScan(dtype=_lib.DTYPE_BF16, n_tokens=n, n_seqs=len(lens), n_heads=heads, n_groups=1, state_dim=N,
                                head_dim=P, n_slots=len(lens), state_in=pool[0].data_ptr() if start else None,
                                state_out=pool[0].data_ptr())
            need = _lib.load().gdn_scan_prefill_workspace(ctypes.byref(args))
            out, got = [torch.zeros_like(a["x"]) for _ in pool], []
            for p, o, fill in zip(pool, out, (0xFF, 0x3C)):  # NaN; small numbers
                room = torch.full((need + 8192,), fill, dtype=torch.uint8, device="cuda")
                call(g.scan_prefill, a, cu, state_in=p if start else None, state_out=p, out=o, workspace=room[4096:4096 + need])
                assert (room[:4096] == fill).all() and (room[4096 + need:] == fill).all(), (lens, first)
                got.append((o, p))
            assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1]), (lens, first)
            assert torch.isfinite(got[0][0]).all() and torch.isfinite(got[0][1]).all(), (lens, first)
