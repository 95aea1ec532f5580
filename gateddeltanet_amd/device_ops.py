"""The operators on the caller's device tensors (include/gdn_amd.h, "operators
on the caller's device buffers"): the gated delta rule over a batch of
sequences.

Arguments are torch tensors on one GPU; work goes to that GPU's current stream
and is not waited for, and every call can be captured into a graph.  Where a
function makes its output or workspace, it takes them from torch's allocator on
that stream.  Errors raise ``GDNError``, before anything is enqueued.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib as L
from .engine import GDNError

_DTYPES = {torch.bfloat16: L.DTYPE_BF16, torch.float16: L.DTYPE_FP16, torch.float32: L.DTYPE_FP32}


def _fail(what: str) -> None:
    raise GDNError(what)


def _on(device: torch.device, name: str, x, dtype, shape) -> int:
    """The address of contiguous tensor x, or None's; shape with -1 = any."""
    if x is None:
        return 0
    if x.device != device or x.dtype != dtype or len(x.shape) != len(shape) or not x.is_contiguous() or any(
            a != b for a, b in zip(x.shape, shape) if b >= 0):
        _fail(f"{name}: expected a contiguous {dtype} tensor of shape {tuple(shape)} on {device}, got "
              f"{x.dtype} {tuple(x.shape)} on {x.device}")
    return x.data_ptr()


def _launch(device: torch.device, what: str, fn, *args) -> None:
    """fn(*args, stream) with the tensors' device as the current one."""
    if torch.cuda.current_device() == device.index:
        rc = fn(*args, torch.cuda.current_stream().cuda_stream)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch.cuda.current_stream().cuda_stream)
    if rc != 0:
        _fail(f"{what} failed (rc={rc})")


def _heads(name: str, x: torch.Tensor, like: torch.Tensor) -> None:
    if x.device != like.device or x.dtype != like.dtype or x.dim() != 3 or (
            x.shape[0] > 0 and (x.stride(2) != 1 or x.stride(1) != x.shape[2])):
        _fail(f"{name}: expected {like.dtype} [rows][heads][dim] on {like.device} with contiguous heads, got {x.dtype} "
              f"{tuple(x.shape)} strides {x.stride()} on {x.device}")


def _delta(q, k, v, g, beta, out, state_in, state_out, slots, n_seqs, scale, l2norm):
    dtype = _DTYPES.get(q.dtype)
    if dtype is None or not q.is_cuda:
        _fail(f"q: expected a bfloat16, float16 or float32 tensor on a GPU, got {q.dtype} on {q.device}")
    for name, x in (("q", q), ("k", k), ("v", v), ("out", out)):
        _heads(name, x, q)
    n, hq, dk = q.shape
    hv, dv = v.shape[1:]
    if k.shape != q.shape or v.shape[0] != n or out.shape != v.shape:
        _fail(f"shapes do not agree: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}, out {tuple(out.shape)}")
    if g.shape != (n, hv) or beta.shape != (n, hv) or g.dtype != torch.float32 or beta.dtype != torch.float32 or (
            g.device != q.device or beta.device != q.device) or (
            n > 0 and hv > 1 and (g.stride(1) != 1 or beta.stride(1) != 1)) or (n > 1 and g.stride(0) != beta.stride(0)):
        _fail(f"g and beta: expected float32 [{n}][{hv}] of equal row strides on {q.device}")
    pool = state_out if state_out is not None else state_in
    n_slots = pool.shape[0] if pool is not None else n_seqs
    states = [_on(q.device, name, x, torch.float32, (n_slots, hv, dk, dv))
              for name, x in (("state_in", state_in), ("state_out", state_out))]
    where = _on(q.device, "slots", slots, torch.int32, (n_seqs,))
    if slots is None and n_slots < n_seqs:
        _fail(f"{n_seqs} sequences without slots need as many states, got {n_slots}")
    return L.GDNDelta(dtype, n, n_seqs, hq, hv, dk, dv, 1 if l2norm else 0, dk**-0.5 if scale is None else scale,
                      n_slots, q.stride(0), k.stride(0), v.stride(0), out.stride(0), g.stride(0), q.data_ptr(),
                      k.data_ptr(), v.data_ptr(), out.data_ptr(), g.data_ptr(), beta.data_ptr(), 0, where, *states)


def delta_prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                  cu_seqlens: torch.Tensor, *, state_in: Optional[torch.Tensor] = None,
                  state_out: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None,
                  scale: Optional[float] = None, l2norm: bool = True, out: Optional[torch.Tensor] = None,
                  workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """gdn_delta_prefill: the gated delta rule over packed sequences.

    q, k [tokens][qk heads][key dim] and v [tokens][value heads][value dim] of
    one type (rows may be strided, as slices of a fused projection are); g (log
    decay) and beta FP32 [tokens][value heads]; cu_seqlens int32 [sequences +
    1]: sequence i is rows cu_seqlens[i] .. cu_seqlens[i + 1] - 1.  state_in
    (None: zeros) and state_out (None: not kept) FP32 [slots][value heads][key
    dim][value dim], may be one tensor; sequence i's is slot slots[i] (int32;
    None: i), and a sequence with a slot outside the tensor is left out.
    scale: None for key dim^-1/2.  Returns out, [tokens][value heads][value
    dim]; where it is made here, rows of no sequence hold nothing defined.
    workspace: uint8, gdn_delta_prefill_workspace bytes (None: allocated).
    """
    if out is None:
        out = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    n_seqs = cu_seqlens.shape[0] - 1 if cu_seqlens.dim() == 1 else -1
    if n_seqs < 0:
        _fail("cu_seqlens: expected int32 [sequences + 1]")
    args = _delta(q, k, v, g, beta, out, state_in, state_out, slots, n_seqs, scale, l2norm)
    args.cu_seqlens = _on(q.device, "cu_seqlens", cu_seqlens, torch.int32, (n_seqs + 1,))
    lib, ref = L.load(), ctypes.byref(args)
    if workspace is None:
        workspace = torch.empty(lib.gdn_delta_prefill_workspace(ref), dtype=torch.uint8, device=q.device)
    ws = _on(q.device, "workspace", workspace, torch.uint8, (-1,))
    _launch(q.device, "gdn_delta_prefill", lib.gdn_delta_prefill, ref, ws, workspace.numel())
    return out


def delta_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
               state: torch.Tensor, *, state_out: Optional[torch.Tensor] = None,
               slots: Optional[torch.Tensor] = None, scale: Optional[float] = None, l2norm: bool = True,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """gdn_delta_step: one token of every sequence; row i of q, k, v, g, beta
    is sequence i's, its state slot slots[i] of ``state``, updated in place (or
    written to state_out).  Shapes and the rest as delta_prefill's."""
    if out is None:
        out = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    args = _delta(q, k, v, g, beta, out, state, state if state_out is None else state_out, slots, q.shape[0], scale,
                  l2norm)
    _launch(q.device, "gdn_delta_step", L.load().gdn_delta_step, ctypes.byref(args))
    return out
