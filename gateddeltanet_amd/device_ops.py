"""The operators on the caller's device tensors (include/gdn_amd.h, "operators
on the caller's device buffers"): the gated delta rule over a batch of
sequences, and the way from a batch's logits to its tokens.

Arguments are torch tensors on one GPU; work goes to that GPU's current stream
and is not waited for, and every call can be captured into a graph.  Where a
function makes its output or workspace, it takes them from torch's allocator on
that stream.  Errors raise ``GDNError``, before anything is enqueued.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

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


def _logits(x: torch.Tensor, name: str = "logits") -> int:
    dtype = _DTYPES.get(x.dtype)
    if dtype is None or not x.is_cuda or x.dim() != 2 or (x.shape[1] > 1 and x.stride(1) != 1):
        _fail(f"{name}: expected a bfloat16, float16 or float32 [rows][vocabulary] on a GPU with contiguous rows, got "
              f"{x.dtype} {tuple(x.shape)} on {x.device}")
    return dtype


def _matrix(device, name: str, x, dtype, rows: int) -> int:
    if x.device != device or x.dtype != dtype or x.dim() != 2 or (rows >= 0 and x.shape[0] != rows) or (
            x.shape[1] > 1 and x.stride(1) != 1):
        _fail(f"{name}: expected {dtype} [{rows if rows >= 0 else 'n'}][n] on {device} with contiguous rows, got "
              f"{x.dtype} {tuple(x.shape)} on {x.device}")
    return x.data_ptr()


def logits_process(logits: torch.Tensor, *, history: Optional[torch.Tensor] = None,
                   history_len: Optional[torch.Tensor] = None, prompt_len: Optional[torch.Tensor] = None,
                   repetition: Optional[torch.Tensor] = None, presence: Optional[torch.Tensor] = None,
                   frequency: Optional[torch.Tensor] = None,
                   bias: Optional[Tuple[torch.Tensor, torch.Tensor, torch.Tensor]] = None,
                   mask: Optional[torch.Tensor] = None, mask_index: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """gdn_logits_process: penalties for repeated tokens, biases and masks.

    logits [rows][vocab]; history int32 [rows][width] with history_len and
    prompt_len int32 [rows]; repetition, presence, frequency FP32 [rows]; bias
    (offsets int32 [rows + 1], ids int32, values FP32); mask int32 words
    [masks][>= vocab / 32] with a set bit for every allowed token, mask_index
    int32 [rows].  out may be logits itself.  Returns out.
    """
    dtype, device, rows = _logits(logits), logits.device, logits.shape[0]
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=device)
    elif _logits(out, "out") != dtype or out.shape != logits.shape or out.device != device:
        _fail(f"out: expected {logits.dtype} {tuple(logits.shape)} on {device}, got {out.dtype} {tuple(out.shape)}")
    a = L.GDNLogits(dtype, rows, logits.shape[1], 0, 0, 0, logits.stride(0), out.stride(0), 0, 0, logits.data_ptr(),
                    out.data_ptr())
    if history is not None:
        if history_len is None:
            _fail("history needs history_len")
        a.history = _matrix(device, "history", history, torch.int32, rows)
        a.history_width, a.history_stride = history.shape[1], history.stride(0)
        a.history_len = _on(device, "history_len", history_len, torch.int32, (rows,))
        a.prompt_len = _on(device, "prompt_len", prompt_len, torch.int32, (rows,))
        a.repetition = _on(device, "repetition", repetition, torch.float32, (rows,))
        a.presence = _on(device, "presence", presence, torch.float32, (rows,))
        a.frequency = _on(device, "frequency", frequency, torch.float32, (rows,))
    elif not (history_len is prompt_len is repetition is presence is frequency is None):
        _fail("penalties need a history")
    if bias is not None:
        offsets, ids, values = bias
        a.bias_offsets = _on(device, "bias offsets", offsets, torch.int32, (rows + 1,))
        a.bias_ids = _on(device, "bias ids", ids, torch.int32, (-1,))
        a.bias_values = _on(device, "bias values", values, torch.float32, (ids.shape[0],))
        a.n_bias = ids.shape[0]
    if mask is not None:
        a.mask = _matrix(device, "mask", mask, torch.int32, -1)
        a.n_masks, a.mask_stride = mask.shape[0], mask.stride(0) if mask.shape[0] > 1 else mask.shape[1]
        if mask.shape[1] * 32 < logits.shape[1]:
            _fail(f"mask: {mask.shape[1]} words are fewer than {logits.shape[1]} tokens")
        a.mask_index = _on(device, "mask_index", mask_index, torch.int32, (rows,))
    elif mask_index is not None:
        _fail("mask_index needs a mask")
    _launch(device, "gdn_logits_process", L.load().gdn_logits_process, ctypes.byref(a))
    return out


def sample_tokens(logits: torch.Tensor, uniform: Optional[torch.Tensor] = None, *,
                  temperature: Optional[torch.Tensor] = None, top_k: Optional[torch.Tensor] = None,
                  top_p: Optional[torch.Tensor] = None, min_p: Optional[torch.Tensor] = None,
                  tokens: Optional[torch.Tensor] = None,
                  logprobs: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """gdn_sample_tokens: a token of every row and its log-probability.

    logits [rows][vocab]; uniform (in [0, 1)), temperature, top_p and min_p
    FP32 [rows], top_k int32 [rows].  Without a temperature, or where it is not
    positive: the first of the highest logits.  Returns (tokens int32 [rows],
    logprobs FP32 [rows]); -1 where no logit is above -infinity.
    """
    dtype, device, rows = _logits(logits), logits.device, logits.shape[0]
    if tokens is None:
        tokens = torch.empty(rows, dtype=torch.int32, device=device)
    if logprobs is None:
        logprobs = torch.empty(rows, dtype=torch.float32, device=device)
    a = L.GDNSample(dtype, rows, logits.shape[1], 0, logits.stride(0), logits.data_ptr(),
                    _on(device, "uniform", uniform, torch.float32, (rows,)),
                    _on(device, "temperature", temperature, torch.float32, (rows,)),
                    _on(device, "top_k", top_k, torch.int32, (rows,)),
                    _on(device, "top_p", top_p, torch.float32, (rows,)),
                    _on(device, "min_p", min_p, torch.float32, (rows,)),
                    _on(device, "tokens", tokens, torch.int32, (rows,)),
                    _on(device, "logprobs", logprobs, torch.float32, (rows,)))
    _launch(device, "gdn_sample_tokens", L.load().gdn_sample_tokens, ctypes.byref(a))
    return tokens, logprobs
