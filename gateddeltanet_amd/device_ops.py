"""The operators on the caller's device tensors (include/gdn_amd.h, "operators
on the caller's device buffers"): the gated delta rule over a batch of
sequences, and the way from a batch's logits to its tokens.

Arguments are torch tensors on one GPU; work goes to that GPU's current stream
and is not waited for, and every call can be captured into a graph.  Where a
function makes its output or workspace, it takes them from torch's allocator on
that stream.  Errors raise ``GDNError``, before anything is enqueued.  Nothing
here is recorded for gradients, so where torch records them a floating-point
argument that requires one is an error; a tensor written in place counts as
modified, as after torch's own in-place operations.
"""
from __future__ import annotations

import ctypes
import functools
import struct
from typing import Optional, Tuple

import torch
from torch.autograd.graph import increment_version

from . import _lib as L
from .engine import GDNError

_DTYPES = {torch.bfloat16: L.DTYPE_BF16, torch.float16: L.DTYPE_FP16, torch.float32: L.DTYPE_FP32}


_raw_stream = torch._C._cuda_getCurrentRawStream  # current_stream().cuda_stream without the objects, 2.7 us less
_F32, _I32 = torch.float32, torch.int32


def _fail(what: str) -> None:
    raise GDNError(what)


def _apart_from_gradients(*tensors) -> None:
    if torch.is_grad_enabled():
        for x in tensors:
            if x is not None and x.requires_grad:
                _fail("an argument requires gradients, which these operators do not form: detach it, or call under "
                      "torch.no_grad()")


def _on(dev: int, name: str, x, dtype, shape) -> int:
    """The address of x, contiguous, of this type and shape on GPU dev (None: 0)."""
    if x is None:
        return 0
    if x.dtype is dtype and x.shape == shape and x.get_device() == dev and x.is_contiguous():
        return x.data_ptr()
    _fail(f"{name}: expected a contiguous {dtype} tensor of shape {tuple(shape)} on GPU {dev}, got {x.dtype} "
          f"{tuple(x.shape)} strides {x.stride()} on {x.device}")


# A call's struct as bytes: 0.7 us less than filling a ctypes object, and a value
# that passes its field is an error.
_CODES = {ctypes.c_int32: "i", ctypes.c_uint32: "I", ctypes.c_int64: "q", ctypes.c_float: "f", ctypes.c_void_p: "P"}


def _packer(cls):
    code = struct.Struct("@" + "".join(_CODES[t] for _, t in cls._fields_))
    if code.size != ctypes.sizeof(cls):
        raise TypeError(f"{cls.__name__}: {code.size} bytes packed, {ctypes.sizeof(cls)} wanted")

    def pack(*values) -> bytes:
        try:
            return code.pack(*values)
        except (struct.error, OverflowError) as e:
            raise GDNError(f"{cls.__name__}: {e}") from None

    return pack


_pack_delta, _pack_logits, _pack_sample = _packer(L.GDNDelta), _packer(L.GDNLogits), _packer(L.GDNSample)


@functools.lru_cache(maxsize=None)
def _entry(name: str):
    """The library's entry point, its struct taken as bytes."""
    fn = L.load()[name]  # (an object apart from the attribute's)
    fn.restype, args = L.SIGNATURES[name]
    fn.argtypes = [ctypes.c_char_p, *args[1:]]
    return fn


def _launch(dev: int, what: str, *args) -> None:
    """The entry point `what` (*args, stream) with GPU dev as the current one."""
    fn = _entry(what)
    if torch.cuda.current_device() == dev:
        rc = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(dev))
    if rc != 0:
        _fail(f"{what} failed (rc={rc})")


def _delta(q, k, v, g, beta, out, state_in, state_out, slots, n_seqs, cu, scale, l2norm):
    """(GPU, GDNDelta) of a call, checked."""
    _apart_from_gradients(q, k, v, g, beta, out, state_in, state_out)
    qt, dev = q.dtype, q.get_device()
    dtype = _DTYPES.get(qt)
    if dtype is None or dev < 0:
        _fail(f"q: expected a bfloat16, float16 or float32 tensor on a GPU, got {qt} on {q.device}")
    for name, x in (("q", q), ("k", k), ("v", v), ("out", out)):
        if x.dtype is not qt or x.dim() != 3 or x.get_device() != dev:
            _fail(f"{name}: expected {qt} [rows][heads][dim] on {q.device}, got {x.dtype} {tuple(x.shape)} on {x.device}")
    n, hq, dk = qs = q.shape
    _, hv, dv = vs = v.shape
    if k.shape != qs or vs[0] != n or out.shape != vs:
        _fail(f"shapes do not agree: q {tuple(qs)}, k {tuple(k.shape)}, v {tuple(vs)}, out {tuple(out.shape)}")
    sq, sk, sv, so = q.stride(), k.stride(), v.stride(), out.stride()
    heads, values = (dk, 1), (dv, 1)
    if n and (sq[1:] != heads or sk[1:] != heads or sv[1:] != values or so[1:] != values) and not (
            # (a single head's stride is not used)
            sq[2] == sk[2] == sv[2] == so[2] == 1 and (hq == 1 or sq[1] == sk[1] == dk) and (
                hv == 1 or sv[1] == so[1] == dv)):
        _fail(f"heads must be contiguous in a row: strides q {sq}, k {sk}, v {sv}, out {so}")
    gates, sg, sb = (n, hv), g.stride(), beta.stride()
    if g.shape != gates or beta.shape != gates or g.dtype is not _F32 or beta.dtype is not _F32 or (
            g.get_device() != dev or beta.get_device() != dev) or (
            n > 0 and hv > 1 and (sg[1] != 1 or sb[1] != 1)) or (n > 1 and sg[0] != sb[0]):
        _fail(f"g and beta: expected float32 [{n}][{hv}] of equal row strides on {q.device}")
    pool = state_in if state_out is None else state_out
    n_slots = n_seqs if pool is None else pool.shape[0] if pool.dim() else -1
    states = (n_slots, hv, dk, dv)
    at_in = _on(dev, "state_in", state_in, _F32, states)
    at_out = at_in if state_out is state_in else _on(dev, "state_out", state_out, _F32, states)
    if slots is None and n_slots < n_seqs:
        _fail(f"{n_seqs} sequences without slots need as many states, got {n_slots}")
    return dev, _pack_delta(
        dtype, n, n_seqs, hq, hv, dk, dv, 1 if l2norm else 0, dk**-0.5 if scale is None else scale, n_slots, sq[0],
        sk[0], sv[0], so[0], sg[0], q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), g.data_ptr(),
        beta.data_ptr(), _on(dev, "cu_seqlens", cu, _I32, (n_seqs + 1,)), _on(dev, "slots", slots, _I32, (n_seqs,)),
        at_in, at_out)


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
    dim], apart from every input; where it is made here, rows of no sequence
    hold nothing defined.
    workspace: uint8, gdn_delta_prefill_workspace bytes (None: allocated).
    """
    made = out is None
    if made:
        out = torch.empty_like(v, memory_format=torch.contiguous_format)
    n_seqs = cu_seqlens.shape[0] - 1 if cu_seqlens.dim() == 1 else -1
    if n_seqs < 0:
        _fail("cu_seqlens: expected int32 [sequences + 1]")
    dev, args = _delta(q, k, v, g, beta, out, state_in, state_out, slots, n_seqs, cu_seqlens, scale, l2norm)
    if workspace is None:
        workspace = torch.empty(_entry("gdn_delta_prefill_workspace")(args), dtype=torch.uint8, device=q.device)
    size = workspace.numel()
    _launch(dev, "gdn_delta_prefill", args,
            _on(dev, "workspace", workspace, torch.uint8, (size,)), size)
    if not made:
        increment_version(out)
    if state_out is not None:
        increment_version(state_out)
    return out


def delta_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
               state: torch.Tensor, *, state_out: Optional[torch.Tensor] = None,
               slots: Optional[torch.Tensor] = None, scale: Optional[float] = None, l2norm: bool = True,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """gdn_delta_step: one token of every sequence; row i of q, k, v, g, beta
    is sequence i's, its state slot slots[i] of ``state``, updated in place (or
    written to state_out).  Shapes and the rest as delta_prefill's."""
    made = out is None
    if made:
        out = torch.empty_like(v, memory_format=torch.contiguous_format)
    into = state if state_out is None else state_out
    dev, args = _delta(q, k, v, g, beta, out, state, into, slots, q.shape[0], None, scale, l2norm)
    _launch(dev, "gdn_delta_step", args)
    if not made:
        increment_version(out)
    if into is not None:
        increment_version(into)
    return out


def _logits(x: torch.Tensor, name: str = "logits"):
    """(GPU, type, rows, vocabulary, row stride) of a batch of logits."""
    dtype, dev = _DTYPES.get(x.dtype), x.get_device()
    if dtype is None or dev < 0 or x.dim() != 2 or (x.shape[1] > 1 and x.stride(1) != 1):
        _fail(f"{name}: expected a bfloat16, float16 or float32 [rows][vocabulary] on a GPU with contiguous rows, got "
              f"{x.dtype} {tuple(x.shape)} strides {x.stride()} on {x.device}")
    rows, vocab = x.shape
    return dev, dtype, rows, vocab, x.stride(0)


def _matrix(dev: int, name: str, x, rows: int):
    """(address, columns, row stride) of an int32 matrix (rows < 0: any)."""
    if x.dtype is not _I32 or x.dim() != 2 or x.get_device() != dev or (rows >= 0 and x.shape[0] != rows) or (
            x.shape[1] > 1 and x.stride(1) != 1):
        _fail(f"{name}: expected int32 [{rows if rows >= 0 else 'n'}][n] on GPU {dev} with contiguous rows, got "
              f"{x.dtype} {tuple(x.shape)} strides {x.stride()} on {x.device}")
    return x.data_ptr(), x.shape[1], x.stride(0) if x.shape[0] > 1 else x.shape[1]


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
    offsets, ids, values = (None, None, None) if bias is None else bias
    _apart_from_gradients(logits, out, repetition, presence, frequency, values)
    dev, dtype, rows, vocab, stride = _logits(logits)
    made = out is None
    if made:
        out = torch.empty_like(logits, memory_format=torch.contiguous_format)
        into = vocab
    else:
        to_dev, to_type, _, _, into = _logits(out, "out")
        if to_dev != dev or to_type != dtype or out.shape != logits.shape:
            _fail(f"out: expected {logits.dtype} {tuple(logits.shape)} on {logits.device}, got {out.dtype} "
                  f"{tuple(out.shape)} on {out.device}")
    one, hist, length, prompt, width, h_stride = (rows,), 0, 0, 0, 0, 0
    rep = pres = freq = 0
    if history is not None:
        if history_len is None:
            _fail("history needs history_len")
        hist, width, h_stride = _matrix(dev, "history", history, rows)
        length, prompt = _on(dev, "history_len", history_len, _I32, one), _on(dev, "prompt_len", prompt_len, _I32, one)
        rep, pres = _on(dev, "repetition", repetition, _F32, one), _on(dev, "presence", presence, _F32, one)
        freq = _on(dev, "frequency", frequency, _F32, one)
    elif not (history_len is prompt_len is repetition is presence is frequency is None):
        _fail("penalties need a history")
    b_at = b_ids = b_values = n_bias = 0
    if bias is not None:
        entries = (ids.numel(),)
        b_at = _on(dev, "bias offsets", offsets, _I32, (rows + 1,))
        b_ids, b_values = _on(dev, "bias ids", ids, _I32, entries), _on(dev, "bias values", values, _F32, entries)
        n_bias = entries[0]
    m_at = m_index = n_masks = m_stride = 0
    if mask is not None:
        m_at, words, m_stride = _matrix(dev, "mask", mask, -1)
        if words * 32 < vocab:
            _fail(f"mask: {words} words are fewer than {vocab} tokens")
        n_masks, m_index = mask.shape[0], _on(dev, "mask_index", mask_index, _I32, one)
        if mask_index is None and n_masks < rows:
            _fail(f"mask: {n_masks} masks for {rows} rows, and no mask_index")
    elif mask_index is not None:
        _fail("mask_index needs a mask")
    a = _pack_logits(dtype, rows, vocab, width, n_bias, n_masks, stride, into, h_stride, m_stride, logits.data_ptr(),
                     out.data_ptr(), hist, length, prompt, rep, pres, freq, b_at, b_ids, b_values, m_at, m_index)
    _launch(dev, "gdn_logits_process", a)
    if not made:
        increment_version(out)
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
    _apart_from_gradients(logits, uniform, temperature, top_p, min_p, logprobs)
    dev, dtype, rows, vocab, stride = _logits(logits)
    one, given = (rows,), [x for x in (tokens, logprobs) if x is not None]
    if tokens is None:
        tokens = torch.empty(one, dtype=_I32, device=logits.device)
    if logprobs is None:
        logprobs = torch.empty(one, dtype=_F32, device=logits.device)
    a = _pack_sample(dtype, rows, vocab, 0, stride, logits.data_ptr(), _on(dev, "uniform", uniform, _F32, one),
                     _on(dev, "temperature", temperature, _F32, one), _on(dev, "top_k", top_k, _I32, one),
                     _on(dev, "top_p", top_p, _F32, one), _on(dev, "min_p", min_p, _F32, one),
                     _on(dev, "tokens", tokens, _I32, one), _on(dev, "logprobs", logprobs, _F32, one))
    size = _entry("gdn_sample_workspace")(a)
    ws = torch.empty(size, dtype=torch.uint8, device=logits.device) if size else None
    _launch(dev, "gdn_sample_tokens", a, ws.data_ptr() if size else 0, size)
    if given:
        increment_version(given)
    return tokens, logprobs
