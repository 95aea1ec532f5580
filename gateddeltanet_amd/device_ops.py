"""The operators on the caller's device tensors (include/gdn_amd.h, "operators
on the caller's device buffers"): the recurrences over a batch of sequences (the
gated delta rule, the selective state space scan), the short convolution in front
of them, the norm around them, and the way from a batch's logits to its tokens.

Arguments are torch tensors on one GPU; work goes to that GPU's current stream
and is not waited for, and every call can be captured into a graph.  Where a
function makes its output or workspace, it takes them from torch's allocator on
that stream.  Errors raise ``GDNError``, before anything is enqueued.  Nothing
here is recorded for gradients, so where torch records them a floating-point
argument that requires one is an error, and so is one with a tangent; a tensor
written in place counts as modified, as after torch's own in-place operations.
"""
from __future__ import annotations

import ctypes
import functools
import struct
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import _lib as L
from .engine import GDNError

_DTYPES = {torch.bfloat16: L.DTYPE_BF16, torch.float16: L.DTYPE_FP16, torch.float32: L.DTYPE_FP32}


_raw_stream = torch._C._cuda_getCurrentRawStream  # current_stream().cuda_stream without the objects, 2.7 us less
_current_device = torch._C._cuda_getDevice  # (a tensor on a GPU is there: torch is initialised), 0.2 us less
_F32, _I32 = torch.float32, torch.int32


def _fail(what: str) -> None:
    raise GDNError(what)


def _apart_from_gradients(*tensors) -> None:
    if torch.is_grad_enabled():
        for x in tensors:
            if x is not None and x.requires_grad:
                _fail("an argument requires gradients, which these operators do not form: detach it, or call under "
                      "torch.no_grad()")
    if forward_ad._current_level >= 0:  # (a level is open, which no_grad() does not close)
        for x in tensors:
            if x is not None and forward_ad.unpack_dual(x).tangent is not None:
                _fail("an argument carries a tangent, which these operators do not pass on: unpack it first")


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
_pack_conv, _pack_scan, _pack_norm = _packer(L.GDNConv), _packer(L.GDNScan), _packer(L.GDNNorm)


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
    if _current_device() == dev:
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


def _sequences(cu) -> int:
    if cu.dim() != 1 or cu.shape[0] < 1:
        _fail("cu_seqlens: expected int32 [sequences + 1]")
    return cu.shape[0] - 1


def _conv(x, weight, bias, silu, out, state_in, state_out, slots, n_seqs, cu):
    """(GPU, GDNConv) of a call, checked."""
    _apart_from_gradients(x, weight, bias, out, state_in, state_out)
    xt, dev = x.dtype, x.get_device()
    dtype = _DTYPES.get(xt)
    if dtype is None or dev < 0 or x.dim() != 2:
        _fail(f"x: expected a bfloat16, float16 or float32 [tokens][channels] on a GPU, got {xt} {tuple(x.shape)} on "
              f"{x.device}")
    n, channels = xs = x.shape
    if out.dtype is not xt or out.shape != xs or out.get_device() != dev:
        _fail(f"out: expected {xt} {tuple(xs)} on {x.device}, got {out.dtype} {tuple(out.shape)} on {out.device}")
    sx, so = x.stride(), out.stride()
    if n and channels > 1 and (sx[1] != 1 or so[1] != 1):
        _fail(f"channels must be contiguous: strides x {sx}, out {so}")
    if weight.dim() != 2:
        _fail(f"weight: expected float32 [channels][width], got {tuple(weight.shape)}")
    width = weight.shape[1]
    pool = state_in if state_out is None else state_out
    n_slots = n_seqs if pool is None else pool.shape[0] if pool.dim() else -1
    tails = (n_slots, width - 1, channels)
    at_in = _on(dev, "state_in", state_in, xt, tails)
    at_out = at_in if state_out is state_in else _on(dev, "state_out", state_out, xt, tails)
    if slots is None and n_slots < n_seqs:
        _fail(f"{n_seqs} sequences without slots need as many states, got {n_slots}")
    return dev, _pack_conv(
        dtype, n, n_seqs, channels, width, 1 if silu else 0, n_slots, 0, sx[0], so[0], x.data_ptr(), out.data_ptr(),
        _on(dev, "weight", weight, _F32, (channels, width)), _on(dev, "bias", bias, _F32, (channels,)),
        _on(dev, "cu_seqlens", cu, _I32, (n_seqs + 1,)), _on(dev, "slots", slots, _I32, (n_seqs,)), at_in, at_out)


def conv_prefill(x: torch.Tensor, weight: torch.Tensor, cu_seqlens: torch.Tensor, *, bias: Optional[torch.Tensor] = None,
                 silu: bool = True, state_in: Optional[torch.Tensor] = None, state_out: Optional[torch.Tensor] = None,
                 slots: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """gdn_conv_prefill: the short causal convolution over packed sequences.

    x [tokens][channels] (rows may be strided, as slices of a fused projection are);
    weight FP32 [channels][width], width 2 to 4, its last column the token's own;
    bias FP32 [channels]; silu: the output through SiLU.  cu_seqlens and slots as
    delta_prefill's.  state_in (None: zeros) and state_out (None: not kept): the tails,
    the width - 1 inputs before (behind) the sequence, oldest first, of x's type
    [slots][width - 1][channels], may be one tensor.  Returns out, [tokens][channels],
    apart from x; where it is made here, rows of no sequence hold nothing defined.
    """
    made = out is None
    if made:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    dev, args = _conv(x, weight, bias, silu, out, state_in, state_out, slots, _sequences(cu_seqlens), cu_seqlens)
    _launch(dev, "gdn_conv_prefill", args)
    if not made:
        increment_version(out)
    if state_out is not None:
        increment_version(state_out)
    return out


def conv_step(x: torch.Tensor, weight: torch.Tensor, state: torch.Tensor, *, bias: Optional[torch.Tensor] = None,
              silu: bool = True, state_out: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """gdn_conv_step: one token of every sequence; row i of x is sequence i's, its
    tail slot slots[i] of ``state``, updated in place (or written to state_out).  out
    may be x.  Shapes and the rest as conv_prefill's."""
    made = out is None
    if made:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    into = state if state_out is None else state_out
    dev, args = _conv(x, weight, bias, silu, out, state, into, slots, x.shape[0] if x.dim() else 0, None)
    _launch(dev, "gdn_conv_step", args)
    if not made:
        increment_version(out)
    if into is not None:
        increment_version(into)
    return out


def _scan(x, dt, A, B, C, D, dt_bias, softplus, out, state_in, state_out, slots, n_seqs, cu):
    """(GPU, GDNScan) of a call, checked."""
    _apart_from_gradients(x, dt, A, B, C, D, dt_bias, out, state_in, state_out)
    xt, dev = x.dtype, x.get_device()
    dtype = _DTYPES.get(xt)
    if dtype is None or dev < 0:
        _fail(f"x: expected a bfloat16, float16 or float32 tensor on a GPU, got {xt} on {x.device}")
    for name, y in (("x", x), ("B", B), ("C", C), ("out", out)):
        if y.dtype is not xt or y.dim() != 3 or y.get_device() != dev:
            _fail(f"{name}: expected {xt} [rows][heads][dim] on {x.device}, got {y.dtype} {tuple(y.shape)} on {y.device}")
    n, heads, P = xs = x.shape
    _, groups, N = bs = B.shape
    if C.shape != bs or bs[0] != n or out.shape != xs:
        _fail(f"shapes do not agree: x {tuple(xs)}, B {tuple(bs)}, C {tuple(C.shape)}, out {tuple(out.shape)}")
    sx, sb, sc, so = x.stride(), B.stride(), C.stride(), out.stride()
    wide, narrow = (P, 1), (N, 1)
    if n and (sx[1:] != wide or so[1:] != wide or sb[1:] != narrow or sc[1:] != narrow) and not (
            # (a single head's or group's stride is not used)
            sx[2] == so[2] == sb[2] == sc[2] == 1 and (heads == 1 or sx[1] == so[1] == P) and (
                groups == 1 or sb[1] == sc[1] == N)):
        _fail(f"heads must be contiguous in a row: strides x {sx}, B {sb}, C {sc}, out {so}")
    sd, of = dt.stride(), dt.dtype
    if dt.shape != (n, heads) or (of is not xt and of is not _F32) or dt.get_device() != dev or (
            n > 0 and heads > 1 and sd[1] != 1):
        _fail(f"dt: expected {xt} or float32 [{n}][{heads}] on {x.device} with contiguous rows, got {of} "
              f"{tuple(dt.shape)} strides {sd} on {dt.device}")
    pool = state_in if state_out is None else state_out
    n_slots = n_seqs if pool is None else pool.shape[0] if pool.dim() else -1
    states, each = (n_slots, heads, N, P), (heads,)
    at_in = _on(dev, "state_in", state_in, _F32, states)
    at_out = at_in if state_out is state_in else _on(dev, "state_out", state_out, _F32, states)
    if slots is None and n_slots < n_seqs:
        _fail(f"{n_seqs} sequences without slots need as many states, got {n_slots}")
    return dev, _pack_scan(
        dtype, _DTYPES[of], n, n_seqs, heads, groups, N, P, 1 if softplus else 0, n_slots, sx[0], sb[0], sc[0], sd[0],
        so[0], x.data_ptr(), B.data_ptr(), C.data_ptr(), dt.data_ptr(), out.data_ptr(), _on(dev, "A", A, _F32, each),
        _on(dev, "D", D, _F32, each), _on(dev, "dt_bias", dt_bias, _F32, each),
        _on(dev, "cu_seqlens", cu, _I32, (n_seqs + 1,)), _on(dev, "slots", slots, _I32, (n_seqs,)), at_in, at_out)


def scan_prefill(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                 cu_seqlens: torch.Tensor, *, D: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None,
                 softplus: bool = False, state_in: Optional[torch.Tensor] = None,
                 state_out: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """gdn_scan_prefill: the selective state space scan over packed sequences.

    x [tokens][heads][head dim], B and C [tokens][groups][state dim] of one type
    (rows may be strided); dt [tokens][heads] of that type or FP32, the steps, or
    what dt_bias is added to and (softplus) a softplus makes them of; A (negative in a
    stable model), D and dt_bias FP32 [heads].  cu_seqlens, state_in, state_out and
    slots as delta_prefill's, states FP32 [slots][heads][state dim][head dim].
    Returns out, as x, apart from every input; where it is made here, rows of no
    sequence hold nothing defined.
    workspace: uint8, gdn_scan_prefill_workspace bytes (None: allocated).
    """
    made = out is None
    if made:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    dev, args = _scan(x, dt, A, B, C, D, dt_bias, softplus, out, state_in, state_out, slots, _sequences(cu_seqlens),
                      cu_seqlens)
    at = 0
    if workspace is None:
        size = _entry("gdn_scan_prefill_workspace")(args)
        if size:
            workspace = x.new_empty(size, dtype=torch.uint8)
            at = workspace.data_ptr()
    else:
        size = workspace.numel()
        at = _on(dev, "workspace", workspace, torch.uint8, (size,))
    _launch(dev, "gdn_scan_prefill", args, at, size)
    if not made:
        increment_version(out)
    if state_out is not None:
        increment_version(state_out)
    return out


def scan_step(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, state: torch.Tensor,
              *, D: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None, softplus: bool = False,
              state_out: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """gdn_scan_step: one token of every sequence; row i of x, dt, B and C is
    sequence i's, its state slot slots[i] of ``state``, updated in place (or written
    to state_out).  Shapes and the rest as scan_prefill's."""
    made = out is None
    if made:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    into = state if state_out is None else state_out
    dev, args = _scan(x, dt, A, B, C, D, dt_bias, softplus, out, state, into, slots, x.shape[0] if x.dim() else 0, None)
    _launch(dev, "gdn_scan_step", args)
    if not made:
        increment_version(out)
    if into is not None:
        increment_version(into)
    return out


def _rows(dev: int, name: str, x, dtype, shape):
    """(address, row stride) of rows of this type and shape on GPU dev, the rest of
    a row contiguous (None: 0)."""
    if x is None:
        return 0, 0
    st = x.stride()
    if x.dtype is not dtype or x.shape != shape or x.get_device() != dev or (
            st[-1] != 1 and shape[-1] > 1 and x.numel()) or (
            len(shape) == 3 and shape[1] > 1 and x.numel() and st[1] != shape[2]):
        _fail(f"{name}: expected {dtype} {tuple(shape)} on GPU {dev} with contiguous rows, got {x.dtype} "
              f"{tuple(x.shape)} strides {st} on {x.device}")
    return x.data_ptr(), st[0]


def _norm(x, weight, eps, residual, gate, gate_first, out, out_type, total, scales, block):
    _apart_from_gradients(x, weight, residual, gate, out, total, scales)
    xt, dev, shape = x.dtype, x.get_device(), x.shape
    dtype = _DTYPES.get(xt)
    if dtype is None or dev < 0 or len(shape) not in (2, 3):
        _fail(f"x: expected a bfloat16, float16 or float32 [rows][dim] or [rows][heads][dim] on a GPU, got {xt} "
              f"{tuple(shape)} on {x.device}")
    rows, dim, heads = shape[0], shape[-1], shape[1] if len(shape) == 3 else 1
    if total is not None and residual is None:
        _fail("the sum needs a residual")
    if gate_first and gate is None:
        _fail("gate_first needs a gate")
    shared = weight is None or weight.dim() == 1
    at_x, sx = _rows(dev, "x", x, xt, shape)
    at_r, sr = _rows(dev, "residual", residual, xt, shape)
    at_g, sg = _rows(dev, "gate", gate, xt, shape)
    at_o, so = _rows(dev, "out", out, out_type, shape)
    at_s, ss = _rows(dev, "sum", total, xt, shape)
    _launch(dev, "gdn_rms_norm", _pack_norm(
        dtype, rows, heads, dim, 1 if gate_first else 0, 0 if shared else 1, 0 if scales is None else 1, block, eps, 0,
        sx, sr, sg, so, ss, at_x, at_r, at_g, _on(dev, "weight", weight, _F32, (dim,) if shared else (heads, dim)),
        at_o, at_s, 0 if scales is None else _on(
            dev, "scales", scales, _F32, (rows, heads * dim // block if block else 1))))


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, *, eps: float = 1e-6,
             residual: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, gate_first: bool = False,
             out: Optional[torch.Tensor] = None, sum_out: Optional[torch.Tensor] = None):
    """gdn_rms_norm: the root-mean-square norm over the last dimension.

    x [rows][dim] or [rows][heads][dim] (rows may be strided); weight FP32 [dim], or
    [heads][dim]; residual and gate as x.  x + residual is normed; SiLU of the gate
    multiplies the normed values, or (gate_first) what is normed.  Returns out, as x,
    or with a residual (out, sum_out), the sum rounded to x's type.  out may be x, residual
    or gate, sum_out x or residual.
    Squares are FP32: with an eps below 2^-126 a head below 2^-63 has fewer bits, with 0
    one of values below 2^-75 infinities and NaN.
    """
    given = [y for y in (out, sum_out) if y is not None]
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    if residual is not None and sum_out is None:
        sum_out = torch.empty_like(x, memory_format=torch.contiguous_format)
    _norm(x, weight, eps, residual, gate, gate_first, out, x.dtype, sum_out, None, 0)
    if given:
        increment_version(given)
    return out if residual is None else (out, sum_out)


def rms_norm_fp8(x: torch.Tensor, weight: Optional[torch.Tensor] = None, *, block: int = 0, eps: float = 1e-6,
                 residual: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                 gate_first: bool = False, out: Optional[torch.Tensor] = None, scales: Optional[torch.Tensor] = None,
                 sum_out: Optional[torch.Tensor] = None):
    """gdn_rms_norm with an output in 8 bits: (out, scales), or with a residual (out,
    scales, sum_out).  out, float8_e4m3fn as x, times its scale stands for the normed
    values; scales FP32 [rows][heads * dim / block], a scale for every 32, 64 or 128
    values of a row, or [rows][1] (block 0).  The rest as rms_norm's."""
    given = [y for y in (out, scales, sum_out) if y is not None]
    if out is None:
        out = torch.empty_like(x, dtype=torch.float8_e4m3fn, memory_format=torch.contiguous_format)
    if block not in (0, 32, 64, 128):
        _fail(f"block: expected 0, 32, 64 or 128, got {block}")
    if scales is None:
        wide = x.shape[-1] * (x.shape[1] if x.dim() == 3 else 1) if x.dim() else 0
        scales = x.new_empty((x.shape[0] if x.dim() else 0, wide // block if block else 1), dtype=_F32)
    if residual is not None and sum_out is None:
        sum_out = torch.empty_like(x, memory_format=torch.contiguous_format)
    _norm(x, weight, eps, residual, gate, gate_first, out, torch.float8_e4m3fn, sum_out, scales, block)
    if given:
        increment_version(given)
    return (out, scales) if residual is None else (out, scales, sum_out)


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
