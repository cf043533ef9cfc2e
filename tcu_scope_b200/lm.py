"""Operators of language models next to the reductions and scans: the gated linear recurrence (a scan
whose running sum decays), with its gradient and its form for single tokens, and the norms around a block (sums of
squares of rows, and their use) fused with its gate and its residual, with their gradient, and the log
probabilities of given tokens (sums of exponentials of rows) with entropy and best alternatives, with their gradient.

Like the other operators these take CUDA tensors, call the C ABI on the current stream of the
tensors' device and return at once.  They are plain functions: autograd does not record them, so a tensor
that requires a gradient is refused while autograd records (call under ``torch.no_grad()`` or inside a
``torch.autograd.Function``), and one with a tangent of forward-mode autograd is, too; each operator has a function for its
gradient beside it.  An input may be a view
with any strides as long as the elements of a row (the last dimension) lie side by side; outputs that
the caller passes are contiguous and do not overlap other arguments except where it says so.
"""
from __future__ import annotations

import struct
from typing import NamedTuple

import torch

from . import _lib
from .ops import _check

_TYPE = {torch.float16: 0, torch.float32: 1, torch.bfloat16: 2}
GATE = {"decay": 0, "log": 1, "sigmoid": 2}
ACT = {"none": 0, "sigmoid": 1, "silu": 2}
_INDEX = (torch.int32, torch.int64)


# The current stream and device as plain numbers: the calls behind torch.cuda.current_stream() and
# current_device(), which take 2 us more, as long as a small operator runs.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_device_now = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_forward_ad = torch.autograd.forward_ad
_entries: dict = {}


def _launch(name: str, args: bytes, device: torch.device) -> None:
    """Calls an entry point that takes a struct of 8-byte fields, on the tensors' device and its current stream."""
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(_lib.load(), name)
    index = device.index
    if index == _device_now():
        status = fn(args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            status = fn(args, _raw_stream(index))
    if status:
        _check(status, name)


def _ptr(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def _inputs(device: torch.device, names: tuple, tensors: tuple) -> None:
    """What every input has to be: on the device of the first one, and not recorded by autograd."""
    if device.type != "cuda":
        raise RuntimeError("input must be a CUDA tensor: there is no CPU path in this library")
    duals = getattr(_forward_ad, "_current_level", 0) >= 0  # tensors can have tangents
    for i, t in enumerate(tensors):
        if t is None:
            continue
        if duals and _forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{names[i]} has a tangent, which forward-mode autograd would lose: unpack it, or call inside a "
                               "torch.autograd.Function with a jvp")
        if t.device != device:
            raise RuntimeError(f"{names[i]} is on {t.device}, the other tensors on {device}")
        if t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{names[i]} requires a gradient, which autograd would not get: call under "
                               "torch.no_grad() and use the operator's backward function")


def _rows(t: torch.Tensor, name: str) -> None:
    if t.stride(-1) != 1 and t.size(-1) > 1:
        raise ValueError(f"the last dimension of {name} must be contiguous")


def _result(t: torch.Tensor | None, name: str, shape, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """The caller's output tensor, checked, or a new one."""
    if t is None:
        return torch.empty(shape, dtype=dtype, device=device)
    if t.device != device or t.dtype != dtype or tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on {device}")
    return t


def _result_like(t: torch.Tensor | None, name: str, x: torch.Tensor) -> torch.Tensor:
    """The caller's output tensor, checked, or a new one, of x's shape and type."""
    if t is None:
        return torch.empty_like(x, memory_format=torch.contiguous_format)
    return _result(t, name, x.shape, x.dtype, x.device)


def _like(t: torch.Tensor | None, name: str, shape, dtype: torch.dtype) -> None:
    """Checks an optional contiguous input."""
    if t is not None and (t.dtype != dtype or tuple(t.shape) != tuple(shape) or not t.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)}")


# ------------------------------------------------------------------------------ linear recurrence

_SCAN = struct.Struct("=7Q3q4q5q")
_SCAN_BACKWARD = struct.Struct("=9Q3q6q5q")
_STEP = struct.Struct("=5Q3q2q5q")


def _scan_shape(a, x, gate, offsets):
    """(batch, tokens, dim) of a call, after checking what describes it."""
    if x.dtype not in _TYPE or a.dtype not in (x.dtype, torch.float32):
        raise TypeError("x must be float16, bfloat16 or float32, a of x's type or float32")
    if gate not in GATE:
        raise ValueError(f"gate must be one of {sorted(GATE)}")
    if a.shape != x.shape:
        raise ValueError(f"a and x must have one shape, got {tuple(a.shape)} and {tuple(x.shape)}")
    if offsets is None:
        if x.dim() != 3:
            raise ValueError("x must be (batch, tokens, dim), or (tokens, dim) with offsets")
        batch, tokens, dim = x.shape
    else:
        if x.dim() != 2:
            raise ValueError("x must be (tokens, dim) with offsets")
        if offsets.dtype not in _INDEX or offsets.dim() != 1 or offsets.numel() < 1 or not offsets.is_contiguous():
            raise ValueError("offsets must be a contiguous int32 or int64 tensor of batch + 1 values")
        (tokens, dim), batch = x.shape, offsets.numel() - 1
    _rows(a, "a")
    _rows(x, "x")
    return batch, tokens, dim


def _strides(t: torch.Tensor | None):
    """(batch stride, row stride)."""
    if t is None:
        return 0, 0
    return (t.stride(0), t.stride(1)) if t.dim() == 3 else (0, t.stride(0))


def linear_scan_states(x: torch.Tensor, offsets: torch.Tensor | None = None) -> torch.Tensor:
    """An uninitialised tensor for the ``states`` of :func:`linear_scan`: one row of floats for every 16 tokens."""
    if offsets is None:
        rows = _lib.load().tcu_linear_scan_states_rows(x.size(0), x.size(1), 0)
    else:
        rows = _lib.load().tcu_linear_scan_states_rows(offsets.numel() - 1, x.size(0), 1)
    return torch.empty((rows, x.size(-1)), dtype=torch.float32, device=x.device)


def linear_scan(a: torch.Tensor, x: torch.Tensor, gate: str = "decay", h0: torch.Tensor | None = None,
                offsets: torch.Tensor | None = None, states: torch.Tensor | None = None,
                out: torch.Tensor | None = None, last: torch.Tensor | None = None):
    """The gated linear recurrence ``h[t] = f[t] * h[t-1] + u[t]`` of every channel; returns ``(h, last)``.

    ``gate``: "decay" f = a, u = x; "log" f = exp(a), u = x; "sigmoid" f = sigmoid(a), u = (1 - f) * x.
    Gates are meant to have ``|f| <= 1`` (products of up to 1024 of them must stay within float32).

    x: (batch, tokens, dim), float16, bfloat16 or float32; a: the same shape, x's type or float32; h: x's shape
    and type.  h0: float32 (batch, dim), the states before the first tokens (default 0); last: float32
    (batch, dim), the states behind the last ones (may be h0 itself).

    With ``offsets`` (batch + 1 values, int32 or int64, on the device) x and a are (tokens, dim) and sequence b is their rows
    ``offsets[b] ... offsets[b+1]-1``.  An empty sequence leaves its state as it is.  Rows before the first and behind
    the last sequence are 0 in a new ``h`` and are left as they were in ``out``.  A sequence whose offsets decrease or
    pass the end counts as empty and raises bit 3 of :func:`device_error`; its rows are not written.  So do, but for one
    of them, sequences that then share rows or lie in another order than their numbers.

    states: from :func:`linear_scan_states`, for :func:`linear_scan_backward`.
    """
    device = x.device
    _inputs(device, ("x", "a", "h0", "offsets", "states"), (x, a, h0, offsets, states))
    batch, tokens, dim = _scan_shape(a, x, gate, offsets)
    _like(h0, "h0", (batch, dim), torch.float32)
    clear = out is None
    h = _result_like(out, "out", x)
    last = _result(last, "last", (batch, dim), torch.float32, device)
    if states is not None:
        rows = _lib.load().tcu_linear_scan_states_rows(batch, tokens, 0 if offsets is None else 1)
        _like(states, "states", (rows, dim), torch.float32)
    if offsets is not None and batch == 0:
        return (h.zero_() if clear else h), last
    _launch("tcu_linear_scan", _SCAN.pack(
        _ptr(a), _ptr(x), _ptr(h), _ptr(h0), _ptr(last), _ptr(states), _ptr(offsets), batch, tokens, dim,
        *_strides(a), *_strides(x), GATE[gate], _TYPE[a.dtype], _TYPE[x.dtype],
        offsets is not None and offsets.dtype == torch.int64, clear), device)
    return h, last


def linear_scan_backward(dh: torch.Tensor | None, a: torch.Tensor, x: torch.Tensor, states: torch.Tensor,
                         gate: str = "decay", dlast: torch.Tensor | None = None,
                         offsets: torch.Tensor | None = None, da: torch.Tensor | None = None,
                         dx: torch.Tensor | None = None, dh0: torch.Tensor | None = None):
    """The gradient of :func:`linear_scan`; returns ``(da, dx, dh0)``.

    dh: the gradient of h (x's shape and type; None: zero); dlast: that of ``last`` (None: zero); a, x, gate and
    offsets: as in the forward call, states: as it left them.  da and dx have the types of a and x, dh0 is float32.
    Rows before the first and behind the last sequence have gradient 0 in new tensors and are left as they were in the
    caller's.
    """
    device = x.device
    _inputs(device, ("x", "a", "dh", "states", "dlast", "offsets"), (x, a, dh, states, dlast, offsets))
    batch, tokens, dim = _scan_shape(a, x, gate, offsets)
    if dh is not None:
        if dh.shape != x.shape or dh.dtype != x.dtype:
            raise ValueError("dh must have the shape and type of x")
        _rows(dh, "dh")
    rows = _lib.load().tcu_linear_scan_states_rows(batch, tokens, 0 if offsets is None else 1)
    _like(states, "states", (rows, dim), torch.float32)
    _like(dlast, "dlast", (batch, dim), torch.float32)
    if offsets is not None and (da is None) != (dx is None):
        raise ValueError("with offsets, pass both da and dx or neither")
    clear = da is None
    da = _result_like(da, "da", a)
    dx = _result_like(dx, "dx", x)
    dh0 = _result(dh0, "dh0", (batch, dim), torch.float32, device)
    if offsets is not None and batch == 0:
        return (da.zero_(), dx.zero_(), dh0) if clear else (da, dx, dh0)
    _launch("tcu_linear_scan_backward", _SCAN_BACKWARD.pack(
        _ptr(dh), _ptr(a), _ptr(x), _ptr(states), _ptr(dlast), _ptr(da), _ptr(dx), _ptr(dh0), _ptr(offsets),
        batch, tokens, dim, *_strides(dh), *_strides(a), *_strides(x), GATE[gate], _TYPE[a.dtype],
        _TYPE[x.dtype], offsets is not None and offsets.dtype == torch.int64, clear), device)
    return da, dx, dh0


def linear_scan_step(a: torch.Tensor, x: torch.Tensor, state: torch.Tensor, gate: str = "decay",
                     slots: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """One token of :func:`linear_scan` for each of ``batch`` sequences: advances their states in place and returns h.

    a, x: (batch, dim); state: float32 (pool, dim), contiguous; row b advances ``state[slots[b]]`` (slots: int32 or
    int64; default: ``state[b]``).  A negative slot marks a padded row: its row of h is 0 in a new tensor and
    left as it was in ``out``.  The same holds, with bit 3 of :func:`device_error`, for a slot past the pool
    and for a slot that an earlier row names.
    """
    device = x.device
    _inputs(device, ("x", "a", "state", "slots"), (x, a, state, slots))
    if x.dim() != 2 or a.shape != x.shape:
        raise ValueError("a and x must both be (batch, dim)")
    if x.dtype not in _TYPE or a.dtype not in (x.dtype, torch.float32):
        raise TypeError("x must be float16, bfloat16 or float32, a of x's type or float32")
    if gate not in GATE:
        raise ValueError(f"gate must be one of {sorted(GATE)}")
    _rows(a, "a")
    _rows(x, "x")
    batch, dim = x.shape
    if state.dtype != torch.float32 or state.dim() != 2 or state.size(1) != dim or not state.is_contiguous():
        raise ValueError(f"state must be a contiguous float32 tensor of shape (pool, {dim})")
    if slots is None:
        if state.size(0) < batch:
            raise ValueError("state has fewer rows than x")
    elif slots.dtype not in _INDEX or tuple(slots.shape) != (batch,) or not slots.is_contiguous():
        raise ValueError("slots must be a contiguous int32 or int64 tensor of batch values")
    clear = out is None
    h = _result_like(out, "out", x)
    if batch and dim:
        _launch("tcu_linear_scan_step", _STEP.pack(
            _ptr(a), _ptr(x), _ptr(h), _ptr(state), _ptr(slots), batch, state.size(0), dim, a.stride(0),
            x.stride(0), GATE[gate], _TYPE[a.dtype], _TYPE[x.dtype],
            slots is not None and slots.dtype == torch.int64, clear), device)
    return h


# ------------------------------------------------------------------------------ norms, gate, residual

_NORM = struct.Struct("=7Q3q3q3q2d")
_NORM_BACKWARD = struct.Struct("=13Qq3q5q3q2d")


class NormGradients(NamedTuple):
    """What :func:`norm_residual_backward` returns; None for what the call did not have."""
    dz: torch.Tensor
    dresidual: torch.Tensor | None
    dpost_weight: torch.Tensor | None
    dgate: torch.Tensor | None
    dpre_weight: torch.Tensor | None


def _row_stride(t: torch.Tensor | None, name: str) -> int:
    """The stride between the rows of t (all dimensions but the last, one after the other)."""
    if t is None:
        return 0
    _rows(t, name)
    if t.dim() == 2:
        return t.stride(0)
    if t.is_contiguous() or t.numel() == 0:
        return t.size(-1)
    try:
        return t.view(-1, t.size(-1)).stride(0)
    except RuntimeError:
        raise ValueError(f"the rows of {name} must be one stride apart") from None


def _norm_arguments(z, residual, post_weight, gate, gate_act, pre_weight):
    """(rows, dim, gate rows, weight type) of a call, after checking what describes it."""
    if z.dtype not in _TYPE:
        raise TypeError("z must be float16, bfloat16 or float32")
    if z.dim() < 1 or z.size(-1) == 0:
        raise ValueError("z must have rows of at least one element")
    if gate_act not in ACT:
        raise ValueError(f"gate_act must be one of {sorted(ACT)}")
    dim = z.size(-1)
    rows = z.numel() // dim
    if residual is not None and (residual.shape != z.shape or residual.dtype != z.dtype):
        raise ValueError("residual must have the shape and type of z")
    weight = post_weight if post_weight is not None else pre_weight
    w_type = z.dtype if weight is None else weight.dtype
    if w_type not in (z.dtype, torch.float32):
        raise TypeError("weights must have z's type or float32")
    _like(post_weight, "post_weight", (dim,), w_type)
    _like(pre_weight, "pre_weight", (dim,), w_type)
    gate_rows = 1
    if gate is not None:
        if gate.dtype != z.dtype or gate.dim() < 1 or gate.size(-1) != dim:
            raise ValueError("gate must have z's type and last dimension")
        gate_rows = gate.numel() // dim
        if gate_rows == 1 and gate.dim() == 1:
            return rows, dim, 1, w_type
        lead, of = tuple(gate.shape[:-1]), tuple(z.shape[:-1])
        fits = lead == () or (len(of) == 1 and len(lead) == 1 and gate_rows > 0 and rows % gate_rows == 0) or \
            any(lead == of[:k] + (1,) * (len(of) - k) for k in range(len(of) + 1))
        if not fits:
            raise ValueError(f"gate {tuple(gate.shape)} does not give consecutive rows of z {tuple(z.shape)} a gate: "
                             "it is (dim,), (groups, dim) for a z of groups * n rows, or z's shape with trailing "
                             "dimensions before the last of size 1")
    return rows, dim, gate_rows, w_type


def norm_residual(z: torch.Tensor, residual: torch.Tensor | None = None, *,
                  post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                  gate_act: str = "none", scale: float = 1.0, pre_weight: torch.Tensor | None = None,
                  eps: float = 1e-6, out: torch.Tensor | None = None, normed: torch.Tensor | None = None):
    """The norm behind a block, its gate, its residual connection and the next block's norm; returns ``(out, normed)``.

    ``out = residual + scale * act(gate) * z / rms(z) * post_weight`` and
    ``normed = out / rms(out) * pre_weight``, ``rms(y) = sqrt(mean(y * y) + eps)`` of each row (the last dimension, up to
    16384 elements).  Without post_weight z is not normed, without pre_weight ``normed`` is None; without gate it is 1,
    without residual 0.  ``normed`` is made from ``out`` before that is rounded.

    z, residual: one shape; float16, bfloat16 or float32; gate: their type, of shape (dim,), of z's
    shape, of z's shape with 1 in the place of trailing dimensions before the last ((batch, 1, dim) for a z of (batch, tokens, dim)), or,
    for a z of (rows, dim), (groups, dim): a gate for each of groups * n consecutive rows.  gate_act: "none",
    "sigmoid" or "silu" of the gate.  Weights: (dim,), z's type or float32.
    ``out`` may be z or residual themselves, ``normed`` z, if they are contiguous.
    """
    device = z.device
    _inputs(device, ("z", "residual", "post_weight", "gate", "pre_weight"), (z, residual, post_weight, gate, pre_weight))
    rows, dim, gate_rows, w_type = _norm_arguments(z, residual, post_weight, gate, gate_act, pre_weight)
    out = _result_like(out, "out", z)
    if pre_weight is not None:
        normed = _result_like(normed, "normed", z)
    elif normed is not None:
        raise ValueError("normed needs pre_weight")
    if rows:
        _launch("tcu_norm_residual", _NORM.pack(
            _ptr(z), _ptr(residual), _ptr(post_weight), _ptr(gate), _ptr(pre_weight), _ptr(out), _ptr(normed),
            rows, dim, gate_rows, _row_stride(z, "z"), _row_stride(residual, "residual"),
            _row_stride(gate, "gate") if gate_rows > 1 else 0, ACT[gate_act], _TYPE[z.dtype], _TYPE[w_type],
            scale, eps), device)
    return out, normed


def norm_residual_backward(dout: torch.Tensor | None, dnormed: torch.Tensor | None, z: torch.Tensor,
                           residual: torch.Tensor | None = None, *, post_weight: torch.Tensor | None = None,
                           gate: torch.Tensor | None = None, gate_act: str = "none", scale: float = 1.0,
                           pre_weight: torch.Tensor | None = None, eps: float = 1e-6,
                           dz: torch.Tensor | None = None, dresidual: torch.Tensor | None = None,
                           workspace: torch.Tensor | None = None) -> NormGradients:
    """The gradient of :func:`norm_residual`, from those of ``out`` and ``normed`` (None: zero).

    The other arguments are those of the forward call.  Each gradient has the shape and type of what it is the
    gradient of; those of weights and of a gate that rows share are summed over the rows in a fixed order.
    ``dresidual`` may be dout itself; ``dz`` may be z, dnormed, or, if dresidual is not, dout.  workspace: bytes
    (tcu_norm_residual_workspace_bytes), not shared by calls that can run at the same time; default: a new one.
    """
    device = z.device
    _inputs(device, ("z", "residual", "post_weight", "gate", "pre_weight", "dout", "dnormed", "workspace"), (z, residual, post_weight, gate, pre_weight, dout, dnormed, workspace))
    rows, dim, gate_rows, w_type = _norm_arguments(z, residual, post_weight, gate, gate_act, pre_weight)
    for name, t in (("dout", dout), ("dnormed", dnormed)):
        if t is not None and (t.shape != z.shape or t.dtype != z.dtype):
            raise ValueError(f"{name} must have the shape and type of z")
    if dnormed is not None and pre_weight is None:
        raise ValueError("dnormed needs pre_weight")
    dz = _result_like(dz, "dz", z)
    if residual is not None:
        dresidual = _result_like(dresidual, "dresidual", z)
    elif dresidual is not None:
        raise ValueError("dresidual needs residual")
    dpost = None if post_weight is None else torch.empty_like(post_weight)
    dpre = None if pre_weight is None else torch.empty_like(pre_weight)
    dgate = None if gate is None else _result_like(None, "dgate", gate)
    need = _lib.load().tcu_norm_residual_workspace_bytes(rows, dim, gate_rows)
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
    elif not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    _launch("tcu_norm_residual_backward", _NORM_BACKWARD.pack(
        _ptr(dout), _ptr(dnormed), _ptr(z), _ptr(residual), _ptr(post_weight), _ptr(gate), _ptr(pre_weight),
        _ptr(dz), _ptr(dresidual), _ptr(dpost), _ptr(dgate), _ptr(dpre), _ptr(workspace),
        workspace.numel() * workspace.element_size(), rows, dim, gate_rows, _row_stride(dout, "dout"),
        _row_stride(dnormed, "dnormed"), _row_stride(z, "z"), _row_stride(residual, "residual"),
        _row_stride(gate, "gate") if gate_rows > 1 else 0, ACT[gate_act], _TYPE[z.dtype], _TYPE[w_type], scale,
        eps), device)
    return NormGradients(dz, dresidual, dpost, dgate, dpre)


# ------------------------------------------------------------------------------ log probabilities

_LOGPROBS = struct.Struct("=7Q5q2q")
_LOGPROBS_BACKWARD = struct.Struct("=7Q4q2q")


class TokenLogprobs(NamedTuple):
    """What :func:`token_logprobs` returns: float32, top_index int64."""
    logprob: torch.Tensor | None
    entropy: torch.Tensor
    lse: torch.Tensor
    top_logprob: torch.Tensor | None
    top_index: torch.Tensor | None


def _logits_rows(logits, targets):
    """(rows, vocab, row stride) of a call, after checking what describes it."""
    if logits.dtype not in _TYPE:
        raise TypeError("logits must be float16, bfloat16 or float32")
    if logits.dim() < 1 or logits.size(-1) == 0:
        raise ValueError("logits must have rows of at least one element")
    lead = logits.shape[:-1]
    if targets is not None and (targets.dtype not in _INDEX or targets.shape != lead or not targets.is_contiguous()):
        raise ValueError(f"targets must be a contiguous int32 or int64 tensor of shape {tuple(lead)}")
    return lead.numel(), logits.size(-1), _row_stride(logits, "logits")


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor | None = None, top: int = 0,
                   ignore_index: int = -100) -> TokenLogprobs:
    """Log probabilities of the target tokens under softmax(logits), with entropy and the ``top`` best alternatives.

    logits: (..., vocab), float16, bfloat16 or float32; targets: (...), int32 or int64 (None: no ``logprob``).
    Returns ``logprob`` (...), ``entropy`` (...), ``lse`` (...), the log of the sum of exponentials, and, with ``top`` (at most 32)
    above 0, ``top_logprob`` and ``top_index`` (..., top): the most probable tokens, the most probable first, the lowest index first
    where they are equal; NaN counts as the largest.

    Logits of -inf are tokens left out.  A row of nothing else has ``lse`` and log probabilities -inf and entropy 0; a
    row with NaN or +inf gives NaN.  A row whose target is ``ignore_index`` has ``logprob`` 0, and so, with bit
    3 of :func:`device_error`, has one whose target is out of range.
    """
    device = logits.device
    _inputs(device, ("logits", "targets"), (logits, targets))
    rows, vocab, stride = _logits_rows(logits, targets)
    if top > vocab:
        raise ValueError("top is more than the vocabulary")
    lead = logits.shape[:-1]
    lse, entropy, logprob = torch.empty((3, *lead), dtype=torch.float32, device=device).unbind(0)
    if targets is None:
        logprob = None
    top_logprob = torch.empty((*lead, top), dtype=torch.float32, device=device) if top else None
    top_index = torch.empty((*lead, top), dtype=torch.int64, device=device) if top else None
    if rows:
        _launch("tcu_token_logprobs", _LOGPROBS.pack(
            _ptr(logits), _ptr(targets), _ptr(logprob), _ptr(entropy), _ptr(lse), _ptr(top_logprob),
            _ptr(top_index), rows, vocab, stride, top, ignore_index, _TYPE[logits.dtype],
            targets is not None and targets.dtype == torch.int64), device)
    return TokenLogprobs(logprob, entropy, lse, top_logprob, top_index)


def token_logprobs_backward(logits: torch.Tensor, targets: torch.Tensor | None, lse: torch.Tensor,
                            entropy: torch.Tensor | None = None, *, dlogprob: torch.Tensor | None = None,
                            dentropy: torch.Tensor | None = None, ignore_index: int = -100,
                            out: torch.Tensor | None = None) -> torch.Tensor:
    """The gradient of the logits of :func:`token_logprobs`, from those of ``logprob`` and ``entropy`` (None: zero).

    lse and entropy: as the forward call returned them (entropy is wanted with dentropy, targets with dlogprob).
    Probabilities go by lse, whose rounding is their relative error (at most 2^-20 for float32 logits); rows whose |lse| is above
    32 (256 for 16-bit logits) are summed once more instead.
    ``out`` may be the logits themselves, if they are contiguous.
    """
    device = logits.device
    _inputs(device, ("logits", "targets", "lse", "entropy", "dlogprob", "dentropy"), (logits, targets, lse, entropy, dlogprob, dentropy))
    rows, vocab, stride = _logits_rows(logits, targets)
    for name, t in (("lse", lse), ("entropy", entropy), ("dlogprob", dlogprob), ("dentropy", dentropy)):
        _like(t, name, logits.shape[:-1], torch.float32)
    if (dlogprob is not None and targets is None) or (dentropy is not None and entropy is None):
        raise ValueError("dlogprob needs targets, dentropy needs entropy")
    out = _result_like(out, "out", logits)
    if rows:
        _launch("tcu_token_logprobs_backward", _LOGPROBS_BACKWARD.pack(
            _ptr(logits), _ptr(targets), _ptr(lse), _ptr(entropy), _ptr(dlogprob), _ptr(dentropy), _ptr(out),
            rows, vocab, stride, ignore_index, _TYPE[logits.dtype],
            targets is not None and targets.dtype == torch.int64), device)
    return out
