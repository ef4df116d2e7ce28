"""Readout operators over a network's captured outputs, on the GPU.

``learn.capture_signals_cached`` brings out the course of a network's output voltages, and
``learn.replay_grads_from_cached_signals`` takes the loss's gradient by them.  The operators
here stand between the two: what turns that course into answers, the loss that teaches it from
a trained network, and the gradients of both.

  linear_attention, linear_attention_grad   a temporal readout over whole recordings: linear
                                            attention whose state decays as a synapse's does
  linear_attention_step                     the same for one tick of a running network
  gated_recurrence, gated_recurrence_grad   a state for each channel that moves to its input as far as its gate
                                            lets it, over whole recordings
  gated_recurrence_step                     the same for one tick
  layer_norm, layer_norm_grad               rows brought to one mean and size, for recordings and ticks alike
  distill_loss, distill_loss_grad           the loss against a teacher's top logits
  token_logprobs, token_logprobs_grad       log probabilities of given answers, entropies and the top
                                            alternatives, with their gradient
  sample                                    an answer drawn from logits
  adamw_state, adamw_step                   an AdamW step of many parameters at once, moments in 32 bits or 8

They take and return torch tensors on one GPU (fp32, fp16 or bf16), work on torch's current
stream, wait for nothing, and may be captured into a graph.  Sums, softmax statistics and
states are fp32 or wider whatever the inputs are.  Arguments that do not fit raise ValueError
or TypeError; sizes, values and overlaps that the library refuses, and launches that fail, raise
HelioxError.  Results carry no graph for autograd: gradients are calls of their own, and the calls
that have one refuse inputs that require a gradient while torch records.  What a call writes in
place counts as changed: a backward pass that kept its old values is refused by torch.
"""
from __future__ import annotations

import functools
import operator
import struct
from array import array
from typing import NamedTuple, Optional, Sequence, Tuple, Union

import torch

from .sim import HelioxError, lib

# The records of include/heliox.h, field by field (8 bytes each).
_ATTENTION = struct.Struct("=9q 3Q 9q 3Q d Q 3q Q Q 3q Q 3Q Q Q Q q Q q Q")
_DISTILL = struct.Struct("=6q Q q Q q Q q 2Q d Q Q q Q")
_NORM = struct.Struct("=4q Q q 2Q d Q q 2Q Q q Q q 2Q Q q Q")
_RECURRENCE = struct.Struct("=4q 2Q 4q 2Q Q 2q Q Q 2q Q 2Q Q 2Q q Q q Q")
_LOGPROB = struct.Struct("=5q Q q Q d 3Q 2Q 2Q Q q Q q Q")
_ADAMW = struct.Struct("=2q 7Q 2Q 2Q q 5d 2Q Q Q")
_SAMPLE = struct.Struct("=3q Q q Q Q Q 2Q 3d q 2Q Q")

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


# A call's checks are most of a small call's time, so each goes the short way first (attributes
# compared as they are, devices as numbers, 50-80 ns each) and finds out what is wrong only where
# something is.


def _no_graph(call: str, instead: str, *inputs: Optional[torch.Tensor]) -> None:
    """Results here carry no autograd graph: where one is being recorded, a gradient that an input
    asks for would be lost in silence."""
    if torch.is_grad_enabled():
        for x in inputs:
            if x is not None and x.requires_grad:
                raise ValueError(f"{call} records no graph for autograd, and an input requires a gradient: "
                                 f"{instead}, and call {call} under torch.no_grad() or in an autograd.Function")


def _type(x: torch.Tensor, what: str) -> int:
    kind = _TYPES.get(x.dtype)
    if kind is None:
        raise TypeError(f"{what}: {x.dtype} is not float32, float16 or bfloat16")
    return kind


def _on_gpu(x: torch.Tensor, what: str) -> int:
    """The number of the GPU that x is on."""
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{what} has to be a tensor, got {type(x).__name__}")
    device = x.get_device()
    if device < 0:
        raise ValueError(f"{what} has to be on the GPU, it is on {x.device}")
    return device


def _empty(x: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor like x (empty_like is the quicker call, but keeps strides)."""
    return torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x with its last dimension contiguous (a copy only where it is not)."""
    return x if x.stride(-1) == 1 or x.shape[-1] <= 1 else x.contiguous()


def _array(x: Optional[torch.Tensor], what: str, dtype: torch.dtype, shape: tuple,
           device: int) -> Optional[torch.Tensor]:
    """An argument that is handed on as a contiguous array of one type."""
    if x is None:
        return None
    if not isinstance(x, torch.Tensor) or x.get_device() != device:
        if _on_gpu(x, what) != device:
            raise ValueError(f"{what} is on {x.device}, not on cuda:{device}")
    if x.dtype is not dtype:
        raise TypeError(f"{what} is {x.dtype}, expected {dtype}")
    if x.shape != shape:
        raise ValueError(f"{what} has shape {tuple(x.shape)}, expected {tuple(shape)}")
    return x if x.is_contiguous() else x.contiguous()


def _real(x, what: str) -> float:
    if type(x) is float:
        return x
    try:
        if isinstance(x, (str, bytes)):
            raise TypeError
        return float(x)
    except OverflowError:
        raise ValueError(f"{what} is too large a number") from None
    except (TypeError, ValueError):
        raise TypeError(f"{what} has to be a number, got {type(x).__name__}") from None


def _scale(scale, dk: int) -> float:
    return dk ** -0.5 if scale is None else _real(scale, "scale")


def _whole(x, what: str) -> int:
    try:
        x = operator.index(x)
    except TypeError:
        raise TypeError(f"{what} has to be a whole number, got {type(x).__name__}") from None
    if not -2 ** 63 <= x < 2 ** 63:
        raise ValueError(f"{what} is too large a number")
    return x


def _ptr(x: Optional[torch.Tensor]) -> int:
    return 0 if x is None else x.data_ptr()


# torch's current stream on a device as the number that the library takes (torch.cuda's own
# object for it takes 2 us to make).
_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (
    lambda device: torch.cuda.current_stream(device).cuda_stream)

# (the public call takes twice as long for one tensor)
_count_writes = getattr(torch._C, "_increment_version", torch.autograd.graph.increment_version)


def _written(*xs: torch.Tensor) -> None:
    """Counts a write in place, so that a backward pass that kept the old values says so."""
    try:
        _count_writes(xs)
    except RuntimeError:
        _count_writes([x for x in xs if not x.is_inference()])      # inference tensors are never kept


_entries: dict = {}


def _call(name: str, device: int, *args) -> int:
    """The library's answer; on the device of the tensors."""
    entry = _entries.get(name)
    if entry is None:
        entry = _entries[name] = getattr(lib(), name)
    if torch.cuda.current_device() == device:
        got = entry(*args)
    else:
        with torch.cuda.device(device):
            got = entry(*args)
    if got < 0:
        raise HelioxError(lib().hx_readout_error().decode())
    return got


def _like(x: torch.Tensor, what: str, q: torch.Tensor, device: int, other: str = "q") -> None:
    if not isinstance(x, torch.Tensor) or x.get_device() != device:
        if _on_gpu(x, what) != device:
            raise ValueError(f"{what} is on {x.device}, {other} on cuda:{device}")
    if x.dtype is not q.dtype:
        raise TypeError(f"{what} is {x.dtype}, {other} is {q.dtype}")


def _attention_inputs(q, k, v, log_decay, ndim: int):
    """The tensors with contiguous last dimensions (kept by the caller until its call is queued),
    and the record's fields up to log_decay: sizes, pointers, strides."""
    device = _on_gpu(q, "q")
    _like(k, "k", q, device)
    _like(v, "v", q, device)
    kind = _type(q, "q, k and v")
    sq, sk, sv = q.shape, k.shape, v.shape
    if not len(sq) == len(sk) == len(sv) == ndim:
        want = "(batch, time, heads, d)" if ndim == 4 else "(batch, heads, d)"
        raise ValueError(f"q, k and v have to be {want}, got {tuple(sq)}, {tuple(sk)}, {tuple(sv)}")
    if not sq[:-2] == sk[:-2] == sv[:-2]:
        raise ValueError(f"q, k and v differ in batch or time: {tuple(sq)}, {tuple(sk)}, {tuple(sv)}")
    if sq[-1] != sk[-1]:
        raise ValueError(f"q has {sq[-1]} channels, k has {sk[-1]}")
    heads = log_decay.shape[0] if isinstance(log_decay, torch.Tensor) and log_decay.dim() == 1 else -1
    if log_decay is None:
        raise TypeError("log_decay has to be a tensor")
    log_decay = _array(log_decay, "log_decay", torch.float32, (heads,), device)
    rows = q, k, v = _rows(q), _rows(k), _rows(v)
    a, b, c = q.stride(), k.stride(), v.stride()
    if ndim == 4:
        fields = (kind, sq[0], sq[1], heads, sq[2], sk[2], sv[2], sq[3], sv[3], q.data_ptr(), k.data_ptr(),
                  v.data_ptr(), a[0], a[1], a[2], b[0], b[1], b[2], c[0], c[1], c[2], log_decay.data_ptr())
    else:
        fields = (kind, sq[0], 1, heads, sq[1], sk[1], sv[1], sq[2], sv[2], q.data_ptr(), k.data_ptr(),
                  v.data_ptr(), a[0], 0, a[1], b[0], 0, b[1], c[0], 0, c[1], log_decay.data_ptr())
    return device, (rows, log_decay), fields


def _lengths(lengths, batch: int, device) -> Optional[torch.Tensor]:
    return _array(lengths, "lengths", torch.int32, (batch,), device)


def linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, *,
                     scale: Optional[float] = None, initial_state: Optional[torch.Tensor] = None,
                     lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Linear attention with a decay for each head, over whole sequences:

        S_t = e^log_decay S_{t-1} + k_t v_t^T,   o_t = scale S_t^T q_t.

    q (batch, time, q_heads, dk), k (batch, time, k_heads, dk), v (batch, time, v_heads, dv),
    log_decay (heads,) fp32, at most 0; q_heads, k_heads and v_heads each divide heads, and head
    h reads head h * n // heads of them.  scale is dk ** -0.5 unless given.  initial_state is
    (batch, heads, dk, dv) fp32, zero unless given.  Sequence i ends after lengths[i] steps
    (int32; all of time unless given); its outputs beyond are zero, whatever its inputs hold.
    Returns o (batch, time, heads, dv) of q's type and the state at each sequence's end.

    An infinite or NaN input reaches what it reaches in the recurrence, and no earlier step, but as
    NaN where that may have an infinity.
    """
    device, kept, fields = _attention_inputs(q, k, v, log_decay, 4)
    _, batch, time, heads, _, _, _, dk, dv = fields[:9]
    initial_state = _array(initial_state, "initial_state", torch.float32, (batch, heads, dk, dv), device)
    _no_graph("linear_attention", "take it from linear_attention_grad", q, k, v, log_decay, initial_state)
    lengths = _lengths(lengths, batch, device)
    o = torch.empty((batch, time, heads, dv), dtype=q.dtype, device=q.device)
    end = torch.empty((batch, heads, dk, dv), dtype=torch.float32, device=q.device)
    head = (*fields, _ptr(initial_state), _ptr(lengths), _scale(scale, dk), o.data_ptr(),
            time * heads * dv, heads * dv, dv, end.data_ptr(), 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)
    _run_attention("hx_linear_attention", device, head, 0)
    return o, end


@functools.lru_cache(maxsize=1024)
def _attention_space(sizes: tuple, grad: int) -> int:
    """Bytes of workspace, by the sizes alone."""
    record = _ATTENTION.pack(*sizes, *[0] * 15, 1.0, *[0] * 20)
    need = lib().hx_linear_attention_workspace(record, grad)
    if need < 0:
        raise HelioxError(lib().hx_readout_error().decode())
    return need


def _run_attention(name: str, device: int, head: tuple, grad: int) -> None:
    need = _attention_space(head[:9], grad)
    space = torch.empty(need, dtype=torch.uint8, device=f"cuda:{device}") if need else None
    _call(name, device, _ATTENTION.pack(*head, _ptr(space), need, _stream(device)))


def linear_attention_grad(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                          do: torch.Tensor, *, scale: Optional[float] = None,
                          initial_state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                          dstate: Optional[torch.Tensor] = None):
    """Gradients of linear_attention: do is the loss's gradient by o, dstate by the end states
    (zero unless given).  Returns dq, dk, dv of the shapes and type of q, k and v (what heads
    share adds up over them; zero beyond a sequence's length) and the gradient by initial_state
    (None where that is None).  Decays are time constants of the readout: no gradient is made
    for them."""
    device, kept, fields = _attention_inputs(q, k, v, log_decay, 4)
    _, batch, time, heads, _, _, _, dk, dv = fields[:9]
    _like(do, "do", q, device)
    if do.shape != (batch, time, heads, dv):
        raise ValueError(f"do has shape {tuple(do.shape)}, expected {(batch, time, heads, dv)}")
    do = _rows(do)
    initial_state = _array(initial_state, "initial_state", torch.float32, (batch, heads, dk, dv), device)
    dstate = _array(dstate, "dstate", torch.float32, (batch, heads, dk, dv), device)
    lengths = _lengths(lengths, batch, device)
    dq, dk_, dv_ = (torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in (q, k, v))
    dinitial = None if initial_state is None else torch.empty_like(initial_state)
    head = (*fields, _ptr(initial_state), _ptr(lengths), _scale(scale, dk), 0, 0, 0, 0, 0,
            do.data_ptr(), *do.stride()[:3], _ptr(dstate), dq.data_ptr(), dk_.data_ptr(), dv_.data_ptr(),
            _ptr(dinitial), 0, 0, 0)
    _run_attention("hx_linear_attention_grad", device, head, 1)
    return dq, dk_, dv_, dinitial


def linear_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                          state: torch.Tensor, *, scale: Optional[float] = None,
                          slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One step of linear_attention for a batch of running sequences: q (batch, q_heads, dk), k,
    v alike; state (n_slots, heads, dk, dv) fp32, contiguous, is updated in place.  Row i's state
    is slot slots[i] (int32, distinct; a slot outside 0..n_slots-1 leaves the row out and its
    output zero), slot i unless given.  Returns o (batch, heads, dv)."""
    device, kept, fields = _attention_inputs(q, k, v, log_decay, 3)
    _, batch, _, heads, _, _, _, dk, dv = fields[:9]
    if _on_gpu(state, "state") != device or state.dtype is not torch.float32 or not state.is_contiguous():
        raise TypeError(f"state has to be a contiguous float32 tensor on {q.device}")
    if state.dim() != 4 or state.shape[1:] != (heads, dk, dv):
        raise ValueError(f"state has shape {tuple(state.shape)}, expected (n_slots, {heads}, {dk}, {dv})")
    _no_graph("linear_attention_step", "take it from linear_attention_grad over the steps", q, k, v, log_decay, state)
    slots = _array(slots, "slots", torch.int32, (batch,), device)
    o = torch.empty((batch, heads, dv), dtype=q.dtype, device=q.device)
    _call("hx_linear_attention_step", device, _ATTENTION.pack(
        *fields, 0, 0, _scale(scale, dk), o.data_ptr(), heads * dv, 0, dv, 0, 0, 0, 0, 0, 0, 0, 0,
        0, 0, state.data_ptr(), _ptr(slots), state.shape[0], 0, 0, _stream(device)))
    _written(state)
    return o


def _recurrence_inputs(x, gate, ndim: int):
    """The tensors with contiguous last dimensions (kept by the caller until its call is queued),
    and the record's fields up to gate_stride."""
    device = _on_gpu(x, "x")
    _like(gate, "gate", x, device, "x")
    kind = _type(x, "x and gate")
    shape = x.shape
    if len(shape) != ndim or shape[-1] < 1:
        want = "(batch, time, channels)" if ndim == 3 else "(batch, channels)"
        raise ValueError(f"x has to be {want} with at least one channel, got shape {tuple(shape)}")
    if gate.shape != shape:
        raise ValueError(f"gate has shape {tuple(gate.shape)}, x {tuple(shape)}")
    rows = x, gate = _rows(x), _rows(gate)
    a, b = x.stride(), gate.stride()
    if ndim == 3:
        fields = (kind, shape[0], shape[1], shape[2], x.data_ptr(), gate.data_ptr(), a[0], a[1], b[0], b[1])
    else:
        fields = (kind, shape[0], 1, shape[1], x.data_ptr(), gate.data_ptr(), a[0], 0, b[0], 0)
    return device, rows, fields


@functools.lru_cache(maxsize=1024)
def _recurrence_space(sizes: tuple, grad: int) -> int:
    need = lib().hx_gated_recurrence_workspace(_RECURRENCE.pack(*sizes, *[0] * 25), grad)
    if need < 0:
        raise HelioxError(lib().hx_readout_error().decode())
    return need


def gated_recurrence(x: torch.Tensor, gate: torch.Tensor, *, initial_state: Optional[torch.Tensor] = None,
                     lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """A state for each channel that moves to its input as far as its gate lets it, over whole
    sequences: with a = sigmoid(gate),

        h_t = a_t h_{t-1} + (1 - a_t) x_t,   o_t = h_t,

    a membrane's exponential step towards x.  x and gate (batch, time, channels) are of one type;
    initial_state (batch, channels) fp32 is zero unless given.  Sequence i ends after lengths[i]
    steps (int32; all of time unless given); its outputs beyond are zero, whatever its inputs hold.
    Returns o of x's shape and type and the state (batch, channels) fp32 at each sequence's end.

    An infinite or NaN input reaches what it reaches in the recurrence, and no earlier step, but as
    NaN where that may have an infinity."""
    device, kept, fields = _recurrence_inputs(x, gate, 3)
    _, batch, time, channels = sizes = fields[:4]
    initial_state = _array(initial_state, "initial_state", torch.float32, (batch, channels), device)
    _no_graph("gated_recurrence", "take it from gated_recurrence_grad", x, gate, initial_state)
    lengths = _lengths(lengths, batch, device)
    o = _empty(x)
    end = torch.empty((batch, channels), dtype=torch.float32, device=x.device)
    need = _recurrence_space(sizes, 0)
    space = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
    _call("hx_gated_recurrence", device, _RECURRENCE.pack(
        *fields, _ptr(initial_state), _ptr(lengths), o.data_ptr(), time * channels, channels, end.data_ptr(),
        0, 0, 0, 0, 0, 0, 0, 0, 0, 0, _ptr(space), need, _stream(device)))
    return o, end


def gated_recurrence_grad(x: torch.Tensor, gate: torch.Tensor, do: torch.Tensor, *,
                          initial_state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                          dstate: Optional[torch.Tensor] = None):
    """Gradients of gated_recurrence: do is the loss's gradient by o, dstate by the end states (zero
    unless given).  Returns dx and dgate of x's shape and type (zero beyond a sequence's length)
    and the gradient by initial_state (None where that is None)."""
    device, kept, fields = _recurrence_inputs(x, gate, 3)
    _, batch, _, channels = sizes = fields[:4]
    _like(do, "do", x, device, "x")
    if do.shape != x.shape:
        raise ValueError(f"do has shape {tuple(do.shape)}, x {tuple(x.shape)}")
    do = _rows(do)
    initial_state = _array(initial_state, "initial_state", torch.float32, (batch, channels), device)
    dstate = _array(dstate, "dstate", torch.float32, (batch, channels), device)
    lengths = _lengths(lengths, batch, device)
    dx, dgate = _empty(x), _empty(x)
    dinitial = None if initial_state is None else torch.empty_like(initial_state)
    need = _recurrence_space(sizes, 1)
    space = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
    _call("hx_gated_recurrence_grad", device, _RECURRENCE.pack(
        *fields, _ptr(initial_state), _ptr(lengths), 0, 0, 0, 0, do.data_ptr(), *do.stride()[:2], _ptr(dstate),
        dx.data_ptr(), dgate.data_ptr(), _ptr(dinitial), 0, 0, 0, _ptr(space), need, _stream(device)))
    return dx, dgate, dinitial


def gated_recurrence_step(x: torch.Tensor, gate: torch.Tensor, state: torch.Tensor, *,
                          slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One step of gated_recurrence for a batch of running sequences: x and gate (batch, channels);
    state (n_slots, channels) fp32, contiguous, is updated in place.  Row i's state is slot slots[i]
    (int32, distinct; a slot outside 0..n_slots-1 leaves the row out and its output zero), slot i
    unless given.  Returns o (batch, channels)."""
    device, kept, fields = _recurrence_inputs(x, gate, 2)
    batch, channels = x.shape
    if _on_gpu(state, "state") != device or state.dtype is not torch.float32 or not state.is_contiguous():
        raise TypeError(f"state has to be a contiguous float32 tensor on {x.device}")
    if state.dim() != 2 or state.shape[1] != channels:
        raise ValueError(f"state has shape {tuple(state.shape)}, expected (n_slots, {channels})")
    _no_graph("gated_recurrence_step", "take it from gated_recurrence_grad over the steps", x, gate, state)
    slots = _array(slots, "slots", torch.int32, (batch,), device)
    o = _empty(x)
    _call("hx_gated_recurrence_step", device, _RECURRENCE.pack(
        *fields, 0, 0, o.data_ptr(), channels, 0, 0, 0, 0, 0, 0, 0, 0, 0, state.data_ptr(), _ptr(slots), state.shape[0],
        0, 0, _stream(device)))
    _written(state)
    return o


def _flat_rows(x: torch.Tensor) -> torch.Tensor:
    """x as (rows, its last dimension), the last contiguous (a copy only where no view is one)."""
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1]) if x.numel() else x.new_empty(0, x.shape[-1])
    return _rows(x)


def _norm_inputs(x, weight, bias):
    device = _on_gpu(x, "x")
    kind = _type(x, "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x has to be (..., width) with at least one value a row, got shape {tuple(x.shape)}")
    size, weight_kind = x.shape[-1:], 0
    if weight is not None:
        weight = _array(weight, "weight", getattr(weight, "dtype", None), size, device)
        weight_kind = _type(weight, "weight")
    if bias is not None:
        bias = _array(bias, "bias", getattr(bias, "dtype", None), size, device)
        if weight is not None and bias.dtype is not weight.dtype:
            raise TypeError(f"weight is {weight.dtype}, bias is {bias.dtype}")
        weight_kind = _type(bias, "bias")
    return device, kind, weight_kind, _flat_rows(x), weight, bias


@functools.lru_cache(maxsize=1024)
def _norm_space(kind: int, rows: int, width: int) -> int:
    need = lib().hx_layer_norm_workspace(_NORM.pack(kind, 0, rows, width, *[0] * 4, 0.0, *[0] * 8, 1, 1, 0, 0, 0))
    if need < 0:
        raise HelioxError(lib().hx_readout_error().decode())
    return need


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
               eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(x - mean) / sqrt(variance + eps) * weight + bias over the last dimension of x (..., width);
    weight and bias (width,) are of one type, fp32, fp16 or bf16, whatever x's is (1 and 0 unless
    given); eps is 0 or at least 2^-126.  Returns y of x's shape and type, and each row's mean and 1 / sqrt(variance + eps)
    (fp32, x's shape without the last), which layer_norm_grad takes."""
    device, kind, weight_kind, rows, weight, bias = _norm_inputs(x, weight, bias)
    _no_graph("layer_norm", "take it from layer_norm_grad", x, weight, bias)
    y = _empty(x)
    mean, rstd = torch.empty((2, *x.shape[:-1]), dtype=torch.float32, device=x.device).unbind(0)
    n, width = rows.shape
    _call("hx_layer_norm", device, _NORM.pack(
        kind, weight_kind, n, width, rows.data_ptr(), rows.stride(0), _ptr(weight), _ptr(bias), _real(eps, "eps"),
        y.data_ptr(), width, mean.data_ptr(), rstd.data_ptr(), 0, 0, 0, 0, 0, 0, 0, 0, _stream(device)))
    return y, mean, rstd


def layer_norm_grad(x: torch.Tensor, weight: Optional[torch.Tensor], mean: torch.Tensor, rstd: torch.Tensor,
                    dy: torch.Tensor, *, parameters: bool = True):
    """Gradients of layer_norm from its mean and rstd: dy is the loss's gradient by y.  Returns dx of
    x's shape and type, and the gradients by weight and by bias (width,) fp32, summed over the rows
    in an order of the sizes alone (None, None with parameters=False)."""
    device, kind, weight_kind, rows, weight, _ = _norm_inputs(x, weight, None)
    _like(dy, "dy", x, device, "x")
    if dy.shape != x.shape:
        raise ValueError(f"dy has shape {tuple(dy.shape)}, x {tuple(x.shape)}")
    if mean is None or rstd is None:
        raise TypeError("mean and rstd have to be tensors")
    mean = _array(mean, "mean", torch.float32, x.shape[:-1], device)
    rstd = _array(rstd, "rstd", torch.float32, x.shape[:-1], device)
    dy = _flat_rows(dy)
    n, width = rows.shape
    dx = _empty(x)
    dweight = dbias = space = None
    need = 0
    if parameters:
        dweight, dbias = torch.empty((2, width), dtype=torch.float32, device=x.device).unbind(0)
        need = _norm_space(kind, n, width)
        space = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
    _call("hx_layer_norm_grad", device, _NORM.pack(
        kind, weight_kind, n, width, rows.data_ptr(), rows.stride(0), _ptr(weight), 0, 0.0, 0, 0, mean.data_ptr(),
        rstd.data_ptr(), dy.data_ptr(), dy.stride(0), dx.data_ptr(), width, _ptr(dweight), _ptr(dbias), _ptr(space), need,
        _stream(device)))
    return dx, dweight, dbias


def _logits(logits: torch.Tensor):
    device = _on_gpu(logits, "logits")
    if logits.dim() != 2:
        raise ValueError(f"logits have to be (rows, vocab), got shape {tuple(logits.shape)}")
    return device, _type(logits, "logits"), _rows(logits)


def _distill(logits, teacher_index, teacher_logits, temperature, teacher_lse, weight, grad) -> torch.Tensor:
    device, kind, logits = _logits(logits)
    rows, vocab = logits.shape
    for x, name in ((teacher_index, "teacher_index"), (teacher_logits, "teacher_logits")):
        if _on_gpu(x, name) != device:
            raise ValueError(f"{name} is on {x.device}, logits on {logits.device}")
        if x.dim() != 2 or x.shape[0] != rows:
            raise ValueError(f"{name} has to be ({rows}, top), got shape {tuple(x.shape)}")
    if teacher_index.shape != teacher_logits.shape:
        raise ValueError(f"teacher_index has shape {tuple(teacher_index.shape)}, "
                         f"teacher_logits {tuple(teacher_logits.shape)}")
    if teacher_index.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"teacher_index is {teacher_index.dtype}, expected int32 or int64")
    teacher_kind = _type(teacher_logits, "teacher_logits")
    teacher_index, teacher_logits = _rows(teacher_index), _rows(teacher_logits)
    teacher_lse = _array(teacher_lse, "teacher_lse", torch.float32, (rows,), device)
    weight = _array(weight, "weight", torch.float32, (rows,), device)
    loss = torch.empty(rows, dtype=torch.float32, device=logits.device)
    _call("hx_distill_loss", device, _DISTILL.pack(
        kind, teacher_kind, 32 if teacher_index.dtype == torch.int32 else 64, rows, vocab, teacher_index.shape[1],
        _ptr(logits), logits.stride(0), _ptr(teacher_index), teacher_index.stride(0), _ptr(teacher_logits),
        teacher_logits.stride(0), _ptr(teacher_lse), _ptr(weight), _real(temperature, "temperature"), _ptr(loss),
        _ptr(grad), 0 if grad is None else grad.stride(0), _stream(device)))
    return loss


def distill_loss(logits: torch.Tensor, teacher_index: torch.Tensor, teacher_logits: torch.Tensor, *,
                 temperature: float = 1.0, teacher_lse: Optional[torch.Tensor] = None) -> torch.Tensor:
    """temperature^2 KL(teacher | student) of each row, (rows,) fp32, from the teacher's top
    logits alone: teacher_logits (rows, top) stand at the vocabulary places teacher_index (int32
    or int64; a place outside the vocabulary is an absent entry).  Without teacher_lse the
    teacher is the softmax over its entries.  With teacher_lse (rows,) fp32, the logarithm of
    sum exp(logit / temperature) over the teacher's whole vocabulary, its mass on all other
    places is one more class, but where the student's mask leaves none of them (their mass is
    under 2^-1074).  A row without entries has loss 0."""
    for x, name in ((logits, "logits"), (teacher_logits, "teacher_logits")):
        _on_gpu(x, name)
    _no_graph("distill_loss", "take it from distill_loss_grad", logits, teacher_logits, teacher_lse)
    return _distill(logits, teacher_index, teacher_logits, temperature, teacher_lse, None, None)


def distill_loss_grad(logits: torch.Tensor, teacher_index: torch.Tensor, teacher_logits: torch.Tensor, *,
                      temperature: float = 1.0, teacher_lse: Optional[torch.Tensor] = None,
                      weight: Optional[torch.Tensor] = None,
                      out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """distill_loss and, in the same pass, the gradient of sum_i weight_i loss_i by the logits
    (weight (rows,) fp32, 1 unless given), of the logits' type.  The gradient goes to ``out``
    where that is given; it may be the logits themselves, but not overlap them otherwise."""
    if out is None:
        _on_gpu(logits, "logits")
        out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    elif (_on_gpu(out, "out") != _on_gpu(logits, "logits") or out.dtype != logits.dtype or out.shape != logits.shape
          or (out.shape[-1] > 1 and out.stride(-1) != 1)):
        raise ValueError("out has to be like the logits, its last dimension contiguous")
    loss = _distill(logits, teacher_index, teacher_logits, temperature, teacher_lse, weight, out)
    _written(out)
    return loss, out


class TokenLogprobs(NamedTuple):
    """What token_logprobs returns of each row."""

    logprob: torch.Tensor                 # (rows,) fp32
    entropy: torch.Tensor                 # (rows,) fp32
    top_logprob: torch.Tensor             # (rows, top) fp32, the largest first
    top_index: torch.Tensor               # (rows, top) int64
    stats: torch.Tensor                   # (rows, 2) fp32: the largest logit, and log of the sum beside it


def _tokens(tokens, rows: int, device: int) -> torch.Tensor:
    if not isinstance(tokens, torch.Tensor):
        raise TypeError(f"tokens has to be a tensor, got {type(tokens).__name__}")
    if tokens.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"tokens is {tokens.dtype}, expected int32 or int64")
    return _array(tokens, "tokens", tokens.dtype, (rows,), device)


@functools.lru_cache(maxsize=1024)
def _logprob_space(kind: int, rows: int, vocab: int, top: int) -> int:
    need = lib().hx_token_logprobs_workspace(_LOGPROB.pack(kind, 64, rows, vocab, top, 0, 0, 0, 1.0, *[0] * 12))
    if need < 0:
        raise HelioxError(lib().hx_readout_error().decode())
    return need


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, temperature: float = 1.0,
                   top: int = 0) -> TokenLogprobs:
    """Of each row of logits (rows, vocab), with q = softmax(logits / temperature): log q of the row's
    token (tokens (rows,) int32 or int64; 0 for a token outside the vocabulary, as of padding), the
    entropy of q, and the ``top`` most likely places (at most 256; ties: the lowest index first) with
    their log q.  NaN ranks as -inf, and a row with a NaN or +inf has NaN for all of its numbers (but 0 for
    a token outside the vocabulary); a row of nothing but -inf has log q -inf and entropy 0.

    stats holds the largest logit m and log sum exp((logits - m) / temperature), which
    token_logprobs_grad takes; m / temperature plus the latter is the logsumexp."""
    device, kind, logits = _logits(logits)
    _no_graph("token_logprobs", "take it from token_logprobs_grad", logits)
    rows, vocab = logits.shape
    tokens = _tokens(tokens, rows, device)
    top, temperature = _whole(top, "top"), _real(temperature, "temperature")
    need = _logprob_space(kind, rows, vocab, top)
    f32 = {"dtype": torch.float32, "device": logits.device}
    got = TokenLogprobs(torch.empty(rows, **f32), torch.empty(rows, **f32), torch.empty((rows, top), **f32),
                        torch.empty((rows, top), dtype=torch.int64, device=logits.device), torch.empty((rows, 2), **f32))
    space = torch.empty(need, dtype=torch.uint8, device=logits.device) if need else None
    _call("hx_token_logprobs", device, _LOGPROB.pack(
        kind, 32 if tokens.dtype is torch.int32 else 64, rows, vocab, top, logits.data_ptr(), logits.stride(0),
        tokens.data_ptr(), temperature, got.logprob.data_ptr(), got.entropy.data_ptr(), got.stats.data_ptr(),
        got.top_logprob.data_ptr(), got.top_index.data_ptr(), 0, 0, 0, 0, _ptr(space), need, _stream(device)))
    return got


def token_logprobs_grad(logits: torch.Tensor, tokens: torch.Tensor, scored: TokenLogprobs,
                        dlogprob: Optional[torch.Tensor], dentropy: Optional[torch.Tensor] = None, *,
                        temperature: float = 1.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The gradient by the logits, of their type, from what token_logprobs gave for them (``scored``, its
    entropy and stats) and the loss's gradients by logprob and by entropy ((rows,) fp32, 0 where None).
    It goes to ``out`` where that is given; it may be the logits themselves, but not overlap them
    otherwise.  None is made for the top alternatives."""
    device, kind, logits = _logits(logits)
    rows, vocab = logits.shape
    tokens = _tokens(tokens, rows, device)
    if not isinstance(scored, TokenLogprobs):
        raise TypeError(f"scored has to be what token_logprobs returned, got {type(scored).__name__}")
    entropy = _array(scored.entropy, "entropy", torch.float32, (rows,), device)
    stats = _array(scored.stats, "stats", torch.float32, (rows, 2), device)
    dlogprob = _array(dlogprob, "dlogprob", torch.float32, (rows,), device)
    dentropy = _array(dentropy, "dentropy", torch.float32, (rows,), device)
    if out is None:
        out = _empty(logits)
    elif (_on_gpu(out, "out") != device or out.dtype != logits.dtype or out.shape != logits.shape
          or (out.shape[-1] > 1 and out.stride(-1) != 1)):
        raise ValueError("out has to be like the logits, its last dimension contiguous")
    _call("hx_token_logprobs_grad", device, _LOGPROB.pack(
        kind, 32 if tokens.dtype is torch.int32 else 64, rows, vocab, 0, logits.data_ptr(), logits.stride(0),
        tokens.data_ptr(), _real(temperature, "temperature"), 0, entropy.data_ptr(), stats.data_ptr(), 0, 0,
        _ptr(dlogprob), _ptr(dentropy), out.data_ptr(), out.stride(0), 0, 0, _stream(device)))
    _written(out)
    return out


Setting = Union[float, torch.Tensor]


def sample(logits: torch.Tensor, u: torch.Tensor, *, temperature: Setting = 1.0,
           top_k: Union[int, torch.Tensor] = 0, top_p: Setting = 1.0,
           min_p: Setting = 0.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """One token for each row of logits (rows, vocab), from the random numbers u (rows,) fp32 in
    [0, 1): of the places ranked by logit (ties: the lowest index first) the first top_k stay (0:
    all), of those the fewest that hold top_p of their mass, of those the ones with at least
    min_p of the largest probability; the token is the first in index order whose running sum
    passes u of what stays.  temperature 0 takes the largest logit.  Each setting is a number or
    a tensor (rows,), fp32 (top_k: int32).  Returns tokens (int64) and the logarithms of their
    shares of what stays (fp32).

    Masses are whole numbers (2^-40 of the largest), so that an answer does not depend on the
    order of a sum: what is less than 2^-40 times as probable as the largest is never drawn.
    NaN counts as -inf; a row without a finite logit gives token -1.  Neither result carries a
    gradient."""
    device, kind, logits = _logits(logits)
    rows, vocab = logits.shape
    u = _array(u, "u", torch.float32, (rows,), device)
    if u is None:
        raise TypeError("u has to be a tensor")
    pointers, values = [], []
    for x, name, dtype in ((temperature, "temperature", torch.float32), (top_k, "top_k", torch.int32),
                           (top_p, "top_p", torch.float32), (min_p, "min_p", torch.float32)):
        if isinstance(x, torch.Tensor):
            x = _array(x, name, dtype, (rows,), device)
            pointers.append(x)
            values.append(0)
        else:
            pointers.append(None)
            values.append(_whole(x, name) if dtype is torch.int32 else _real(x, name))
    token = torch.empty(rows, dtype=torch.int64, device=logits.device)
    logprob = torch.empty(rows, dtype=torch.float32, device=logits.device)
    _call("hx_sample", device, _SAMPLE.pack(
        kind, rows, vocab, _ptr(logits), logits.stride(0), _ptr(u), *map(_ptr, pointers), values[0], values[2],
        values[3], values[1], _ptr(token), _ptr(logprob), _stream(device)))
    return token, logprob


def _held(name: str, doc: str) -> property:
    """A tensor of a state: what is assigned is copied into it, for its address is what a step, and a captured
    one, writes to."""
    def get(state):
        return getattr(state, name)

    def put(state, x):
        here = getattr(state, name)
        if here is None and x is None:
            return
        if not isinstance(x, torch.Tensor) or here is None:
            raise TypeError(f"{name[1:]} of a state in {state.bits} bits is "
                            f"{'None' if here is None else 'a tensor'}, got {type(x).__name__}")
        if x.dtype is not here.dtype:
            raise TypeError(f"{name[1:]} is {here.dtype}, got {x.dtype}")
        if x.shape != here.shape:
            raise ValueError(f"{name[1:]} has shape {tuple(here.shape)}, got {tuple(x.shape)}")
        here.copy_(x)

    return property(get, put, doc=doc)


class AdamWState:
    """What adamw_step keeps for a list of parameters, made by adamw_state.  Tensor i's moments are
    elements starts[i] to starts[i] + sizes[i] of m and v; starts are multiples of 256.

    bits 32: m and v are fp32.  bits 8: m and the root of v are float8_e4m3fn, each 256 elements
    relative to m_scale and v_scale (fp32, one for each 256).  step, int64 on the GPU, counts the
    steps taken.  All of them may be saved, and copied into another state of the same parameters;
    a tensor that is assigned to one of them, from whichever device, is copied (step: a whole number too)."""

    m = _held("_m", "first moments")
    v = _held("_v", "second moments; with 8 bits their roots")
    m_scale = _held("_m_scale", "what codes of m are relative to; None with 32 bits")
    v_scale = _held("_v_scale", "the same of v")

    def __init__(self, sizes: Sequence[int], bits: int, device: int):
        self.bits, self.device = bits, device
        self.sizes, self.starts = array("q", sizes), array("q")
        whole = 0
        for n in self.sizes:
            self.starts.append(whole)
            whole += -(-n // 256) * 256
        on = {"device": f"cuda:{device}"}
        kind, held = (torch.float32, torch.float32) if bits == 32 else (torch.float8_e4m3fn, torch.uint8)
        self._m, self._v = (torch.zeros(whole, dtype=held, **on).view(kind) for _ in range(2))
        self._m_scale, self._v_scale = (torch.zeros(whole // 256, **on) if bits == 8 else None for _ in range(2))
        # the count, and room that the library uses
        self._count = torch.zeros(2, dtype=torch.int64, **on)
        self._held = [x for x in (self._m, self._v, self._m_scale, self._v_scale, self._count) if x is not None]
        self._elements = [x.numel() for x in self._held]

    @property
    def step(self) -> torch.Tensor:
        """Steps taken, (1,) int64."""
        return self._count[:1]

    @step.setter
    def step(self, x) -> None:
        if not isinstance(x, torch.Tensor):
            x = _whole(x, "step")
            if x < 0:
                raise ValueError(f"step has to be at least 0, got {x}")
            self._count[0] = x
        elif x.dtype is not torch.int64 or x.numel() != 1:
            raise TypeError(f"step has to be one int64, got {tuple(x.shape)} of {x.dtype}")
        else:
            self._count[:1].copy_(x.reshape(1))

    def _check(self) -> None:
        """Its tensors are of the sizes and on the device that they were made with."""
        held = self._held
        if (list(map(_size_of, held)) != self._elements or set(map(_device_of, held)) != {self.device}
                or not all(map(_whole_of, held))):
            raise ValueError(f"the state's tensors were changed: {[tuple(x.shape) for x in held]} on {[str(x.device) for x in held]} "
                             f"where {self._elements} contiguous elements on cuda:{self.device} belong")


# What is asked of hundreds of tensors in a step is asked by map, a tenth of a loop's time each.
_device_of, _address_of, _whole_of = torch.Tensor.get_device, torch.Tensor.data_ptr, torch.Tensor.is_contiguous
_shape_of, _dtype_of, _size_of = operator.attrgetter("shape"), operator.attrgetter("dtype"), torch.Tensor.numel


def _tensors(xs: list, what: str, device: Optional[int]) -> array:
    """The types of tensors that are all on one GPU (`device`, or the first one's)."""
    try:
        places = set(map(_device_of, xs))
        kinds = list(map(_TYPES.get, map(_dtype_of, xs)))
    except (TypeError, AttributeError):
        places, kinds = (), (None,)
    if len(places) != 1 or min(places) < 0 or None in kinds or (device is not None and device not in places):
        for i, x in enumerate(xs):
            here = _on_gpu(x, f"{what}[{i}]")
            _type(x, f"{what}[{i}]")
            device = here if device is None else device
            if here != device:
                raise ValueError(f"{what}[{i}] is on cuda:{here}, others on cuda:{device}")
    return array("q", kinds)


def _parameters(params: list) -> Tuple[int, array]:
    if not params:
        raise ValueError("params has no tensors")
    kinds = _tensors(params, "params", None)
    if not all(map(_whole_of, params)):
        raise ValueError("params have to be contiguous")
    return params[0].get_device(), kinds


def adamw_state(params: Sequence[torch.Tensor], *, bits: int = 32) -> AdamWState:
    """A state of zeros for these parameters (contiguous tensors on one GPU, fp32, fp16 or bf16): 8
    bytes of moments for each of their elements with bits=32, 2 and a 32nd with bits=8."""
    params = list(params)
    device, _ = _parameters(params)
    bits = _whole(bits, "bits")
    if bits not in (8, 32):
        raise ValueError(f"bits has to be 8 or 32, got {bits}")
    return AdamWState(list(map(_size_of, params)), bits, device)


def _one_number(x, what: str, device: int):
    """(a tensor's address or 0, a number): a setting that is either."""
    if isinstance(x, torch.Tensor):
        if x.numel() != 1:
            raise ValueError(f"{what} has to be one number, got shape {tuple(x.shape)}")
        return _array(x, what, torch.float32, x.shape, device).data_ptr(), 0.0
    return 0, _real(x, what)


def _decays(weight_decay, count: int) -> array:
    if isinstance(weight_decay, (list, tuple)):
        if len(weight_decay) != count:
            raise ValueError(f"{len(weight_decay)} weight_decay for {count} params")
        try:
            return array("d", weight_decay)
        except (TypeError, ValueError, OverflowError):
            return array("d", [_real(w, "weight_decay") for w in weight_decay])
    return array("d", [_real(weight_decay, "weight_decay")]) * count


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[Optional[torch.Tensor]], state: AdamWState, *,
               lr: Setting, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
               weight_decay: Union[float, Sequence[float]] = 0.01, grad_scale: Setting = 1.0) -> None:
    """One AdamW step, in place: with t the state's step after it and g = grad_scale grad,

        m = beta1 m + (1 - beta1) g,   v = beta2 v + (1 - beta2) g^2,
        p = p (1 - lr weight_decay) - lr (m / (1 - beta1^t)) / (sqrt(v / (1 - beta2^t)) + eps),

    in fp32, p rounded once to its type.  grads are of the parameters' shapes and of fp32, fp16 or bf16,
    whatever their parameter is; a parameter whose gradient is None stays as it is, with its
    moments.  weight_decay is one number or one for each parameter.  lr and grad_scale (as of a clipped
    norm) are numbers, or fp32 tensors of one on the GPU, which a captured step reads anew at every
    replay, as it does the state's step.

    With 8 bits the moments are rounded after the step has used them: to nearest while t is at most
    1 / (1 - max(betas)), later up or down by a hash of t and the element, so that they follow changes
    smaller than their codes' steps (the same calls give the same state).  An infinite gradient makes
    the moments of the 256 elements that share its scale NaN, a NaN only its own.  Parameters in 16
    bits lose updates under half a step of their own: keep them in fp32 where that matters.
    Parameters that overlap each other or a gradient are refused."""
    if not isinstance(state, AdamWState):
        raise TypeError(f"state has to be what adamw_state returned, got {type(state).__name__}")
    params, grads = list(params), list(grads)
    device, kinds = _parameters(params)
    if device != state.device:
        raise ValueError(f"params are on cuda:{device}, the state on cuda:{state.device}")
    sizes, starts = state.sizes, state.starts
    if len(grads) != len(params) or array("q", map(_size_of, params)) != sizes:
        raise ValueError(f"{len(params)} params and {len(grads)} grads do not fit a state of sizes {list(sizes)}")
    decays = _decays(weight_decay, len(params))
    if not isinstance(betas, (list, tuple)) or len(betas) != 2:
        raise TypeError("betas has to be two numbers")
    beta1, beta2 = (_real(b, "betas") for b in betas)
    lr_ptr, lr = _one_number(lr, "lr", device)
    scale_ptr, scale = _one_number(grad_scale, "grad_scale", device)
    if any(g is None for g in grads):
        there = [i for i, g in enumerate(grads) if g is not None]
        params, grads = [params[i] for i in there], [grads[i] for i in there]
        kinds, sizes, starts = (array("q", [a[i] for i in there]) for a in (kinds, sizes, starts))
        decays = array("d", [decays[i] for i in there])
    grad_kinds = _tensors(grads, "grads", device)
    if list(map(_shape_of, grads)) != list(map(_shape_of, params)):
        raise ValueError("grads have to be of their parameters' shapes, got "
                         + ", ".join(f"{tuple(g.shape)} for {tuple(p.shape)}" for p, g in zip(params, grads) if p.shape != g.shape))
    if not all(map(_whole_of, grads)):
        grads = [g.contiguous() for g in grads]
    state._check()
    lists = kinds, grad_kinds, array("Q", map(_address_of, params)), array("Q", map(_address_of, grads)), sizes, starts, decays
    _call("hx_adamw_step", device, _ADAMW.pack(
        state.bits, len(params), *[a.buffer_info()[0] for a in lists], state._m.data_ptr(), state._v.data_ptr(),
        _ptr(state._m_scale), _ptr(state._v_scale), state._elements[0], lr, beta1, beta2, _real(eps, "eps"), scale, scale_ptr,
        lr_ptr, state._count.data_ptr(), _stream(device)))
    _written(*params)
