"""Readout operators over a network's captured outputs, on the GPU.

``learn.capture_signals_cached`` brings out the course of a network's output voltages, and
``learn.replay_grads_from_cached_signals`` takes the loss's gradient by them.  The operators
here stand between the two: what turns that course into answers, the loss that teaches it from
a trained network, and the gradients of both.

  linear_attention, linear_attention_grad   a temporal readout over whole recordings: linear
                                            attention whose state decays as a synapse's does
  linear_attention_step                     the same for one tick of a running network
  distill_loss, distill_loss_grad           the loss against a teacher's top logits
  sample                                    an answer drawn from logits

They take and return torch tensors on one GPU (fp32, fp16 or bf16), work on torch's current
stream, wait for nothing, and may be captured into a graph.  Sums, softmax statistics and
states are fp32 or wider whatever the inputs are.  Arguments that do not fit raise ValueError
or TypeError; sizes, values and overlaps that the library refuses, and launches that fail, raise
HelioxError.  Results carry no graph for autograd: gradients are calls of their own, and the calls
that have one refuse inputs that require a gradient while torch records.
"""
from __future__ import annotations

import functools
import operator
import struct
from typing import Optional, Tuple, Union

import torch

from .sim import HelioxError, lib

# The records of include/heliox.h, field by field (8 bytes each).
_ATTENTION = struct.Struct("=9q 3Q 9q 3Q d Q 3q Q Q 3q Q 3Q Q Q Q q Q q Q")
_DISTILL = struct.Struct("=6q Q q Q q Q q 2Q d Q Q q Q")
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


def _like(x: torch.Tensor, what: str, q: torch.Tensor, device: int) -> None:
    if not isinstance(x, torch.Tensor) or x.get_device() != device:
        if _on_gpu(x, what) != device:
            raise ValueError(f"{what} is on {x.device}, q on cuda:{device}")
    if x.dtype is not q.dtype:
        raise TypeError(f"{what} is {x.dtype}, q is {q.dtype}")


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
    return o


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
    return _distill(logits, teacher_index, teacher_logits, temperature, teacher_lse, weight, out), out


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
