"""Gated linear recurrence on the GPU: the layer of a prediction network or an encoder whose
outputs the losses of this package take, over whole sequences with its gradients and, for
decoding, one token at a time.  No counterpart in the reference, which leaves both networks
to the caller.  The arithmetic runs in libfrnnt_sm100.so (csrc/recurrence.cu)."""
from typing import Optional, Tuple

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import _c_int, _c_longlong

_CODES = {torch.float32: _lib.F32, torch.float64: _lib.F64, torch.float16: _lib.F16,
          torch.bfloat16: _lib.BF16}


def _code(dtype) -> int:
    if dtype not in _CODES:
        raise TypeError(f"only float32, float64, float16 and bfloat16 are supported, got {dtype}")
    return _CODES[dtype]


def _state_type(dtype):
    """States are 32 bits wide (64 for float64), whatever the inputs' type."""
    return torch.float64 if dtype == torch.float64 else torch.float32


def _rows(t: Tensor) -> Tensor:
    """`t`, or a copy where its channels do not lie side by side."""
    return t if t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def _strided(t: Optional[Tensor]):
    """(pointer, batch stride, step stride) of a [B][T][D] tensor whose channels lie side by side"""
    if t is None:
        return None, _c_longlong(0), _c_longlong(0)
    return _lib._c_vp(t.data_ptr()), _c_longlong(t.stride(0)), _c_longlong(t.stride(1))


def _forward(x, gate, initial, lengths, keep_states):
    B, T, D = x.shape
    dev, code = x.device, _code(x.dtype)
    state = _state_type(x.dtype)
    saved = None
    with _lib.on_device(dev):
        h = torch.empty(B, T, D, dtype=x.dtype, device=dev)
        last = torch.empty(B, D, dtype=state, device=dev)
        if keep_states:
            saved = torch.empty(max(_lib.size_of("frnnt_recurrence_saved_bytes", code, B, T, D), 1),
                                dtype=torch.uint8, device=dev)
        _lib.call("frnnt_recurrence_forward", _c_int(code), *_strided(x), *_strided(gate),
                  _lib.ptr(initial), _lib.ptr(lengths), _lib.ptr(h), _lib.ptr(last),
                  _lib.ptr(saved), B, T, D, _lib.stream_ptr(dev))
    return h, last, saved


class _GatedRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, initial, lengths):
        x, gate = _rows(x), _rows(gate)
        h, last, saved = _forward(x, gate, initial, lengths, True)
        ctx.save_for_backward(x, gate, lengths, saved)
        ctx.set_materialize_grads(False)
        return h, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dh, dlast):
        x, gate, lengths, saved = ctx.saved_tensors
        B, T, D = x.shape
        dev, code = x.device, _code(x.dtype)
        dh = None if dh is None else _rows(dh)
        dlast = None if dlast is None else dlast.contiguous()
        with _lib.on_device(dev):
            dx = torch.empty(B, T, D, dtype=x.dtype, device=dev)
            dgate = torch.empty(B, T, D, dtype=x.dtype, device=dev)
            dinitial = (torch.empty(B, D, dtype=_state_type(x.dtype), device=dev)
                        if ctx.needs_input_grad[2] else None)
            _lib.call("frnnt_recurrence_backward", _c_int(code), *_strided(x), *_strided(gate),
                      _lib.ptr(lengths), _lib.ptr(saved), *_strided(dh), _lib.ptr(dlast),
                      _lib.ptr(dx), _lib.ptr(dgate), _lib.ptr(dinitial), B, T, D,
                      _lib.stream_ptr(dev))
        return dx, dgate, dinitial, None


def gated_recurrence(x: Tensor, gate: Tensor, initial: Optional[Tensor] = None,
                     lengths: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """(h, last) of the recurrence, for every channel on its own::

        f = sigmoid(gate)
        h[:, t] = f[:, t] * h[:, t - 1] + (1 - f[:, t]) * x[:, t]       # h[:, -1] = initial, or 0

    x and gate are [B][T][D] CUDA tensors of one type (float32, float64, float16 or bfloat16),
    with any strides between batches and steps, so that both may be halves of one projection;
    initial is [B][D] and lengths int64 [B].  h [B][T][D] has the type of x; last [B][D], the
    state after the last step, is float32 (float64 for float64 inputs), as is all arithmetic.

    Steps t >= lengths[b] of a padded batch are not read and leave the state alone: h is zero
    there and so are the gradients of x and gate; last[b] is the state after lengths[b] steps,
    which is initial[b] for an empty sequence.  Lengths below 0 or above T count as 0 and T.
    A gate of -inf drops the state (h[:, t] = x[:, t]) and one of +inf keeps it.

    Differentiable once with respect to x, gate and initial.  No counterpart in the reference."""
    assert x.ndim == 3, x.ndim
    assert gate.shape == x.shape, (gate.shape, x.shape)
    assert gate.dtype == x.dtype, (gate.dtype, x.dtype)
    _code(x.dtype)
    (B, T, D) = x.shape
    state = _state_type(x.dtype)
    assert x.is_cuda and gate.device == x.device, (x.device, gate.device)
    if initial is not None:
        assert initial.shape == (B, D), (initial.shape, (B, D))
        assert initial.device == x.device, (initial.device, x.device)
        assert initial.dtype in (state, x.dtype), initial.dtype
        initial = initial.to(state).contiguous()
    if lengths is not None:
        assert lengths.shape == (B,) and lengths.dtype == torch.int64, (lengths.shape, lengths.dtype)
        assert lengths.device == x.device, (lengths.device, x.device)
        lengths = lengths.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad or
                                    (initial is not None and initial.requires_grad)):
        return _GatedRecurrence.apply(x, gate, initial, lengths)
    return _forward(_rows(x), _rows(gate), initial, lengths, False)[:2]


def gated_recurrence_step(x: Tensor, gate: Tensor, state: Tensor,
                          parents: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """One step of ``gated_recurrence`` for decoding: (h, new state), where h is the new state
    in the type of x (the same tensor where the types agree).

    Without ``parents``, x, gate and state are [...][D] and every row goes on from its own state.
    With ``parents`` (int64 [B][k], as beam_select returns them) x and gate are [B][k][D], state
    is [B][K][D] and row [b][j] goes on from state[b][parents[b][j]]: the reordering of the
    states costs no pass of its own.  A parent outside 0 .. K-1 (-1: no hypothesis) counts as a
    state of zeros.  state is float32 (float64 for float64 inputs) and is left as it is.

    Not differentiable: gated_recurrence is for training.  No counterpart in the reference."""
    assert x.ndim >= 1 and gate.shape == x.shape, (gate.shape, x.shape)
    assert gate.dtype == x.dtype, (gate.dtype, x.dtype)
    code, kind = _code(x.dtype), _state_type(x.dtype)
    assert state.dtype == kind, (state.dtype, kind)
    D = x.shape[-1]
    if parents is None:
        assert state.shape == x.shape, (state.shape, x.shape)
        beams = K = 1
    else:
        assert x.ndim == 3 and state.ndim == 3, (x.ndim, state.ndim)
        beams, K = x.shape[1], state.shape[1]
        assert parents.shape == x.shape[:2], (parents.shape, x.shape)
        assert parents.dtype == torch.int64, parents.dtype
        assert state.shape == (x.shape[0], K, D), (state.shape, x.shape)
        assert parents.device == x.device, (parents.device, x.device)
        parents = parents.contiguous()
    dev = x.device
    assert x.is_cuda and gate.device == dev and state.device == dev, (dev, gate.device, state.device)
    assert not (torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad or
                                             state.requires_grad)), \
        "gated_recurrence_step has no gradients: use gated_recurrence, or torch.no_grad()"
    x2, gate2 = _rows(x.reshape(-1, D)), _rows(gate.reshape(-1, D))
    state = state.contiguous()
    rows = x2.shape[0]
    with _lib.on_device(dev):
        new = torch.empty(x.shape, dtype=kind, device=dev)
        h = new if kind == x.dtype else torch.empty(x.shape, dtype=x.dtype, device=dev)
        if rows > 0 and D > 0:
            _lib.call("frnnt_recurrence_step", _c_int(code), _lib._c_vp(x2.data_ptr()),
                      _c_longlong(x2.stride(0)), _lib._c_vp(gate2.data_ptr()),
                      _c_longlong(gate2.stride(0)), _lib.ptr(state), _lib.ptr(parents),
                      None if h is new else _lib.ptr(h), _lib.ptr(new), _c_longlong(rows), beams, K, D,
                      _lib.stream_ptr(dev))
    return h, new
