"""Gated linear recurrence on the GPU: the layer of a prediction network or an encoder whose
outputs the losses of this package take, over whole sequences with its gradients and, for
decoding, one token at a time.  No counterpart in the reference, which leaves both networks
to the caller.  The arithmetic runs in libfrnnt_sm100.so (csrc/recurrence.cu)."""
from typing import Optional, Tuple

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _lib

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
    t = _lib.plain(t)
    return t if t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def _forward(x, gate, initial, lengths, keep_states):
    B, T, D = x.shape
    dev, code = x.device, _CODES[x.dtype]
    saved = None
    with _lib.on_device(dev):
        h = torch.empty_like(x, memory_format=torch.contiguous_format)
        last = x.new_empty((B, D), dtype=_state_type(x.dtype))
        if keep_states:
            n = _lib.size_of("frnnt_recurrence_saved_bytes", code, B, T, D)
            saved = x.new_empty(n, dtype=torch.uint8) if n else initial   # none: a short sequence
        xs, gs = x.stride(), gate.stride()
        _lib.call("frnnt_recurrence_forward", code, x.data_ptr(), xs[0], xs[1], gate.data_ptr(), gs[0],
                  gs[1], None if initial is None else initial.data_ptr(),
                  None if lengths is None else lengths.data_ptr(), h.data_ptr(), last.data_ptr(),
                  None if saved is None or saved is initial else saved.data_ptr(), B, T, D,
                  _lib.stream_ptr(dev))
    return h, last, saved


def _backward(ctx, dh, dlast):
    x, gate, lengths, saved = ctx.saved_tensors
    B, T, D = x.shape
    dev, code = x.device, _CODES[x.dtype]
    if dh is not None:
        dh = _rows(dh)
    if dlast is not None:
        dlast = _lib.plain(dlast).contiguous()
    with _lib.on_device(dev):
        dx = torch.empty_like(x, memory_format=torch.contiguous_format)
        dgate = torch.empty_like(dx)
        dinitial = (x.new_empty((B, D), dtype=_state_type(x.dtype))
                    if ctx.needs_input_grad[2] else None)
        xs, gs, ds = x.stride(), gate.stride(), (0, 0) if dh is None else dh.stride()
        _lib.call("frnnt_recurrence_backward", code, x.data_ptr(), xs[0], xs[1], gate.data_ptr(), gs[0],
                  gs[1], None if lengths is None else lengths.data_ptr(),
                  None if saved is None else saved.data_ptr(),
                  None if dh is None else dh.data_ptr(), ds[0], ds[1],
                  None if dlast is None else dlast.data_ptr(), dx.data_ptr(), dgate.data_ptr(),
                  None if dinitial is None else dinitial.data_ptr(), B, T, D, _lib.stream_ptr(dev))
    return dx, dgate, dinitial, None


_backward_once = once_differentiable(_backward)


class _GatedRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, initial, lengths):
        h, last, saved = _forward(x, gate, initial, lengths, True)
        ctx.save_for_backward(x, gate, lengths, saved)
        ctx.set_materialize_grads(False)
        return h, last

    @staticmethod
    def backward(ctx, dh, dlast):
        # the wrapper that refuses a second derivative costs microseconds: only where one is recorded
        return (_backward_once if torch.is_grad_enabled() else _backward)(ctx, dh, dlast)


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
    A gate of -inf drops the state (h[:, t] = x[:, t]) and one of +inf keeps it.  x and the states
    are finite numbers: behind an infinite one, its channel holds infinities or NaN.

    B is at most 65535.  A sequence has the same bits in any batch whose tensors are aligned alike
    (rows on 16 bytes, on 4, or on neither).  Differentiable once with
    respect to x, gate and initial, in reverse mode (tensors with a forward-mode tangent are refused).  No counterpart in the reference."""
    assert x.ndim == 3, x.ndim
    shape, dtype, dev = x.shape, x.dtype, x.device
    assert gate.shape == shape, (gate.shape, shape)
    assert gate.dtype == dtype, (gate.dtype, dtype)
    _code(dtype)
    assert x.is_cuda and gate.device == dev, (dev, gate.device)
    if initial is not None:
        state = _state_type(dtype)
        assert initial.shape == (shape[0], shape[2]), (initial.shape, shape)
        assert initial.device == dev, (initial.device, dev)
        assert initial.dtype in (state, dtype), initial.dtype
        initial = _lib.plain(initial if initial.dtype == state else initial.to(state)).contiguous()
    if lengths is not None:
        assert lengths.shape == shape[:1] and lengths.dtype == torch.int64, (lengths.shape, lengths.dtype)
        assert lengths.device == dev, (lengths.device, dev)
        lengths = lengths.contiguous()
    x, gate = _rows(x), _rows(gate)
    if (torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad or
                                     (initial is not None and initial.requires_grad))
            or (_lib.tangents_possible() and _lib.has_tangent(x, gate, initial))):   # the autograd function refuses tangents
        return _GatedRecurrence.apply(x, gate, initial, lengths)
    return _forward(x, gate, initial, lengths, False)[:2]


def gated_recurrence_step(x: Tensor, gate: Tensor, state: Tensor,
                          parents: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """One step of ``gated_recurrence`` for decoding: (h, new state), where h is the new state
    in the type of x (the same tensor where the types agree).

    Without ``parents``, x, gate and state are [...][D] and every row goes on from its own state.
    With ``parents`` (int64 [B][k], as beam_select returns them) x and gate are [B][k][D], state
    is [B][K][D] and row [b][j] goes on from state[b][parents[b][j]]: the reordering of the
    states costs no pass of its own.  A parent outside 0 .. K-1 (-1: no hypothesis) counts as a
    state of zeros.  A row whose gate is +inf everywhere keeps its parent's state, bit for bit, and
    h is that state in the type of x: what a transducer's blank leaves behind.  state is float32 (float64 for float64 inputs) and is left as it is.

    Not differentiable: gated_recurrence is for training.  No counterpart in the reference."""
    assert x.ndim >= 1 and gate.shape == x.shape, (gate.shape, x.shape)
    assert gate.dtype == x.dtype, (gate.dtype, x.dtype)
    code = _code(x.dtype)
    kind = torch.float64 if code == _lib.F64 else torch.float32
    assert state.dtype == kind, (state.dtype, kind)
    D, dev = x.shape[-1], x.device
    index = dev.index
    if parents is None:
        assert state.shape == x.shape, (state.shape, x.shape)
        beams = K = 1
    else:
        assert x.ndim == 3 and state.ndim == 3, (x.ndim, state.ndim)
        beams, K = x.shape[1], state.shape[1]
        assert parents.shape == x.shape[:2], (parents.shape, x.shape)
        assert parents.dtype == torch.int64, parents.dtype
        assert state.shape == (x.shape[0], K, D), (state.shape, x.shape)
        assert parents.get_device() == (-1 if index is None else index), (parents.device, dev)
        parents = parents.contiguous()
    assert x.is_cuda and gate.get_device() == index and state.get_device() == index, (dev, gate.device, state.device)
    assert not (torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad or
                                             state.requires_grad)), \
        "gated_recurrence_step has no gradients: use gated_recurrence, or torch.no_grad()"
    assert not (_lib.tangents_possible() and _lib.has_tangent(x, gate, state)), "gated_recurrence_step has no forward-mode derivative"
    if x.is_neg() or gate.is_neg() or state.is_neg():
        x, gate, state = x.resolve_neg(), gate.resolve_neg(), state.resolve_neg()
    # rows at one distance from the next
    x2 = x if x.is_contiguous() else _rows(x.reshape(-1, D))
    gate2 = gate if gate.is_contiguous() else _rows(gate.reshape(-1, D))
    state = state.contiguous()
    rows = x.numel() // D if D > 0 else 0
    with _lib.on_device(dev):
        new = torch.empty_like(x, dtype=kind, memory_format=torch.contiguous_format)
        h = new if kind == x.dtype else torch.empty_like(x, memory_format=torch.contiguous_format)
        if rows > 0:
            _lib.call("frnnt_recurrence_step", code, x2.data_ptr(), D if x2 is x else x2.stride(0),
                      gate2.data_ptr(), D if gate2 is gate else gate2.stride(0), state.data_ptr(),
                      None if parents is None else parents.data_ptr(),
                      None if h is new else h.data_ptr(), new.data_ptr(), rows, beams, K, D,
                      _lib.raw_stream(index))
    return h, new
