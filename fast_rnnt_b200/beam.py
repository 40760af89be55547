"""Beam search on the GPU: the best continuations of every hypothesis by the trained joiner's
logits, and the reordering of the hypotheses' states.  No counterpart in the reference, which
ends with the losses.  The work runs in libfrnnt_sm100.so (csrc/beam.cu)."""
import math
from typing import List, Optional, Sequence, Tuple, Union

import torch
from torch import Tensor

from . import _lib
from ._lib import _c_longlong


def beam_select(logits: Tensor, scores: Tensor, beam: int, termination_symbol: int = 0,
                finished: Optional[Tensor] = None) -> Tuple[Tensor, Tensor, Tensor]:
    """The ``beam`` best continuations of every utterance: (scores, parents, tokens), each
    [B][beam], best first.

    logits [B][K][V] (float32, float16 or bfloat16, the vocabulary side by side, any strides
    between rows) are the joiner's outputs for the K hypotheses of an utterance and scores
    [B][K] (float32) their log-probabilities so far.  Hypothesis i goes on with symbol v at::

        scores[b, i] + log_softmax(logits[b, i])[v]

    and where ``finished`` (bool [B][K]) is set it only goes on with termination_symbol, at no
    cost, whatever its logits.  parents and tokens are int64: what continuation [b][j] goes on
    from, and with what.  A hypothesis offers the ``beam`` symbols of its largest logits (of equal
    ones the lowest symbols), and of all offers the best scores win, compared in 64 bits; equal
    scores go to the lower hypothesis and then to the lower symbol.  The log-sums come from
    exponentials and sums in 32 bits, off by no more than 2^-21 + (V / 256 + 16) 2^-24 (1.6e-6 for
    500 symbols, 1.3e-5 for 50 000; measured 3e-7 and 1.2e-6).  Equal rows, and rows that differ by
    a constant, have equal log-softmaxes to the last bit.

    Two hypotheses with the same symbols and another place of their blanks are two: nothing here
    merges them.

    A hypothesis with a score of -inf, +inf or NaN is none, whatever its logits; a symbol whose
    logit is -inf is never chosen, and a row whose log-sum-exp is not a finite number (a NaN or
    +inf in it, or nothing but -inf) offers nothing.  Where fewer than ``beam`` continuations are
    left, the slots behind them hold a score of -inf and -1 as parent and token, which
    beam_reorder and gated_recurrence_step take as no hypothesis.

    B is at most 65535, K at most 1024, beam at most 32.  Not differentiable."""
    assert logits.ndim == 3, logits.ndim
    (B, K, V) = logits.shape
    beam, termination_symbol = int(beam), int(termination_symbol)
    assert K >= 1 and V >= 1, logits.shape
    assert scores.shape == (B, K), (scores.shape, logits.shape)
    if logits.dtype != torch.float32 and not _lib.is_16bit(logits):
        raise TypeError(f"only float32, float16 and bfloat16 logits are supported, got {logits.dtype}")
    assert scores.dtype == torch.float32, scores.dtype
    dev = logits.device
    assert logits.is_cuda and scores.get_device() == dev.index, (dev, scores.device)
    if finished is not None:
        assert finished.shape == (B, K) and finished.dtype == torch.bool, (finished.shape, finished.dtype)
        assert finished.device == dev, (dev, finished.device)
        assert 0 <= termination_symbol < V, (termination_symbol, V)
        finished = finished.contiguous()
    assert not (torch.is_grad_enabled() and (logits.requires_grad or scores.requires_grad)), \
        "beam_select has no gradients: call it under torch.no_grad()"
    assert not (_lib.tangents_possible() and _lib.has_tangent(logits, scores)), "beam_select has no forward-mode derivative"
    if logits.is_neg() or scores.is_neg():
        logits, scores = logits.resolve_neg(), scores.resolve_neg()
    if V > 1 and logits.stride(2) != 1:
        logits = logits.contiguous()
    scores = scores.contiguous()
    code, (sb, sk, _) = _lib.input_code(logits.dtype), logits.stride()
    with _lib.on_device(dev):
        best = torch.empty_like(scores) if beam == K else scores.new_empty((B, beam))
        parents = torch.empty_like(best, dtype=torch.int64)
        tokens = torch.empty_like(parents)
        n = _lib.size_of("frnnt_beam_select_scratch_bytes", code, B, K, V, beam)
        scratch = scores.new_empty(n, dtype=torch.uint8)
        _lib.call("frnnt_beam_select", code, logits.data_ptr(), sb, sk, scores.data_ptr(),
                  None if finished is None else finished.data_ptr(), termination_symbol,
                  best.data_ptr(), parents.data_ptr(), tokens.data_ptr(), scratch.data_ptr(), B, K, V,
                  beam, _lib.raw_stream(dev.index))
    return best, parents, tokens


def beam_reorder(states: Union[Tensor, Sequence[Tensor]], parents: Tensor) -> Union[Tensor, List[Tensor]]:
    """``states[b, parents[b, j]]`` for every tensor of ``states`` ([B][K][...], any types and
    sizes), in one pass over all of them: new tensors [B][k][...], a list for a sequence of
    tensors.  parents is int64 [B][k], as beam_select returns it; a parent outside 0 .. K-1 (-1:
    no hypothesis) gives zeros.  Not differentiable."""
    one = isinstance(states, Tensor)
    tensors = [states] if one else list(states)
    assert parents.ndim == 2 and parents.dtype == torch.int64, (parents.shape, parents.dtype)
    (B, k) = parents.shape
    dev = parents.device
    assert parents.is_cuda, "fast_rnnt_b200 runs on CUDA tensors only (no CPU path)"
    parents = parents.contiguous()
    if not tensors:
        return []
    assert tensors[0].ndim >= 2 and tensors[0].shape[1] >= 1, tensors[0].shape
    K, index = tensors[0].shape[1], dev.index
    grad, dual = torch.is_grad_enabled(), _lib.tangents_possible()
    empty_like, contiguous = torch.empty_like, torch.contiguous_format
    rows, out = [], []   # rows: from, to, batch and beam strides, bytes of every tensor
    held = []            # copies stay until the launch
    shape = dtype = None
    with _lib.on_device(dev):
        for t in tensors:
            if t.shape != shape or t.dtype != dtype:   # tensors of one kind come in rows
                shape, dtype = t.shape, t.dtype
                assert len(shape) >= 2 and shape[0] == B and shape[1] == K, (shape, parents.shape, K)
                size, complex_ = t.element_size(), t.is_complex()
                bytes_ = size * math.prod(shape[2:])
            assert t.get_device() == index, (t.device, dev)
            assert not (grad and t.requires_grad), \
                "beam_reorder has no gradients: call it under torch.no_grad()"
            assert not (dual and _lib.has_tangent(t)), "beam_reorder has no forward-mode derivative"
            if t.is_neg() or (complex_ and t.is_conj()):   # memory that holds something else
                t = t.resolve_conj().resolve_neg()
                held.append(t)
            pitch, step = K * bytes_, bytes_
            if not t.is_contiguous():   # a row of a state has to lie in one piece; rows may lie anywhere
                if B > 0 and not t[0, 0].is_contiguous():
                    t = t.contiguous()
                pitch, step = size * t.stride(0), size * t.stride(1)
                held.append(t)
            new = empty_like(t, memory_format=contiguous) if k == K else t.new_empty((B, k) + shape[2:])
            out.append(new)
            rows += (t.data_ptr(), new.data_ptr(), pitch, step, bytes_)
        _lib.call("frnnt_beam_reorder", len(out), (_c_longlong * len(rows))(*rows), parents.data_ptr(), B, k, K,
                  _lib.raw_stream(index))
    return out[0] if one else out
