"""Tensors with a forward-mode tangent: the recurrence and the beam search refuse them, none drops
the tangent without a word."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

pytestmark = pytest.mark.gpu


def dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


@pytest.mark.parametrize("graph", [False, True])
def test_tangents_are_refused(graph):
    import fast_rnnt_b200 as fr
    x, gate, initial = torch.randn(2, 5, 8).cuda(), torch.randn(2, 5, 8).cuda(), torch.randn(2, 8).cuda()
    scores, parents = torch.zeros(2, 5).cuda(), torch.zeros(2, 5, dtype=torch.int64).cuda()
    with forward_ad.dual_level(), torch.set_grad_enabled(graph):
        for n in range(3):
            args = [x, gate, initial]
            args[n] = dual(args[n])
            with pytest.raises((NotImplementedError, RuntimeError)):
                fr.gated_recurrence(*args)
            args = [x, gate, x.clone()]
            args[n] = dual(args[n])
            with pytest.raises(AssertionError, match="forward-mode"):
                fr.gated_recurrence_step(*args)
        for args in ((dual(x), scores), (x, dual(scores))):
            with pytest.raises(AssertionError, match="forward-mode"):
                fr.beam_select(*args, 3)
        for states in (dual(x), [x, dual(gate)]):
            with pytest.raises(AssertionError, match="forward-mode"):
                fr.beam_reorder(states, parents)


def test_plain_tensors_inside_a_dual_level():
    import fast_rnnt_b200 as fr
    x, gate = torch.randn(2, 5, 8).cuda(), torch.randn(2, 5, 8).cuda()
    scores = torch.zeros(2, 5).cuda()

    def calls():
        h, last = fr.gated_recurrence(x, gate)
        best, parents, tokens = fr.beam_select(x, scores, 3)
        return [h, last, best, parents, tokens, *fr.gated_recurrence_step(x, gate, x), fr.beam_reorder(x, parents)]

    want = calls()
    with forward_ad.dual_level():
        other = dual(x)
        for a, b in zip(calls(), want):
            assert torch.equal(a, b) and forward_ad.unpack_dual(a).tangent is None
        primal = fr.gated_recurrence(forward_ad.unpack_dual(other).primal, gate)[0]
        assert torch.equal(primal, want[0])
