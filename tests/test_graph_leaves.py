"""What GraphedStep does to leaves that an eager graph holds, without a GPU."""
import torch

from fast_rnnt_b200.graphs import _held, _renew


def test_accumulators_that_are_held():
    x = torch.randn(3, requires_grad=True)
    assert not _held(x) and not _held(x)
    x.register_hook(lambda g: g)
    x.register_post_accumulate_grad_hook(lambda t: None)
    assert not _held(x)
    y = (x * x).sum()
    assert _held(x) and _held(x)
    del y
    assert not _held(x)


def test_new_accumulator():
    for make in (lambda: torch.nn.Parameter(torch.randn(4, 3)),
                 lambda: torch.randn(5, 6, dtype=torch.float64)[1:, ::2].requires_grad_(True),
                 lambda: torch.randn(6).half().requires_grad_(True)):
        x = make()
        calls = []
        x.register_hook(lambda g: calls.append(1))
        before = (type(x), x.data_ptr(), x.stride(), x.dtype, x._version, x.detach().clone())
        old = (x * x).sum()
        _renew(x)
        assert not _held(x)
        after = (type(x), x.data_ptr(), x.stride(), x.dtype, x._version, x.detach().clone())
        assert before[:-1] == after[:-1] and torch.equal(before[-1], after[-1]) and x.requires_grad
        (x * 3).sum().backward()
        assert torch.equal(x.grad, torch.full_like(x, 3)) and len(calls) == 1
        x.grad = None
        old.backward()      # the graph that was alive
        assert torch.equal(x.grad, 2 * x.detach()) and len(calls) == 2
