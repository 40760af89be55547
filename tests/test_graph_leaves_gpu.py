"""GraphedStep captures over the caller's own leaves: whoever else holds them, or has hooks on
them, gets from a replay what an eager step gives, also where an eager graph of the same leaves
is alive, on whatever stream it was built."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def make(seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(2, 40, 24, generator=g).cuda() for _ in range(2)]


def loss_of(x, gate):
    import fast_rnnt_b200 as fr
    return fr.gated_recurrence(x, gate)[0].square().sum()


def plain_gradients(x, gate):
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, gate)]
    return torch.autograd.grad(loss_of(*leaves), leaves)


@pytest.fixture(params=["released", "alive", "alive on a stream"])
def eager(request):
    """Builds an eager graph of the leaves that lives as long as the test."""
    kept = []

    def build(*leaves):
        stream = torch.cuda.Stream() if request.param == "alive on a stream" else torch.cuda.current_stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            kept.append(loss_of(*leaves))
        torch.cuda.current_stream().wait_stream(stream)
        if request.param == "released":
            kept.clear()
        return kept

    yield build
    kept.clear()


def replayed(graph, static, batch):
    with torch.no_grad():
        for t, value in zip(static, batch):
            t.copy_(value)
    graph()
    torch.cuda.synchronize()


def test_hooks_of_a_leaf(eager):
    from fast_rnnt_b200.graphs import GraphedStep
    x, gate = (t.requires_grad_(True) for t in make(1))
    seen = []
    x.register_hook(lambda grad: grad * 0.5)
    gate.register_post_accumulate_grad_hook(lambda leaf: seen.append(leaf))
    eager(x, gate)

    def step(t):
        loss = loss_of(t["x"], t["gate"])
        loss.backward()
        return loss

    graph = GraphedStep(step, dict(x=x, gate=gate), warmup=2)
    assert len(seen) == 3 and all(t is gate for t in seen)
    batch = make(2)
    dx, dgate = plain_gradients(*batch)
    replayed(graph, (x, gate), batch)
    assert torch.equal(x.grad, dx * 0.5) and torch.equal(gate.grad, dgate)


def test_leaves_reached_otherwise_than_through_the_inputs(eager):
    from fast_rnnt_b200.graphs import GraphedStep

    class Layer(torch.nn.Module):
        def __init__(self, *values):
            super().__init__()
            self.x, self.gate = (torch.nn.Parameter(v) for v in values)

        def forward(self):
            return loss_of(self.x, self.gate)

    layer = Layer(*make(3))
    eager(layer.x, layer.gate)
    kinds = []

    def step(t):
        kinds.append({type(v) for v in t.values()})
        loss = layer()
        loss.backward()
        return loss

    graph = GraphedStep(step, dict(layer.named_parameters()))
    assert all(k == {torch.nn.Parameter} for k in kinds)
    batch = make(4)
    replayed(graph, (layer.x, layer.gate), batch)
    for leaf, want in zip((layer.x, layer.gate), plain_gradients(*batch)):
        assert torch.equal(leaf.grad, want)


def test_optimizer_step_inside(eager):
    """p - lr grad with lr a power of two: one rounding, the same in any order of its two factors."""
    from fast_rnnt_b200.graphs import GraphedStep
    x, gate = (t.requires_grad_(True) for t in make(5))
    optimizer = torch.optim.SGD([x, gate], lr=2.0 ** -10)
    kept = eager(x, gate)

    def step(t):
        optimizer.zero_grad(set_to_none=True)
        loss = loss_of(t["x"], t["gate"])
        loss.backward()
        optimizer.step()
        return loss

    graph = GraphedStep(step, dict(x=x, gate=gate))
    kept.clear()
    for seed in (6, 7):
        batch = make(seed)
        replayed(graph, (x, gate), batch)
        for leaf, old, grad in zip((x, gate), batch, plain_gradients(*batch)):
            assert torch.equal(leaf.grad, grad)
            assert torch.equal(leaf, old - 2.0 ** -10 * grad)


def test_eager_graph_goes_on_after_the_capture(eager):
    """What was alive still gives its gradients, to the same leaves."""
    from fast_rnnt_b200.graphs import GraphedStep
    x, gate = (t.requires_grad_(True) for t in make(8))
    where = [t.data_ptr() for t in (x, gate)]
    kept = eager(x, gate)

    def step(t):
        loss = loss_of(t["x"], t["gate"])
        loss.backward()
        return loss

    graph = GraphedStep(step, dict(x=x, gate=gate))
    want = plain_gradients(x, gate)
    graph()
    torch.cuda.synchronize()
    assert all(torch.equal(t.grad, w) for t, w in zip((x, gate), want))
    assert [t.data_ptr() for t in (x, gate)] == where
    x.grad = gate.grad = None
    if kept:
        kept[0].backward()
        assert all(torch.equal(t.grad, w) for t, w in zip((x, gate), want))


def test_part_of_a_leaf_as_an_input_of_its_own():
    """A leaf and a view of it: the gradient of the leaf holds the shares of both."""
    from fast_rnnt_b200.graphs import GraphedStep
    both = torch.cat(make(9), -1).requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x, gate = both.chunk(2, -1)

    def step(t):
        loss = loss_of(t["x"], t["gate"]) + t["both"].sum()
        loss.backward()
        return loss

    graph = GraphedStep(step, dict(both=both, x=x, gate=gate), leaves=["both"])
    graph()
    torch.cuda.synchronize()
    want = torch.cat(plain_gradients(x, gate), -1) + 1
    assert torch.equal(both.grad, want)


def test_second_capture_of_the_same_leaves():
    """The first one's loss holds their accumulators, on the stream of the captures."""
    from fast_rnnt_b200.graphs import GraphedStep
    x, gate = (t.requires_grad_(True) for t in make(10))

    def step(t):
        loss = loss_of(t["x"], t["gate"])
        loss.backward()
        return loss

    first = GraphedStep(step, dict(x=x, gate=gate))
    second = GraphedStep(step, dict(x=x, gate=gate))
    batch = make(11)
    replayed(second, (x, gate), batch)
    assert all(torch.equal(t.grad, w) for t, w in zip((x, gate), plain_gradients(*batch)))
    first()
    torch.cuda.synchronize()
    assert torch.equal(first.loss, second.loss)
