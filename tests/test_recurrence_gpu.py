"""gated_recurrence and gated_recurrence_step against the formula in 64 bits."""
import pytest
import torch

from tests.recurrence_oracle import check, recurrence

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f64": torch.float64, "f16": torch.float16, "bf16": torch.bfloat16}


def make(B, T, D, dtype, seed=0, layout="apart"):
    """x and gate: tensors of their own, halves of one projection, or with time first"""
    g = torch.Generator().manual_seed(seed)
    x, gate = torch.randn(B, T, D, generator=g), torch.randn(B, T, D, generator=g) * 2 + 1.5
    if layout == "views":
        x, gate = torch.cat([x, gate], -1).to("cuda", dtype).chunk(2, -1)
    elif layout == "time first":
        x, gate = (t.transpose(0, 1).contiguous().to("cuda", dtype).transpose(0, 1) for t in (x, gate))
    else:
        x, gate = x.to("cuda", dtype), gate.to("cuda", dtype)
    state = torch.float64 if dtype == torch.float64 else torch.float32
    more = {"initial": torch.randn(B, D, generator=g).to("cuda", state),
            "dh": torch.randn(B, T, D, generator=g).to("cuda", dtype),
            "dlast": torch.randn(B, D, generator=g).to("cuda", state)}
    return x, gate, more


def run(x, gate, initial=None, lengths=None, dh=None, dlast=None):
    import fast_rnnt_b200 as fr
    leaves = [t.detach().requires_grad_(True) for t in (x, gate, initial) if t is not None]
    h, last = fr.gated_recurrence(leaves[0], leaves[1], leaves[2] if initial is not None else None, lengths)
    assert h.dtype == x.dtype and last.dtype == (torch.float64 if x.dtype == torch.float64 else torch.float32)
    out = {"h": h.detach(), "last": last.detach()}
    pairs = [(o, d) for o, d in ((h, dh), (last, dlast)) if d is not None]
    if pairs:
        grads = torch.autograd.grad([p[0] for p in pairs], leaves, [p[1] for p in pairs])
        out.update(zip(("dx", "dgate", "dinitial"), grads))
    return out


def compare(got, want, names=None):
    for name in names or got:
        check(got[name], want[name], name)


SIZES = [(1, 1, 1), (2, 1, 7), (3, 2, 64), (2, 31, 33), (1, 32, 128), (2, 33, 8), (3, 127, 40), (2, 128, 72),
         (2, 129, 65), (1, 257, 264), (2, 300, 24), (1, 1500, 16), (2, 2500, 34), (1, 3000, 33)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("B,T,D", SIZES)
def test_sequence_and_gradients(B, T, D, dtype):
    x, gate, m = make(B, T, D, TYPES[dtype], seed=T)
    compare(run(x, gate, **m), recurrence(x, gate, **m))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("layout", ["views", "time first"])
@pytest.mark.parametrize("D", [64, 37])
def test_strided_inputs(layout, D, dtype):
    x, gate, m = make(3, 150, D, TYPES[dtype], seed=1, layout=layout)
    compare(run(x, gate, **m), recurrence(x, gate, **m))
    # channels that do not lie side by side, and a gate that all channels share
    y = x.transpose(1, 2).contiguous().transpose(1, 2)
    shared = gate[..., :1].expand(-1, -1, D)
    compare(run(y, shared, **m), recurrence(y, shared, **m))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T", [1, 40, 200, 700])
def test_lengths(T, dtype):
    """A padded batch: what lies behind a sequence is not read, whatever it holds."""
    lengths = torch.tensor([T, 0, 1, T // 2, max(0, T - 1), T + 3, -2])
    x, gate, m = make(7, T, 48, TYPES[dtype], seed=2)
    pad = torch.arange(T)[None] >= lengths[:, None]
    for t in (x, gate, m["dh"]):
        t[pad.cuda()] = float("nan")
    got = run(x, gate, lengths=lengths.cuda(), **m)
    clean = [torch.nan_to_num(t) for t in (x, gate)]
    want = recurrence(*clean, m["initial"], lengths, torch.nan_to_num(m["dh"]), m["dlast"])
    compare(got, want)
    for name in ("h", "dx", "dgate"):
        assert (got[name][pad.cuda()] == 0).all(), name
    assert torch.equal(got["last"][1], m["initial"][1])


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_gradients_of_one_output_alone(dtype):
    x, gate, m = make(2, 140, 40, TYPES[dtype], seed=3)
    for keep in ("dh", "dlast"):
        some = {"initial": m["initial"], keep: m[keep]}
        compare(run(x, gate, **some), recurrence(x, gate, **some))
    # the gradient of a sum is one number seen by every element
    some = {"dh": torch.ones((), device="cuda", dtype=x.dtype).expand(2, 140, 40)}
    compare(run(x, gate, **some), recurrence(x, gate, **some))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_gates_at_their_limits(dtype):
    """+inf keeps the state, -inf drops it; very large gates do the same without overflow."""
    x, gate, m = make(2, 300, 40, TYPES[dtype], seed=4)
    big = 60000.0
    gate[:, 10:20], gate[:, 30:35], gate[0, 40], gate[1, 41:260] = float("inf"), float("-inf"), -big, big
    got, want = run(x, gate, **m), recurrence(x, gate, **m)
    compare(got, want)
    # the state that a run of steps starts from is a product of gates times an earlier state, not
    # the rounded chain, so that a kept state may differ between runs by its bound on either side
    kept = (got["h"][:, 10:20] - got["h"][:, 9:10]).abs().cpu().double()
    assert (kept <= want["h"][1][:, 10:20] + want["h"][1][:, 9:10]).all()
    assert torch.equal(got["h"][:, 30:35], x[:, 30:35])
    assert (got["dgate"][:, 10:20] == 0).all() and (got["dgate"][:, 30:35] == 0).all()


def test_one_nan_stays_in_its_channel():
    import fast_rnnt_b200 as fr
    x, gate, _ = make(2, 300, 40, torch.float32, seed=5)
    ref = fr.gated_recurrence(x, gate)[0]
    x[1, 150, 7] = float("nan")
    h, last = fr.gated_recurrence(x, gate)
    assert torch.isnan(h[1, 150:, 7]).all() and torch.isnan(last[1, 7])
    keep = torch.ones_like(h, dtype=torch.bool)
    keep[1, 150:, 7] = False
    assert torch.equal(h[keep], ref[keep])


@pytest.mark.parametrize("B,T,D", [(0, 5, 8), (2, 0, 8), (2, 5, 0)])
def test_empty(B, T, D):
    import fast_rnnt_b200 as fr
    x, gate, m = make(B, T, D, torch.float32)
    h, last = fr.gated_recurrence(x, gate, m["initial"])
    assert h.shape == (B, T, D) and torch.equal(last, m["initial"] if T == 0 else last)
    got = run(x, gate, **m)
    assert got["dx"].shape == (B, T, D)
    if T == 0:
        assert torch.equal(got["dinitial"], m["dlast"])
        assert (fr.gated_recurrence(x, gate)[1] == 0).all()


def test_gradients_against_differences():
    import fast_rnnt_b200 as fr
    x, gate, m = make(2, 9, 5, torch.float64, seed=6)
    lengths = torch.tensor([9, 4]).cuda()
    leaves = [t.detach().requires_grad_(True) for t in (x, gate, m["initial"])]
    assert torch.autograd.gradcheck(lambda *a: fr.gated_recurrence(*a, lengths), leaves)
    x, gate, _ = make(1, 140, 2, torch.float64, seed=7)
    leaves = [t.detach().requires_grad_(True) for t in (x, gate)]
    assert torch.autograd.gradcheck(fr.gated_recurrence, leaves)


def test_without_gradients_the_same_bits_and_twice_the_same():
    import fast_rnnt_b200 as fr
    x, gate, m = make(3, 500, 136, torch.bfloat16, seed=8)
    a, b = run(x, gate, **m), run(x, gate, **m)
    for name in a:
        assert torch.equal(a[name], b[name]), name
    with torch.no_grad():
        h, last = fr.gated_recurrence(x.requires_grad_(True), gate, m["initial"])
    assert torch.equal(h, a["h"]) and torch.equal(last, a["last"])


@pytest.mark.parametrize("T", [100, 700, 2300])
def test_a_sequence_alone_has_the_bits_it_has_in_a_batch(T):
    """However many tiles of it are taken at once."""
    x, gate, m = make(40, T, 96, torch.float32, seed=19)
    batch = run(x, gate, **m)
    for b in (0, 39):
        alone = run(x[b:b + 1], gate[b:b + 1], **{k: v[b:b + 1] for k, v in m.items()})
        for name in alone:
            assert torch.equal(alone[name][0], batch[name][b]), name


def test_state_carried_between_pieces():
    """A sequence in pieces, each from the state of the one before, as a streaming encoder runs."""
    import fast_rnnt_b200 as fr
    x, gate, m = make(2, 411, 72, torch.float32, seed=9)
    state, parts = m["initial"], []
    for lo, hi in ((0, 1), (1, 130), (130, 300), (300, 411)):
        h, state = fr.gated_recurrence(x[:, lo:hi], gate[:, lo:hi], state)
        parts.append(h)
    want = recurrence(x, gate, m["initial"])
    check(torch.cat(parts, 1), want["h"], "h")
    check(state, want["last"], "last")


def test_refusals():
    import fast_rnnt_b200 as fr
    x, gate, m = make(2, 5, 8, torch.float16)
    lengths = torch.tensor([5, 5])
    for args in [(x, gate.cpu()), (x, gate.float()), (x, gate, m["initial"].cpu()), (x, gate, m["initial"].double()),
                 (x, gate, m["initial"][:1]), (x, gate, None, lengths), (x, gate, None, lengths.cuda().int()),
                 (x, gate, None, lengths[:1].cuda())]:
        with pytest.raises(AssertionError):
            fr.gated_recurrence(*args)
    state = m["initial"]
    for args in [(x[:, 0], gate[:, 0], state.cpu()), (x[:, 0], gate[:, 0], state.half()),
                 (x[:, 0], gate[:, 0], state.clone().requires_grad_(True)),
                 (x, gate, state[:, None], torch.zeros(2, 5, dtype=torch.int64))]:
        with pytest.raises(AssertionError):
            fr.gated_recurrence_step(*args)
    wide = torch.zeros(65536, 1, 1, device="cuda")
    with pytest.raises(fr.FrnntError, match="too large"):
        fr.gated_recurrence(wide, wide)


def test_initial_state_changed_before_the_backward_pass():
    """The state that gradients are computed from is the one of the forward pass, or an error."""
    import fast_rnnt_b200 as fr
    for T in (100, 300):
        x, gate, m = make(2, T, 16, torch.float32, seed=20)
        want = run(x, gate, m["initial"], dh=m["dh"])
        leaf = x.clone().requires_grad_(True)
        buffer = m["initial"].clone()
        h, last = fr.gated_recurrence(leaf, gate, buffer)
        buffer.zero_()
        try:
            (dx,) = torch.autograd.grad(h, leaf, m["dh"])
        except RuntimeError as e:
            assert "modified by an inplace operation" in str(e)
        else:
            assert torch.equal(dx, want["dx"])


def test_second_derivative_is_refused():
    import fast_rnnt_b200 as fr
    x, gate, _ = make(1, 4, 4, torch.float32)
    x = x.requires_grad_(True)
    h, _ = fr.gated_recurrence(x, gate)
    (dx,) = torch.autograd.grad(h.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.sum(), x)


def test_other_stream():
    import fast_rnnt_b200 as fr
    x, gate, m = make(4, 900, 64, torch.float32, seed=10)
    want = run(x, gate, **m)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y = x * 1.0     # produced on the side stream just before
        got = run(y, gate, **m)
    side.synchronize()
    for name in want:
        assert torch.equal(got[name], want[name]), name


def test_captured_step():
    import fast_rnnt_b200 as fr
    from fast_rnnt_b200.graphs import GraphedStep
    x, gate, m = make(3, 260, 40, torch.bfloat16, seed=11)
    x2, gate2, _ = make(3, 260, 40, torch.bfloat16, seed=12)

    def step(t):
        h, last = fr.gated_recurrence(t["x"], t["gate"], t["initial"])
        loss = (h.float() * t["dh"].float()).sum() + (last * t["dlast"]).sum()
        loss.backward()
        return loss

    static = {k: v.clone() for k, v in dict(m, x=x, gate=gate).items()}
    for k in ("x", "gate", "initial"):
        static[k].requires_grad_(True)
    g = GraphedStep(step, static)
    assert g.launches == 2
    for a, b in ((x2, gate2), (x, gate)):
        with torch.no_grad():
            static["x"].copy_(a)
            static["gate"].copy_(b)
        g()
        torch.cuda.synchronize()
        want = run(a, b, **m)
        for k in ("x", "gate", "initial"):
            assert torch.equal(static[k].grad, want["d" + k]), k


def test_offsets_beyond_32_bits():
    """More than 2^31 elements before the last steps."""
    import fast_rnnt_b200 as fr
    D, T = 1024, (1 << 21) + 70
    x = torch.zeros(1, T, D, dtype=torch.bfloat16, device="cuda")
    tail, gate, _ = make(1, 300, D, torch.bfloat16, seed=13)
    x[:, -300:] = tail
    gates = gate[:, :1].expand(1, T, D)
    h, last = fr.gated_recurrence(x, gates)
    want = recurrence(tail, gate[:, :1].expand(1, 300, D))
    check(h[:, -300:], want["h"], "h")
    check(last, want["last"], "last")
    assert (h[:, : T - 300] == 0).all()
    del h
    x.requires_grad_(True)
    h, last = fr.gated_recurrence(x, gates)
    (dx,) = torch.autograd.grad(last.sum(), x)
    want = recurrence(tail, gate[:, :1].expand(1, 300, D), dlast=torch.ones(1, D))
    check(dx[:, -300:], want["dx"], "dx")


@pytest.mark.parametrize("tries", [-1, 0])
def test_waits_of_a_cluster_that_run_out(tries):
    """Nothing is withheld: with no looks at all every wait gives up, and the outputs say so."""
    from fast_rnnt_b200 import _lib
    B, T, D = 2, 1000, 40
    x, gate, m = make(B, T, D, torch.float32, seed=21)
    h, dx, dgate = (torch.empty_like(x) for _ in range(3))
    last = torch.empty(B, D, device="cuda")
    saved = torch.empty(_lib.size_of("frnnt_recurrence_saved_bytes", 0, B, T, D), dtype=torch.uint8, device="cuda")
    _lib.call("frnnt_recurrence_limited", *[_lib.ptr(t) for t in (x, gate, h, last, saved, m["dh"], dx, dgate)],
              B, T, D, tries, _lib.stream_ptr(x.device))
    torch.cuda.synchronize()
    if tries < 0:
        want = recurrence(x, gate, dh=m["dh"])
        compare(dict(h=h, last=last, dx=dx, dgate=dgate), want)
    else:
        for t in (h, last, dx, dgate):
            assert torch.isnan(t).all()
    # and the next call is none the worse for it
    compare(run(x, gate, dh=m["dh"]), recurrence(x, gate, dh=m["dh"]))


# ------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [(1,), (7,), (5, 64), (3, 4, 37), (1, 1, 1), (2, 3, 4, 8)])
def test_step_without_parents(shape, dtype):
    import fast_rnnt_b200 as fr
    rows = max(1, torch.Size(shape).numel() // shape[-1])
    x, gate, m = make(rows, 1, shape[-1], TYPES[dtype], seed=14)
    h, state = fr.gated_recurrence_step(x.reshape(shape), gate.reshape(shape), m["initial"].reshape(shape))
    want = recurrence(x, gate, m["initial"])
    check(h.reshape(rows, 1, -1), want["h"], "h")
    check(state.reshape(rows, -1), want["last"], "state")
    assert h.dtype == TYPES[dtype] and h.shape == shape and state.shape == shape


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("B,K,k,D", [(1, 1, 4, 5), (3, 4, 4, 64), (2, 5, 3, 33), (4, 2, 7, 520)])
def test_step_from_parents(B, K, k, D, dtype):
    """States read through the parents, the same parent twice, and -1 for no hypothesis."""
    import fast_rnnt_b200 as fr
    both, gate, _ = make(B, k, 2 * D, TYPES[dtype], seed=15)
    x, gate = both[..., :D], both[..., D:]
    state = make(B, K, D, TYPES[dtype], seed=16)[0].to(torch.float64 if dtype == "f64" else torch.float32)
    parents = torch.randint(0, K, (B, k), generator=torch.Generator().manual_seed(17))
    parents[0, 0], parents[-1, -1] = -1, K
    if k > 2:
        parents[0, 1] = parents[0, 2]
    keep = state.clone()
    h, new = fr.gated_recurrence_step(x, gate, state, parents.cuda())
    padded = torch.cat([state.cpu(), torch.zeros(B, 1, D, dtype=state.dtype)], 1)
    old = padded[torch.arange(B)[:, None], torch.where(parents < 0, K, parents)]
    want = recurrence(x.reshape(B * k, 1, D), gate.reshape(B * k, 1, D), old.reshape(B * k, D))
    check(h.reshape(B * k, 1, D), want["h"], "h")
    check(new.reshape(B * k, D), want["last"], "state")
    assert torch.equal(state, keep)


def test_steps_are_the_sequence():
    import fast_rnnt_b200 as fr
    x, gate, m = make(2, 40, 24, torch.float32, seed=18)
    state = m["initial"]
    hs = []
    for t in range(40):
        h, state = fr.gated_recurrence_step(x[:, t], gate[:, t], state)
        hs.append(h)
    want = recurrence(x, gate, m["initial"])
    check(torch.stack(hs, 1), want["h"], "h")
    check(state, want["last"], "last")


@pytest.mark.parametrize("B,T,D", [(2, 1000, 40), (1, 5000, 33), (3, 400, 300), (1, 30011, 64)])
def test_waits_that_run_out_now_and_then(B, T, D):
    """However few looks a wait is given: every value is that of waits without a limit, or NaN."""
    from fast_rnnt_b200 import _lib
    x, gate, m = make(B, T, D, torch.float32, seed=22)

    def limited(tries):
        out = dict(h=torch.empty_like(x), last=torch.empty(B, D, device="cuda"), dx=torch.empty_like(x),
                   dgate=torch.empty_like(x))
        saved = torch.empty(_lib.size_of("frnnt_recurrence_saved_bytes", 0, B, T, D), dtype=torch.uint8, device="cuda")
        _lib.call("frnnt_recurrence_limited", *[_lib.ptr(t) for t in (x, gate, out["h"], out["last"], saved, m["dh"],
                                                                      out["dx"], out["dgate"])],
                  B, T, D, tries, _lib.stream_ptr(x.device))
        torch.cuda.synchronize()
        return out

    want = limited(-1)
    assert all(torch.isfinite(t).all() for t in want.values())
    for tries in (0, 1, 2, 3, 5, 9, 20, 50, 0, -1):
        got = limited(tries)
        for name, t in got.items():
            lost = torch.isnan(t)
            assert torch.equal(torch.where(lost, want[name], t), want[name]), (tries, name)
        if tries < 0:
            assert not any(torch.isnan(t).any() for t in got.values())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_gates_of_long_memory(dtype):
    """What a step keeps of the state, off by one rounding below 1 (2^-25) and by what the other share
    is off by: its exponential (2 units in the last place; for 16-bit types those of ex2, the rounding
    of its argument and that of log2(e), 1.3 |g| units of 2^-24), a sum (half a unit) and a
    reciprocal (one)."""
    import fast_rnnt_b200 as fr
    gate = torch.linspace(0, 17, 40001).to("cuda", TYPES[dtype])[None]
    zero, one = torch.zeros_like(gate), torch.ones(gate.shape, device="cuda")
    g = gate.cpu().double()
    take = torch.sigmoid(-g)
    bound = 2.0 ** -25 + take * (7 + (0 if dtype == "f32" else 1.3 * g)) * 2.0 ** -24
    for sign in (1, -1):
        # a step that keeps the state, and one that takes the input
        x, state = (zero, one) if sign == 1 else (zero + 1, 0 * one)
        off = fr.gated_recurrence_step(x, sign * gate, state)[1].cpu().double() - torch.sigmoid(g)
        assert (off.abs() <= bound).all(), (sign, float((off.abs() / bound).max()))
        off = fr.gated_recurrence(x[:, None], sign * gate[:, None], state)[1].cpu().double() - torch.sigmoid(g)
        assert (off.abs() <= bound).all(), (sign, float((off.abs() / bound).max()))
