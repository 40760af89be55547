"""beam_select and beam_reorder against their definitions in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
INF = math.inf


def keys_of(logits, scores, finished=None, symbol=0):
    """Every continuation's score in 64 bits, -inf where it is none."""
    x, s = logits.detach().cpu().double(), scores.cpu().double()
    top = x.amax(-1, keepdim=True)
    logp = (x - top) - torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    if finished is not None:
        f = finished.cpu()
        logp[f] = -INF
        logp[..., symbol] = torch.where(f, 0.0, logp[..., symbol])
    key = s[:, :, None] + logp
    return torch.where(torch.isnan(key), -INF, key).flatten(1)


def tolerance(V):
    """Of a score before its rounding to 32 bits: exponentials of 2^-21 relative error and no more
    than V / 256 + 16 additions one after the other in 32 bits, each off by 2^-24 of the sum."""
    return 2.0 ** -21 + (V / 256 + 16) * 2.0 ** -24


def verify(logits, scores, beam, finished=None, symbol=0, out=None):
    import fast_rnnt_b200 as fr
    B, K, V = logits.shape
    got, parents, tokens = fr.beam_select(logits, scores, beam, symbol, finished) if out is None else out
    assert got.shape == parents.shape == tokens.shape == (B, beam)
    key = keys_of(logits, scores, finished, symbol)
    best, at = torch.sort(key, dim=1, descending=True, stable=True)
    n = min(beam, K * V)
    best, at = best[:, :n], at[:, :n]
    got, parents, tokens = got.cpu(), parents.cpu(), tokens.cpu()
    tol = tolerance(V)
    for b in range(B):
        m = int((best[b] > -INF).sum())
        assert (got[b, m:] == -INF).all() and (parents[b, m:] == -1).all() and (tokens[b, m:] == -1).all(), b
        p, t = parents[b, :m], tokens[b, :m]
        assert ((p >= 0) & (p < K) & (t >= 0) & (t < V)).all(), (b, p, t)
        index = p * V + t
        assert len(set(index.tolist())) == m, (b, index)
        off = (got[b, :m].double() - best[b, :m]).abs()
        assert (off <= tol + 2.0 ** -24 * best[b, :m].abs()).all(), (b, off.max(), tol)
        assert ((key[b, index] - best[b, :m]).abs() <= 2 * tol).all(), b
        # the very continuation wherever its neighbours are further away than the tolerance, or
        # equal to the last digit
        for j in range(m):
            near = (key[b] - best[b, j]).abs() <= 2 * tol
            if not (near & (key[b] != best[b, j])).any():
                assert index[j] == at[b, j], (b, j, index[j], at[b, j])
    return got, parents, tokens


def make(B, K, V, dtype, seed=0, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(B, K, V, generator=g) * scale).to("cuda", TYPES[dtype])
    return logits, (-8 * torch.rand(B, K, generator=g)).cuda()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("B,K,V,beam", [(1, 1, 1, 1), (2, 1, 3, 8), (1, 4, 500, 4), (3, 4, 500, 10), (2, 3, 4233, 5),
                                        (5, 16, 31, 16), (2, 8, 5000, 8), (1, 1, 50001, 32), (40, 5, 77, 3),
                                        (3, 32, 1025, 32), (1, 3, 2049, 32), (2, 100, 40, 20), (600, 2, 130, 2)])
def test_selection(B, K, V, beam, dtype):
    logits, scores = make(B, K, V, dtype, seed=V)
    verify(logits, scores, beam)


def test_most_hypotheses():
    logits, scores = make(2, 1024, 65, "f32", seed=8)
    verify(logits, scores, 32)
    logits, scores = make(0, 3, 9, "f32")
    import fast_rnnt_b200 as fr
    assert [t.shape for t in fr.beam_select(logits, scores, 4)] == [(0, 4)] * 3


def test_refusals():
    import fast_rnnt_b200 as fr
    logits, scores = make(2, 3, 40, "f32")
    for beam in (0, 33):
        with pytest.raises(fr.FrnntError, match="beam"):
            fr.beam_select(logits, scores, beam)
    many = torch.zeros(1, 1025, 4, device="cuda")
    with pytest.raises(fr.FrnntError, match="beams"):
        fr.beam_select(many, many[..., 0].contiguous(), 2)
    for args in [(logits, scores.cpu(), 3), (logits.cpu(), scores, 3),
                 (logits.clone().requires_grad_(True), scores, 3), (logits, scores.clone().requires_grad_(True), 3),
                 (logits, scores, 3, 40, torch.zeros(2, 3, dtype=torch.bool, device="cuda")),
                 (logits, scores, 3, 0, torch.zeros(2, 3, device="cuda")),
                 (logits, scores, 3, 0, torch.zeros(2, 3, dtype=torch.bool))]:
        with pytest.raises(AssertionError):
            fr.beam_select(*args)
    parents = torch.zeros(2, 4, dtype=torch.int64, device="cuda")
    for states in ([logits, logits[:, :2]], [logits, logits[:1]], [logits.cpu()], [scores[0]],
                   [logits.clone().requires_grad_(True)]):
        with pytest.raises(AssertionError):
            fr.beam_reorder(states, parents)
    with torch.no_grad():    # gradients are not wanted: the same tensors are taken
        fr.beam_reorder([logits.clone().requires_grad_(True)], parents)
        fr.beam_select(logits.clone().requires_grad_(True), scores, 3)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_dead_and_finished_hypotheses(dtype):
    logits, scores = make(6, 7, 333, dtype, seed=1)
    scores[0, 2:], scores[1, :], scores[2, 0], scores[2, 3] = -INF, -INF, float("nan"), -INF
    logits[0, 3] = float("nan")             # not read: the hypothesis is none
    finished = torch.zeros(6, 7, dtype=torch.bool)
    finished[3], finished[4, ::2], finished[0, 0], finished[0, 3] = True, True, True, True
    logits[4, 0] = float("nan")             # not read: the hypothesis is finished
    verify(logits.masked_fill(torch.isnan(logits), 0.0), scores, 9, finished.cuda(), 17)
    a = verify(logits.masked_fill(torch.isnan(logits), 0.0), scores, 9, finished.cuda())
    import fast_rnnt_b200 as fr
    b = fr.beam_select(logits, scores, 9, finished=finished.cuda())
    assert all(torch.equal(u, v.cpu()) for u, v in zip(a, b))
    assert (b[1][1] == -1).all() and (b[2][3, :7] == 0).all()
    # a score of +inf is as little a hypothesis as one of -inf
    for value in (INF, -INF, float("nan")):
        scores[5, 3] = value
        got = fr.beam_select(logits, scores, 9)
        assert (got[1][5] != 3).all() and torch.isfinite(got[0][5]).all()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("K", range(1, 20))
def test_every_number_of_hypotheses(K, dtype):
    """Rows split over CTAs, one each, or several each: sizes on either side of every choice."""
    for V in (1100, 2050, 17001):
        logits, scores = make(2, K, V, dtype, seed=K)
        scores[1, K // 2] = -INF
        verify(logits, scores, 6)
        finished = torch.zeros(2, K, dtype=torch.bool, device="cuda")
        finished[:, -1] = True
        verify(logits, scores, 6, finished, V - 1)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_masked_and_bad_logits(dtype):
    logits, scores = make(7, 4, 700, dtype, seed=2)
    logits[0, :, 5:] = -INF                  # few symbols allowed
    logits[1, 1] = -INF                      # none
    logits[2, 2, 11] = float("nan")          # the row offers nothing
    logits[3, 0, 699] = INF
    logits[4, :, 1:] = torch.finfo(TYPES[dtype]).min     # masked by the lowest number
    logits[5] = torch.finfo(TYPES[dtype]).min
    logits[6, :, :690] = -INF
    verify(logits, scores, 12)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("V", [5, 64, 4233, 30000])
def test_ties_go_to_the_lowest(V, dtype):
    import fast_rnnt_b200 as fr
    logits = torch.zeros(2, 3, V, dtype=TYPES[dtype], device="cuda")
    logits[1] = 7
    logits[1, :, 1::2] = 7.5
    logits[0, :, 0] = -0.0
    scores = torch.zeros(2, 3, device="cuda")
    _, p, t = verify(logits, scores, min(32, V))
    n = min(32, V)
    assert (p[0] == 0).all() and torch.equal(t[0], torch.arange(n))
    # equal hypotheses, wherever their rows lie
    g = torch.Generator().manual_seed(3)
    row = (torch.randn(V, generator=g) * 3).to("cuda", TYPES[dtype])
    rows = row.expand(1, 9, V).contiguous()
    s, p, t = fr.beam_select(rows, torch.zeros(1, 9, device="cuda"), 9)
    assert torch.equal(p[0].cpu(), torch.arange(9)), p
    assert (t == t[0, 0]).all() and (s == s[0, 0]).all()
    # and rows that differ by a constant
    whole = torch.randint(-9, 9, (V,), generator=g).to("cuda", TYPES[dtype])
    rows = whole + torch.tensor([0, 5, -3, 64, 1], dtype=TYPES[dtype], device="cuda")[None, :, None]
    s, p, t = fr.beam_select(rows, torch.zeros(1, 5, device="cuda"), 5)
    n = min(5, int((whole == whole.max()).sum()))
    ties = (whole == whole.max()).nonzero()[:n, 0]
    assert (p[0, :n] == 0).all() and torch.equal(t[0, :n], ties) and (s[0, :n] == s[0, 0]).all()
    if n == 1:
        assert torch.equal(p[0].cpu(), torch.arange(5)) and (s == s[0, 0]).all()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("V", [9, 300, 4233, 31999])
def test_many_equal_logits(V, dtype):
    """A few symbols allowed, the others masked by the lowest number; a plateau that begins late,
    a plateau of every n-th symbol, and one behind all others."""
    low = torch.finfo(TYPES[dtype]).min
    n = torch.arange(V)
    g = torch.Generator().manual_seed(V)
    some = torch.randperm(V, generator=g)[:5]
    x = torch.full((7, V), low, dtype=torch.float64)
    x[0, some] = 1.5
    x[1, some] = torch.randn(5, generator=g).double()
    x[2] = torch.where(n > V // 2, 0.25, -1.0).double()
    x[3] = torch.where(n % 611 == 7, 2.0, -2.0).double()
    x[4] = torch.where(n >= V - 3, 3.0, 1.0).double()
    x[5] = torch.where(n < 3, 3.0, 1.0).double()
    x[6] = torch.where(n % 128 == 5, 4.0 + (n % 3) / 4, 1.0).double()
    logits = x.to("cuda", TYPES[dtype])[:, None].repeat(1, 2, 1)
    for beam in (1, 12, 32):
        verify(logits, torch.zeros(7, 2, device="cuda"), beam)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("V", [3000, 70001])
def test_orders_that_come_in_clumps(V, dtype):
    """Ascending, descending and periodic logits: the best ones lie side by side, or all in a few
    threads' shares."""
    n = torch.arange(V, dtype=torch.float64)
    step = 8.0 / V
    for x in (n * step, -n * step, torch.where(n % 2048 < 8, 5 + n * step, n * 0.0),
              torch.where(n % 2048 < 256, (n % 7) * 0.5, n * 0.0), torch.where(n % 256 == 3, 4.0 + n % 3, n * 0.0)):
        logits = x.to("cuda", TYPES[dtype])[None, None].repeat(2, 2, 1)
        logits[1, 1] += 1
        scores = torch.tensor([[0.0, -0.25], [-0.5, 0.0]], device="cuda")
        verify(logits, scores, 32)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_strided_logits(dtype):
    wide, scores = make(3, 5, 1001, dtype, seed=4)
    verify(wide[:, :, :997], scores, 7)
    verify(wide[:, :, 3:998], scores, 7)
    verify(wide[:, ::2], scores[:, ::2], 7)
    verify(wide.transpose(0, 1), scores.t(), 7)
    verify(wide.transpose(1, 2)[:, :5], torch.zeros(3, 5, device="cuda"), 7)
    verify(wide[:, :1].expand(3, 5, 1001), scores, 7)


def test_select_offsets_beyond_32_bits():
    V, K = 1 << 20, 9
    logits = torch.zeros(240, K, V, dtype=torch.bfloat16, device="cuda")   # 2.2e9 elements
    logits[-1] = make(1, K, V, "bf16", seed=5)[0][0]
    scores = make(240, K, 4, "bf16", seed=6)[1]
    import fast_rnnt_b200 as fr
    got = fr.beam_select(logits, scores, 6)
    # both against the definition and not against one another: a row alone is summed in parts
    verify(logits[-1:], scores[-1:], 6, out=[g[-1:] for g in got])
    verify(logits[-1:], scores[-1:], 6)


# ------------------------------------------------------------------------------
def reordered(t, parents):
    t, p = t.cpu(), parents.cpu()
    B, K = t.shape[:2]
    rows = torch.cat([t, torch.zeros_like(t[:, :1])], 1)
    return rows[torch.arange(B)[:, None], torch.where((p < 0) | (p >= K), K, p)]


@pytest.mark.parametrize("B,K,k", [(1, 1, 1), (3, 4, 4), (5, 2, 7), (2, 9, 1), (64, 8, 8)])
def test_reorder(B, K, k):
    import fast_rnnt_b200 as fr
    g = torch.Generator().manual_seed(B)
    parents = torch.randint(-1, K + 1, (B, k), generator=g).cuda()
    states = [torch.randn(B, K, 37, generator=g).cuda(),
              torch.randn(B, K, 512, generator=g).cuda().half(),
              torch.randint(0, 9, (B, K, 65), generator=g).cuda(),
              torch.randint(0, 2, (B, K), generator=g).bool().cuda(),
              torch.randn(B, K, 3, 5, generator=g).cuda().bfloat16(),
              torch.randn(B, K, 1, generator=g).cuda().double(),
              torch.randn(B, K, 0, generator=g).cuda(),
              torch.randn(B, K, 2, 64, generator=g).cuda()[:, :, 1],
              torch.randn(K, B, 33, generator=g).cuda().transpose(0, 1),
              torch.randn(B, K, 9, 4, generator=g).cuda().transpose(2, 3),
              torch.randn(B, 1, 20, generator=g).cuda().expand(B, K, 20),
              torch.randn(B, K, 5001, generator=g).cuda()[..., 1:]]
    got = fr.beam_reorder(states, parents)
    assert isinstance(got, list) and len(got) == len(states)
    for t, u in zip(states, got):
        assert u.dtype == t.dtype and torch.equal(u.cpu(), reordered(t, parents))
    assert torch.equal(fr.beam_reorder(states[0], parents), got[0])
    assert fr.beam_reorder([], parents) == []


@pytest.mark.parametrize("dtype", [torch.uint8, torch.bfloat16, torch.float32, torch.int64])
def test_reorder_rows_of_every_length_and_place(dtype):
    """Rows that begin anywhere, source and destination each on its own."""
    import fast_rnnt_b200 as fr
    g = torch.Generator().manual_seed(9)
    parents = torch.randint(-1, 5, (3, 4), generator=g).cuda()
    wide = torch.randint(0, 120, (3, 5, 300), generator=g).to("cuda", dtype)
    states = [wide[:, :, o:o + n] for n in (1, 2, 3, 7, 15, 16, 17, 31, 33, 63, 64, 65, 79, 97, 255, 280) for o in (0, 1, 5)]
    for t, u in zip(states, fr.beam_reorder(states, parents)):
        assert torch.equal(u.cpu(), reordered(t, parents)), t.shape


def test_reorder_many_and_large():
    import fast_rnnt_b200 as fr
    g = torch.Generator().manual_seed(7)
    parents = torch.randint(-1, 3, (2, 5), generator=g).cuda()
    states = [torch.randn(2, 3, 1 + 7 * n, generator=g).cuda() for n in range(70)]
    for t, u in zip(states, fr.beam_reorder(tuple(states), parents)):
        assert torch.equal(u.cpu(), reordered(t, parents))
    # rows that begin beyond 2^31 elements
    big = torch.zeros(2, 3, 400_000_001, dtype=torch.uint8, device="cuda")
    big[1, 2, -1000:] = torch.arange(1000).cuda() % 251
    out = fr.beam_reorder(big, torch.tensor([[0, 1], [1, 2]]).cuda())
    assert torch.equal(out[1, 1], big[1, 2]) and not out[0].any() and not out[1, 0].any()


def test_captured_search_step():
    """Selection, reordering and the recurrence's step in one graph, replayed on other inputs."""
    import fast_rnnt_b200 as fr

    def step(logits, scores, states, x, gate, state):
        with torch.no_grad():
            best, parents, tokens = fr.beam_select(logits, scores, 4)
            return (best, parents, tokens, *fr.beam_reorder(states, parents),
                    *fr.gated_recurrence_step(x, gate, state, parents))

    def inputs(seed):
        logits, scores = make(3, 4, 500, "f32", seed=seed)
        rest = [make(3, 4, n, "f32", seed=seed + n)[0] for n in (40, 7, 64, 64, 64)]
        return [logits, scores, rest[:2], *rest[2:]]

    static = inputs(1)
    step(*static)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*static)
    for seed in (2, 1):
        for s, t in zip(static, inputs(seed)):
            for a, b in zip(s if isinstance(s, list) else [s], t if isinstance(t, list) else [t]):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step(*inputs(seed))):
            assert torch.equal(a, b)


def test_reorder_of_lazily_conjugated_and_negated_states():
    """Tensors whose memory holds the conjugate, or the negative, of what they are."""
    import fast_rnnt_b200 as fr
    g = torch.Generator().manual_seed(11)
    z = torch.complex(torch.randn(3, 4, 6, generator=g), torch.randn(3, 4, 6, generator=g)).cuda()
    parents = torch.randint(-1, 4, (3, 4), generator=g).cuda()
    states = [z, z.conj(), z.conj()[:, :, 1:], z.conj().imag, z.conj().imag[..., 0], z.conj().real,
              torch._neg_view(z.real.contiguous())]
    assert [t.is_conj() or t.is_neg() for t in states] == [False, True, True, True, True, False, True]
    for t, u in zip(states, fr.beam_reorder(states, parents)):
        assert torch.equal(u.cpu(), reordered(t.resolve_conj().resolve_neg(), parents))


def test_other_inputs_that_are_lazily_negated():
    """A single channel or symbol, whose memory no copy would set right on the way."""
    import fast_rnnt_b200 as fr
    g = torch.Generator().manual_seed(12)
    for width in (1, 8):
        z, gate = (torch.complex(*torch.randn(2, 2, 5, width, generator=g)).cuda() for _ in range(2))
        x, f = z.conj().imag, torch._neg_view(gate.real.contiguous())
        lazy = [x, f, x[:, 0], f[:, 0]]
        assert all(t.is_neg() for t in lazy)
        plain = [t.resolve_neg().contiguous() for t in lazy]
        for a, b in zip(fr.gated_recurrence(*lazy[:3]), fr.gated_recurrence(*plain[:3])):
            assert torch.equal(a, b)
        for a, b in zip(fr.gated_recurrence_step(lazy[2], lazy[3], torch._neg_view(plain[3])),
                        fr.gated_recurrence_step(plain[2], plain[3], -plain[3])):
            assert torch.equal(a, b)
        leaves = [t.clone().requires_grad_(True) for t in plain[:2]]
        out = fr.gated_recurrence(*leaves)
        d = [torch._neg_view(t.detach().clone()) for t in out]
        for a, b in zip(torch.autograd.grad(out, leaves, d, retain_graph=True),
                        torch.autograd.grad(out, leaves, [t.resolve_neg() for t in d])):
            assert torch.equal(a, b)
        for a, b in zip(fr.beam_select(x, torch._neg_view(plain[1][..., 0].contiguous()), 4),
                        fr.beam_select(plain[0], -plain[1][..., 0], 4)):
            assert torch.equal(a, b)


def test_rows_that_differ_by_a_constant_rescale_alike():
    """Logits whose distance is within a rounding of where a thread's sum of exponentials is rescaled:
    whether it is may not hang on where the row lies."""
    import fast_rnnt_b200 as fr
    u = 2.0 ** -20
    V = 4 * (1 + 128 * 4 + 2)
    g = torch.Generator().manual_seed(13)
    # multiples of 2^-20 that a shift by 8 leaves exact
    base = (torch.randn(V, generator=g, dtype=torch.float64).clamp(-4, 0.5) / u).round() * u - 1
    rows = []
    for low, high in ((1.5, 2), (0.5, 1), (2.5, 3), (1.5, 1), (3.5, 3)):
        row = base.clone()
        for thread in range(0, 128, 3):
            row[4 + 4 * thread] = low * u                     # first vector of the thread
            row[4 + 4 * (thread + 128 * 2)] = 10 + high * u   # a later one, in the same thread's share
        rows.append(row)
    for row in rows:
        for order in ((0.0, -8.0), (-8.0, 0.0)):
            logits = torch.stack([row + s for s in order]).float()
            assert torch.equal(logits.double(), torch.stack([row + s for s in order]))
            _, parents, tokens = fr.beam_select(logits[None].cuda(), torch.zeros(1, 2, device="cuda"), 6)
            assert not parents.any(), parents
            assert torch.equal(tokens[0].cpu(), torch.sort(logits[0], descending=True, stable=True).indices[:6])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_scores_and_logits_at_the_ends_of_the_range(dtype):
    """A score less its row's largest logit may leave 32 bits; the continuation's own score does not."""
    for top, low in ((1e38, -1e38), (-2e38, -3e38), (1e38, 0.0)):
        logits = torch.full((1, 3, 500), low, dtype=torch.float64)
        for i in range(3):
            logits[0, i, [7 * i + 3, 100 + i]] = top
        logits = logits.to("cuda", TYPES[dtype])
        for scores in ([-3e38, -2.9e38, -math.inf], [-3.4e38, -3.4e38, -3.3e38], [0.0, -1e38, -2e38]):
            scores = torch.tensor([scores], device="cuda")
            verify(logits, scores, 2 * int((scores > -INF).sum()))
