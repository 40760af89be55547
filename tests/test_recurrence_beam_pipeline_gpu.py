"""The recurrence, the losses and the beam search together, as a transducer's training and decoding
use them: recurrent encoder and prediction network into the losses with gradients for every
weight, and a frame by frame search whose states are reordered."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

B, T, S, C, D, F = 3, 37, 9, 48, 32, 20      # utterances, frames, symbols, vocabulary, channels, features


def network(seed):
    g = torch.Generator().manual_seed(seed)

    def w(*shape):
        return (torch.randn(*shape, generator=g) / math.sqrt(shape[-1])).cuda()

    p = dict(embed=w(C, D) * 4, enc=w(2 * D, F), dec=w(2 * D, D), am=w(C, D), lm=w(C, D), out=w(C, D), bias=w(C))
    for k in ("enc", "dec"):
        p[k][D:] += 0.1
    batch = dict(feats=torch.randn(B, T, F, generator=g).cuda(),
                 symbols=torch.randint(1, C, (B, S), generator=g).cuda(),
                 frames=torch.tensor([T, T - 6, T - 11]).cuda(), lengths=torch.tensor([S, S - 2, S - 4]).cuda())
    batch["boundary"] = torch.stack([torch.zeros(B).long().cuda(), torch.zeros(B).long().cuda(),
                                     batch["lengths"], batch["frames"]], 1)
    return p, batch


def plain_recurrence(x, gate, initial, lengths):
    """the formula, a step at a time"""
    state = x.new_zeros(x.shape[0], x.shape[2]) if initial is None else initial
    f, out = torch.sigmoid(gate), []
    for t in range(x.shape[1]):
        live = (t < lengths)[:, None] if lengths is not None else torch.ones_like(state[:, :1], dtype=torch.bool)
        state = torch.where(live, f[:, t] * state + (1 - f[:, t]) * x[:, t], state)
        out.append(torch.where(live, state, torch.zeros_like(state)))
    return torch.stack(out, 1), state


def losses(p, b, recurrence, pruned):
    import fast_rnnt_b200 as fr
    x, g = fr.linear(b["feats"], p["enc"]).chunk(2, -1)
    enc, _ = recurrence(x, g, None, b["frames"])
    history = torch.nn.functional.pad(b["symbols"], (1, 0))
    x, g = fr.linear(p["embed"][history], p["dec"]).chunk(2, -1)
    dec, _ = recurrence(x, g, None, b["lengths"] + 1)
    am, lm = fr.linear(enc, p["am"]), fr.linear(dec, p["lm"])
    loss, occupancies = fr.rnnt_loss_simple(lm, am, b["symbols"], 0, boundary=b["boundary"], reduction="sum",
                                            return_grad=True)
    if not pruned:
        return loss
    ranges = fr.get_rnnt_prune_ranges(*occupancies, b["boundary"], 4)
    return loss + fr.rnnt_loss_pruned_joiner(enc, dec, ranges, p["out"], p["bias"], b["symbols"], 0,
                                             boundary=b["boundary"], reduction="sum")


def test_training_step():
    """Loss and gradients with the operator and with the formula in its place.  The two differ by
    the roundings of at most 37 steps of either (16 units of 2^-24 a step, 1200 in all) and by what
    the rest of the step makes of them: bounded by 64 times as much of the largest gradient."""
    import fast_rnnt_b200 as fr
    p, b = network(1)
    out = []
    for recurrence in (fr.gated_recurrence, plain_recurrence):
        leaves = {k: v.clone().requires_grad_(True) for k, v in p.items()}
        loss = losses(leaves, b, recurrence, False)
        used = [k for k in leaves if k not in ("out", "bias")]
        out.append((loss, dict(zip(used, torch.autograd.grad(loss, [leaves[k] for k in used])))))
    (la, ga), (lb, gb) = out
    tol = 64 * 37 * 32 * 2.0 ** -24
    assert abs(la - lb) <= tol * abs(lb)
    for k in ga:
        assert (ga[k] - gb[k]).abs().max() <= tol * gb[k].abs().max(), k


def test_pruned_training_step_runs_and_is_captured():
    import fast_rnnt_b200 as fr
    from fast_rnnt_b200.graphs import GraphedStep
    p, b = network(2)
    fr.provide_boundary_rows(b["boundary"], b["boundary"].tolist())
    leaves = {k: v.clone().requires_grad_(True) for k, v in p.items()}
    eager = losses(leaves, b, fr.gated_recurrence, True)
    eager.backward()
    grads = {k: v.grad.clone() for k, v in leaves.items()}
    assert torch.isfinite(eager) and all(torch.isfinite(g).all() and g.abs().max() > 0 for g in grads.values())

    def step(t):
        loss = losses(t, b, fr.gated_recurrence, True)
        loss.backward()
        return loss

    for v in leaves.values():
        v.grad = None
    # an eager graph of the same leaves that is still alive
    alive = losses(leaves, b, fr.gated_recurrence, True)
    step_graph = GraphedStep(step, leaves)
    loss = step_graph()
    torch.cuda.synchronize()
    assert torch.equal(loss, eager.detach()) and torch.equal(alive, loss)
    for k in leaves:
        assert torch.equal(leaves[k].grad, grads[k]), k


def test_captured_leaf_with_two_names():
    import fast_rnnt_b200 as fr
    from fast_rnnt_b200.graphs import GraphedStep
    g = torch.Generator().manual_seed(5)
    x = torch.randn(2, 40, 24, generator=g).cuda().requires_grad_(True)

    def step(t):
        loss = fr.gated_recurrence(t["x"], t["gate"])[0].square().sum()
        loss.backward()
        return loss

    step(dict(x=x, gate=x))
    want, x.grad = x.grad, None
    graph = GraphedStep(step, dict(x=x, gate=x))
    graph()
    torch.cuda.synchronize()
    assert torch.equal(x.grad, want)


def test_search():
    """A search over the frames: at most one symbol a frame (blank 0 keeps the state), four
    hypotheses.  The formula in 64 bits follows the search's own choices; at every frame the kept
    scores are those of the best continuations to within the tolerance of their computation."""
    import fast_rnnt_b200 as fr
    K = 4
    p, b = network(3)
    d = {k: v.double().cpu() for k, v in p.items()}
    with torch.no_grad():
        x, g = fr.linear(b["feats"], p["enc"]).chunk(2, -1)
        enc, _ = fr.gated_recurrence(x, g, None, b["frames"])
        # states and joiner inputs of the hypotheses: a start symbol, then the symbols found
        start = fr.linear(p["embed"][torch.zeros(B, K, dtype=torch.long, device="cuda")], p["dec"])
        dec, state = fr.gated_recurrence_step(*start.chunk(2, -1), torch.zeros(B, K, D, device="cuda"))
        scores = torch.full((B, K), -math.inf, device="cuda")
        scores[:, 0] = 0
        history = torch.full((B, K, T), -1, dtype=torch.int64, device="cuda")
        every = torch.arange(K, device="cuda").expand(B, 1, K).contiguous()

        dstart = (d["embed"][torch.zeros(B, K, dtype=torch.long)] @ d["dec"].T).chunk(2, -1)
        want_state = torch.sigmoid(-dstart[1]) * dstart[0]
        want_scores = scores.double().cpu()
        denc, _ = plain_recurrence(*(b["feats"].double().cpu() @ d["enc"].T).chunk(2, -1), None, b["frames"].cpu())
        path = torch.zeros(B, K, 0, dtype=torch.long)
        # scores: sums of up to T log-probabilities whose logits (below 16 in size) carry the roundings
        # of the networks: up to 64 units of 2^-24 of 16 each
        tol = T * 64 * 16 * 2.0 ** -24
        for t in range(T):
            logits = fr.pruned_joiner(enc[:, t:t + 1], dec, every, p["out"], p["bias"])[:, 0]
            finished = (t >= b["frames"])[:, None].expand(B, K)
            scores, parents, tokens = fr.beam_select(logits, scores, K, finished=finished)
            state, dec, history = fr.beam_reorder([state, dec, history], parents)
            history[:, :, t] = tokens
            emitted = tokens > 0
            xs, gs = fr.linear(p["embed"][tokens.clamp(min=0)], p["dec"]).chunk(2, -1)
            new_dec, new_state = fr.gated_recurrence_step(xs, gs, state)
            state, dec = (torch.where(emitted[..., None], n, o) for n, o in ((new_state, state), (new_dec, dec)))

            # the same frame by the formula
            lg = torch.tanh(denc[:, t:t + 1] + want_state) @ d["out"].T + d["bias"]
            logp = torch.log_softmax(lg, -1)
            done = finished.cpu()
            logp[done] = -math.inf
            logp[..., 0] = torch.where(done, 0.0, logp[..., 0])
            key = (want_scores[..., None] + logp).flatten(1)
            par, tok = parents.cpu(), tokens.cpu()
            assert (par >= 0).all() or t == 0
            best = torch.sort(key, 1, descending=True).values[:, :K]
            chosen = key.gather(1, par.clamp(min=0) * C + tok.clamp(min=0))
            chosen = torch.where(par >= 0, chosen, -math.inf)
            fin = torch.isfinite(best)
            assert torch.equal(fin, par >= 0)
            assert ((chosen - best)[fin].abs() <= 2 * tol).all(), (t, (chosen - best)[fin].abs().max())
            assert ((scores.cpu().double() - chosen)[fin].abs() <= tol).all(), t
            want_scores = chosen
            rows = torch.arange(B)[:, None]
            prev = want_state[rows, par.clamp(min=0)]
            dx, dg = (d["embed"][tok.clamp(min=0)] @ d["dec"].T).chunk(2, -1)
            after = torch.sigmoid(dg) * prev + torch.sigmoid(-dg) * dx
            want_state = torch.where((tok > 0)[..., None], after, prev)
            path = torch.cat([path[rows, par.clamp(min=0)], tok[..., None]], -1)
    assert torch.equal(history.cpu(), path)
    assert (path[2, :, int(b["frames"][2]):] == 0).all()       # nothing after an utterance's end
    # the hypotheses of an utterance are different paths
    assert all(len({tuple(h.tolist()) for h in path[i]}) == K for i in range(B))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_search_whose_step_keeps_the_state_on_blank(dtype):
    """A gate of +inf where a hypothesis goes on with blank: its state and output, read through the
    parents, stay as they are, bit for bit as if they were reordered and selected."""
    import fast_rnnt_b200 as fr
    K = 4
    g = torch.Generator().manual_seed(7)
    embed, w = (torch.randn(*s, generator=g).cuda().to(dtype) for s in ((C, D), (2 * D, D)))
    out = torch.randn(C, D, generator=g).cuda()
    out[0] *= 4      # blank often enough
    with torch.no_grad():
        network = lambda tokens: (embed[tokens.clamp(min=0)] @ w.T).chunk(2, -1)   # noqa: E731
        zero = torch.zeros(B, K, D, device="cuda")
        dec, state = fr.gated_recurrence_step(*network(torch.zeros(B, K, dtype=torch.int64, device="cuda")), zero)
        ref_dec, ref_state = dec, state
        scores = torch.full((B, K), -math.inf, device="cuda")
        scores[:, 0] = 0
        seen = set()
        for t in range(12):
            frame = torch.randn(B, 1, D, generator=g).cuda()
            scores, parents, tokens = fr.beam_select(torch.tanh(frame + dec) @ out.T, scores, K)
            x, gate = network(tokens)
            emitted = (tokens > 0)[..., None]
            dec, state = fr.gated_recurrence_step(x, gate.masked_fill(~emitted, math.inf), state, parents)
            old_dec, old_state = fr.beam_reorder([ref_dec, ref_state], parents)
            new_dec, new_state = fr.gated_recurrence_step(x, gate, old_state)
            ref_dec, ref_state = (torch.where(emitted, n, o) for n, o in ((new_dec, old_dec), (new_state, old_state)))
            assert torch.equal(dec, ref_dec) and torch.equal(state, ref_state), t
            seen |= set((tokens > 0).flatten().tolist()) | ({None} if (parents < 0).any() else set())
        assert {True, False} <= seen
