"""The operators next to the losses, as measurable cases: the gated linear recurrence of a
prediction network or an encoder (a whole sequence with its gradients, and one token), and
beam search's selection and reordering of states.

A case is a dict of plain values; ``prepare`` makes its inputs on the GPU from a seed,
``run`` is one pass: the operators in their plain form where ``own`` is false, the calls of
the library where it is true.  ``exact`` is the same from the definition, in 64 bits.

Operators:

  scan      gated_recurrence: forward, with ``train`` its backward pass too
  step      gated_recurrence_step: one token of every beam, state read through the parents
  select    beam_select: log-softmax of every beam's logits and the best continuations
  reorder   beam_reorder: states and histories of the beams that survive
"""
import math
import random

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # the prediction network on two short utterances: latency of a training step
        dict(name="scan tiny", op="scan", B=2, T=14, D=128, dtype="f32", train=True, ragged=False,
             views=False, initial=False),
        # the prediction network of the benchmark's batch: 64 utterances of up to 100 symbols
        dict(name="scan prediction network", op="scan", B=64, T=101, D=512, dtype="bf16", train=True,
             ragged=True, views=True, initial=False),
        # an encoder layer over long utterances, both halves of one projection as inputs
        dict(name="scan encoder", op="scan", B=16, T=2000, D=1024, dtype="bf16", train=True,
             ragged=True, views=True, initial=True),
        # odd sizes in 32 bits: no row starts on a 16-byte boundary
        dict(name="scan odd", op="scan", B=6, T=2211, D=423, dtype="f32", train=True, ragged=True,
             views=False, initial=True),
        # one long recording, evaluated in one go from a carried state
        dict(name="scan recording", op="scan", B=1, T=30011, D=512, dtype="f16", train=False,
             ragged=False, views=False, initial=True),
        # one stream's beams between two frames: latency of decoding
        dict(name="step stream", op="step", B=1, K=4, D=512, dtype="f32", parents=True),
        # many streams with a state each of eight beams
        dict(name="step batch", op="step", B=512, K=8, D=1024, dtype="bf16", parents=True),
        # one stream, 500 symbols: latency of decoding
        dict(name="select stream", op="select", B=1, K=4, V=500, beam=4, dtype="f32", finished=False),
        # the validation set's batch, 5000 symbols
        dict(name="select batch", op="select", B=64, K=8, V=5000, beam=8, dtype="bf16", finished=True),
        # wide beams over a large vocabulary of no round size
        dict(name="select wide", op="select", B=96, K=16, V=31999, beam=16, dtype="f16", finished=True),
        # one stream's states and its symbols so far
        dict(name="reorder stream", op="reorder", B=1, K=4, layers=2, D=512, L=64, dtype="f32"),
        # many streams, a deep network's states and long histories
        dict(name="reorder batch", op="reorder", B=256, K=8, layers=12, D=1024, L=500, dtype="f32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges above; batches shrink until a case costs no more than the
    largest listed one of its operator."""
    op = rng.choice(["scan", "scan", "scan", "step", "select", "select", "reorder"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "scan":
        train = rng.random() < 0.7
        D = rng.choice([8 * _log_int(rng, 4, 192), _log_int(rng, 20, 1500)])
        c = dict(op=op, B=_log_int(rng, 1, 64), T=_log_int(rng, 1, 30000), D=D, dtype=dtype,
                 train=train, ragged=rng.random() < 0.6, views=rng.random() < 0.5,
                 initial=rng.random() < 0.5)
    elif op == "step":
        c = dict(op=op, B=_log_int(rng, 1, 512), K=rng.randint(1, 16), D=_log_int(rng, 20, 1500),
                 dtype=dtype, parents=rng.random() < 0.7)
    elif op == "select":
        beam = rng.randint(1, 16)
        c = dict(op=op, B=_log_int(rng, 1, 96), K=rng.choice([1, beam, beam, beam]),
                 V=_log_int(rng, 28, 50000), beam=beam, dtype=dtype, finished=rng.random() < 0.5)
    else:
        c = dict(op=op, B=_log_int(rng, 1, 256), K=rng.randint(1, 16), layers=rng.randint(1, 16),
                 D=_log_int(rng, 20, 1500), L=_log_int(rng, 8, 500), dtype=dtype)
    top = [work(x) for x in listed() if x["op"] == op]
    most = {k: max(w[k] for w in top) for k in ("bytes", "flops")}
    while c["B"] > 1 and any(work(c)[k] > most[k] for k in most):
        c["B"] -= max(1, c["B"] // 8)
    while any(work(c)[k] > most[k] for k in most):
        long = "T" if op == "scan" else "V" if op == "select" else "D"
        c[long] -= max(1, c[long] // 8)
    return c


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    r = random.Random(seed)
    dt = _DTYPES[case["dtype"]]
    B = case["B"]

    def normal(*shape, mean=0.0, scale=1.0, dtype=dt):
        return torch.randn(*shape, generator=g, device=dev).mul_(scale).add_(mean).to(dtype)

    def parents_of(K):
        p = torch.randint(0, K, (B, K), generator=g, device=dev)
        if K > 1:  # the search ran out of hypotheses here and there
            p.masked_fill_(torch.rand(B, K, generator=g, device=dev) < 0.05, -1)
        return p

    st = dict(case=case)
    if case["op"] == "scan":
        T, D = case["T"], case["D"]
        if case["views"]:   # one projection gives the values and the gates
            both = torch.cat([normal(B, T, D), normal(B, T, D, mean=2.0, scale=1.5)], dim=-1)
            x, gate = both.chunk(2, dim=-1)
        else:
            x, gate = normal(B, T, D), normal(B, T, D, mean=2.0, scale=1.5)
        st["x"], st["gate"] = x, gate
        st["initial"] = normal(B, D, dtype=torch.float32) if case["initial"] else None
        st["lengths"] = None
        if case["ragged"]:
            rows = [T] + [r.randint((T + 1) // 2, T) for _ in range(B - 1)]
            st["lengths"] = torch.tensor(rows, dtype=torch.int64).to(dev)
        if case["train"]:
            st["dh"], st["dlast"] = normal(B, T, D), normal(B, D, dtype=torch.float32)
            st["leaves"] = [t.requires_grad_(True) for t in (x, gate, st["initial"]) if t is not None]
    elif case["op"] == "step":
        K, D = case["K"], case["D"]
        st["x"], st["gate"] = normal(B, K, D), normal(B, K, D, mean=2.0, scale=1.5)
        st["state"] = normal(B, K, D, dtype=torch.float32)
        st["parents"] = parents_of(K) if case["parents"] else None
    elif case["op"] == "select":
        K, V = case["K"], case["V"]
        st["logits"] = normal(B, K, V, scale=3.0)
        st["scores"] = torch.rand(B, K, generator=g, device=dev).mul_(-8.0)
        if K > 1:           # fewer hypotheses than beams here and there, never none
            dead = torch.rand(B, K, generator=g, device=dev) < 0.1
            dead[:, 0] = False
            st["scores"].masked_fill_(dead, -math.inf)
        st["finished"] = None
        if case["finished"]:  # some hypotheses are complete
            st["finished"] = torch.rand(B, K, generator=g, device=dev) < 0.1
    else:
        K, D = case["K"], case["D"]
        st["states"] = [normal(B, K, D) for _ in range(case["layers"])]
        st["states"].append(torch.randint(0, 500, (B, K, case["L"]), generator=g, device=dev))
        st["parents"] = parents_of(K)
    return st


# ------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------
def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1, by doubling: every pass joins each element with the
    one `step` before it, so that the number of passes is the logarithm of the length."""
    step = 1
    while step < b.shape[1]:
        b = torch.cat([b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]], dim=1)
        a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], dim=1)
        step *= 2
    return b


def _sigmoids(gate):
    """sigmoid(gate) and 1 - sigmoid(gate), the latter without cancellation"""
    return 1.0 / (1.0 + torch.exp(-gate)), 1.0 / (1.0 + torch.exp(gate))


def _plain_scan(st):
    x, gate, initial, lengths = st["x"].detach(), st["gate"].detach(), st["initial"], st["lengths"]
    B, T, D = x.shape
    valid = torch.ones(B, T, 1, dtype=torch.bool, device=x.device)
    if lengths is not None:
        valid = (torch.arange(T, device=x.device) < lengths[:, None])[:, :, None]
    keep, take = _sigmoids(gate.float())
    keep, take = torch.where(valid, keep, 1.0), torch.where(valid, take, 0.0)
    x32 = x.float()
    h0 = torch.zeros(B, D, device=x.device) if initial is None else initial.detach()
    b = take * x32
    b[:, 0] += keep[:, 0] * h0
    h = _scan(keep, b)
    out = dict(h=torch.where(valid, h, 0.0).to(x.dtype), last=h[:, -1].clone())
    if "dh" not in st:
        return out
    dh = torch.where(valid, st["dh"].float(), 0.0)
    dh[:, -1] += st["dlast"]
    # the gradient of h_t also comes through keep_{t+1}: the same recurrence from the other end
    after = torch.cat([keep[:, 1:], torch.ones_like(keep[:, :1])], dim=1)
    lam = _scan(after.flip(1), dh.flip(1)).flip(1)
    before = torch.cat([h0[:, None], h[:, :-1]], dim=1)
    out["dx"] = (lam * take).to(x.dtype)
    out["dgate"] = (lam * (before - x32) * keep * take).to(x.dtype)
    if initial is not None:
        out["dinitial"] = keep[:, 0] * lam[:, 0]
    return out


def _gathered(t, parents):
    rows = torch.arange(t.shape[0], device=t.device)[:, None]
    picked = t[rows, parents.clamp(min=0)]
    return torch.where((parents >= 0).reshape(parents.shape + (1,) * (t.ndim - 2)), picked,
                       torch.zeros_like(picked))


def _plain_step(st):
    state = st["state"] if st["parents"] is None else _gathered(st["state"], st["parents"])
    keep, take = _sigmoids(st["gate"].float())
    new = keep * state + take * st["x"].float()
    return dict(h=new.to(st["x"].dtype), state=new)


def _plain_select(st):
    # 64 bits: the order of two continuations may hang on their last digits
    x, scores, beam = st["logits"].double(), st["scores"].double(), st["case"]["beam"]
    B, K, V = x.shape
    top = x.amax(dim=-1, keepdim=True)
    logp = (x - top) - torch.log(torch.exp(x - top).sum(dim=-1, keepdim=True))
    if st["finished"] is not None:
        only = torch.full((V,), -math.inf, dtype=torch.float64, device=x.device)
        only[0] = 0.0
        logp = torch.where(st["finished"][:, :, None], only, logp)
    key = (scores[:, :, None] + logp).reshape(B, K * V)
    key = torch.where(torch.isnan(key), -math.inf, key)
    best, at = torch.sort(key, dim=1, descending=True, stable=True)
    best, at = best[:, :beam], at[:, :beam]
    none = best == -math.inf
    return dict(scores=best.float(), parents=torch.where(none, -1, at // V),
                tokens=torch.where(none, -1, at % V))


def run(state):
    st, op = state, state["case"]["op"]
    if not own:
        if op == "scan":
            return _plain_scan(st)
        if op == "step":
            return _plain_step(st)
        if op == "select":
            return _plain_select(st)
        return [_gathered(t, st["parents"]) for t in st["states"]]
    import fast_rnnt_b200 as fr
    if op == "scan":
        h, last = fr.gated_recurrence(st["x"], st["gate"], st["initial"], st["lengths"])
        if "dh" not in st:
            return dict(h=h, last=last)
        grads = torch.autograd.grad([h, last], st["leaves"], [st["dh"], st["dlast"]])
        return dict(zip(("h", "last", "dx", "dgate", "dinitial"), (h.detach(), last.detach()) + grads))
    if op == "step":
        h, new = fr.gated_recurrence_step(st["x"], st["gate"], st["state"], st["parents"])
        return dict(h=h, state=new)
    if op == "select":
        scores, parents, tokens = fr.beam_select(st["logits"], st["scores"], st["case"]["beam"],
                                                 finished=st["finished"])
        return dict(scores=scores, parents=parents, tokens=tokens)
    return list(fr.beam_reorder(st["states"], st["parents"]))


def work(case):
    """Every input read once, every output written once; the operations of the formulas, an
    exponential counted as one."""
    B = case["B"]
    if case["op"] == "scan":
        n, es = B * case["T"] * case["D"], _SIZE[case["dtype"]]
        states = 4 * B * case["D"] * (1 + int(case["initial"]))
        if case["train"]:       # x, gate, dh and h, dx, dgate
            return {"bytes": 6 * n * es + 2 * states, "flops": 24 * n}
        return {"bytes": 3 * n * es + states, "flops": 9 * n}
    if case["op"] == "step":
        n = B * case["K"] * case["D"]
        return {"bytes": n * (3 * _SIZE[case["dtype"]] + 8) + 8 * B * case["K"] * int(case["parents"]),
                "flops": 9 * n}
    if case["op"] == "select":
        n = B * case["K"] * case["V"]
        return {"bytes": n * _SIZE[case["dtype"]] + B * (5 * case["K"] + 20 * case["beam"]), "flops": 4 * n}
    row = case["layers"] * case["D"] * _SIZE[case["dtype"]] + 8 * case["L"]
    return {"bytes": B * case["K"] * (2 * row + 8), "flops": 0}


# ------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "scan":
        B, T, D = st["x"].shape
        x, gate = (st[k].detach().double().transpose(0, 1).contiguous() for k in ("x", "gate"))
        h = torch.zeros(B, D, dtype=torch.float64, device=x.device)
        if st["initial"] is not None:
            h = st["initial"].detach().double()
        leaves = [x, gate, h] if case["initial"] else [x, gate]
        if case["train"]:
            leaves = [t.requires_grad_(True) for t in leaves]
        seq = []
        for t, (value, f) in enumerate(zip(x.unbind(0), torch.sigmoid(gate).unbind(0))):
            new = torch.lerp(value, h, f)
            if st["lengths"] is not None:
                live = (st["lengths"] > t)[:, None]
                h = torch.where(live, new, h)
                seq.append(torch.where(live, new, 0.0))
            else:
                h = new
                seq.append(new)
        out = torch.stack(seq, dim=1)
        res = dict(h=out.detach(), last=h.detach())
        if case["train"]:
            grads = torch.autograd.grad([out, h], leaves, [st["dh"].double(), st["dlast"].double()])
            res["dx"], res["dgate"] = (d.transpose(0, 1).contiguous() for d in grads[:2])
            if case["initial"]:
                res["dinitial"] = grads[2]
        return res
    if case["op"] == "step":
        state, parents = st["state"].double(), st["parents"]
        if parents is not None:
            K = state.shape[1]
            pick = (parents[:, :, None] == torch.arange(K, device=state.device)).double()
            state = pick @ state
        new = torch.lerp(st["x"].double(), state, torch.sigmoid(st["gate"].double()))
        return dict(h=new, state=new)
    if case["op"] == "select":
        logp = torch.log_softmax(st["logits"].double(), dim=-1)
        if st["finished"] is not None:
            logp[st["finished"]] = -math.inf
            logp[..., 0].masked_fill_(st["finished"], 0.0)
        key = (logp + st["scores"].double()[:, :, None]).flatten(1)
        return dict(scores=torch.topk(key, case["beam"], dim=1).values, parents=None, tokens=None)
    K = case["K"]   # a row of zeros behind the last beam is what a slot without a parent gets
    at = torch.where(st["parents"] < 0, K, st["parents"])[:, :, None]
    wide = [torch.nn.functional.pad(t.double(), (0, 0, 0, 1)) for t in st["states"][:-1]]
    return [t.gather(1, at.expand(-1, -1, t.shape[2])) for t in wide] + [None]
