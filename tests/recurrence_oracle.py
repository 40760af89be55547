"""The gated recurrence and its gradients from the formula, step by step in 64 bits on the CPU,
with a bound on what arithmetic of unit roundoff u may be off by.

The bound follows the recurrence: every step multiplies by keep and take, which carry a few
roundings (the exponential 2 units in the last place, a sum, a division, a product: 16 u with
room for another order of the same products), and the sums have no larger terms than those of
the same recurrence on absolute values."""
import torch


def bounds_of(dtype):
    """(unit roundoff of the arithmetic, half a step of the output type, its smallest step / 2)"""
    u = 2.0 ** -53 if dtype == torch.float64 else 2.0 ** -24
    info = torch.finfo(dtype)
    half = 0.0 if dtype in (torch.float32, torch.float64) else info.eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else info.tiny
    return u, half, tiny


def recurrence(x, gate, initial=None, lengths=None, dh=None, dlast=None):
    """dict name -> (value, bound) of h, last and, where dh or dlast is given, dx, dgate, dinitial"""
    dtype = x.dtype
    u, half, tiny = bounds_of(dtype)
    c = 16 * u * (2 if dtype == torch.float64 else 1)   # the oracle's own arithmetic is no finer
    x, gate = x.detach().cpu().double(), gate.detach().cpu().double()
    B, T, D = x.shape
    zero = torch.zeros(B, D, dtype=torch.float64)
    n = torch.full((B,), T) if lengths is None else lengths.cpu().clamp(0, T)
    f, i = torch.sigmoid(gate), torch.sigmoid(-gate)
    state = zero if initial is None else initial.detach().cpu().double()
    mag, err = state.abs(), zero
    H, E, M = [], [], [mag]
    before, before_err = [], []
    for t in range(T):
        live = (n > t)[:, None]
        before.append(state)
        before_err.append(err)
        xt = torch.where(live, x[:, t], 0.0)
        ft, it = torch.where(live, f[:, t], 1.0), torch.where(live, i[:, t], 0.0)
        # a gate of +-inf: 0 * inf does not occur with finite values and states
        new_err = ft * (err + c * mag) + c * it * xt.abs()
        state = torch.where(live, ft * state + it * xt, state)
        mag = torch.where(live, ft * mag + it * xt.abs(), mag)
        err = torch.where(live, new_err, err)
        H.append(torch.where(live, state, 0.0))
        E.append(torch.where(live, err, 0.0))
    out = {"last": (state, err + tiny)}
    if T:
        h = torch.stack(H, 1)
        out["h"] = (h, torch.stack(E, 1) * (1 + half) + half * h.abs() + tiny)
    else:
        out["h"] = (torch.zeros(B, 0, D, dtype=torch.float64),) * 2
    if dh is None and dlast is None:
        return out
    dh = torch.zeros(B, T, D, dtype=torch.float64) if dh is None else dh.detach().cpu().double()
    flow = zero if dlast is None else dlast.detach().cpu().double()
    flow_mag, flow_err = flow.abs(), zero
    DX, DG = [None] * T, [None] * T
    for t in reversed(range(T)):
        live = (n > t)[:, None]
        d = torch.where(live, dh[:, t], 0.0)
        xt = torch.where(live, x[:, t], 0.0)
        ft, it = torch.where(live, f[:, t], 1.0), torch.where(live, i[:, t], 0.0)
        lam, lam_mag = flow + d, flow_mag + d.abs()
        lam_err = flow_err + c * lam_mag
        diff, size = before[t] - xt, before[t].abs() + xt.abs()
        dx = (torch.where(live, it * lam, 0.0), it * (lam_err + c * lam_mag))
        dg = (torch.where(live, lam * diff * ft * it, 0.0),
              ft * it * (lam_err * size + lam_mag * before_err[t] + 2 * c * lam_mag * size))
        DX[t], DG[t] = dx, dg
        flow = torch.where(live, ft * lam, flow)
        flow_err = torch.where(live, ft * (lam_err + c * lam_mag), flow_err)
        flow_mag = torch.where(live, ft * lam_mag, flow_mag)
    for name, got in (("dx", DX), ("dgate", DG)):
        if T:
            v, e = torch.stack([g[0] for g in got], 1), torch.stack([g[1] for g in got], 1)
            out[name] = (v, e * (1 + half) + half * v.abs() + tiny)
        else:
            out[name] = (torch.zeros(B, 0, D, dtype=torch.float64),) * 2
    out["dinitial"] = (flow, flow_err + tiny)
    return out


def check(got, want, what):
    value, bound = want
    got = got.detach().cpu().double()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    assert torch.isfinite(got).all(), what
    off = (got - value).abs()
    bad = off > bound
    if bad.any():
        at = tuple(int(k) for k in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {at}: "
                             f"{float(got[at])} for {float(value[at])}, bound {float(bound[at])}")
