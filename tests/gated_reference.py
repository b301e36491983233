"""The gated linear recurrence in float64, step by step from its formulas, with the error that float32
arithmetic may leave in each result.

U is one rounding, 2^-24.  Every result comes with a bound: a running first-order analysis in which an
exponential is off by 4 U and by one U for each unit of its argument, a reciprocal or square root by 2 U, a
product or sum by one.  A step's decay lies next to one, so 1 - a is followed by itself: where a = 1 - m, a is
off by m's error and its own rounding.  Sums that the kernel may associate in another order count each term's
absolute value.
"""
import torch

U = 2.0 ** -24


def double(t):
    return None if t is None else t.detach().double().cpu()


def check(got, want, bound, name):
    """|got - want| <= bound + half a step of got's type, element by element; non-finite values are equal."""
    assert tuple(got.shape) == tuple(want.shape), (name, got.shape, want.shape)
    info = torch.finfo(got.dtype)
    step = info.eps / 2 if got.dtype != torch.float32 else 0.0  # float32's own rounding is in the bound
    got = got.detach().double().cpu()
    allowed = (bound + step * (want.abs() + bound)) * 1.01 + info.tiny  # (second-order terms)
    if got.numel() and step:  # below the type's normal range a step is a fixed one
        allowed = allowed + info.tiny * info.eps
    bad = ~(((got - want).abs() <= allowed) | (got == want))
    if bad.any():
        i = int(((got - want).abs() / allowed).nan_to_num(nan=float("inf")).argmax())
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} off; at {i}: got {got.flatten()[i].item()}, "
                             f"want {want.flatten()[i].item()}, allowed {allowed.flatten()[i].item():.3g}")


def _gate(v):
    """sigmoid(v), sigmoid(-v), their product; relative errors of the first two (in U) and of the product."""
    r, rest = torch.sigmoid(v), torch.sigmoid(-v)
    k = 10 + torch.where(v.isinf(), 0.0, v.abs())  # (exp(-infinity) is exact)
    return r, rest, r * rest, k


def gated_scan(x, gate, decay=None, input_gate=None, state=None, lengths=None, dy=None, dfinal=None):
    """(results, bounds): y, final and, with dy, dx, dgate, ddecay, dinput_gate, dstate."""
    T, N, D = x.shape
    x, gate, decay, input_gate, state, dy, dfinal = map(double, (x, gate, decay, input_gate, state, dy, dfinal))
    lens = torch.full((N,), T) if lengths is None else lengths.cpu().clamp(0, T)
    live = (torch.arange(T)[:, None] < lens[None])[..., None].expand(T, N, D)
    x, gate = torch.where(live, x, 0.0), torch.where(live, gate, 0.0)
    r, rest, slope, kr = _gate(gate)
    if decay is not None:
        open_ = decay <= 0
        dec = torch.where(open_, decay, 0.0)
        l = dec * r
        a, m = torch.exp(l), -torch.expm1(l)
        slow_dm = (kr + 6) * U * m
        far_da = (6 + l.abs() * (kr + 3)) * U * a
        # which way the kernel takes changes at l = -0.35; both bounds next to it
        slow, far = l > -0.36, l < -0.34
        dm = torch.maximum(torch.where(slow, slow_dm, 0.0), torch.where(far, far_da + U * m, 0.0))
        da = torch.maximum(torch.where(slow, slow_dm + U * a, 0.0), torch.where(far, far_da, 0.0))
        w = torch.sqrt(m * (1 + a))
        ew = 0.5 * (torch.where(m > 0, dm / m, 0.0) + da / (1 + a) + 2 * U) + 4 * U
        over = torch.where(w > 0, 1 / w, 0.0)
        # Where r is below 2^-125 it may come out as zero or as that: w = sqrt(-2 decay r) to first order is off by the most
        # that it is there.
        lost = torch.where(r < 2.0 ** -124, torch.sqrt(-2 * dec * 2.0 ** -124), 0.0)
    else:
        lost = 0.0
        a, w = r, rest
        da = torch.where(gate > 0, kr * U * rest + U * a, kr * U * a)
        ew = kr * U
    if input_gate is not None:
        input_gate = torch.where(live, input_gate, 0.0)
        i, irest, islope, ki = _gate(input_gate)
    else:
        i, islope, ki = torch.ones_like(x), torch.zeros_like(x), torch.zeros_like(x)
    u, eu = x * i, (ki + 1) * U
    b = torch.where(live, w * u, 0.0)
    eb = ew + eu + U
    # a sigmoid below 2^-125 may come out as zero or as that: both factors of a step are off by as much
    lost = torch.where(live, lost * u.abs() + 2.0 ** -124 * x.abs(), 0.0)
    a, da = torch.where(live, a, 1.0), torch.where(live, da + 2.0 ** -125, 0.0)
    three = torch.where(live, 3 * U, 0.0)
    h = torch.zeros(N, D, dtype=torch.float64) if state is None else state
    E, H = torch.zeros_like(h), h.abs()
    hs, Es, Hs, ys, Ys = [], [], [], [], []
    for t in range(T):
        hs.append(h); Es.append(E); Hs.append(H)  # in front of step t
        E = a[t] * E + (da[t] + three[t] * a[t]) * H + (eb[t] + three[t]) * b[t].abs() + lost[t]
        H = a[t] * H + b[t].abs()
        h = a[t] * h + b[t]
        ys.append(h); Ys.append(E)
    out = {"y": torch.where(live, torch.stack(ys), 0.0) if T else x, "final": h}
    bound = {"y": torch.where(live, torch.stack(Ys), 0.0) if T else x, "final": E}
    if dy is None:
        return out, bound
    dy = torch.where(live, dy, 0.0)
    mu = torch.zeros(N, D, dtype=torch.float64) if dfinal is None else dfinal
    F, M = torch.zeros_like(mu), mu.abs()
    g = {k: torch.zeros_like(x) for k in ("dx", "dgate", "dinput_gate", "ddecay")}
    e = {k: torch.zeros_like(x) for k in g}
    size = torch.zeros_like(x)
    for t in reversed(range(T)):
        lam, L, F = dy[t] + mu, dy[t].abs() + M, F + 3 * U * (dy[t].abs() + M)
        g["dx"][t] = lam * w[t] * i[t]
        e["dx"][t] = F * w[t] * i[t] + L * w[t] * i[t] * (ew[t] + ki[t] * U + 3 * U)
        g["dinput_gate"][t] = lam * w[t] * x[t] * islope[t]
        scale = (w[t] * x[t] * islope[t]).abs()
        e["dinput_gate"][t] = F * scale + L * scale * (ew[t] + 2 * ki[t] * U + 4 * U)
        if decay is None:
            z, zs = hs[t] - u[t], Hs[t] + u[t].abs()
            ez = Es[t] + eu[t] * u[t].abs() + 3 * U * zs
            g["dgate"][t] = lam * z * slope[t]
            e["dgate"][t] = (F * zs + L * ez + L * zs * (2 * kr[t] + 4) * U) * slope[t]
        else:
            part = u[t].abs() * a[t] * over[t]
            z, zs = a[t] * (hs[t] - u[t] * a[t] * over[t]), a[t] * (Hs[t] + part)
            ez = da[t] * (Hs[t] + part) + a[t] * (Es[t] + part * (da[t] / a[t].clamp(min=1e-300) + ew[t] + eu[t] + 3 * U)) + 3 * U * zs
            dl, edl, ldl = lam * z, F * zs + L * ez + U * L * zs, L * zs
            g["dgate"][t] = dl * dec * slope[t]
            e["dgate"][t] = (edl + ldl * (2 * kr[t] + 4) * U) * dec.abs() * slope[t]
            g["ddecay"][t] = dl * r[t]
            e["ddecay"][t] = edl * r[t] + ldl * r[t] * (kr[t] + 1) * U
            size[t] = ldl * r[t]
        mu = torch.where(live[t], a[t] * lam, mu)
        F = torch.where(live[t], a[t] * F + (da[t] + 3 * U * a[t]) * L, F)
        M = torch.where(live[t], a[t] * L, M)
    for k in ("dx", "dgate", "dinput_gate"):
        out[k], bound[k] = torch.where(live, g[k], 0.0), torch.where(live, e[k], 0.0)
    if decay is not None:
        terms = T * N + 8
        out["ddecay"] = torch.where(open_, torch.where(live, g["ddecay"], 0.0).sum((0, 1)), 0.0)
        bound["ddecay"] = torch.where(live, e["ddecay"] + terms * U * size, 0.0).sum((0, 1))
    out["dstate"], bound["dstate"] = mu, F
    return out, bound
