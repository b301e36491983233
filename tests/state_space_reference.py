"""The state space operators in float64, step by step from their formulas, with error bounds.

Every function returns (results, majorant): the majorant of a result is the same formula with the
absolute value of each term, so K roundings of 2^-24 along a path of the computation put the float32
result off by at most K 2^-24 majorant (to first order).  `roundings` counts K; `check` adds the one
rounding to the output's type, half a step: finfo.eps / 2 relative.
"""
import torch

U = 2.0 ** -24


def double(t):
    return None if t is None else t.detach().double().cpu()


def silu(v):
    return v * torch.sigmoid(v)


def slope(v):
    s = torch.sigmoid(v)
    return s * (1 + v * (1 - s))


def check(got, want, majorant, K, name):
    """|got - want| <= half a step of got's type + K 2^-24 majorant, element by element."""
    assert tuple(got.shape) == tuple(want.shape), (name, got.shape, want.shape)
    info = torch.finfo(got.dtype)
    step = info.eps / 2 if got.dtype != torch.float32 else 0.0  # float32's own rounding is one of K
    bound = step * want.abs() + (K * U) * majorant * (1 + step) + info.tiny
    off = (got.detach().double().cpu() - want).abs()
    bad = ~(off <= bound)
    if bad.any():
        i = int((off / bound).nan_to_num(nan=float("inf")).argmax())
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} off; at {i}: got {got.flatten()[i].item()}, "
                             f"want {want.flatten()[i].item()}, bound {bound.flatten()[i].item():.3g}")


# An exponential is off by 2^-22 = 4 roundings and by one for each unit of its argument; with the
# reciprocal and the products a SiLU or its slope has 16 roundings and 2 |v| more.  The majorant of
# silu(v) and of its slope (which is below 1.1) is taken with that factor.
def _act_major(v):
    return v.abs() * (1 + v.abs() / 8), 1.1 * (1 + v.abs() / 8)


def conv(x, weight, bias, state, lengths, use_silu, dy=None, dfinal=None):
    """(results, majorants, K): y, final, and with dy: dx, dweight, dbias, dstate."""
    T, N, D = x.shape
    W = weight.shape[1]
    x, weight, bias, state, dy, dfinal = map(double, (x, weight, bias, state, dy, dfinal))
    lens = [T] * N if lengths is None else [min(max(int(v), 0), T) for v in lengths]
    K = 4 * W + 24 + T + N  # products and sums of p, SiLU, and the sums over steps and rows one after the other
    out, major = {}, {}
    y, ym = torch.zeros(T, N, D, dtype=torch.float64), torch.zeros(T, N, D, dtype=torch.float64)
    final = torch.zeros(N, W - 1, D, dtype=torch.float64)
    grads = {"dx": torch.zeros_like(y), "dweight": torch.zeros(D, W, dtype=torch.float64),
             "dbias": torch.zeros(D, dtype=torch.float64), "dstate": torch.zeros_like(final)}
    gmajor = {k: torch.zeros_like(v) for k, v in grads.items()}
    for n in range(N):
        past = state[n] if state is not None else torch.zeros(W - 1, D, dtype=torch.float64)
        rows = torch.cat([past, x[:lens[n], n]])  # row r is step r - (W-1)
        final[n] = rows[lens[n]:]
        drows, dmajor = torch.zeros_like(rows), torch.zeros_like(rows)
        if dfinal is not None:
            drows[lens[n]:] += dfinal[n]
            dmajor[lens[n]:] += dfinal[n].abs()
        for t in range(lens[n]):
            window = rows[t:t + W]
            p, pm = (window * weight.t()).sum(0), (window * weight.t()).abs().sum(0)
            if bias is not None:
                p, pm = p + bias, pm + bias.abs()
            # an error e of p moves silu by at most 1.1 e and its slope by at most e / 2
            y[t, n] = silu(p) if use_silu else p
            ym[t, n] = _act_major(p)[0] + 1.1 * pm if use_silu else pm
            if dy is None:
                continue
            g = dy[t, n] * (slope(p) if use_silu else 1.0)
            gm = dy[t, n].abs() * (_act_major(p)[1] + pm / 2 if use_silu else 1.0)
            drows[t:t + W] += g * weight.t()
            dmajor[t:t + W] += gm * weight.t().abs()
            grads["dweight"] += (g * window).t()
            gmajor["dweight"] += (gm * window.abs()).t()
            grads["dbias"] += g
            gmajor["dbias"] += gm
        grads["dstate"][n], gmajor["dstate"][n] = drows[:W - 1], dmajor[:W - 1]
        grads["dx"][:lens[n], n], gmajor["dx"][:lens[n], n] = drows[W - 1:], dmajor[W - 1:]
    out, major = {"y": y, "final": final}, {"y": ym, "final": torch.zeros_like(final)}
    if dy is not None:
        out, major = out | grads, major | gmajor
    return out, major, K


def scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, state=None, lengths=None, softplus=True, dy=None, dfinal=None):
    """(results, majorants, K): y, final, and with dy: dx, ddt, dA, dB, dC, dD, dz, ddt_bias, dstate."""
    T, N, Dn = x.shape
    S, G = A.shape[1], B.shape[2]
    x, dt, A, B, C, D, z, dt_bias, state, dy, dfinal = map(double, (x, dt, A, B, C, D, z, dt_bias, state, dy, dfinal))
    live = torch.ones(T, N, 1, dtype=torch.float64)
    if lengths is not None:
        live = (torch.arange(T)[:, None] < torch.as_tensor(lengths).cpu()[None])[..., None].double()
    dead = live.expand(T, N, Dn) == 0
    x, dt = x.masked_fill(dead, 0.0), dt.masked_fill(dead, 0.0)
    over = live[..., None].expand(T, N, G, S) == 0
    wide = lambda m: m.masked_fill(over, 0.0).repeat_interleave(Dn // G, 2)  # noqa: E731  [T,N,D,S]
    Bw, Cw = wide(B), wide(C)
    raw = dt if dt_bias is None else dt + dt_bias
    delta = (torch.logaddexp(raw, torch.zeros(())) if softplus else raw) * live
    a = torch.exp(delta[..., None] * A)
    skip = torch.zeros(Dn, dtype=torch.float64) if D is None else D
    h0 = torch.zeros(N, Dn, S, dtype=torch.float64) if state is None else state
    # A decay has the error of its exponential and of its argument: 4 + 4 |delta A| roundings, at most
    # as many as 4 + 4 max|delta A|, and a state has met at most T of them, each with a product and a sum.
    # |delta A| only matters where the decay does not vanish: v exp(-v) <= 1/e, so 4 |v| counts 2.
    # delta itself: 8 (softplus).  Backward, a second such chain; then the sums over S, T, N and D.
    K = 16 * T + 2 * S + T + N + Dn + 64
    hs, hm = [h0], [h0.abs()]
    for t in range(T):
        b = (delta[t] * x[t])[..., None] * Bw[t]
        hs.append(a[t] * hs[-1] + b)
        hm.append(a[t] * hm[-1] + b.abs())
    h, hmaj = torch.stack(hs), torch.stack(hm)
    y = (h[1:] * Cw).sum(-1) + skip * x
    ym = (hmaj[1:] * Cw.abs()).sum(-1) + (skip * x).abs()
    out, major = {"final": h[-1].clone()}, {"final": hmaj[-1].clone()}
    if z is None:
        out["y"], major["y"] = y * live, ym * live
    else:
        z = z.masked_fill(dead, 0.0)
        gate, act = silu(z), _act_major(z)
        out["y"], major["y"] = y * gate * live, ym * act[0] * live
    if dy is None:
        return out, major, K
    dy = dy.masked_fill(dead, 0.0)
    gm = dy.abs()
    if z is not None:
        out["dz"], major["dz"] = dy * y * slope(z), dy.abs() * ym * act[1]
        dy, gm = dy * gate, dy.abs() * act[0]
    lam = torch.zeros(N, Dn, S, dtype=torch.float64) if dfinal is None else dfinal
    lm = lam.abs()
    sums = {k: torch.zeros_like(v) for k, v in (("dA", A), ("dB", B), ("dC", C), ("dx", x), ("ddt", x))}
    smajor = {k: torch.zeros_like(v) for k, v in sums.items()}
    group = lambda m: m.reshape(N, G, Dn // G, S).sum(2)  # noqa: E731
    for t in range(T - 1, -1, -1):
        lam, lm = lam + dy[t][..., None] * Cw[t], lm + gm[t][..., None] * Cw[t].abs()
        sums["dC"][t], smajor["dC"][t] = group(dy[t][..., None] * h[t + 1]), group(gm[t][..., None] * hmaj[t + 1])
        dx = (delta[t] * x[t])[..., None]
        sums["dB"][t], smajor["dB"][t] = group(lam * dx), group(lm * dx.abs())
        lb, lbm = (lam * Bw[t]).sum(-1), (lm * Bw[t].abs()).sum(-1)
        lam, lm = lam * a[t], lm * a[t]  # what the step before takes
        u, um = lam * h[t], lm * hmaj[t]
        sums["dA"] += (u * delta[t][..., None]).sum(0)
        smajor["dA"] += (um * delta[t].abs()[..., None]).sum(0)
        sums["dx"][t] = delta[t] * lb + skip * dy[t]
        smajor["dx"][t] = delta[t].abs() * lbm + skip.abs() * gm[t]
        dd = ((lb * x[t]) + (u * A).sum(-1)) * live[t]
        ddm = ((lbm * x[t].abs()) + (um * A.abs()).sum(-1)) * live[t]
        s = torch.sigmoid(raw[t]) if softplus else 1.0
        sums["ddt"][t], smajor["ddt"][t] = dd * s, ddm * s * (1 + raw[t].abs() / 8)
    out |= sums | {"dstate": lam, "ddt_bias": sums["ddt"].sum((0, 1)), "dD": (dy * x).sum((0, 1))}
    major |= smajor | {"dstate": lm, "ddt_bias": smajor["ddt"].sum((0, 1)), "dD": (gm * x.abs()).sum((0, 1))}
    return out, major, K


def norm(x, weight, bias=None, gate=None, residual=None, scale=None, eps=1e-5, kind="rms", dy=None, dr=None):
    """(results, majorants, K): y, r, and with dy: dx, dweight, dbias, dgate, dresidual, dscale."""
    H, rows = x.shape[-1], x.shape[0] * x.shape[1]
    x, weight, bias, gate, residual, scale, dy, dr = map(double, (x, weight, bias, gate, residual, scale, dy, dr))
    g, gm = (1.0, 1.0) if gate is None else (silu(gate), _act_major(gate)[0])
    u, um = x * g, x.abs() * gm
    r, rm = (u, um) if scale is None else (scale * u, scale.abs() * um)
    if residual is not None:
        r, rm = residual + r, residual.abs() + rm
    layer = kind == "layer"
    mean = r.mean(-1, keepdim=True) if layer else 0.0
    c = r - mean
    inv = (c.square().mean(-1, keepdim=True) + eps) ** -0.5
    n = c * inv
    # Errors e of the row's values (e = K u major) move n by at most inv (e + mean e) + |n| inv max e:
    # inv changes by inv^2 mean(|n| e) <= inv^2 max e.
    cm = rm + (rm.mean(-1, keepdim=True) if layer else 0.0)
    nm = (cm + n.abs() * cm.amax(-1, keepdim=True)) * inv
    y, ym = n * weight, nm * weight.abs()
    if bias is not None:
        y, ym = y + bias, ym + bias.abs()
    # a thread adds at most 16 values, a warp 32 lanes, a block 16 warps; the sums over rows: one after the other
    K = 96 + rows
    out, major = {"y": y, "r": r}, {"y": ym, "r": rm}
    if dy is None:
        return out, major, K
    dn = dy * weight
    over, overm = (dn * n).mean(-1, keepdim=True), (dn.abs() * (n.abs() + nm)).mean(-1, keepdim=True)
    d, dm = dn - n * over, dn.abs() + (n.abs() + nm) * overm
    if layer:
        d, dm = d - dn.mean(-1, keepdim=True), dm + dn.abs().mean(-1, keepdim=True)
    # the relative error of inv: inv max e
    d, dm = d * inv, dm * inv * (1 + inv * cm.amax(-1, keepdim=True))
    out["dweight"], major["dweight"] = (dy * n).sum((0, 1)), (dy.abs() * (n.abs() + nm)).sum((0, 1))
    out["dbias"], major["dbias"] = dy.sum((0, 1)), dy.abs().sum((0, 1))
    if dr is not None:
        d, dm = d + dr, dm + dr.abs()
    out["dresidual"], major["dresidual"] = d, dm
    out["dscale"], major["dscale"] = (d * u).sum((0, 1)), (dm * um).sum((0, 1))
    if scale is not None:
        d, dm = d * scale, dm * scale.abs()
    if gate is not None:
        out["dgate"], major["dgate"] = d * x * slope(gate), dm * x.abs() * _act_major(gate)[1]
    out["dx"], major["dx"] = d * g, dm * gm
    return out, major, K
