"""Performance cases of the selective state space operators: the short causal convolution, the
selective scan and the norm around a block, each for whole sequences (forward, forward and
backward) and the first two for single tokens.

`run` computes a case's plain form in elementary torch operations, or, with `own`, calls
`haste_b200.ssm`.  All sequences are time-major [T,N,...]; `batch_first` cases hand over views of
[N,T,...] tensors.  Inner widths are twice the layers' hidden sizes, as a block with an expansion
of two has them.
"""
import math

import torch

own = False  # True: the framework's operators instead of the plain forms

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _conv(task, dtype, T, N, D, W, batch_first=False, lengths=False, state=False, **name):
    return dict(op="conv", task=task, dtype=dtype, T=T, N=N, D=D, W=W, batch_first=batch_first,
                lengths=lengths, state=state, **name)


def _scan(task, dtype, T, N, D, S, G=1, batch_first=False, lengths=False, state=False, gate=True, **name):
    return dict(op="scan", task=task, dtype=dtype, T=T, N=N, D=D, S=S, G=G, batch_first=batch_first,
                lengths=lengths, state=state, gate=gate, **name)


def _norm(task, dtype, T, N, H, kind, gate=False, residual=False, scale=False, bias=False, **name):
    return dict(op="norm", task=task, dtype=dtype, T=T, N=N, H=H, kind=kind, gate=gate,
                residual=residual, scale=scale, bias=bias, **name)


def listed():
    return [
        # One stream that answers token by token: nothing but latency.
        _conv("step", "bf16", 1, 1, 1024, 4, name="conv-step-n1"),
        # Prompts of a batch of requests; x is one half of the block's input projection.
        _conv("infer", "bf16", 1000, 8, 2048, 4, name="conv-prompt"),
        # Training at the sequence length and batch of the layer-normalised stack's configuration.
        _conv("train", "fp32", 400, 64, 1024, 4, name="conv-train"),
        # Batch-first utterances of unequal length that go on from a state, at sizes nobody rounded.
        _conv("train", "bf16", 333, 37, 250, 3, batch_first=True, lengths=True, state=True, name="conv-train-odd"),
        # Token by token: one stream, and a server that batches its streams.
        _scan("step", "fp32", 1, 1, 1024, 16, state=True, name="scan-step-n1"),
        _scan("step", "bf16", 1, 128, 2048, 16, state=True, name="scan-step-n128"),
        # One long prompt: few channels, many steps.
        _scan("infer", "fp32", 2000, 1, 1024, 16, name="scan-prompt-n1"),
        # Prompts of unequal length that go on from a state, two groups of B and C.
        _scan("infer", "bf16", 237, 19, 640, 16, G=2, lengths=True, state=True, name="scan-prompt-ragged"),
        # Training at the headline's batch and length, forward and backward.
        _scan("train", "bf16", 1000, 64, 1024, 16, name="scan-train"),
        # Training in full precision on sizes that fit no tile, without the gate.
        _scan("train", "fp32", 333, 7, 250, 24, G=2, batch_first=True, lengths=True, state=True, gate=False,
              name="scan-train-odd"),
        # The gated norm behind a block while serving a batch of streams.
        _norm("infer", "bf16", 1, 32, 1024, "rms", gate=True, name="norm-step"),
        # Training: the norm in front of a block, with the residual stream and its scale.
        _norm("train", "bf16", 1000, 64, 1024, "layer", residual=True, scale=True, bias=True, name="norm-train"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _width(rng, lo, hi):
    """A multiple of 8 two times out of three, else as it falls."""
    w = _log_int(rng, lo, hi)
    return w if rng.random() < 1 / 3 else max(lo, w // 8 * 8)


def _draw_once(rng):
    op = rng.choice(["conv", "scan", "scan", "norm"])
    task = rng.choice(["step", "infer", "train", "train"])
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    T, N = (1, _log_int(rng, 1, 256)) if task == "step" else (_log_int(rng, 2, 4000), _log_int(rng, 1, 128))
    if op == "norm":
        residual = rng.random() < 0.6
        return _norm("infer" if task == "step" else task, dtype, T, N, _width(rng, 64, 4096), rng.choice(["rms", "layer"]),
                     gate=rng.random() < 0.5, residual=residual, scale=residual and rng.random() < 0.5,
                     bias=rng.random() < 0.4)
    flags = dict(batch_first=rng.random() < 0.4 and T > 1, lengths=rng.random() < 0.4 and T > 1,
                 state=rng.random() < 0.4 or T == 1)
    if op == "conv":
        return _conv(task, dtype, T, N, _width(rng, 64, 4096), rng.choice([2, 3, 4, 4, 4]), **flags)
    G = rng.choice([1, 1, 1, 2, 4])
    return _scan(task, dtype, T, N, G * _width(rng, 64 // G, 4096 // G), rng.choice([4, 8, 16, 16, 16, 24, 32, 64]), G=G,
                 gate=rng.random() < 0.7, **flags)


def draw(rng):
    most = {k: max(work(c)[k] for c in listed()) for k in ("bytes", "flops")}
    values = 1000 * 64 * 1024 * 16  # (t, n, d, s) of the largest listed scan
    while True:
        case = _draw_once(rng)
        w = work(case)
        if all(w[k] <= most[k] for k in most) and (case["op"] != "scan" or case["T"] * case["N"] * case["D"] * case["S"] <= values):
            return case


def _values(c):
    return c["T"] * c["N"] * (c["H"] if c["op"] == "norm" else c["D"])


def work(c):
    e, n, train = (4 if c["dtype"] == "fp32" else 2), _values(c), c["task"] == "train"
    if c["op"] == "conv":
        state = 2 * (c["W"] - 1) * c["N"] * c["D"] * e
        streams, flops = (4, 6 * c["W"] + 14) if train else (2, 2 * c["W"] + 5)  # x, y; dy, dx
        return {"bytes": n * streams * e + state + c["W"] * c["D"] * e, "flops": n * flops}
    if c["op"] == "scan":
        gate = 1 if c["gate"] else 0
        bc = c["T"] * c["N"] * c["G"] * c["S"] * 2 * e
        state = 2 * c["N"] * c["D"] * c["S"] * 4
        streams = (3 + gate) + ((3 + gate) if train else 0)  # x, dt, z, y; dy, dx, ddt, dz
        per = 7 + (19 if train else 0)  # (t, n, d, s): one exponential, products and sums
        return {"bytes": n * streams * e + bc * (2 if train else 1) + state + c["D"] * c["S"] * 4,
                "flops": n * c["S"] * per}
    extra = int(c["gate"]) + 2 * int(c["residual"])  # gate; residual and the new residual
    back = 2 + int(c["gate"]) + 2 * int(c["residual"])  # dy, dx; dgate; dr, dresidual
    return {"bytes": n * (2 + extra + (back if train else 0)) * e, "flops": n * (32 if train else 12)}


# ------------------------------------------------------------------ inputs
def _sequence(g, c, width, dtype, scale=1.0):
    """[T,N,width], a view of [N,T,width] with batch_first."""
    T, N = c["T"], c["N"]
    if c.get("batch_first"):
        return (torch.randn(N, T, width, generator=g, device="cuda") * scale).to(dtype).transpose(0, 1)
    return (torch.randn(T, N, width, generator=g, device="cuda") * scale).to(dtype)


def _lengths(g, c):
    if not c.get("lengths"):
        return None
    n = torch.randint(1, c["T"] + 1, (c["N"],), generator=g, device="cuda")
    n[0] = c["T"]
    return n


def _prepare_conv(c, g, t):
    D, W, N = c["D"], c["W"], c["N"]
    s = {"x": _sequence(g, c, 2 * D, t)[..., :D],  # the other half is the gate
         "weight": ((torch.rand(D, W, generator=g, device="cuda") * 2 - 1) / math.sqrt(W)).to(t),
         "bias": (0.1 * torch.randn(D, generator=g, device="cuda")).to(t), "lengths": _lengths(g, c),
         "state": torch.randn(N, W - 1, D, generator=g, device="cuda").to(t) if c["state"] or c["task"] == "step" else None}
    if c["task"] == "step":
        s["x"] = s["x"][0]
    if c["task"] == "train":
        s["dy"] = _sequence(g, c, D, t)
    return s


def _prepare_scan(c, g, t):
    D, S, G, N = c["D"], c["S"], c["G"], c["N"]
    rank = max(8, D // 32)  # B and C lie behind the step sizes' low-rank projection
    proj = _sequence(g, c, rank + 2 * G * S, t)
    B, C = proj[..., rank:rank + G * S].unflatten(-1, (G, S)), proj[..., rank + G * S:].unflatten(-1, (G, S))
    x = _sequence(g, c, D, torch.float32)
    step = torch.exp(torch.rand(D, generator=g, device="cuda") * math.log(100.0) + math.log(1e-3))  # 0.001 .. 0.1
    s = {"x": (x * torch.sigmoid(x)).to(t), "dt": _sequence(g, c, D, t, 0.5), "B": B, "C": C,
         "A": -torch.arange(1, S + 1, device="cuda") * (1 + 0.05 * torch.randn(D, S, generator=g, device="cuda")).abs(),
         "D": 1 + 0.1 * torch.randn(D, generator=g, device="cuda"), "dt_bias": step + torch.log(-torch.expm1(-step)),
         "z": _sequence(g, c, 2 * D, t)[..., D:] if c["gate"] else None, "lengths": _lengths(g, c),
         "state": 0.3 * torch.randn(N, D, S, generator=g, device="cuda") if c["state"] else None}
    if c["task"] == "step":
        for k in ("x", "dt", "B", "C", "z"):
            s[k] = None if s[k] is None else s[k][0]
    if c["task"] == "train":
        s["dy"] = _sequence(g, c, D, t)
    return s


def _prepare_norm(c, g, t):
    H = c["H"]
    s = {"x": _sequence(g, c, H, t), "weight": (1 + 0.1 * torch.randn(H, generator=g, device="cuda")).to(t),
         "bias": (0.1 * torch.randn(H, generator=g, device="cuda")).to(t) if c["bias"] else None,
         "gate": _sequence(g, c, H, t) if c["gate"] else None,
         "residual": _sequence(g, c, H, t, 2.0) if c["residual"] else None,
         "scale": (0.5 + 0.1 * torch.randn(H, generator=g, device="cuda")).to(t) if c["scale"] else None}
    if c["task"] == "train":
        s["dy"] = _sequence(g, c, H, t)
        s["dr"] = _sequence(g, c, H, t) if c["residual"] else None
    return s


# what a training step returns the gradients of
LEAVES = {"conv": ("x", "weight", "bias", "state"),
          "scan": ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "state"),
          "norm": ("x", "weight", "bias", "gate", "residual", "scale")}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    make = {"conv": _prepare_conv, "scan": _prepare_scan, "norm": _prepare_norm}[case["op"]]
    s = make(case, g, DTYPES[case["dtype"]])
    if case["task"] == "train":
        for k in LEAVES[case["op"]]:
            if s[k] is not None:
                s[k].requires_grad_(True)
    s["case"] = case
    return s


# ------------------------------------------------------------------ plain forms
def _f(t):
    return None if t is None else t.detach().float()


def _valid(lengths, T):
    """[T,N,1]: 1 where a step belongs to its row."""
    return (torch.arange(T, device=lengths.device)[:, None] < lengths[None])[..., None].float()


def _silu_and_slope(p):
    s = 1 / (1 + torch.exp(-p))
    return p * s, s * (1 + p * (1 - s))


def _conv_plain(s, c):
    x, w, b, state, t = _f(s["x"]), _f(s["weight"]), _f(s["bias"]), _f(s["state"]), s["x"].dtype
    if c["task"] == "step":
        window = torch.cat([state, x[:, None]], 1)  # [N,W,D]
        y, _ = _silu_and_slope((window * w.t()).sum(1) + b)
        return {"y": y.to(t), "state": window[:, 1:].to(t)}
    T, W, N, D = c["T"], c["W"], c["N"], c["D"]
    if state is None:
        state = x.new_zeros(N, W - 1, D)
    padded = torch.cat([state.transpose(0, 1), x], 0)  # [W-1+T,N,D]
    windows = padded.unfold(0, W, 1)  # [T,N,D,W]
    p = (windows * w).sum(-1) + b
    y, slope = _silu_and_slope(p)
    lengths = s["lengths"] if c["lengths"] else torch.full((N,), T, device=x.device)
    valid = _valid(lengths, T)
    rows = lengths[:, None] + torch.arange(W - 1, device=x.device)  # last W-1 inputs of each row
    out = {"y": (y * valid).to(t),
           "state": padded[rows, torch.arange(N, device=x.device)[:, None]].to(t)}
    if c["task"] == "train":
        dp = _f(s["dy"]) * valid * slope
        taps = torch.cat([dp, dp.new_zeros(W - 1, N, D)], 0)
        late = torch.cat([dp.new_zeros(W - 1, N, D), taps], 0).unfold(0, W, 1)  # gradient of padded row r: dp_{r-W+1..r}
        dpadded = (late * w.flip(1)).sum(-1)
        out |= {"dx": dpadded[W - 1:].to(t), "dweight": (windows * dp[..., None]).sum((0, 1)).to(t),
                "dbias": dp.sum((0, 1)).to(t)}
        if c["state"]:
            out["dstate"] = dpadded[:W - 1].transpose(0, 1).to(t)
    return out


def _linear_scan(a, b):
    """h_t = a_t h_{t-1} + b_t along the first axis, by doubling."""
    step = 1
    while step < len(a):
        b = torch.cat([b[:step], torch.addcmul(b[step:], a[step:], b[:-step])])
        a = torch.cat([a[:step], a[step:] * a[:-step]])
        step *= 2
    return b


def _softplus(v):
    return v.clamp(min=0) + torch.log1p(torch.exp(-v.abs()))


def _scan_plain(s, c):
    t, S, G, N, D = s["x"].dtype, c["S"], c["G"], c["N"], c["D"]
    one = c["task"] == "step"
    x, dt, B, C, z = (None if s[k] is None else _f(s[k])[None] if one else _f(s[k]) for k in ("x", "dt", "B", "C", "z"))
    T = x.shape[0]
    split = lambda v: v.reshape(T, N, G, D // G)  # noqa: E731
    A, skip = _f(s["A"]).reshape(G, D // G, S), _f(s["D"])
    raw = dt + _f(s["dt_bias"])
    valid = _valid(s["lengths"], T) if c["lengths"] else x.new_ones(1, 1, 1)
    delta = split(_softplus(raw) * valid)
    xs = split(x)
    Bg, Cg = B[:, :, :, None], C[:, :, :, None]  # [T,N,G,1,S]
    a = torch.exp(delta[..., None] * A)
    b = (delta * xs)[..., None] * Bg
    h0 = x.new_zeros(N, G, D // G, S) if s["state"] is None else _f(s["state"]).reshape(N, G, D // G, S)
    b[0] += a[0] * h0
    h = _linear_scan(a, b)
    del b
    y = (h * Cg).sum(-1).reshape(T, N, D) + skip * x
    gate, slope = (None, None) if z is None else _silu_and_slope(z)
    out = (y if z is None else y * gate) * valid
    last = h[-1].reshape(N, D, S)
    if one:
        return {"y": out[0].to(t), "state": last.clone()}
    res = {"y": out.to(t), "state": last.clone()}
    if c["task"] == "train":
        dy = _f(s["dy"]) * valid
        if z is not None:
            res["dz"] = (dy * y * slope).to(t)
            dy = dy * gate
        dyg = split(dy)
        res["dC"] = (dyg[..., None] * h).sum(3).to(t)
        # the adjoint runs from the last step: lam_t = C_t dy_t + a_{t+1} lam_{t+1}
        lam = _linear_scan(torch.cat([a[1:], a[:1]]).flip(0), (dyg[..., None] * Cg).flip(0)).flip(0)
        h = torch.cat([h0[None], h[:-1]])
        h *= a
        h *= lam  # lam a h_{t-1}
        res["dstate"] = (a[0] * lam[0]).reshape(N, D, S) if c["state"] else None
        del a
        res["dA"] = (h * delta[..., None]).sum((0, 1)).reshape(D, S)
        ddelta = (h * A).sum(-1)
        del h
        res["dB"] = (lam * (delta * xs)[..., None]).sum(3).to(t)
        lb = (lam * Bg).sum(-1)
        del lam
        ddelta = ((ddelta + lb * xs).reshape(T, N, D) * valid) / (1 + torch.exp(-raw))
        res |= {"dx": ((lb * delta).reshape(T, N, D) + skip * dy).to(t), "ddt": ddelta.to(t),
                "ddt_bias": ddelta.sum((0, 1)), "dD": (dy * x).sum((0, 1))}
        if not c["state"]:
            del res["dstate"]
    return res


def _norm_plain(s, c):
    t, H = s["x"].dtype, c["H"]
    x, w, b, gate, residual, scale = (_f(s[k]) for k in ("x", "weight", "bias", "gate", "residual", "scale"))
    g, slope = (None, None) if gate is None else _silu_and_slope(gate)
    u = x if gate is None else x * g
    r = u if scale is None else scale * u
    r = r if residual is None else residual + r
    m = r.mean(-1, keepdim=True) if c["kind"] == "layer" else 0.0
    inv = 1 / torch.sqrt(((r - m) ** 2).mean(-1, keepdim=True) + 1e-5)
    n = (r - m) * inv
    res = {"y": (n * w if b is None else n * w + b).to(t)}
    if residual is not None:
        res["r"] = r.to(t)
    if c["task"] == "train":
        dy = _f(s["dy"])
        dn = dy * w
        over = (dn * n).mean(-1, keepdim=True)
        dr = inv * (dn - n * over - (dn.mean(-1, keepdim=True) if c["kind"] == "layer" else 0.0))
        res["dweight"] = (dy * n).sum((0, 1)).to(t)
        if b is not None:
            res["dbias"] = dy.sum((0, 1)).to(t)
        if residual is not None:
            dr = dr + _f(s["dr"])
            res["dresidual"] = dr.to(t)
        if scale is not None:
            res["dscale"] = (dr * u).sum((0, 1)).to(t)
            dr = dr * scale
        if gate is not None:
            res["dgate"] = (dr * x * slope).to(t)
            dr = dr * g
        res["dx"] = dr.to(t)
    return res


# ------------------------------------------------------------------ the framework's operators
def _gradients(s, c, outputs, incoming):
    names = [k for k in LEAVES[c["op"]] if s[k] is not None]
    return dict(zip(("d" + k for k in names), torch.autograd.grad(outputs, [s[k] for k in names], incoming)))


def _conv_own(s, c):
    from haste_b200 import ssm
    if c["task"] == "step":
        y, state = ssm.causal_conv1d_step(s["x"], s["state"], s["weight"], s["bias"])
        return {"y": y, "state": state}
    y, state = ssm.causal_conv1d(s["x"], s["weight"], s["bias"], initial_state=s["state"], lengths=s["lengths"])
    out = {"y": y.detach(), "state": state.detach()}
    return out | _gradients(s, c, [y], [s["dy"]]) if c["task"] == "train" else out


def _scan_own(s, c):
    from haste_b200 import ssm
    if c["task"] == "step":
        y, state = ssm.selective_scan_step(s["x"], s["dt"], s["A"], s["B"], s["C"], s["state"], D=s["D"], z=s["z"],
                                           dt_bias=s["dt_bias"])
        return {"y": y, "state": state}
    y, state = ssm.selective_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"],
                                  initial_state=s["state"], lengths=s["lengths"])
    out = {"y": y.detach(), "state": state.detach()}
    return out | _gradients(s, c, [y], [s["dy"]]) if c["task"] == "train" else out


def _norm_own(s, c):
    from haste_b200 import ssm
    y, r = ssm.fused_norm(s["x"], s["weight"], s["bias"], gate=s["gate"], residual=s["residual"], scale=s["scale"],
                          kind=c["kind"])
    out = {"y": y.detach()} | ({} if r is None else {"r": r.detach()})
    if c["task"] != "train":
        return out
    return out | _gradients(s, c, [y] + ([] if r is None else [r]), [s["dy"]] + ([] if r is None else [s["dr"]]))


def run(state):
    c = state["case"]
    if own:
        if c["task"] != "train":
            with torch.no_grad():
                return {"conv": _conv_own, "scan": _scan_own, "norm": _norm_own}[c["op"]](state, c)
        return {"conv": _conv_own, "scan": _scan_own, "norm": _norm_own}[c["op"]](state, c)
    with torch.no_grad():
        return {"conv": _conv_plain, "scan": _scan_plain, "norm": _norm_plain}[c["op"]](state, c)


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    """Step by step as the formulas have it, gradients by automatic differentiation."""
    c, s = case, prepare(case, seed)
    leaf = {k: v.detach().double().requires_grad_(c["task"] == "train") for k, v in s.items()
            if torch.is_tensor(v) and v.is_floating_point() and k not in ("dy", "dr")}
    with torch.set_grad_enabled(c["task"] == "train"):
        out, into = {"conv": _conv_exact, "scan": _scan_exact, "norm": _norm_exact}[c["op"]](leaf, s, c)
    if c["task"] == "train":
        names = [k for k in LEAVES[c["op"]] if k in leaf]
        grads = torch.autograd.grad([o for o, _ in into], [leaf[k] for k in names], [d.double() for _, d in into])
        out |= dict(zip(("d" + k for k in names), grads))
    return {k: v.detach() for k, v in out.items()}


def _conv_exact(v, s, c):
    x = v["x"][None] if c["task"] == "step" else v["x"]
    T, N, D = x.shape
    W = c["W"]
    past = [v["state"][:, k] for k in range(W - 1)] if "state" in v else [x.new_zeros(N, D)] * (W - 1)
    live = [torch.ones(N, 1, dtype=torch.bool, device=x.device) if s["lengths"] is None else (t < s["lengths"])[:, None]
            for t in range(T)]
    ys = []
    for t in range(T):
        now = past + [x[t]]
        p = v["bias"] + sum(now[k] * v["weight"][:, k] for k in range(W))
        ys.append(torch.where(live[t], torch.nn.functional.silu(p), 0.0))
        past = [torch.where(live[t], n, o) for n, o in zip(now[1:], past)]
    y = torch.stack(ys)
    out = {"y": y[0] if c["task"] == "step" else y, "state": torch.stack(past, 1)}
    return out, [(y, s["dy"])] if c["task"] == "train" else []


def _scan_exact(v, s, c):
    one = c["task"] == "step"
    x, dt, B, C = (v[k][None] if one else v[k] for k in ("x", "dt", "B", "C"))
    T, N, D = x.shape
    per = D // c["G"]
    h = v["state"] if "state" in v else x.new_zeros(N, D, c["S"])
    delta = torch.nn.functional.softplus(dt + v["dt_bias"], threshold=700.0)
    if s["lengths"] is not None:
        live = torch.arange(T, device=x.device)[:, None] < s["lengths"]
        delta = torch.where(live[..., None], delta, 0.0)
    dx = delta * x
    ys = []
    for t in range(T):
        Bt, Ct = (m[t].repeat_interleave(per, 1) for m in (B, C))
        h = torch.exp(delta[t, :, :, None] * v["A"]) * h + dx[t, :, :, None] * Bt
        ys.append(torch.einsum("nds,nds->nd", h, Ct))
    y = torch.stack(ys) + v["D"] * x
    if "z" in v:
        y = y * torch.nn.functional.silu(v["z"][None] if one else v["z"])
    if s["lengths"] is not None:
        y = torch.where(live[..., None], y, 0.0)
    out = {"y": y[0] if one else y, "state": h}
    return out, [(y, s["dy"])] if c["task"] == "train" else []


def _norm_exact(v, s, c):
    u = v["x"] * torch.nn.functional.silu(v["gate"]) if "gate" in v else v["x"]
    r = v["scale"] * u if "scale" in v else u
    r = v["residual"] + r if "residual" in v else r
    d = r - r.mean(-1, keepdim=True) if c["kind"] == "layer" else r
    y = d * torch.rsqrt(d.square().mean(-1, keepdim=True) + 1e-5) * v["weight"]
    y = y + v["bias"] if "bias" in v else y
    out = {"y": y} | ({"r": r} if "residual" in v else {})
    if c["task"] != "train":
        return out, []
    return out, [(y, s["dy"])] + ([(r, s["dr"])] if "residual" in v else [])
