"""Performance cases of the operators of a gated linear recurrence block: the recurrence's scan over
whole sequences (forward, forward and backward) and for single tokens, the projections around it with
bias, activation and residual, and the global gradient norm and clipping that end a training step.

`run` computes a case's plain form in elementary torch operations, or, with `own`, calls
`haste_b200.ssm` and `haste_b200.gradients`.  All sequences are time-major [T,N,...]; `batch_first`
cases hand over views of [N,T,...] tensors.  Gradients have the shapes of a stack of LSTM layers.
"""
import math

import torch

own = False  # True: the framework's operators instead of the plain forms

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _scan(task, dtype, T, N, D, decay=False, input_gate=False, batch_first=False, lengths=False, state=False, **name):
    return dict(op="scan", task=task, dtype=dtype, T=T, N=N, D=D, decay=decay, input_gate=input_gate,
                batch_first=batch_first, lengths=lengths, state=state, **name)


def _linear(task, dtype, T, N, C, H, activation="none", bias=True, residual=False, batch_first=False, **name):
    return dict(op="linear", task=task, dtype=dtype, T=T, N=N, C=C, H=H, activation=activation, bias=bias,
                residual=residual, batch_first=batch_first, **name)


def _clip(dtype, layers, H, out, clips, **name):
    return dict(op="clip", task="train", dtype=dtype, layers=layers, H=H, out=out, clips=clips, **name)


def listed():
    return [
        # One stream that answers token by token: nothing but latency.
        _scan("step", "bf16", 1, 1, 1024, decay=True, input_gate=True, state=True, name="gated-scan-step-n1"),
        # One long prompt: few channels, many steps.
        _scan("infer", "fp32", 2000, 1, 1024, decay=True, input_gate=True, name="gated-scan-prompt-n1"),
        # Training at the headline's batch and length, forward and backward, with both gates.
        _scan("train", "bf16", 1000, 64, 1024, decay=True, input_gate=True, name="gated-scan-train"),
        # Batch-first utterances of unequal length that go on from a state, one gate, sizes that nobody rounded.
        _scan("train", "fp16", 333, 37, 250, batch_first=True, lengths=True, state=True, name="gated-scan-train-odd"),
        # The projection into the block for one stream: the weights are read once, nothing else counts.
        _linear("step", "bf16", 1, 1, 1024, 4096, "silu", name="linear-step-n1"),
        # The projection back for a server that batches its streams.
        _linear("step", "bf16", 1, 32, 4096, 1024, residual=True, name="linear-step-n32"),
        # Prompts of a batch of requests.
        _linear("infer", "fp16", 250, 8, 2048, 4096, "gelu", name="linear-prompt"),
        # Training at the headline's batch and length, forward and backward.
        _linear("train", "bf16", 1000, 64, 1024, 2048, "silu", name="linear-train"),
        # Training in full precision on sizes that fit no tile.
        _linear("train", "fp32", 333, 7, 250, 1000, "gelu", residual=True, batch_first=True, name="linear-train-odd"),
        # The headline's one layer, late in training: the norm is below the bound, nothing is scaled.
        _clip("fp32", 1, 512, out=False, clips=False, name="clip-layer"),
        # A stack's bf16 gradients, clipped into the float32 ones that the optimiser reads.
        _clip("bf16", 6, 2048, out=True, clips=True, name="clip-stack"),
        # Many small tensors of odd sizes.
        _clip("fp32", 20, 97, out=True, clips=True, name="clip-many"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _width(rng, lo, hi):
    """A multiple of 8 two times out of three, else as it falls."""
    w = _log_int(rng, lo, hi)
    return w if rng.random() < 1 / 3 else max(lo, w // 8 * 8)


def _draw_once(rng):
    op = rng.choice(["scan", "scan", "linear", "linear", "clip"])
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    if op == "clip":
        clips = rng.random() < 0.6
        return _clip(dtype, _log_int(rng, 1, 20), _log_int(rng, 16, 2048), out=clips or rng.random() < 0.5, clips=clips)
    task = rng.choice(["step", "infer", "train", "train"])
    T, N = (1, _log_int(rng, 1, 256)) if task == "step" else (_log_int(rng, 2, 4000), _log_int(rng, 1, 128))
    batch_first = rng.random() < 0.4 and T > 1
    if op == "linear":
        return _linear(task, dtype, T, N, _width(rng, 64, 4096), _width(rng, 64, 4096),
                       rng.choice(["none", "relu", "silu", "silu", "gelu", "tanh", "sigmoid"]), bias=rng.random() < 0.7,
                       residual=rng.random() < 0.4, batch_first=batch_first)
    return _scan(task, dtype, T, N, _width(rng, 64, 4096), decay=rng.random() < 0.6, input_gate=rng.random() < 0.6,
                 batch_first=batch_first, lengths=rng.random() < 0.4 and T > 1, state=rng.random() < 0.4 or T == 1)


def draw(rng):
    while True:
        case = _draw_once(rng)
        w = work(case)
        most = [work(c) for c in listed() if c["op"] == case["op"]]
        if all(w[k] <= max(m[k] for m in most) for k in w):
            return case


def _shapes(c):
    """Of the gradients: kernel, recurrent kernel and bias of each layer."""
    H = c["H"]
    return [s for _ in range(c["layers"]) for s in ((H, 4 * H), (H, 4 * H), (4 * H,))]


def work(c):
    e, train = (4 if c["dtype"] == "fp32" else 2), c["task"] == "train"
    if c["op"] == "scan":
        n, streams = c["T"] * c["N"] * c["D"], 3 + int(c["input_gate"])  # x, gates; y
        back = streams if train else 0  # dy; dx, the gates' gradients
        state = 2 * c["N"] * c["D"] * 4 * (2 if train and c["state"] else 1)
        per = 12 + (14 if c["decay"] else 0) + (6 if c["input_gate"] else 0)
        return {"bytes": n * (streams + back) * e + state, "flops": n * per * (3 if train else 1)}
    if c["op"] == "linear":
        M, C, H = c["T"] * c["N"], c["C"], c["H"]
        rows, extra = M * (C + H), M * H * int(c["residual"])  # x, y; residual
        return {"bytes": (rows * (2 if train else 1) + extra + C * H * (2 if train else 1)) * e,
                "flops": 2 * M * C * H * (3 if train else 1)}
    n = sum(math.prod(s) for s in _shapes(c))
    return {"bytes": n * (e + (4 if c["out"] else 0)), "flops": n * (3 if c["clips"] else 2)}


# ------------------------------------------------------------------ inputs
def _sequence(g, c, width, dtype, scale=1.0):
    """[T,N,width], a view of [N,T,width] with batch_first."""
    T, N = c["T"], c["N"]
    if c.get("batch_first"):
        return (torch.randn(N, T, width, generator=g, device="cuda") * scale).to(dtype).transpose(0, 1)
    return (torch.randn(T, N, width, generator=g, device="cuda") * scale).to(dtype)


def _prepare_scan(c, g, t):
    D, N = c["D"], c["N"]
    gates = _sequence(g, c, 2 * D, t)  # both gates come from one projection
    lam = torch.rand(D, generator=g, device="cuda") * 0.099 + 0.9  # half open, a gate decays by 0.9 .. 0.999 a step
    s = {"x": _sequence(g, c, D, t), "gate": gates[..., :D], "input_gate": gates[..., D:] if c["input_gate"] else None,
         "decay": 2 * torch.log(lam) if c["decay"] else None, "lengths": None,
         "state": 0.5 * torch.randn(N, D, generator=g, device="cuda") if c["state"] else None}
    if c["lengths"]:
        s["lengths"] = torch.randint(1, c["T"] + 1, (N,), generator=g, device="cuda")
        s["lengths"][0] = c["T"]
    if c["task"] == "step":
        for k in ("x", "gate", "input_gate"):
            s[k] = None if s[k] is None else s[k][0]
    if c["task"] == "train":
        s["dy"] = _sequence(g, c, D, t)
    return s


def _prepare_linear(c, g, t):
    C, H = c["C"], c["H"]
    s = {"x": _sequence(g, c, C, t), "weight": ((torch.rand(H, C, generator=g, device="cuda") * 2 - 1) / math.sqrt(C)).to(t),
         "bias": (0.1 * torch.randn(H, generator=g, device="cuda")).to(t) if c["bias"] else None,
         "residual": _sequence(g, c, H, t, 2.0) if c["residual"] else None}
    if c["task"] == "step":
        for k in ("x", "residual"):
            s[k] = None if s[k] is None else s[k][0]
    if c["task"] == "train":
        s["dy"] = _sequence(g, c, H, t)
    return s


def _prepare_clip(c, g, t):
    # layers' gradients differ in size; a step that is clipped has a norm far above 1, the other one below
    n = sum(math.prod(s) for s in _shapes(c))
    rms = (5.0 if c["clips"] else 0.1) / math.sqrt(n)
    scale = torch.exp(torch.rand(len(_shapes(c)), generator=g, device="cuda") - 0.5) * rms
    grads = [(torch.randn(s, generator=g, device="cuda") * k).to(t) for s, k in zip(_shapes(c), scale)]
    if c["out"]:
        return {"gradients": grads, "into": [torch.empty_like(v, dtype=torch.float32) for v in grads]}
    parameters = [torch.nn.Parameter(torch.zeros_like(v)) for v in grads]
    for p, v in zip(parameters, grads):
        p.grad = v
    return {"gradients": grads, "parameters": parameters}


# what a training step returns the gradients of
LEAVES = {"scan": ("x", "gate", "decay", "input_gate", "state"), "linear": ("x", "weight", "bias", "residual"), "clip": ()}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    make = {"scan": _prepare_scan, "linear": _prepare_linear, "clip": _prepare_clip}[case["op"]]
    s = make(case, g, DTYPES[case["dtype"]])
    if case["task"] == "train":
        for k in LEAVES[case["op"]]:
            if s[k] is not None:
                s[k] = s[k].detach().requires_grad_(True)
    s["case"] = case
    return s


# ------------------------------------------------------------------ plain forms
def _f(t):
    return None if t is None else t.detach().float()


def _sigmoid(v):
    return 1 / (1 + torch.exp(-v))


def _linear_scan(a, b):
    """h_t = a_t h_{t-1} + b_t along the first axis, by doubling."""
    step = 1
    while step < len(a):
        b = torch.cat([b[:step], torch.addcmul(b[step:], a[step:], b[:-step])])
        a = torch.cat([a[:step], a[step:] * a[:-step]])
        step *= 2
    return b


def _scan_plain(s, c):
    t, one = s["x"].dtype, c["task"] == "step"
    x, gate, inner = (None if s[k] is None else _f(s[k])[None] if one else _f(s[k]) for k in ("x", "gate", "input_gate"))
    decay, T = _f(s["decay"]), x.shape[0]
    r = _sigmoid(gate)
    if c["decay"]:
        log_a = decay * r
        # (rounded from 64 bits: a step's decay lies next to one, and an error of one sign adds up over 1 / (1 - a) steps)
        a, w = torch.exp(log_a.double()).float(), torch.sqrt(-torch.expm1(2 * log_a))
    else:
        a, w = r, _sigmoid(-gate)
    i = 1.0 if inner is None else _sigmoid(inner)
    u = x * i
    b = w * u
    if c["lengths"]:
        valid = (torch.arange(T, device=x.device)[:, None] < s["lengths"][None])[..., None]
        a, b = torch.where(valid, a, 1.0), torch.where(valid, b, 0.0)
    h0 = x.new_zeros(x.shape[1:]) if s["state"] is None else _f(s["state"])
    b[0] += a[0] * h0
    h = _linear_scan(a, b)
    y = torch.where(valid, h, 0.0) if c["lengths"] else h
    if one:
        return {"y": y[0].to(t), "state": h[-1].clone()}
    out = {"y": y.to(t), "state": h[-1].clone()}
    if c["task"] == "train":
        dy = _f(s["dy"])
        if c["lengths"]:
            dy = torch.where(valid, dy, 0.0)
        # the adjoint runs from the last step: lam_t = dy_t + a_{t+1} lam_{t+1}
        lam = _linear_scan(torch.cat([a[1:], a[:1]]).flip(0), dy.flip(0)).flip(0)
        before = torch.cat([h0[None], h[:-1]])
        if c["lengths"]:
            out_lam = torch.where(valid, lam, 0.0)
        else:
            out_lam = lam
        if c["decay"]:
            dlog = out_lam * (a * before - a * a / w * u)
            out |= {"ddecay": (dlog * r).sum((0, 1), dtype=torch.float64).float(), "dgate": (dlog * decay * r * _sigmoid(-gate)).to(t)}
        else:
            out["dgate"] = (out_lam * (before - u) * r * _sigmoid(-gate)).to(t)
        out["dx"] = (out_lam * w * i).to(t)
        if inner is not None:
            out["dinput_gate"] = (out_lam * w * x * i * _sigmoid(-inner)).to(t)
        if c["state"]:
            out["dstate"] = a[0] * lam[0]
    return out


def _act(name, p):
    if name == "relu":
        return torch.where(p > 0, p, 0.0)
    if name == "silu":
        return p * _sigmoid(p)
    if name == "gelu":
        return 0.5 * p * (1 + torch.erf(p / math.sqrt(2)))
    if name == "tanh":
        return torch.tanh(p)
    return _sigmoid(p) if name == "sigmoid" else p


def _slope(name, p):
    if name == "relu":
        return (p > 0).to(p.dtype)
    if name == "silu":
        s = _sigmoid(p)
        return s * (1 + p * (1 - s))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(p / math.sqrt(2))) + p * torch.exp(-0.5 * p * p) / math.sqrt(2 * math.pi)
    if name == "tanh":
        return 1 - torch.tanh(p) ** 2
    s = _sigmoid(p)
    return s * (1 - s)


def _linear_plain(s, c):
    t, C, H = s["x"].dtype, c["C"], c["H"]
    x, w, b, residual = (_f(s[k]) for k in ("x", "weight", "bias", "residual"))
    p = x @ w.t()
    if b is not None:
        p = p + b
    y = _act(c["activation"], p)
    if residual is not None:
        y = y + residual
    out = {"y": y.to(t)}
    if c["task"] == "train":
        dp = _f(s["dy"])
        if c["activation"] != "none":
            dp = dp * _slope(c["activation"], p)
        flat = dp.reshape(-1, H)
        out |= {"dx": (dp @ w).to(t), "dweight": (flat.t() @ x.reshape(-1, C)).to(t)}
        if b is not None:
            out["dbias"] = flat.sum(0).to(t)
        if residual is not None:
            out["dresidual"] = s["dy"].detach()
    return out


def _clip_plain(s, c):
    grads = s["gradients"]
    norm = torch.sqrt(torch.stack([(v.float() ** 2).sum() for v in grads]).sum())
    factor = torch.clamp(1.0 / (norm + 1e-6), max=1.0)
    t = torch.float32 if c["out"] else grads[0].dtype
    return {"norm": norm, "gradients": [(v.float() * factor).to(t) for v in grads]}


# ------------------------------------------------------------------ the framework's operators
def _gradients(s, c, outputs, incoming):
    names = [k for k in LEAVES[c["op"]] if s[k] is not None]
    return dict(zip(("d" + k for k in names), torch.autograd.grad(outputs, [s[k] for k in names], incoming)))


def _scan_own(s, c):
    from haste_b200 import ssm
    if c["task"] == "step":
        y, state = ssm.gated_scan_step(s["x"], s["gate"], s["state"], decay=s["decay"], input_gate=s["input_gate"])
        return {"y": y, "state": state}
    y, state = ssm.gated_scan(s["x"], s["gate"], decay=s["decay"], input_gate=s["input_gate"], initial_state=s["state"],
                              lengths=s["lengths"])
    out = {"y": y.detach(), "state": state.detach()}
    return out | _gradients(s, c, [y], [s["dy"]]) if c["task"] == "train" else out


def _linear_own(s, c):
    from haste_b200 import ssm
    y = ssm.fused_linear(s["x"], s["weight"], s["bias"], activation=None if c["activation"] == "none" else c["activation"],
                         residual=s["residual"])
    return {"y": y.detach()} | (_gradients(s, c, [y], [s["dy"]]) if c["task"] == "train" else {})


def _clip_own(s, c):
    from haste_b200 import gradients
    if not c["out"]:
        return {"norm": gradients.clip_grad_norm_(s["parameters"], 1.0), "gradients": s["gradients"]}
    return {"norm": gradients.clip_gradients(s["gradients"], 1.0, out=s["into"]), "gradients": s["into"]}


def run(state):
    c = state["case"]
    if own:
        call = {"scan": _scan_own, "linear": _linear_own, "clip": _clip_own}[c["op"]]
        if c["task"] == "train":
            return call(state, c)
        with torch.no_grad():
            return call(state, c)
    with torch.no_grad():
        return {"scan": _scan_plain, "linear": _linear_plain, "clip": _clip_plain}[c["op"]](state, c)


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    """Step by step as the formulas have it, gradients by automatic differentiation."""
    c, s = case, prepare(case, seed)
    if c["op"] == "clip":
        grads = [v.double() for v in s["gradients"]]
        norm = sum(v.square().sum() for v in grads).sqrt()
        factor = min(1.0, 1.0 / (norm.item() + 1e-6))
        return {"norm": norm, "gradients": [v * factor for v in grads]}
    train = c["task"] == "train"
    leaf = {k: s[k].detach().double().requires_grad_(train) for k in LEAVES[c["op"]] if s[k] is not None}
    with torch.set_grad_enabled(train):
        out = {"scan": _scan_exact, "linear": _linear_exact}[c["op"]](leaf, s, c)
        if train:
            grads = torch.autograd.grad([out["y"]], list(leaf.values()), [s["dy"].double()])
            out |= dict(zip(("d" + k for k in leaf), grads))
    return {k: v.detach() for k, v in out.items()}


def _scan_exact(v, s, c):
    one = c["task"] == "step"
    x, gate = (v[k][None] if one else v[k] for k in ("x", "gate"))
    T = x.shape[0]
    r = torch.sigmoid(gate)
    a = torch.exp(v["decay"] * r) if "decay" in v else r
    w = torch.sqrt(1 - a * a) if "decay" in v else 1 - a
    b = w * x
    if "input_gate" in v:
        b = b * torch.sigmoid(v["input_gate"][None] if one else v["input_gate"])
    live = None if s["lengths"] is None else torch.arange(T, device=x.device)[:, None, None] < s["lengths"][None, :, None]
    h = v["state"] if "state" in v else torch.zeros_like(x[0])
    hs = []
    for at, bt, t in zip(a.unbind(0), b.unbind(0), range(T)):
        new = at * h + bt
        h = new if live is None else torch.where(live[t], new, h)
        hs.append(h)
    y = torch.stack(hs)
    if live is not None:
        y = torch.where(live, y, 0.0)
    return {"y": y[0] if one else y, "state": h}


def _linear_exact(v, s, c):
    p = torch.nn.functional.linear(v["x"], v["weight"], v.get("bias"))
    act = {"none": lambda p: p, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
           "tanh": torch.tanh, "sigmoid": torch.sigmoid}[c["activation"]]
    y = act(p)
    return {"y": y + v["residual"] if "residual" in v else y}
