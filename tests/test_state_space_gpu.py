"""The state space operators against their float64 reference, element by element within the roundings
that the arithmetic may make (state_space_reference.py)."""
import pytest
import torch

import state_space_reference as ref

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def seq(g, T, N, D, dtype, batch_first=False, half=False, scale=1.0, step=1):
    """[T,N,D]: dense, a view of a batch-first tensor, one half of a wider one, or strided along D."""
    D2 = (2 * D if half else D) * step
    t = torch.randn((N, T, D2) if batch_first else (T, N, D2), generator=g, device="cuda") * scale
    t = t.to(dtype)
    t = t.transpose(0, 1) if batch_first else t
    return (t[..., D * step:] if half else t)[..., ::step]


def leaves(d, names):
    for k in names:
        if d.get(k) is not None:
            d[k] = d[k].detach().requires_grad_(True)
    return [k for k in names if d.get(k) is not None]


def lens(g, T, N, kind):
    if kind is None:
        return None
    n = torch.randint(0, T + 1, (N,), generator=g, device="cuda")
    n[0] = 0
    n[-1] = T
    return n.to(kind)


def poison(t, lengths):
    """NaN and infinity behind the rows' ends: nothing may read them."""
    if lengths is None:
        return t
    T, N = t.shape[:2]
    dead = torch.arange(T, device="cuda")[:, None] >= lengths[None]
    t = t.clone() if t.is_contiguous() else t
    with torch.no_grad():
        t[dead] = float("nan")
        t[dead & (torch.arange(N, device="cuda")[None] % 2 == 0)] = float("inf")
    return t


# ------------------------------------------------------------------ causal_conv1d
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("T,N,D,W,opt", [
    (1, 1, 1, 4, {}), (1, 3, 64, 4, dict(state=True)), (2, 2, 7, 3, dict(state=True)), (3, 1, 33, 2, {}),
    (2, 2, 16, 4, dict(state=True, bias=False)), (17, 2, 130, 4, dict(batch_first=True)),
    (70, 3, 250, 3, dict(lengths=torch.int64, state=True, batch_first=True)), (65, 2, 1024, 4, dict(half=True)),
    (40, 5, 96, 4, dict(lengths=torch.int32)), (130, 1, 8, 2, dict(silu=False, state=True)),
    (64, 2, 520, 4, dict(params=F32, state=True)), (9, 2, 12, 4, dict(step=2)), (257, 4, 36, 4, dict(half=True, state=True)),
])
def test_causal_conv1d(T, N, D, W, opt, dtype):
    from haste_b200 import ssm
    g = torch.Generator(device="cuda").manual_seed(T * 1000 + N * 100 + D + W)
    p = opt.get("params", dtype)
    d = dict(x=seq(g, T, N, D, dtype, opt.get("batch_first"), opt.get("half"), step=opt.get("step", 1)),
             weight=torch.randn(D, W, generator=g, device="cuda").to(p),
             bias=torch.randn(D, generator=g, device="cuda").to(p) if opt.get("bias", True) else None,
             initial_state=torch.randn(N, W - 1, D, generator=g, device="cuda").to(dtype) if opt.get("state") else None)
    lengths = lens(g, T, N, opt.get("lengths"))
    d["x"] = poison(d["x"], lengths)
    names = leaves(d, ["x", "weight", "bias", "initial_state"])
    dy = poison(seq(g, T, N, D, dtype), lengths)
    dfinal = torch.randn(N, W - 1, D, generator=g, device="cuda").to(dtype)
    y, final = ssm.causal_conv1d(**d, lengths=lengths, silu=opt.get("silu", True))
    got = dict(zip(names, torch.autograd.grad([y, final], [d[k] for k in names], [dy, dfinal])))
    want, major, K = ref.conv(d["x"], d["weight"], d["bias"], d["initial_state"], lengths, opt.get("silu", True), dy, dfinal)
    assert y.dtype == final.dtype == dtype and (y.stride(0) < y.stride(1)) == bool(opt.get("batch_first") and T > 1)
    ref.check(y, want["y"], major["y"], K, "y")
    assert torch.equal(final.double().cpu(), want["final"])  # copies
    for k, name in (("x", "dx"), ("weight", "dweight"), ("bias", "dbias"), ("initial_state", "dstate")):
        if k in got:
            ref.check(got[k], want[name], major[name], K, name)
    # without gradients: the same bits
    with torch.no_grad():
        again = ssm.causal_conv1d(**d, lengths=lengths, silu=opt.get("silu", True))
    assert torch.equal(again[0], y) and torch.equal(again[1], final)


# ------------------------------------------------------------------ selective_scan
def scan_inputs(g, T, N, D, S, G, dtype, opt):
    bf = opt.get("batch_first")
    bc = seq(g, T, N, 2 * G * S + 3, dtype, bf)
    step = torch.rand(D, generator=g, device="cuda") * 0.3 + 0.01
    d = dict(x=seq(g, T, N, D, dtype, bf, opt.get("half")), dt=seq(g, T, N, D, dtype, bf, scale=0.5),
             A=-(torch.rand(D, S, generator=g, device="cuda") * 4 + 0.05),
             B=bc[..., 3:3 + G * S].unflatten(-1, (G, S)), C=bc[..., 3 + G * S:].unflatten(-1, (G, S)))
    if opt.get("D", True):
        d["D"] = torch.randn(D, generator=g, device="cuda")
    if opt.get("z", True):
        d["z"] = seq(g, T, N, D, dtype, bf, opt.get("half"), scale=2.0)
    if opt.get("bias", True):
        d["dt_bias"] = step + torch.log(-torch.expm1(-step))
    if not opt.get("softplus", True):  # steps of the size that softplus would give
        d["dt"] = (d["dt"].float().abs() * 0.3).to(dtype)
        d["dt_bias"] = step
    if opt.get("state"):
        d["initial_state"] = torch.randn(N, D, S, generator=g, device="cuda")
    return d


SCANS = [
    (1, 1, 1, 1, 1, {}), (1, 2, 5, 16, 1, dict(state=True)), (2, 1, 3, 4, 1, dict(z=False, D=False, bias=False)),
    (7, 2, 33, 16, 1, {}), (8, 1, 32, 16, 2, dict(state=True)), (9, 3, 40, 5, 1, dict(state=True, lengths=torch.int64)),
    (16, 2, 64, 8, 1, dict(batch_first=True)), (17, 1, 130, 16, 1, dict(half=True)), (40, 2, 12, 24, 2, dict(state=True)),
    (33, 2, 20, 32, 1, dict(z=False)), (70, 3, 50, 16, 2, dict(lengths=torch.int32, state=True, batch_first=True)),
    (25, 1, 9, 64, 3, dict(D=False)), (66, 1, 7, 128, 1, dict(state=True)), (20, 2, 6, 100, 1, dict(lengths=torch.int64)),
    (37, 2, 48, 16, 1, dict(softplus=False, state=True)), (200, 1, 24, 16, 1, dict(state=True)), (24, 1, 300, 3, 1, {}),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("T,N,D,S,G,opt", SCANS)
def test_selective_scan(T, N, D, S, G, opt, dtype):
    from haste_b200 import ssm
    g = torch.Generator(device="cuda").manual_seed(T * 1000 + N * 100 + D + S)
    d = scan_inputs(g, T, N, D, S, G, dtype, opt)
    lengths = lens(g, T, N, opt.get("lengths"))
    for k in ("x", "dt", "z"):
        if k in d:
            d[k] = poison(d[k], lengths)
    poison(d["B"], lengths)
    poison(d["C"], lengths)
    names = leaves(d, ["x", "dt", "A", "B", "C", "D", "z", "dt_bias", "initial_state"])
    dy = poison(seq(g, T, N, D, dtype, half=True), lengths)
    dfinal = torch.randn(N, D, S, generator=g, device="cuda")
    sp = opt.get("softplus", True)
    y, final = ssm.selective_scan(**d, lengths=lengths, softplus=sp)
    got = dict(zip(names, torch.autograd.grad([y, final], [d[k] for k in names], [dy, dfinal])))
    want, major, K = ref.scan(d["x"], d["dt"], d["A"], d["B"], d["C"], d.get("D"), d.get("z"), d.get("dt_bias"),
                              d.get("initial_state"), lengths, sp, dy, dfinal)
    assert y.dtype == dtype and final.dtype == F32 and (y.stride(0) < y.stride(1)) == bool(opt.get("batch_first") and T > 1)
    ref.check(y, want["y"], major["y"], K, "y")
    ref.check(final, want["final"], major["final"], K, "final")
    for k in names:
        name = "dstate" if k == "initial_state" else "d" + k
        ref.check(got[k], want[name], major[name], K, name)
    with torch.no_grad():
        again = ssm.selective_scan(**d, lengths=lengths, softplus=sp)
    ref.check(again[0], want["y"], major["y"], K, "y without gradients")
    ref.check(again[1], want["final"], major["final"], K, "final without gradients")


# ------------------------------------------------------------------ fused_norm
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("T,N,H,opt", [
    (1, 1, 1, {}), (1, 3, 64, dict(gate=True)), (3, 2, 7, dict(residual=True, bias=True)),
    (5, 1, 250, dict(gate=True, residual=True, scale=True, batch_first=True)), (4, 3, 1024, dict(residual=True, scale=True, bias=True)),
    (3, 2, 1000, dict(gate=True, half=True)), (2, 2, 2050, dict(residual=True, wide=True)), (2, 1, 4096, dict(gate=True, bias=True)),
    (3, 1, 4099, dict(residual=True, scale=True)), (2, 1, 8192, dict(gate=True, residual=True, scale=True, bias=True)),
    (700, 8, 40, dict(residual=True, scale=True, wide=True, params=F32)), (1, 2, 8191, {}),
])
def test_fused_norm(T, N, H, opt, kind, dtype):
    from haste_b200 import ssm
    g = torch.Generator(device="cuda").manual_seed(T * 1000 + N * 100 + H)
    p, bf, half = opt.get("params", dtype), opt.get("batch_first"), opt.get("half")
    rdtype = F32 if opt.get("wide") else dtype
    vec = lambda: torch.randn(H, generator=g, device="cuda").to(p)  # noqa: E731
    d = dict(x=seq(g, T, N, H, dtype, bf, half), weight=vec(), bias=vec() if opt.get("bias") else None,
             gate=seq(g, T, N, H, dtype, bf) if opt.get("gate") else None,
             residual=seq(g, T, N, H, rdtype, False, half) if opt.get("residual") else None,
             scale=vec() if opt.get("scale") else None)
    names = leaves(d, list(d))
    y, r = ssm.fused_norm(**d, kind=kind)
    dy = seq(g, T, N, H, dtype)
    dr = seq(g, T, N, H, rdtype) if r is not None else None
    got = dict(zip(names, torch.autograd.grad([y] + ([] if r is None else [r]), [d[k] for k in names],
                                              [dy] + ([] if r is None else [dr]))))
    want, major, K = ref.norm(d["x"], d["weight"], d["bias"], d["gate"], d["residual"], d["scale"], 1e-5, kind, dy, dr)
    ref.check(y, want["y"], major["y"], K, "y")
    assert (r is None) == (d["residual"] is None)
    if r is not None:
        assert r.dtype == rdtype
        ref.check(r, want["r"], major["r"], K, "r")
    for k in names:
        ref.check(got[k], want["d" + k], major["d" + k], K, "d" + k)
    with torch.no_grad():
        again = ssm.fused_norm(**d, kind=kind)
    assert torch.equal(again[0], y) and (r is None or torch.equal(again[1], r))


# ------------------------------------------------------------------ single tokens
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("N,D,S,G,W", [(1, 1, 1, 1, 2), (1, 1024, 16, 1, 4), (5, 33, 5, 1, 3), (3, 60, 24, 2, 4), (2, 10, 128, 1, 4)])
def test_steps(N, D, S, G, W, dtype):
    from haste_b200 import ssm
    g = torch.Generator(device="cuda").manual_seed(N + D + S)
    x, w, b = seq(g, 1, N, D, dtype, half=True)[0], torch.randn(D, W, generator=g, device="cuda").to(dtype), None
    state = torch.randn(N, W - 1, D, generator=g, device="cuda").to(dtype)
    before = state.clone()
    y, new = ssm.causal_conv1d_step(x, state, w, b)
    want, major, K = ref.conv(x[None], w, b, state, None, True)
    ref.check(y[None], want["y"], major["y"], K, "conv y")
    assert torch.equal(new.double().cpu(), want["final"]) and torch.equal(state, before)
    y2, same = ssm.causal_conv1d_step(x, state, w, b, out_state=state)  # in place
    assert same is state or same.data_ptr() == state.data_ptr()
    assert torch.equal(y2, y) and torch.equal(state, new)

    d = scan_inputs(g, 1, N, D, S, G, dtype, dict(state=True, half=True))
    h = d.pop("initial_state")
    want, major, K = ref.scan(d["x"], d["dt"], d["A"], d["B"], d["C"], d["D"], d["z"], d["dt_bias"], h)
    one = {k: v[0] if k in ("x", "dt", "B", "C", "z") else v for k, v in d.items()}
    y, new = ssm.selective_scan_step(**one, state=h)
    ref.check(y[None], want["y"], major["y"], K, "scan y")
    ref.check(new, want["final"], major["final"], K, "scan state")
    y2, same = ssm.selective_scan_step(**one, state=h, out_state=h)
    assert torch.equal(y2, y) and torch.equal(h, new) and same.data_ptr() == h.data_ptr()
    if G == 1:
        y3, _ = ssm.selective_scan_step(**(one | {k: one[k][:, 0] for k in "BC"}), state=h)
        assert y3.shape == (N, D)


def test_a_step_with_gradients():
    from haste_b200 import ssm
    g = torch.Generator(device="cuda").manual_seed(3)
    x = seq(g, 1, 2, 6, F32)[0].requires_grad_()
    w = torch.randn(6, 4, generator=g, device="cuda")
    state = torch.randn(2, 3, 6, generator=g, device="cuda").requires_grad_()
    y, new = ssm.causal_conv1d_step(x, state, w)
    dy = torch.randn(2, 6, generator=g, device="cuda")
    dx, ds = torch.autograd.grad(y, [x, state], dy)
    want, major, K = ref.conv(x[None], w, None, state, None, True, dy[None])
    ref.check(dx[None], want["dx"], major["dx"], K, "dx")
    ref.check(ds, want["dstate"], major["dstate"], K, "dstate")


# ------------------------------------------------------------------ cut sequences, edges
@pytest.mark.parametrize("cut", [1, 3, 8, 19])
def test_a_sequence_may_be_cut_anywhere(cut):
    """A prompt, the rest of it, and then steps: within the roundings of the whole."""
    from haste_b200 import ssm
    T, N, D, S = 23, 2, 40, 16
    g = torch.Generator(device="cuda").manual_seed(cut)
    d = scan_inputs(g, T, N, D, S, 1, F32, dict(state=True))
    x, w = d["x"], torch.randn(D, 4, generator=g, device="cuda")
    y0, s = ssm.causal_conv1d(x[:cut], w)
    y1, s = ssm.causal_conv1d(x[cut:-2], w, initial_state=s)
    ys = [y0, y1]
    for t in (T - 2, T - 1):
        y, s = ssm.causal_conv1d_step(x[t], s, w)
        ys.append(y[None])
    want, major, K = ref.conv(x, w, None, None, None, True)
    ref.check(torch.cat(ys), want["y"], major["y"], K, "conv")

    h = d.pop("initial_state")
    want, major, K = ref.scan(d["x"], d["dt"], d["A"], d["B"], d["C"], d["D"], d["z"], d["dt_bias"], h)
    part = lambda t: {k: v[t] if k in ("x", "dt", "B", "C", "z") else v for k, v in d.items()}  # noqa: E731
    y0, h = ssm.selective_scan(**part(slice(0, cut)), initial_state=h)
    y1, h = ssm.selective_scan(**part(slice(cut, T - 2)), initial_state=h)
    ys = [y0, y1]
    for t in (T - 2, T - 1):
        y, h = ssm.selective_scan_step(**part(t), state=h)
        ys.append(y[None])
    ref.check(torch.cat(ys), want["y"], major["y"], K, "scan")
    ref.check(h, want["final"], major["final"], K, "scan state")


@pytest.mark.parametrize("T,N", [(0, 2), (3, 0)])
def test_nothing_to_do(T, N):
    from haste_b200 import ssm
    g = torch.Generator(device="cuda").manual_seed(1)
    d = scan_inputs(g, T, N, 6, 4, 1, F32, dict(state=True))
    names = leaves(d, list(d))
    y, final = ssm.selective_scan(**d)
    assert y.shape == (T, N, 6) and torch.equal(final, d["initial_state"])
    dfinal = torch.randn_like(final)
    got = dict(zip(names, torch.autograd.grad([y, final], [d[k] for k in names], [torch.zeros_like(y), dfinal])))
    assert torch.equal(got["initial_state"], dfinal)
    for k in ("A", "D", "dt_bias"):
        assert not got[k].any()
    w = torch.randn(6, 4, device="cuda", requires_grad=True)
    s = torch.randn(N, 3, 6, device="cuda", requires_grad=True)
    y, last = ssm.causal_conv1d(d["x"], w, initial_state=s)
    assert torch.equal(last, s)
    df = torch.randn_like(last)
    dw, ds = torch.autograd.grad([y, last], [w, s], [torch.zeros_like(y), df])
    assert not dw.any() and torch.equal(ds, df)
    weight = torch.ones(6, device="cuda", requires_grad=True)
    y, r = ssm.fused_norm(d["x"], weight, residual=torch.zeros_like(d["x"]))
    assert y.shape == r.shape == (T, N, 6)
    assert not torch.autograd.grad([y], [weight], [torch.zeros_like(y)])[0].any()


def test_only_the_final_state_is_used():
    from haste_b200 import ssm
    g = torch.Generator(device="cuda").manual_seed(5)
    d = scan_inputs(g, 11, 2, 6, 4, 1, F32, {})
    names = leaves(d, list(d))
    _, final = ssm.selective_scan(**d)
    df = torch.randn_like(final)
    got = torch.autograd.grad(final, [d["x"], d["A"]], df)
    want, major, K = ref.scan(d["x"], d["dt"], d["A"], d["B"], d["C"], d["D"], d["z"], d["dt_bias"],
                              dy=torch.zeros(11, 2, 6), dfinal=df)
    ref.check(got[0], want["dx"], major["dx"], K, "dx")
    ref.check(got[1], want["dA"], major["dA"], K, "dA")


def test_broadcast_inputs_get_their_gradients():
    """Expanded inputs (stride 0): autograd sums what the operators return for every place."""
    from haste_b200 import ssm
    g = torch.Generator(device="cuda").manual_seed(6)
    x1 = torch.randn(9, 1, 8, generator=g, device="cuda").requires_grad_()
    w = torch.randn(8, 4, generator=g, device="cuda")
    dy = torch.randn(9, 3, 8, generator=g, device="cuda")
    y, _ = ssm.causal_conv1d(x1.expand(9, 3, 8), w)
    got, = torch.autograd.grad(y, x1, dy)
    want, major, K = ref.conv(x1.expand(9, 3, 8), w, None, None, None, True, dy)
    ref.check(got, want["dx"].sum(1, keepdim=True), major["dx"].sum(1, keepdim=True), K, "dx")


# ------------------------------------------------------------------ streams, graphs, order
def _block(d, w, weight):
    """A run of them as a block has it; returns outputs and all gradients."""
    from haste_b200 import ssm
    u, _ = ssm.causal_conv1d(d["x"], w)
    y, _ = ssm.selective_scan(u, d["dt"], d["A"], d["B"], d["C"], d["D"], None, d["dt_bias"], d["initial_state"])
    o, r = ssm.fused_norm(y, weight, gate=d["z"], residual=d["x"])
    names = [d[k] for k in d] + [w, weight]
    return [o, r, *torch.autograd.grad([o, r], names, [torch.ones_like(o), torch.ones_like(r)])]


def _block_inputs(seed, dtype=F32, T=70, N=3, D=72, S=16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    d = scan_inputs(g, T, N, D, S, 1, dtype, dict(state=True))
    w = torch.randn(D, 4, generator=g, device="cuda").to(dtype).requires_grad_()
    weight = torch.randn(D, generator=g, device="cuda").to(dtype).requires_grad_()
    leaves(d, list(d))
    return d, w, weight


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_block_is_deterministic_on_any_stream(dtype):
    a, b = _block_inputs(1, dtype), _block_inputs(2, dtype)
    torch.cuda.synchronize()
    want_a, want_b = _block(*a), _block(*b)
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(sa):
            got_a = _block(*a)
        with torch.cuda.stream(sb):
            got_b = _block(*b)
        torch.cuda.synchronize()
        for got, want in ((got_a, want_a), (got_b, want_b)):
            for x, y in zip(got, want):
                assert torch.equal(x, y)


def test_a_block_against_the_formulas():
    d, w, weight = _block_inputs(3, T=21, N=2, D=24)
    got = _block(d, w, weight)
    v = {k: t.detach().double().cpu().requires_grad_() for k, t in d.items()}
    wr, nr = (t.detach().double().cpu().requires_grad_() for t in (w, weight))
    T, N, D = v["x"].shape
    padded = torch.cat([torch.zeros(3, N, D, dtype=torch.float64), v["x"]])
    u = torch.nn.functional.silu(sum(padded[k:k + T] * wr[:, k] for k in range(4)))
    delta = torch.nn.functional.softplus(v["dt"] + v["dt_bias"])
    h, ys = v["initial_state"], []
    for t in range(T):
        h = torch.exp(delta[t][..., None] * v["A"]) * h + (delta[t] * u[t])[..., None] * v["B"][t]
        ys.append((h * v["C"][t]).sum(-1) + v["D"] * u[t])
    p = torch.stack(ys) * torch.nn.functional.silu(v["z"])
    r = v["x"] + p
    o = r * torch.rsqrt(r.square().mean(-1, keepdim=True) + 1e-5) * nr
    want = [o, r, *torch.autograd.grad([o.sum() + r.sum()], list(v.values()) + [wr, nr])]
    for x, y in zip(got, want):
        # three operators after one another, each within a few hundred roundings of its terms
        assert (x.double().cpu() - y).abs().max() <= 2000 * ref.U * y.abs().max()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_captured_block_replays(dtype):
    a, b = _block_inputs(4, dtype), _block_inputs(5, dtype)
    # detached: an eager graph of the same leaves must not live while torch captures their backward pass
    want_a, want_b = ([t.detach().clone() for t in _block(*v)] for v in (a, b))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _block(*a)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for inputs in (a, b):  # two graphs side by side: nothing that they work on is shared
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _block(*inputs)
        graphs.append((graph, out))
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        torch.cuda.synchronize()
        with torch.cuda.stream(s1):
            graphs[0][0].replay()
        with torch.cuda.stream(s2):
            graphs[1][0].replay()
        torch.cuda.synchronize()
        for (_, out), want in zip(graphs, (want_a, want_b)):
            for x, y in zip(out, want):
                assert torch.equal(x, y)


def test_captured_steps_update_their_state_in_place():
    from haste_b200 import ssm
    g = torch.Generator(device="cuda").manual_seed(8)
    N, D, S, steps = 3, 40, 16, 5
    d = scan_inputs(g, steps, N, D, S, 1, F32, dict(state=True))
    h = d.pop("initial_state")
    w, cs = torch.randn(D, 4, generator=g, device="cuda"), torch.zeros(N, 3, D, device="cuda")
    at = lambda t: {k: v[t] if k in ("x", "dt", "B", "C", "z") else v for k, v in d.items()}  # noqa: E731
    now = {k: v.clone() for k, v in at(0).items()}

    def step(h, cs):
        u, _ = ssm.causal_conv1d_step(now["x"], cs, w, out_state=cs)
        return ssm.selective_scan_step(**(now | {"x": u}), state=h, out_state=h)[0]

    hw, cw = h.clone(), cs.clone()
    want = []
    for t in range(steps):
        for k, v in at(t).items():
            now[k].copy_(v)
        want.append(step(hw, cw).clone())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(h.clone(), cs.clone())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step(h, cs)
    for t in range(steps):
        for k, v in at(t).items():
            now[k].copy_(v)
        graph.replay()
        assert torch.equal(y, want[t])
    assert torch.equal(h, hw) and torch.equal(cs, cw)


def test_saved_tensors_that_changed_are_noticed():
    from haste_b200 import ssm
    d, w, weight = _block_inputs(7)
    y, _ = ssm.causal_conv1d(d["x"], w)
    with torch.no_grad():
        d["x"].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_offsets_beyond_32_bits():
    """The last rows of sequences of more than 2^31 values, against the same rows on their own."""
    from haste_b200 import ssm
    T, D = (1 << 20) + 40, 2056  # 2.16 G values
    x = torch.empty(T, 1, D, dtype=BF16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(11)
    for i in range(0, T, 1 << 17):
        x[i:i + (1 << 17)] = torch.randn(min(1 << 17, T - i), 1, D, generator=g, device="cuda").to(BF16)
    w = torch.randn(D, 4, generator=g, device="cuda").to(BF16)
    y, state = ssm.causal_conv1d(x, w)
    assert torch.equal(state[0], x[-3:, 0])
    tail, _ = ssm.causal_conv1d(x[-100:], w, initial_state=x[-103:-100].transpose(0, 1))
    assert torch.equal(y[-100:], tail)
    del y
    weight = torch.randn(D, generator=g, device="cuda").to(BF16)
    o, _ = ssm.fused_norm(x, weight)
    assert torch.equal(o[-100:], ssm.fused_norm(x[-100:], weight)[0])
    del o
    A = -torch.rand(D, 4, generator=g, device="cuda") - 2.0
    bc = torch.randn(T, 1, 4, generator=g, device="cuda").to(BF16)
    bias = torch.full((D,), 3.0, device="cuda")  # steps of 3: a state is gone (exp(-6 a step)) after 20
    y, state = ssm.selective_scan(x, x, A, bc, bc, dt_bias=bias)
    tail, last = ssm.selective_scan(x[-200:], x[-200:], A, bc[-200:], bc[-200:], dt_bias=bias)
    off = (y[-100:].float() - tail[-100:].float()).abs().max()
    assert off <= 2 ** -7 * tail[-100:].float().abs().max()
    assert (state - last).abs().max() <= 1e-5 * last.abs().max()


# ------------------------------------------------------------------ automatic differentiation
def _calls(g, dtype=F32):
    """One call of each operator: (function of its first input, that input)."""
    from haste_b200 import ssm
    d = scan_inputs(g, 5, 2, 8, 4, 1, dtype, {})
    x = d.pop("x")
    w, weight = torch.randn(8, 4, generator=g, device="cuda").to(dtype), torch.randn(8, generator=g, device="cuda").to(dtype)
    return [(lambda v: ssm.causal_conv1d(v, w)[0], x), (lambda v: ssm.selective_scan(v, **d)[0], x),
            (lambda v: ssm.fused_norm(v, weight, gate=d["z"])[0], x)]


def test_a_second_derivative_is_refused():
    g = torch.Generator(device="cuda").manual_seed(1)
    for call, x in _calls(g):
        x = x.detach().requires_grad_()
        dx, = torch.autograd.grad(call(x).square().sum(), x, create_graph=True)
        again, = torch.autograd.grad(call(x).square().sum(), x)
        assert torch.equal(dx, again)
        with pytest.raises(RuntimeError, match="differentiate.* twice"):
            dx.sum().backward()


def test_forward_mode_and_tracing_are_refused_or_right():
    import torch.autograd.forward_ad as forward_ad
    g = torch.Generator(device="cuda").manual_seed(2)
    for call, x in _calls(g):
        with forward_ad.dual_level():
            call(x)
            with pytest.raises(NotImplementedError):
                call(forward_ad.make_dual(x, torch.ones_like(x)))
        try:
            traced = torch.jit.trace(call, x, check_trace=False)
        except RuntimeError:
            continue
        other = torch.randn_like(x)
        torch.testing.assert_close(traced(other), call(other))


def test_saved_tensors_may_move():
    d, w, weight = _block_inputs(9)
    want = _block(d, w, weight)
    with torch.autograd.graph.save_on_cpu():
        got = _block(d, w, weight)
    for x, y in zip(got, want):
        assert torch.equal(x, y)


def test_frozen_parameters():
    """Only some inputs want gradients; the others' are dropped."""
    from haste_b200 import ssm
    g = torch.Generator(device="cuda").manual_seed(4)
    d = scan_inputs(g, 19, 2, 24, 16, 1, BF16, dict(state=True))
    full = {k: v.detach().requires_grad_() for k, v in d.items()}
    dy = seq(g, 19, 2, 24, BF16)
    want = torch.autograd.grad(ssm.selective_scan(**full)[0], [full["dt"], full["B"]], dy)
    some = d | {"dt": d["dt"].detach().requires_grad_(), "B": d["B"].detach().requires_grad_()}
    got = torch.autograd.grad(ssm.selective_scan(**some)[0], [some["dt"], some["B"]], dy)
    for x, y in zip(got, want):
        assert torch.equal(x, y)


def test_checkpointed_and_repeated_backward():
    from torch.utils.checkpoint import checkpoint
    g = torch.Generator(device="cuda").manual_seed(5)
    for call, x in _calls(g):
        x = x.detach().requires_grad_()
        y = call(x)
        a, = torch.autograd.grad(y.sum(), x, retain_graph=True)
        b, = torch.autograd.grad(y.sum(), x)
        c, = torch.autograd.grad(checkpoint(call, x, use_reentrant=False).sum(), x)
        assert torch.equal(a, b) and torch.equal(a, c)


def test_library_errors_keep_their_type():
    from haste_b200 import _C
    with pytest.raises(_C.HasteError, match="dtype"):
        _C.call("haste_b200_causal_conv1d_forward", b"\x07" * 512, None)


# ------------------------------------------------------------------ buffers of the caller's, large scratch
def test_out_state_is_checked_and_counted():
    from haste_b200 import ssm
    g = torch.Generator(device="cuda").manual_seed(6)
    w = torch.randn(8, 4, generator=g, device="cuda")
    pool = torch.randn(4, 3, 8, generator=g, device="cuda")
    x = torch.randn(2, 8, generator=g, device="cuda")
    with pytest.raises(ValueError, match="lies over"):  # one row further than the state
        ssm.causal_conv1d_step(x, pool[:2], w, out_state=pool[1:3])
    with pytest.raises(ValueError, match="contiguous"):
        ssm.causal_conv1d_step(x, pool[:2], w, out_state=torch.empty(3, 2, 8, device="cuda").transpose(0, 1))
    with pytest.raises(ValueError, match="wrong shape"):
        ssm.causal_conv1d_step(x, pool[:2], w, out_state=pool)
    y0, s0 = ssm.causal_conv1d_step(x, pool[:2], w)
    y1, s1 = ssm.causal_conv1d_step(x, pool[:2], w, out_state=pool[2:])  # another part of the pool
    assert torch.equal(y0, y1) and torch.equal(s0, pool[2:]) and s1.data_ptr() == pool[2:].data_ptr()
    y, _ = ssm.causal_conv1d(x[None], w.requires_grad_(), initial_state=pool[:2])
    with torch.no_grad():
        ssm.causal_conv1d_step(x, pool[:2], w, out_state=pool[:2])
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()
    with torch.inference_mode():
        s = pool[:2].clone()
        ssm.causal_conv1d_step(x, s, w, out_state=s)
    h = torch.randn(2, 8, 4, generator=g, device="cuda")
    A = -torch.rand(8, 4, generator=g, device="cuda")
    with pytest.raises(ValueError, match="lies over"):
        ssm.selective_scan_step(x, x, A, h[:, 0], h[:, 1], h, out_state=h)


def test_many_states_take_the_rows_in_turn():
    """dB and dC of 128 states: more than a GB of partial sums for the whole batch."""
    from haste_b200 import ssm
    T, N, D, S = 1900, 26, 256, 128
    g = torch.Generator(device="cuda").manual_seed(12)
    d = scan_inputs(g, T, N, D, S, 1, BF16, dict(z=False))
    leaves(d, ["B", "C", "A", "dt"])
    dy = seq(g, T, N, D, BF16)
    got = torch.autograd.grad(ssm.selective_scan(**d)[0], [d["B"], d["C"], d["dt"], d["A"]], dy)
    total = 0.0
    for rows in (slice(0, 3), slice(3, 20), slice(20, 26)):
        part = {k: v[:, rows].detach().requires_grad_() if k in ("B", "C", "dt") else v.detach().requires_grad_(k == "A") if k == "A"
                else v[:, rows] if v.dim() > 2 else v for k, v in d.items()}
        want = torch.autograd.grad(ssm.selective_scan(**part)[0], [part["B"], part["C"], part["dt"], part["A"]], dy[:, rows])
        for x, y in zip(got[:3], want[:3]):
            # pieces differ with the batch: both within their roundings of bf16's half step, twice 2^-9
            assert (x[:, rows].float() - y.float()).abs().max() <= 2 ** -8 * y.float().abs().max()
        total = total + want[3]
    assert (got[3] - total).abs().max() <= 1e-4 * total.abs().max()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("T,N,H,opt", [
    (37, 5, 100, dict(gate=True, residual=True, scale=True, bias=True)), (9, 3, 128, dict(residual=True, scale=True)),
    (50, 7, 33, dict(gate=True, batch_first=True)), (1, 17, 63, dict(bias=True)), (600, 40, 64, dict(residual=True, scale=True)),
    (4, 9, 129, dict(gate=True)), (3, 5, 2, dict(residual=True, wide=True)),
])
def test_fused_norm_of_short_rows(T, N, H, opt, kind, dtype):
    """Rows that share a warp, and blocks whose last rows do not exist."""
    test_fused_norm(T, N, H, opt, kind, dtype)


# ------------------------------------------------------------------ rows that end early, pieces, states in place
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,N,D,S,G,opt", [
    (300, 3, 24, 16, 1, dict(lengths=torch.int64, state=True)), (260, 5, 10, 5, 1, dict(lengths=torch.int64, batch_first=True)),
    (530, 2, 33, 32, 1, dict(lengths=torch.int32, state=True, z=False)), (400, 4, 6, 100, 2, dict(lengths=torch.int64, state=True)),
    (333, 2, 250, 3, 1, dict(state=True)),
])
def test_selective_scan_in_pieces(T, N, D, S, G, opt, dtype):
    """Few channels, long sequences: pieces, some of them behind the rows' ends."""
    test_selective_scan(T, N, D, S, G, opt, dtype)


@pytest.mark.parametrize("T", [24, 200, 5000])
def test_steps_behind_the_end_leave_the_state_alone(T):
    """However many there are.  A row without steps keeps its bits: a piece of no steps multiplies by
    exp(0) and adds zero.  A row with steps keeps them only while one piece holds the whole sequence: joined
    pieces take exp(A (d1 + d2 + ..)) h + e, rounded elsewhere than the product of the steps' decays."""
    from haste_b200 import ssm
    g = torch.Generator(device="cuda").manual_seed(13)
    N, D, S = 3, 20, 16
    d = scan_inputs(g, 5000, N, D, S, 1, F32, dict(state=True))
    short = {k: v[:16] if v.dim() > 2 and v.shape[0] == 5000 else v for k, v in d.items()}
    cut = {k: v[:T] if v.dim() > 2 and v.shape[0] == 5000 else v for k, v in d.items()}
    lengths = torch.tensor([11, 0, 16], device="cuda")
    want = ssm.selective_scan(**short, lengths=lengths)
    y, final = ssm.selective_scan(**cut, lengths=lengths)
    assert torch.equal(final[1], d["initial_state"][1])
    exact, major, K = ref.scan(*[short[k] for k in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "initial_state")], lengths)
    ref.check(final, exact["final"], major["final"], K, "final_state")
    assert T > 24 or torch.equal(final, want[1])
    assert torch.equal(y[:16], want[0]) and not y[16:].any()
    h = d["initial_state"].clone().requires_grad_()
    df = torch.randn(N, D, S, generator=g, device="cuda")
    cut["initial_state"] = h
    dh, = torch.autograd.grad(ssm.selective_scan(**cut, lengths=torch.zeros(N, dtype=torch.long, device="cuda"))[1], h, df)
    assert torch.equal(dh, df)


def test_a_long_prompt_may_leave_its_state_in_place():
    """Through the native call: pieces all start from the initial state, so it must outlive them."""
    from haste_b200 import _C
    g = torch.Generator(device="cuda").manual_seed(14)
    T, N, D, S = 900, 1, 64, 16
    d = scan_inputs(g, T, N, D, S, 1, F32, dict(state=True))
    h = d["initial_state"]
    args = [d["x"], d["dt"], d["A"], d["B"], d["C"], d["D"], d["z"], d["dt_bias"]]
    want, major, K = ref.scan(*args, h)
    for _ in range(5):
        state = h.clone()
        y, last, _ = _C.native().selective_scan_forward(*args, state, None, True, False, state)
        assert last.data_ptr() == state.data_ptr()
        ref.check(y, want["y"], major["y"], K, "y")
        ref.check(state, want["final"], major["final"], K, "state")
    x = torch.randn(900, 2, 8, generator=g, device="cuda")
    w = torch.randn(8, 4, generator=g, device="cuda")
    s = torch.randn(2, 3, 8, generator=g, device="cuda")
    y0, last = _C.native().causal_conv1d_forward(x, w, None, s, None, True, None)
    y1, _ = _C.native().causal_conv1d_forward(x, w, None, s, None, True, s)
    assert torch.equal(y0, y1) and torch.equal(s, last)


# ------------------------------------------------------------------ values that are not numbers, overflow
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,D,W", [(5, 7, 4), (40, 64, 3), (33, 20, 2)])
def test_a_row_without_steps_adds_nothing_to_the_taps_gradients(T, D, W, dtype):
    """Its state goes through to the final state, whatever it holds, and takes part in nothing else."""
    from haste_b200 import ssm
    g = torch.Generator(device="cuda").manual_seed(15)
    N = 3
    lengths = torch.tensor([T, 0, T // 2], device="cuda")
    x = poison(seq(g, T, N, D, dtype), lengths)
    state = torch.randn(N, W - 1, D, generator=g, device="cuda").to(dtype)
    state[1] = float("nan")
    state[1, 0, ::2] = float("inf")
    w, b = torch.randn(D, W, generator=g, device="cuda").to(dtype), torch.randn(D, generator=g, device="cuda").to(dtype)
    d = dict(x=x, weight=w, bias=b, initial_state=state)
    names = leaves(d, list(d))
    dy = seq(g, T, N, D, dtype)
    y, final = ssm.causal_conv1d(**d, lengths=lengths)
    got = dict(zip(names, torch.autograd.grad(y, [d[k] for k in names], dy)))
    want, major, K = ref.conv(x, w, b, state, lengths, True, dy)
    ref.check(y, want["y"], major["y"], K, "y")
    assert torch.equal(final[1].isnan(), state[1].isnan()) and torch.equal(final[1].isinf(), state[1].isinf())
    for k, name in (("x", "dx"), ("weight", "dweight"), ("bias", "dbias"), ("initial_state", "dstate")):
        ref.check(got[k], want[name], major[name], K, name)


def test_the_last_input_meets_no_step_behind_it():
    """Without SiLU an infinite last input reaches the gradient of the last tap alone."""
    from haste_b200 import ssm
    g = torch.Generator(device="cuda").manual_seed(16)
    T, N, D, W = 12, 2, 8, 4
    lengths = torch.tensor([T, 6], device="cuda")
    x, w, dy = seq(g, T, N, D, F32), torch.randn(D, W, generator=g, device="cuda").requires_grad_(), seq(g, T, N, D, F32)
    x[5, 1, 3] = float("inf")
    got, = torch.autograd.grad(ssm.causal_conv1d(x, w, lengths=lengths, silu=False)[0], w, dy)
    want, major, K = ref.conv(x, w, None, None, lengths, False, dy)
    assert got[3, 3].isinf()
    got[3, 3] = 0.0
    for r in (want, major):
        r["dweight"][3, 3] = 0.0
    ref.check(got, want["dweight"], major["dweight"], K, "dweight")


@pytest.mark.parametrize("S,gate", [(16, True), (5, False)])
def test_pieces_with_states_that_grow(S, gate):
    """Decays above one: over a piece their product may leave float32 although no state does.  Nothing
    comes in before the last steps, no gradient behind the first ones: all results are finite, those
    of the pieces in between zero."""
    from haste_b200 import ssm
    g = torch.Generator(device="cuda").manual_seed(17)
    T, N, D = 900, 1, 64
    x, z, dy = (torch.randn(T, N, D, generator=g, device="cuda") for _ in range(3))
    B, C = (torch.randn(T, N, 1, S, generator=g, device="cuda") for _ in range(2))
    x[:-10] = 0.0
    dy[10:] = 0.0
    d = dict(x=x, dt=torch.rand(T, N, D, generator=g, device="cuda") * 0.1 + 0.95, B=B, C=C,
             A=torch.rand(D, S, generator=g, device="cuda") * 0.5 + 2.0)
    if gate:
        d["z"] = z
    names = leaves(d, list(d))
    y, final = ssm.selective_scan(**d, softplus=False)
    got = dict(zip(names, torch.autograd.grad(y, [d[k] for k in names], dy)))
    want, major, K = ref.scan(x, d["dt"], d["A"], B, C, None, d.get("z"), softplus=False, dy=dy)
    ref.check(y, want["y"], major["y"], K, "y")
    ref.check(final, want["final"], major["final"], K, "final")
    for k in names:
        ref.check(got[k], want["d" + k], major["d" + k], K, "d" + k)


def test_a_small_state_that_grows_through_pieces():
    """exp(A sum of delta) of a piece beyond float32 (e^110), the state that it meets e^-60."""
    from haste_b200 import ssm
    T, N, D, S = 192, 1, 8, 4
    one = torch.ones(T, N, D, device="cuda")
    A = torch.full((D, S), 110.0 / 64, device="cuda")  # 64 steps of 1
    h = torch.full((N, D, S), 1e-26, device="cuda")
    dt = one.clone()
    dt[64:] = -0.5  # and back: e^(110 - 60 - 110) in the end
    bc = torch.ones(T, N, 1, S, device="cuda")
    y, final = ssm.selective_scan(0 * one, dt, A, bc, bc, initial_state=h, softplus=False)
    want, major, K = ref.scan(0 * one, dt, A, bc, bc, state=h, softplus=False)
    ref.check(y, want["y"], major["y"], K, "y")
    ref.check(final, want["final"], major["final"], K, "final")


@pytest.mark.parametrize("D", [6, 40])
@pytest.mark.parametrize("gate", [True, False])
def test_gradients_behind_the_end_are_zero_whatever_the_state(gate, D):
    """A state that overflowed at the last step: the gradients behind it stay zero, and no other channel
    notices.  (The channel's own dA takes 0 times that state from the steps behind, as the formula does.)"""
    from haste_b200 import ssm
    g = torch.Generator(device="cuda").manual_seed(18)
    T, N, S = 24, 2, 16
    d = scan_inputs(g, T, N, D, S, 1, F32, dict(z=gate))
    lengths = torch.tensor([13, T], device="cuda")
    d["x"][12, 0, 1] = float("inf")
    names = leaves(d, list(d))
    dy = seq(g, T, N, D, F32)
    y, final = ssm.selective_scan(**d, lengths=lengths)
    assert final[0, 1].isinf().any() and not y[13:, 0].any()
    got = dict(zip(names, torch.autograd.grad(y, [d[k] for k in names], dy)))
    for k in ("x", "dt", "B", "C") + (("z",) if gate else ()):
        assert not got[k][13:, 0].any(), k
    d["x"].detach()[12, 0, 1] = 0.0
    rest = [n for n in range(D) if n != 1]
    want, major, K = ref.scan(d["x"], d["dt"], d["A"], d["B"], d["C"], d["D"], d.get("z"), d["dt_bias"], None, lengths, dy=dy)
    ref.check(got["A"][rest], want["dA"][rest], major["dA"][rest], K, "dA")
    ref.check(got["x"][..., rest], want["dx"][..., rest], major["dx"][..., rest], K, "dx")


def test_traced_calls_follow_their_input():
    """The tracer records the call itself: another input gives that input's results and gradients."""
    g = torch.Generator(device="cuda").manual_seed(19)
    for call, x in _calls(g):
        traced = torch.jit.trace(call, x, check_trace=False)
        other = torch.randn(x.shape, generator=g, device="cuda").requires_grad_()
        got, want = traced(other), call(other)
        assert torch.equal(got, want) and not torch.equal(got, call(x))
        for a, b in zip(torch.autograd.grad(got.sum(), other), torch.autograd.grad(want.sum(), other)):
            assert torch.equal(a, b)


def test_outputs_lie_like_batch_first_inputs_of_any_stride():
    """Batch-first, every second channel: the copy that the kernels read is batch-first too."""
    from haste_b200 import ssm
    g = torch.Generator(device="cuda").manual_seed(20)
    T, N, D, S = 6, 3, 8, 4
    x = seq(g, T, N, D, F32, batch_first=True, step=2).requires_grad_()
    w, weight = torch.randn(D, 3, generator=g, device="cuda"), torch.randn(D, generator=g, device="cuda")
    A, bc = -torch.rand(D, S, generator=g, device="cuda"), seq(g, T, N, 2 * S, F32, batch_first=True, step=2)
    dense = x.detach().contiguous().requires_grad_()
    for call in (lambda v: ssm.causal_conv1d(v, w)[0], lambda v: ssm.fused_norm(v, weight, residual=v)[0],
                 lambda v: ssm.selective_scan(v, v, A, bc[..., :S], bc[..., S:])[0]):
        y, want = call(x), call(dense)
        assert torch.equal(y, want) and y.transpose(0, 1).is_contiguous() and want.is_contiguous()
        for a, b in zip(torch.autograd.grad(y.square().sum(), x), torch.autograd.grad(want.square().sum(), dense)):
            assert torch.equal(a, b)
