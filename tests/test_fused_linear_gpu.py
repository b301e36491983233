"""Projections with bias, activation and residual against float64, element by element within the roundings that float32
sums, the activations and the types may make."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24
# (gelu by the complementary error function: 1 + erf has no digits left at -9, in 64 bits too)
ACTS = {None: lambda p: p, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": lambda p: 0.5 * p * torch.erfc(-p / math.sqrt(2)),
        "tanh": torch.tanh, "sigmoid": torch.sigmoid}
CURVE = {None: 0.0, "relu": 0.0, "silu": 0.5, "gelu": 0.8, "tanh": 0.77, "sigmoid": 0.1}  # most of the second derivative


def half(t):
    return torch.finfo(t).eps / 2 if t != F32 else U


def sums(n):
    """Roundings of a sum of n products on the tensor cores, which cut sums off: twice a rounding each.  fp32 operands in three
    bf16 planes drop products of 2^-24 of a term; the 32 hold that and what the planes and parts add."""
    return (n + 32) * 2 * U


def reference(x, w, b, act, residual, dy, dtype, out):
    """(results, errors) in float64 on the device, rows flattened."""
    x, w, dy = (t.detach().double() for t in (x, w, dy))
    rows = x.reshape(-1, x.shape[-1])
    p = rows @ w.t() + (b.detach().double() if b is not None else 0.0)
    ep = sums(x.shape[-1]) * (rows.abs() @ w.t().abs()) + 2 * U * p.abs() + (U * b.detach().double().abs() if b is not None else 0.0)
    q = p.clone().requires_grad_()
    f = ACTS[act](q)
    d1 = torch.autograd.grad(f.sum(), q)[0]
    f = f.detach()
    # exponentials: 4 U and the rounding of their argument, |p| U (gelu: p^2 U), and the few operations around them, the
    # approximation of the normal distribution (1.2e-7 of its value) among them
    own = (24 + 2 * p.abs() + (p * p if act == "gelu" else 0.0)) * U
    ey = d1.abs() * ep + 0.5 * CURVE[act] * ep * ep + (own * f.abs() if act not in (None, "relu") else 0.0)
    if act == "gelu":
        ey = ey + 2 * U * p.abs() * torch.exp(-p * p / 2)  # 1 - tail
    y = f
    if residual is not None:
        y = y + residual.detach().double().reshape(y.shape)
        ey = ey + U * (f.abs() + y.abs())
    ey = ey + half(out) * (y.abs() + ey) + (torch.finfo(out).smallest_normal * torch.finfo(out).eps if out != F32 else 0.0)
    dyr = dy.reshape(y.shape)
    dp = dyr * d1
    kept = (half(dtype) if dtype != F32 else 0.0) * p.abs() + (torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps if dtype != F32 else 0.0)
    if act == "relu":
        es = (p.abs() <= ep).double()
    elif act is None:
        es = torch.zeros_like(p)
    else:
        es = CURVE[act] * (ep + kept) + own * (1.0 + p.abs() * torch.exp(-p * p / 2) if act == "gelu" else 1.0)
        if act in ("tanh", "sigmoid"):  # products of exponentials: relative
            es = CURVE[act] * (ep + kept) + 2 * own * d1.abs()
    ed = dyr.abs() * es + U * dp.abs()
    if act is not None or out != dtype:
        ed = ed + half(dtype) * (dp.abs() + ed) + (torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps if dtype != F32 else 0.0)
    got = {"y": y, "dx": dp @ w, "dweight": dp.t() @ rows, "dbias": dp.sum(0)}
    H, M = w.shape[0], rows.shape[0]
    big = dp.abs() + ed
    err = {"y": ey, "dx": ed @ w.abs() + sums(H) * (big @ w.abs()), "dweight": ed.t() @ rows.abs() + sums(M) * (big.t() @ rows.abs()),
           "dbias": ed.sum(0) + (M + 8) * U * big.sum(0)}
    return got, err


def check(name, got, want, err, dtype):
    want, err = want.reshape(got.shape), err.reshape(got.shape)
    if name != "y" and dtype != F32:
        err = err + half(dtype) * (want.abs() + err) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    off = (got.detach().double() - want).abs()
    bad = ~(off <= err * 1.01 + 2.0 ** -140)
    if bad.any():
        i = int((off / err).nan_to_num(nan=math.inf).argmax())
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} off; at {i}: got {got.flatten()[i].item()}, want "
                             f"{want.flatten()[i].item()}, allowed {err.flatten()[i].item():.3g}")


def run(shape, C, H, act, dtype, opt, seed=0):
    from haste_b200 import ssm
    g = torch.Generator(device="cuda").manual_seed(seed + 7 * C + H)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    layout = opt.get("layout")

    def rows(width, t, scale=1.0):
        if layout == "batch_first":
            return (rand(shape[1], shape[0], width) * scale).to(t).transpose(0, 1)
        if layout == "half":
            return (rand(*shape, 2 * width) * scale).to(t)[..., width:]
        if layout == "odd":
            return (rand(*shape, width + 3) * scale).to(t)[..., 1:1 + width]
        if layout == "strided":
            return (rand(*shape, 2 * width) * scale).to(t)[..., ::2]
        return (rand(*shape, width) * scale).to(t)

    out = F32 if opt.get("residual") == "fp32" else dtype
    x, w = rows(C, dtype), (rand(H, C) / math.sqrt(C)).to(dtype)
    b = rand(H).to(F32 if opt.get("bias") == "fp32" else dtype) if opt.get("bias", True) else None
    residual = rows(H, out, 2.0) if opt.get("residual") else None
    leaf = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b, residual)]
    dy = rows(H, out)
    y = ssm.fused_linear(leaf[0], leaf[1], leaf[2], activation=act, residual=leaf[3])
    assert y.shape == (*shape, H) and y.dtype == out
    if layout == "batch_first" and shape[0] > 1 and shape[1] > 1:
        assert y.stride(0) < y.stride(1)
    given = [t for t in leaf if t is not None]
    grads = iter(torch.autograd.grad(y, given, dy))
    got = dict(zip(("dx", "dweight", "dbias", "dresidual"), (None if t is None else next(grads) for t in leaf)))
    want, err = reference(x, w, b, act, residual, dy, dtype, out)
    check("y", y, want["y"], err["y"], out)
    for k in ("dx", "dweight", "dbias"):
        if got[k] is not None:
            check(k, got[k], want[k], err[k], got[k].dtype)
    if residual is not None:
        assert torch.equal(got["dresidual"], dy)
    with torch.no_grad():
        again = ssm.fused_linear(x, w, b, activation=act, residual=residual)
    assert torch.equal(again, y)
    return y


CASES = [
    ((1,), 1, 1, None, {}), ((1,), 8, 16, "relu", dict(residual=True)), ((2,), 7, 5, "silu", {}), ((3, 2), 64, 100, "gelu", dict(residual=True)),
    ((8,), 1024, 250, "tanh", dict(bias="fp32")), ((9,), 250, 1000, "sigmoid", dict(residual="fp32")), ((16,), 512, 33, "silu", dict(layout="half")),
    ((31,), 100, 128, None, dict(residual=True, layout="half")), ((4, 8), 4096, 1024, "silu", dict(residual=True)), ((33,), 40, 17, "gelu", dict(layout="odd")),
    ((64,), 33, 65, "relu", {}), ((1,), 1024, 4096, "silu", {}), ((65,), 64, 64, "silu", dict(residual="fp32")), ((5, 13, 2), 96, 200, "gelu", {}),
    ((130,), 1, 70, "tanh", dict(bias=False)), ((150,), 70, 1, "sigmoid", {}), ((70, 3), 129, 257, "silu", dict(layout="batch_first", residual=True)),
    ((300,), 512, 384, "relu", dict(layout="strided")), ((77, 4), 1000, 24, None, dict(bias=False, residual="fp32", layout="odd")),
    ((1000,), 250, 333, "gelu", dict(bias="fp32", layout="half")), ((40, 9), 2048, 130, "tanh", dict(layout="batch_first")),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape,C,H,act,opt", CASES)
def test_fused_linear(shape, C, H, act, opt, dtype):
    run(shape, C, H, act, dtype, opt)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape,C,H,act,opt", [
    ((2050,), 1024, 2048, "silu", {}), ((500, 9), 1032, 1000, "gelu", dict(residual=True, layout="batch_first")),
    ((3000,), 1537, 2047, "tanh", dict(residual="fp32")), ((16000,), 512, 512, None, {}), ((300,), 8192, 256, "relu", {}),
])
def test_sizes_that_pairs_and_splits_take(shape, C, H, act, opt, dtype):
    run(shape, C, H, act, dtype, opt)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("act", [a for a in ACTS if a])
@pytest.mark.parametrize("M", [8, 300])
def test_sums_far_from_zero(M, act, dtype):
    """Sums up to hundreds, and infinite and NaN ones: what the formulas have there (minus infinity times zero is a NaN)."""
    from haste_b200 import ssm
    v = torch.tensor([0.0, 1e-6, -1e-6, 0.2, -0.3, 3.0, -4.0, 9.0, -9.0, 30.0, -30.0, 100.0, -100.0, math.inf, -math.inf, math.nan], device="cuda")
    x = torch.zeros(M, 16, device="cuda", dtype=dtype)
    x[:, 0] = 1
    w = torch.zeros(16, 16, device="cuda", dtype=dtype).requires_grad_()
    bias = v.clone().requires_grad_()
    y = ssm.fused_linear(x, w, bias, activation=act)
    want = ACTS[act](bias.double())
    (d,) = torch.autograd.grad(want.sum(), bias)
    lines = y.detach().double()
    assert torch.equal(lines, lines[:1].expand_as(lines)) or lines.isnan().any()
    finite = want.isfinite()
    # (the roundings of the derivation above; 16 bits keep v itself to half a step, which moves a slope by that times 0.8)
    size = v.abs().nan_to_num(nan=0.0, posinf=0.0)  # (an infinite sum leaves no rounding)
    allowed = (24 + size ** 2) * U * want.abs() + half(dtype) * want.abs() + 1e-37
    assert ((lines[0] - want).abs() <= allowed)[finite].all(), (lines[0], want)
    assert torch.equal(lines[0][~finite].isnan(), want[~finite].isnan()) and torch.equal(lines[0][13], want[13])
    (db,) = torch.autograd.grad(y.sum(), bias)
    d, size = d[:13], size[:13]
    allowed = M * (0.8 * size * half(dtype) + (half(dtype) + 300 * U) * (d.abs() + 0.01))
    assert ((db[:13].double() - M * d).abs() <= allowed).all(), (db, M * d)
    assert db[15].isnan()


def test_one_dimension_rows_that_repeat_and_no_rows():
    from haste_b200 import ssm
    g = torch.Generator(device="cuda").manual_seed(1)
    w, b = torch.randn(24, 40, generator=g, device="cuda"), torch.randn(24, generator=g, device="cuda")
    x = torch.randn(40, generator=g, device="cuda")
    one = ssm.fused_linear(x, w, b, activation="silu")
    assert one.shape == (24,)
    many = ssm.fused_linear(x.expand(5, 40), w, b, activation="silu")
    assert torch.equal(many, one.expand(5, 24))
    for rows in (3, 100):
        x3, w2 = torch.randn(rows, 1, 40, device="cuda", requires_grad=True), w.clone().requires_grad_()
        y = ssm.fused_linear(x3, w2, b)
        dx, dw = torch.autograd.grad(y.sum(), [x3, w2])  # a gradient that is one value, expanded
        assert torch.allclose(dx, w.sum(0).expand_as(x3), atol=1e-4) and torch.allclose(dw, x3.sum((0, 1)).expand_as(w), atol=1e-3)
    x0, w0, b0 = torch.zeros(0, 7, 40, device="cuda", requires_grad=True), w.clone().requires_grad_(), b.clone().requires_grad_()
    y = ssm.fused_linear(x0, w0, b0, activation="gelu")
    assert y.shape == (0, 7, 24)
    dx, dw, db = torch.autograd.grad(y.sum(), [x0, w0, b0])
    assert dx.shape == x0.shape and not dw.any() and not db.any()


def test_only_wanted_gradients_and_second_derivatives():
    from haste_b200 import ssm
    x, w, b = (torch.randn(*s, device="cuda", requires_grad=True) for s in ((70, 32), (48, 32), (48,)))
    full = torch.autograd.grad(ssm.fused_linear(x, w, b, activation="silu").sum(), [x, w, b])
    for which in range(3):
        leaf = [t.detach().requires_grad_(i == which) for i, t in enumerate((x, w, b))]
        (d,) = torch.autograd.grad(ssm.fused_linear(*leaf, activation="silu").sum(), [leaf[which]])
        assert torch.equal(d, full[which])
    (dx,) = torch.autograd.grad(ssm.fused_linear(x, w, b, activation="silu").sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="twice|once_differentiable"):
        dx.sum().backward()
    # (a tensor that requires grad cannot be a constant of a trace)
    traced = torch.jit.trace(lambda a, v, c: ssm.fused_linear(a, v, c, activation="silu"), (x, w, b), check_trace=False)
    other = torch.randn(70, 32, device="cuda")
    assert torch.equal(traced(other, w, b), ssm.fused_linear(other, w, b, activation="silu"))


@pytest.mark.parametrize("M,C,H", [(4, 512, 1024), (48, 1000, 520), (2100, 1024, 2048), (200, 4096, 256), (333, 250, 100)])
def test_graphs_and_streams_share_nothing(M, C, H):
    """Two captured calls, replayed side by side on two streams, give what the calls by themselves give."""
    from haste_b200 import ssm
    g = torch.Generator(device="cuda").manual_seed(M)

    def make():
        x, w, r, dy = (torch.randn(*s, generator=g, device="cuda").to(BF16) for s in ((M, C), (H, C), (M, H), (M, H)))
        return x, w / 32, r, dy

    def step(x, w, r, dy):
        leaf = [t.detach().requires_grad_() for t in (x, w, r)]
        y = ssm.fused_linear(leaf[0], leaf[1], activation="silu", residual=leaf[2])
        return [y.detach(), *torch.autograd.grad(y, leaf, dy)]

    data = [make(), make()]
    alone = [step(*d) for d in data]
    held, graphs, outs = [], [], []
    for d in data:
        static = [t.clone() for t in d]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(*static))
        held.append(static)
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(3):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for a, o in zip(alone, outs):
        assert all(torch.equal(p, q) for p, q in zip(a, o))


@pytest.mark.parametrize("M", [2, 40])
@pytest.mark.parametrize("C,H", [(8, (1 << 20) - 1), ((1 << 20) - 1, 8)])
def test_the_most_inputs_and_outputs(C, H, M):
    """Ones, whose sums are exact: at most 2^20."""
    from haste_b200 import ssm
    x, w = torch.ones(M, C, device="cuda", dtype=BF16), torch.ones(H, C, device="cuda", dtype=BF16)
    w[-1] = 2
    residual = torch.zeros(M, H, device="cuda")
    y = ssm.fused_linear(x, w, residual=residual)
    assert (y[:, :-1] == C).all() and (y[:, -1] == 2 * C).all()


def test_more_elements_than_32_bits_count():
    from haste_b200 import ssm
    M, C, H = 1050000, 8, 2056
    x = torch.randn(M, C, device="cuda").to(BF16)
    w = (torch.randn(H, C, device="cuda") / 3).to(BF16).requires_grad_()
    y = ssm.fused_linear(x, w, activation="silu")
    assert torch.equal(y[-100:], ssm.fused_linear(x[-100:], w, activation="silu"))
    dy = torch.zeros_like(y)
    dy[-1] = 1
    (dw,) = torch.autograd.grad(y, w, dy)
    (want,) = torch.autograd.grad(ssm.fused_linear(x[-1:], w, activation="silu").sum(), w)
    assert torch.equal(dw, want)  # one term beside zeros
