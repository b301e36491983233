"""The operators of a gated linear recurrence block as they are used together: norm, projections, scan and projection back
onto the residual stream, a training step that ends with clipping, and token by token from the prompt's state."""
import math

import pytest
import torch

import gated_reference as ref

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def parameters(g, H, D, dtype):
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    p = dict(norm=1 + 0.1 * rand(H), inward=rand(2 * D, H) / math.sqrt(H), gates=rand(2 * D, D) / math.sqrt(D),
             gate_bias=rand(2 * D), back=rand(H, D) / math.sqrt(D))
    p = {k: v.to(dtype) for k, v in p.items()}
    p["decay"] = -torch.rand(D, generator=g, device="cuda") - 0.05
    return p


def block(p, r, state=None, lengths=None):
    """r [T,N,H] -> (r + block(r), state)."""
    from haste_b200 import ssm
    D = p["decay"].numel()
    n, _ = ssm.fused_norm(r, p["norm"])
    u = ssm.fused_linear(n, p["inward"], activation="silu")
    x, side = u[..., :D], u[..., D:]
    gates = ssm.fused_linear(x, p["gates"], p["gate_bias"])
    y, state = ssm.gated_scan(x, gates[..., :D], decay=p["decay"], input_gate=gates[..., D:], initial_state=state, lengths=lengths)
    return ssm.fused_linear(y * side, p["back"], residual=r), state


def token(p, r, state):
    from haste_b200 import ssm
    D = p["decay"].numel()
    n, _ = ssm.fused_norm(r[None], p["norm"])
    u = ssm.fused_linear(n[0], p["inward"], activation="silu")
    x, side = u[..., :D], u[..., D:]
    gates = ssm.fused_linear(x, p["gates"], p["gate_bias"])
    y, state = ssm.gated_scan_step(x, gates[..., :D], state, decay=p["decay"], input_gate=gates[..., D:], out_state=state)
    return ssm.fused_linear(y * side, p["back"], residual=r), state


def plain(p, r, state=None):
    """The same from the formulas, in the parameters' type."""
    D = p["decay"].numel()
    n = r * torch.rsqrt(r.square().mean(-1, keepdim=True) + 1e-5) * p["norm"]
    u = torch.nn.functional.silu(n @ p["inward"].t())
    x, side = u[..., :D], u[..., D:]
    gates = x @ p["gates"].t() + p["gate_bias"]
    a = torch.exp(p["decay"] * torch.sigmoid(gates[..., :D]))
    b = torch.sqrt(1 - a * a) * x * torch.sigmoid(gates[..., D:])
    h = r.new_zeros(r.shape[1], D) if state is None else state
    ys = []
    for t in range(r.shape[0]):
        h = a[t] * h + b[t]
        ys.append(h)
    return r + (torch.stack(ys) * side) @ p["back"].t(), h


@pytest.mark.parametrize("T,N,H,D", [(37, 3, 64, 96), (130, 2, 50, 70)])
def test_block_and_its_gradients(T, N, H, D):
    g = torch.Generator(device="cuda").manual_seed(T)
    p = parameters(g, H, D, F32)
    r, dy = torch.randn(T, N, H, generator=g, device="cuda"), torch.randn(T, N, H, generator=g, device="cuda")
    leaf = {k: v.clone().requires_grad_() for k, v in dict(p, r=r).items()}
    wide = {k: v.double().requires_grad_() for k, v in dict(p, r=r).items()}
    y, state = block({k: v for k, v in leaf.items() if k != "r"}, leaf["r"])
    want, last = plain({k: v for k, v in wide.items() if k != "r"}, wide["r"])
    # every operator is held to its own bound elsewhere; through five of them float32's roundings stay below 2000 U of the size
    def near(a, b):
        return (a.detach().double() - b.detach()).norm() <= 2000 * ref.U * b.detach().norm()
    assert near(y, want) and near(state, last)
    for (k, a), b in zip(leaf.items(), torch.autograd.grad(want, list(wide.values()), dy.double())):
        (got,) = torch.autograd.grad(y, a, dy, retain_graph=True)
        assert near(got, b), k


def test_tokens_follow_a_prompt():
    g = torch.Generator(device="cuda").manual_seed(1)
    T, N, H, D = 40, 5, 128, 192
    p = parameters(g, H, D, BF16)
    r = torch.randn(T, N, H, generator=g, device="cuda").to(BF16)
    with torch.no_grad():
        whole, last = block(p, r)
        some, state = block(p, r[:25])
        got = [some]
        for t in range(25, T):
            y, state = token(p, r[t], state)
            got.append(y[None])
        want, _ = plain({k: v.double() for k, v in p.items()}, r.double())
    # roundings to bfloat16: the norm's, u's, the gates', y's, the product's and the result's, half a step each, and none of
    # what lies behind them makes more of one than a few times itself
    for y in (whole, torch.cat(got)):
        assert (y.double() - want).norm() <= 12 * 2.0 ** -8 * want.norm()
    assert (state - last).norm() <= 12 * 2.0 ** -8 * last.norm()


def test_a_training_step_ends_with_clipping_and_may_be_captured():
    import haste_b200
    g = torch.Generator(device="cuda").manual_seed(2)
    T, N, H, D = 70, 4, 96, 128
    p = {k: torch.nn.Parameter(v) for k, v in parameters(g, H, D, BF16).items()}
    r = torch.randn(T, N, H, generator=g, device="cuda").to(BF16)
    lengths = torch.tensor([70, 3, 0, 41], device="cuda")

    def step():
        for q in p.values():
            q.grad = None
        y, _ = block(p, r, lengths=lengths)
        y.float().square().sum().backward()
        return haste_b200.clip_grad_norm_(p.values(), 1.0)

    norm = step()
    first = {k: q.grad.clone() for k, q in p.items()}
    assert torch.isfinite(norm) and norm > 1
    clipped = math.sqrt(sum(v.double().square().sum().item() for v in first.values()))
    assert abs(clipped - 1) <= 2.0 ** -8  # each value is rounded by half a step at most
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    for q in p.values():
        q.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    graph.replay()
    assert torch.equal(captured, norm) and all(torch.equal(q.grad, first[k]) for k, q in p.items())
