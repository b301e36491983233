"""The gated linear recurrence against its float64 reference, element by element within the roundings that
float32 arithmetic may make (gated_reference.py)."""
import pytest
import torch

import gated_reference as ref
from test_state_space_gpu import leaves, lens, poison, seq

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def inputs(g, T, N, D, dtype, opt):
    bf = opt.get("batch_first")
    d = dict(x=seq(g, T, N, D, dtype, bf, opt.get("half"), step=opt.get("step", 1)),
             gate=seq(g, T, N, D, dtype, bf, opt.get("half"), scale=opt.get("scale", 1.5)))
    if opt.get("decay"):
        d["decay"] = -torch.rand(D, generator=g, device="cuda") * opt["decay"]
    if opt.get("inner"):
        d["input_gate"] = seq(g, T, N, D, dtype, bf, scale=2.0)
    if opt.get("state"):
        d["initial_state"] = torch.randn(N, D, generator=g, device="cuda")
    return d


def reference(d, lengths, dy=None, dfinal=None):
    return ref.gated_scan(d["x"], d["gate"], d.get("decay"), d.get("input_gate"), d.get("initial_state"), lengths, dy, dfinal)


NAMES = {"x": "dx", "gate": "dgate", "decay": "ddecay", "input_gate": "dinput_gate", "initial_state": "dstate"}


def compare(d, lengths, dy, dfinal):
    from haste_b200 import ssm
    names = leaves(d, list(NAMES))
    y, final = ssm.gated_scan(**d, lengths=lengths)
    got = dict(zip(names, torch.autograd.grad([y, final], [d[k] for k in names], [dy, dfinal])))
    want, bound = reference(d, lengths, dy, dfinal)
    ref.check(y, want["y"], bound["y"], "y")
    ref.check(final, want["final"], bound["final"], "final")
    for k in names:
        assert got[k].dtype == d[k].dtype
        ref.check(got[k], want[NAMES[k]], bound[NAMES[k]], NAMES[k])
    with torch.no_grad():
        again = ssm.gated_scan(**d, lengths=lengths)
    ref.check(again[0], want["y"], bound["y"], "y without gradients")
    ref.check(again[1], want["final"], bound["final"], "final without gradients")
    return y, final, got


CASES = [
    (1, 1, 1, dict(decay=2.0)), (1, 3, 40, dict(state=True, inner=True)), (2, 2, 7, dict(decay=0.5, inner=True)),
    (5, 1, 64, {}), (31, 2, 33, dict(state=True)), (32, 1, 66, dict(decay=0.2, state=True)),
    (33, 3, 130, dict(decay=3.0, inner=True, lengths=torch.int64)), (63, 2, 64, dict(inner=True, half=True)),
    (64, 1, 250, dict(decay=0.1, batch_first=True)), (65, 2, 96, dict(state=True, lengths=torch.int32, batch_first=True)),
    (130, 1, 8, dict(decay=0.05, inner=True, state=True)), (128, 2, 31, dict(step=2)), (257, 2, 65, dict(decay=0.3, half=True)),
    (300, 3, 70, dict(state=True, lengths=torch.int64, inner=True)), (700, 2, 40, dict(decay=0.01, inner=True, state=True)),
    (1000, 1, 66, dict(lengths=torch.int64, decay=0.02)), (513, 1, 64, dict(scale=8.0)), (321, 2, 34, dict(scale=8.0, decay=8.0)),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("T,N,D,opt", CASES)
def test_gated_scan(T, N, D, opt, dtype):
    g = torch.Generator(device="cuda").manual_seed(T * 1000 + N * 100 + D)
    d = inputs(g, T, N, D, dtype, opt)
    lengths = lens(g, T, N, opt.get("lengths"))
    for k in ("x", "gate", "input_gate"):
        if k in d:
            d[k] = poison(d[k], lengths)
    dy = poison(seq(g, T, N, D, dtype, half=True), lengths)
    dfinal = torch.randn(N, D, generator=g, device="cuda")
    y, final, got = compare(d, lengths, dy, dfinal)
    assert y.dtype == dtype and final.dtype == F32
    assert (y.stride(0) < y.stride(1)) == bool(opt.get("batch_first") and T > 1 and N > 1)


@pytest.mark.parametrize("decay", [None, 1.0])
def test_gates_at_their_ends(decay):
    """Open, closed and infinite gates; decays of zero, above zero and far below."""
    g = torch.Generator(device="cuda").manual_seed(3)
    T, N, D = 70, 2, 32
    d = inputs(g, T, N, D, F32, dict(inner=True, state=True))
    edge = torch.tensor([0.0, 30.0, -30.0, 100.0, -100.0, float("inf"), -float("inf"), 1e-30], device="cuda")
    d["gate"] = edge[torch.randint(0, 8, (T, N, D), generator=g, device="cuda")]
    d["input_gate"] = edge[torch.randint(0, 8, (T, N, D), generator=g, device="cuda")]
    if decay:
        d["decay"] = torch.tensor([0.0, -1e-30, -1e-8, -1e-3, -0.35, -1.0, -60.0, 0.5], device="cuda").repeat(4)
    dy, dfinal = torch.randn(T, N, D, generator=g, device="cuda"), torch.randn(N, D, generator=g, device="cuda")
    from haste_b200 import ssm
    names = leaves(d, list(NAMES))
    y, final = ssm.gated_scan(**d)
    grads = torch.autograd.grad([y, final], [d[k] for k in names], [dy, dfinal])
    want, bound = reference(d, None, dy, dfinal)
    ref.check(y, want["y"], bound["y"], "y")
    ref.check(final, want["final"], bound["final"], "final")
    assert all(torch.isfinite(v).all() for v in grads)
    if decay:
        assert not grads[names.index("decay")][7::8].any()  # counts as zero


def test_a_state_that_lasts_keeps_its_bits():
    """A thousandth of a decay a step, over thousands: an error of one sign in a would add up to 1e-5."""
    from haste_b200 import ssm
    g = torch.Generator(device="cuda").manual_seed(4)
    T, N, D = 6000, 1, 32
    d = dict(x=1 + 0.1 * torch.randn(T, N, D, generator=g, device="cuda"), gate=torch.randn(T, N, D, generator=g, device="cuda"),
             decay=torch.full((D,), -1e-3, device="cuda"))
    y, _ = ssm.gated_scan(**d)
    r = torch.sigmoid(d["gate"].double())
    a, w = torch.exp(-1e-3 * r), torch.sqrt(-torch.expm1(-2e-3 * r))
    h = torch.zeros(N, D, dtype=torch.float64, device="cuda")
    for t in range(T):
        h = a[t] * h + w[t] * d["x"][t].double()
    # roundings to either side: 2000 steps of memory, a standard deviation of sqrt(2000 / 3) U = 26 U, six of them
    assert ((y[-1].double() - h).abs() / h.abs()).max() < 6 * 26 * ref.U


def test_rows_of_length_zero_keep_any_state():
    from haste_b200 import ssm
    T, N, D = 70, 3, 40
    g = torch.Generator(device="cuda").manual_seed(5)
    d = inputs(g, T, N, D, BF16, dict(decay=1.0, inner=True))
    state = torch.full((N, D), float("inf"), device="cuda")
    state[1] = 2.0
    lengths = torch.tensor([0, 5, -3], device="cuda")
    for v in (d["x"], d["gate"], d["input_gate"]):
        poison(v, lengths.clamp(min=0))
    leaf = {k: v.detach().requires_grad_() for k, v in dict(d, initial_state=state).items()}
    y, final = ssm.gated_scan(**leaf, lengths=lengths)
    assert torch.equal(final[0], state[0]) and torch.equal(final[2], state[2]) and torch.isfinite(final[1]).all()
    assert not y[:, 0].any() and not y[:, 2].any() and not y[5:, 1].any() and torch.isfinite(y).all()
    dy = torch.full_like(y, float("nan"))
    dy[:5, 1] = 1.0
    dx, dgate, dstate = torch.autograd.grad([y, final], [leaf["x"], leaf["gate"], leaf["initial_state"]],
                                            [dy, torch.ones_like(final)])
    assert not dx[:, 0].any() and not dgate[5:, 1].any() and torch.isfinite(dx).all()
    assert torch.equal(dstate[0], torch.ones(D, device="cuda"))


@pytest.mark.parametrize("T,N,D", [(0, 2, 8), (5, 0, 8), (5, 2, 0)])
def test_empty(T, N, D):
    from haste_b200 import ssm
    x = torch.randn(T, N, D, device="cuda", requires_grad=True)
    state = torch.randn(N, D, device="cuda", requires_grad=True)
    decay = -torch.rand(D, device="cuda").requires_grad_()
    y, final = ssm.gated_scan(x, torch.zeros_like(x), decay, initial_state=state)
    assert y.shape == x.shape and final.shape == state.shape
    dx, ddecay, dstate = torch.autograd.grad([y.sum() + final.sum()], [x, decay, state])
    assert dx.shape == x.shape and not ddecay.any()
    if T == 0:
        assert torch.equal(final, state) and torch.equal(dstate, torch.ones_like(state))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("N,D,opt", [(1, 1, {}), (3, 33, dict(decay=1.0)), (2, 64, dict(inner=True)), (130, 512, dict(decay=0.1, inner=True))])
def test_step(N, D, opt, dtype):
    from haste_b200 import ssm
    g = torch.Generator(device="cuda").manual_seed(N + D)
    d = inputs(g, 1, N, D, dtype, dict(opt, state=True, half=True))
    want, bound = reference(d, None)
    one = {k: v[0] for k, v in d.items() if k in ("x", "gate", "input_gate")}
    state = d["initial_state"].clone()
    y, new = ssm.gated_scan_step(**one, state=state, decay=d.get("decay"))
    ref.check(y, want["y"][0], bound["y"][0], "y")
    ref.check(new, want["final"], bound["final"], "state")
    version = state._version
    y2, same = ssm.gated_scan_step(**one, state=state, decay=d.get("decay"), out_state=state)
    assert same.data_ptr() == state.data_ptr() and torch.equal(y2, y) and torch.equal(state, new) and state._version > version
    buffer = torch.zeros(2 * N * D, device="cuda")
    with pytest.raises(ValueError, match="lies over"):  # one value behind another state of the same size, or over the input
        ssm.gated_scan_step(**one, state=buffer[:N * D].view(N, D), out_state=buffer[1:N * D + 1].view(N, D)) if N * D > 1 else \
            ssm.gated_scan_step(buffer.view(N, -1)[:, 1:], buffer.view(N, -1)[:, 1:], buffer[:1].view(N, D), out_state=buffer[1:].view(N, D))
    # with gradients: the same call as one step of a sequence
    x = one["x"].detach().requires_grad_()
    y3, _ = ssm.gated_scan_step(x, one["gate"], d["initial_state"], decay=d.get("decay"), input_gate=one.get("input_gate"))
    assert torch.autograd.grad(y3.sum(), x)[0].shape == x.shape
    ref.check(y3, want["y"][0], bound["y"][0], "y with gradients")


def test_a_prompt_may_be_cut_and_followed_by_steps():
    from haste_b200 import ssm
    g = torch.Generator(device="cuda").manual_seed(6)
    T, N, D = 150, 2, 70
    d = inputs(g, T, N, D, F32, dict(decay=0.3, inner=True))
    want, bound = reference(d, None)
    decay = d.pop("decay")
    state = None
    got = []
    for a, b in ((0, 1), (1, 64), (64, 140)):
        y, state = ssm.gated_scan(**{k: v[a:b] for k, v in d.items()}, decay=decay, initial_state=state)
        got.append(y)
    for t in range(140, T):
        y, state = ssm.gated_scan_step(d["x"][t], d["gate"][t], state, decay, d["input_gate"][t], out_state=state)
        got.append(y[None])
    ref.check(torch.cat(got), want["y"], bound["y"], "y")
    ref.check(state, want["final"], bound["final"], "state")


def test_repeats_bit_for_bit_on_any_stream_and_in_a_graph():
    from haste_b200 import ssm
    g = torch.Generator(device="cuda").manual_seed(7)
    T, N, D = 600, 2, 96
    d = inputs(g, T, N, D, BF16, dict(decay=0.2, inner=True, state=True))
    dy = torch.randn(T, N, D, generator=g, device="cuda").to(BF16)

    def run(v):
        leaf = {k: t.detach().requires_grad_() for k, t in v.items()}
        y, final = ssm.gated_scan(**leaf)
        return [y.detach(), final.detach(), *torch.autograd.grad(y, list(leaf.values()), dy)]

    first = run(d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(d)
        second = run(d)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    static = {k: torch.zeros_like(v) for k, v in d.items()}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run(static)
    for k, v in d.items():
        static[k].copy_(v)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(first, captured))


def test_more_elements_than_32_bits_count():
    """4.3 GB a sequence: the last rows' steps against the same steps by themselves, which see all that a state of so fast
    a decay remembers."""
    from haste_b200 import ssm
    T, N, D = 33000, 64, 1024
    x = torch.empty(T, N, D, device="cuda", dtype=BF16).uniform_(-1, 1)
    gate = torch.full((1, 1, 1), -3.0, device="cuda", dtype=BF16).expand(T, N, D).contiguous()
    y, final = ssm.gated_scan(x, gate)
    y2, final2 = ssm.gated_scan(x[-256:], gate[-256:])
    # 0.047^64 is far below a rounding.  The two calls' tiles start at other steps, so sums are associated in another order:
    # three roundings a step of terms that add up to less than 1 / (1 - 0.05), in either, and each y is rounded by itself
    apart = 2 * 3 * 1.06 * ref.U
    assert (final - final2).abs().max() < apart
    a, b = y[-192:].float(), y2[-192:].float()
    assert ((a - b).abs() <= torch.finfo(BF16).eps * a.abs() + apart).all() and (a != b).float().mean() < 1e-4


def test_second_derivatives_and_tracing():
    from haste_b200 import ssm
    x = torch.randn(4, 2, 8, device="cuda", requires_grad=True)
    gate = torch.randn(4, 2, 8, device="cuda", requires_grad=True)
    y, _ = ssm.gated_scan(x, gate)
    (dx,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="twice|once_differentiable"):
        dx.sum().backward()
    traced = torch.jit.trace(lambda a, b: ssm.gated_scan(a, b)[0], (x, gate), check_trace=False)
    other = torch.randn(4, 2, 8, device="cuda")
    assert torch.equal(traced(other, gate), ssm.gated_scan(other, gate)[0])
