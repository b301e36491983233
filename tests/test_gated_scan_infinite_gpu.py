"""The gated linear recurrence with infinite states and adjoints: a decay is never zero, so an infinity stays what it is for the
rest of the sequence, whatever the product of the decays rounds to and however the sequence is cut."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
INF = math.inf


# one channel a lane and two; in pieces (few channels) and whole; decays whose products over a step, a warp's four steps, a
# tile, a piece leave float32's range
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("gate,decay", [(-2.0, None), (-8.0, None), (-30.0, None), (-100.0, None), (3.0, -2.0), (3.0, -30.0), (8.0, -60.0),
                                        (8.0, -300.0)])
@pytest.mark.parametrize("T,N,D", [(300, 2, 33), (301, 2, 64), (70, 75, 250), (65, 40, 251)])
def test_an_infinite_state_stays_infinite(T, N, D, gate, decay, dtype):
    from haste_b200 import ssm
    g = torch.Generator(device="cuda").manual_seed(T + D)
    x = torch.randn(T, N, D, generator=g, device="cuda").to(dtype)
    gates = (gate + 0.1 * torch.randn(T, N, D, generator=g, device="cuda")).to(dtype)
    dec = None if decay is None else torch.full((D,), decay, device="cuda")
    state = torch.randn(N, D, generator=g, device="cuda")
    calm = x.clone(), state.clone()
    first = torch.full((N, D), T, device="cuda")  # the step from which on the state is infinite
    sign = torch.ones(N, D, device="cuda")
    state[:, 0::7], state[:, 1::7] = INF, -INF
    first[:, :] = torch.where(state.isinf(), -1, first)
    for c, (t, s) in {2: (0, 1), 3: (5, -1), 4: (16, 1), 5: (T - 1, -1)}.items():
        x[t, :, c::7] = s * INF
        first[:, c::7] = t
    sign[:, 1::7] = sign[:, 3::7] = sign[:, 5::7] = -1
    y, final = ssm.gated_scan(x, gates, dec, initial_state=state)
    quiet, last = ssm.gated_scan(calm[0], gates, dec, initial_state=calm[1])
    live = torch.arange(T, device="cuda")[:, None, None] >= first
    want = torch.where(live, (sign * INF).expand_as(live), quiet.float())
    assert torch.equal(y.float(), want) and torch.equal(final, torch.where(first < T, sign * INF, last))
    # step by step
    h = state
    for t in range(20):
        one, h = ssm.gated_scan_step(x[t], gates[t], h, dec)
        assert torch.equal(one.float().isinf(), want[t].isinf()) and not one.isnan().any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("gate,decay", [(-2.0, None), (-8.0, None), (-30.0, None), (3.0, -2.0), (3.0, -30.0), (8.0, -300.0)])
@pytest.mark.parametrize("T,N,D", [(300, 2, 33), (301, 2, 64), (70, 75, 250), (65, 40, 251)])
def test_an_infinite_adjoint_stays_infinite(T, N, D, gate, decay, dtype):
    from haste_b200 import ssm
    g = torch.Generator(device="cuda").manual_seed(T + D)
    x = torch.randn(T, N, D, generator=g, device="cuda").to(dtype).requires_grad_()
    gates = (gate + 0.1 * torch.randn(T, N, D, generator=g, device="cuda")).to(dtype)
    dec = None if decay is None else torch.full((D,), decay, device="cuda")
    state = torch.randn(N, D, generator=g, device="cuda").requires_grad_()
    dy = torch.randn(T, N, D, generator=g, device="cuda").to(dtype)
    dfinal = torch.randn(N, D, generator=g, device="cuda")
    out = ssm.gated_scan(x, gates, dec, initial_state=state)
    dx0, ds0 = torch.autograd.grad(out, [x, state], [dy, dfinal], retain_graph=True)
    last = torch.full((N, D), -1, device="cuda")  # the step up to which the adjoint is infinite
    dfinal[:, 0::5], last[:, 0::5] = INF, T
    dy[T - 1, :, 1::5], last[:, 1::5] = INF, T - 1
    dy[T // 2, :, 2::5], last[:, 2::5] = -INF, T // 2
    dx, ds = torch.autograd.grad(out, [x, state], [dy, dfinal])
    sign = torch.where(torch.arange(D, device="cuda") % 5 == 2, -INF, INF).expand(N, D)
    live = torch.arange(T, device="cuda")[:, None, None] <= last
    assert torch.equal(dx.float(), torch.where(live, sign.expand_as(live), dx0.float()))
    assert torch.equal(ds, torch.where(last >= 0, sign, ds0))
