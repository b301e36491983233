"""State space operators at the sizes where another kernel, or another turn of a kernel's loop, takes over:
many rows and channels, few steps, so that the float64 reference stays quick."""
import pytest
import torch

import state_space_reference as ref
import test_state_space_gpu as base
from test_state_space_gpu import BF16, F16, F32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("T,N,D,S,G,opt", [
    (9, 128, 1001, 4, 1, dict(state=True)), (17, 128, 1001, 3, 1, dict(lengths=torch.int64, z=False)),
    (11, 128, 1280, 4, 1, dict(lengths=torch.int64, state=True)), (9, 128, 1280, 2, 1, dict(half=True, z=False)),
    (10, 64, 1538, 1, 2, dict(lengths=torch.int32, batch_first=True)),
])
def test_selective_scan_of_many_channels_with_few_states(T, N, D, S, G, opt, dtype):
    """One lane a channel: blocks of 128 and 256 channels, staged one by one or in fours."""
    base.test_selective_scan(T, N, D, S, G, opt, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("T,N,D,S,G,opt", [
    (10, 150, 516, 8, 1, dict(state=True)), (9, 150, 517, 7, 1, dict(lengths=torch.int64, z=False)),
    (20, 64, 640, 16, 1, dict(lengths=torch.int64, state=True)), (9, 64, 646, 16, 1, dict(half=True)),
    (17, 64, 640, 13, 1, dict(z=False, batch_first=True)), (12, 40, 1200, 16, 2, dict(lengths=torch.int32, state=True)),
    (10, 64, 352, 24, 1, dict(state=True)), (9, 48, 430, 32, 2, dict(lengths=torch.int64, z=False)),
    (9, 64, 161, 64, 1, dict(state=True, lengths=torch.int64)), (11, 64, 176, 50, 1, dict(half=True)),
    (9, 64, 80, 128, 1, dict(state=True, lengths=torch.int64)), (8, 64, 81, 100, 1, dict(z=False)),
])
def test_selective_scan_of_many_channels(T, N, D, S, G, opt, dtype):
    """Above 592 (forward) and 444 (backward) blocks a thread takes two channels."""
    base.test_selective_scan(T, N, D, S, G, opt, dtype)


def test_a_slow_state_has_no_bias():
    """Decays of 0.985 to 0.998, inputs of one sign: an error of the decays that is not random adds up over
    1 / (1 - a) steps, 120 on average.  One of 2.4e-8 would be seen as 3e-6; the states' own roundings (each up to
    6e-8, random) leave less than 1e-8 in the mean over 10240 channels and 16 states.  Rows in one walk and in pieces."""
    from haste_b200 import ssm
    g = torch.Generator(device="cuda").manual_seed(21)
    T, N, D, S = 2000, 16, 640, 16
    x, dt = (torch.rand(T, N, D, generator=g, device="cuda") for _ in range(2))
    dt = dt * 0.012 + 0.002
    B, C = torch.ones(T, N, 1, S, device="cuda"), torch.ones(T, N, 1, S, device="cuda")
    A = -(torch.rand(D, S, generator=g, device="cuda") * 0.2 + 0.9)
    want = torch.zeros(N, D, S, dtype=torch.float64, device="cuda")
    A64 = A.double()
    for t in range(T):
        d = dt[t].double()[..., None]
        want = torch.exp(d * A64) * want + d * x[t].double()[..., None]
    for rows in (N, 1):
        _, final = ssm.selective_scan(x[:, :rows], dt[:, :rows], A, B[:, :rows], C[:, :rows], softplus=False)
        off = (final.double() / want[:rows] - 1).mean().abs().item()
        assert off < 1e-6, (rows, off)


# ------------------------------------------------------------------ single tokens of large batches
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("N,D,S,G", [(3, 64, 16, 1), (129, 1024, 16, 1), (130, 1200, 8, 2), (131, 700, 24, 1), (70, 1001, 20, 1), (1217, 256, 4, 1)])
def test_steps_of_large_batches(N, D, S, G, packed, dtype):
    """From 2048 threads an SM on a thread takes four rows; B and C go in fours where they lie so."""
    from haste_b200 import ssm
    g = torch.Generator(device="cuda").manual_seed(N + D + S)
    d = base.scan_inputs(g, 1, N, D, S, G, dtype, dict(state=True, half=True))
    h = d.pop("initial_state")
    one = {k: v[0] if k in ("x", "dt", "B", "C", "z") else v for k, v in d.items()}
    if packed:
        one |= {k: one[k].contiguous() for k in "BC"}
    want, major, K = ref.scan(d["x"], d["dt"], d["A"], d["B"], d["C"], d["D"], d["z"], d["dt_bias"], h)
    before = h.clone()
    y, new = ssm.selective_scan_step(**one, state=h)
    ref.check(y[None], want["y"], major["y"], K, "y")
    ref.check(new, want["final"], major["final"], K, "state")
    assert torch.equal(h, before)
    y2, same = ssm.selective_scan_step(**one, state=h, out_state=h)
    assert torch.equal(y2, y) and torch.equal(h, new) and same.data_ptr() == h.data_ptr()


# ------------------------------------------------------------------ blocks that take several rows or items
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("T,N,H,opt", [
    (1583, 3, 250, dict(residual=True, scale=True, bias=True)), (1583, 3, 129, dict(gate=True, batch_first=True)),
    (397, 3, 1024, dict(gate=True, residual=True, scale=True, bias=True)), (301, 1, 4096, dict(residual=True, scale=True, bias=True)),
    (151, 2, 4099, dict(gate=True, residual=True, wide=True)), (101, 3, 5000, dict(residual=True, scale=True, params=F32)),
    (301, 1, 8192, dict(gate=True, residual=True, scale=True, bias=True)),
])
def test_fused_norm_of_many_rows(T, N, H, opt, kind, dtype):
    """More than twice as many rows as blocks, and a remainder."""
    from haste_b200 import ssm
    g = torch.Generator(device="cuda").manual_seed(T + N + H)
    p, bf = opt.get("params", dtype), opt.get("batch_first")
    rdtype = F32 if opt.get("wide") else dtype
    vec = lambda: torch.randn(H, generator=g, device="cuda").to(p)  # noqa: E731
    d = dict(x=base.seq(g, T, N, H, dtype, bf), weight=vec(), bias=vec() if opt.get("bias") else None,
             gate=base.seq(g, T, N, H, dtype, bf) if opt.get("gate") else None,
             residual=base.seq(g, T, N, H, rdtype) if opt.get("residual") else None, scale=vec() if opt.get("scale") else None)
    names = base.leaves(d, list(d))
    y, r = ssm.fused_norm(**d, kind=kind)
    out = [y] + ([] if r is None else [r])
    dy, dr = base.seq(g, T, N, H, dtype), base.seq(g, T, N, H, rdtype) if r is not None else None
    got = dict(zip(names, torch.autograd.grad(out, [d[k] for k in names], [dy] + ([] if r is None else [dr]))))
    want, major, K = ref.norm(d["x"], d["weight"], d["bias"], d["gate"], d["residual"], d["scale"], 1e-5, kind, dy, dr)
    own = K - T * N  # a row's results do not know the others; the sums over rows take one rounding each
    ref.check(y, want["y"], major["y"], own, "y")
    if r is not None:
        ref.check(r, want["r"], major["r"], own, "r")
    for k in names:
        ref.check(got[k], want["d" + k], major["d" + k], own if k in ("x", "gate", "residual") else K, "d" + k)
    again = torch.autograd.grad(ssm.fused_norm(**d, kind=kind)[0], [d[k] for k in names], dy)
    more = torch.autograd.grad(ssm.fused_norm(**d, kind=kind)[0], [d[k] for k in names], dy)
    for a, b in zip(again, more):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("T,N,D,W,opt", [
    (5, 1500, 20, 4, dict(state=True)), (5, 1500, 19, 4, dict(lengths=torch.int64, state=True)), (3, 1301, 250, 3, dict(silu=False)),
    (7, 1499, 64, 2, dict(lengths=torch.int32, state=True, params=F32)),
])
def test_causal_conv1d_of_many_rows(T, N, D, W, opt, dtype):
    """More rows than resident blocks: in the backward pass a block takes several."""
    base.test_causal_conv1d(T, N, D, W, opt, dtype)
