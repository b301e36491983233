"""The gated linear recurrence's gradients where no sequence is cut into pieces (there are channels enough), and with gates and
decays at their ends."""
import pytest
import torch

import gated_reference as ref
from test_gated_scan_gpu import NAMES, compare, inputs
from test_state_space_gpu import leaves, lens, poison, seq

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


# 300 blocks and more: two an SM and beyond, one channel a lane (odd) and two
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("T,N,D,opt", [
    (150, 75, 250, dict(decay=0.3, inner=True, lengths=torch.int64, batch_first=True)), (170, 40, 251, dict(state=True, lengths=torch.int32)),
    (161, 79, 256, dict(decay=1.0, state=True)), (200, 150, 65, dict(inner=True, half=True, state=True)),
    (133, 41, 257, dict(decay=0.02, inner=True, state=True, lengths=torch.int64)),
])
def test_whole_sequences(T, N, D, opt, dtype):
    g = torch.Generator(device="cuda").manual_seed(T + N + D)
    d = inputs(g, T, N, D, dtype, opt)
    lengths = lens(g, T, N, opt.get("lengths"))
    for k in ("x", "gate", "input_gate"):
        if k in d:
            d[k] = poison(d[k], lengths)
    dy = poison(seq(g, T, N, D, dtype, half=True), lengths)
    compare(d, lengths, dy, torch.randn(N, D, generator=g, device="cuda"))


# (few channels: in pieces; 5 x 2048: whole)
@pytest.mark.parametrize("N,repeat", [(2, 4), (5, 2560)])
@pytest.mark.parametrize("decay", [None, 1.0])
def test_gradients_with_gates_at_their_ends(decay, N, repeat):
    """Sigmoids are held at 2^-125: the reference gets the gates that have that.  Where w^2 = -2 decay r is below 1e-23, 1 / w is
    taken with 1e-30 added to w^2 (what is lost is at most the term itself, |lam u w / 2| and the like); a decay of -1e-30, of
    whose own gradient such terms are all, is left out of it."""
    from haste_b200 import ssm
    g = torch.Generator(device="cuda").manual_seed(3)
    T, D = 70, 8 * repeat
    d = inputs(g, T, N, D, F32, dict(inner=True, state=True))
    edge = torch.tensor([0.0, 30.0, -30.0, 100.0, -100.0, float("inf"), -float("inf"), 1e-30], device="cuda")
    for k in ("gate", "input_gate"):
        d[k] = edge[torch.randint(0, 8, (T, N, D), generator=g, device="cuda")]
    if decay:
        d["decay"] = torch.tensor([0.0, -1e-30, -1e-8, -1e-3, -0.35, -1.0, -60.0, 0.5], device="cuda").repeat(repeat)
    dy, dfinal = torch.randn(T, N, D, generator=g, device="cuda"), torch.randn(N, D, generator=g, device="cuda")
    names = leaves(d, list(NAMES))
    y, final = ssm.gated_scan(**d)
    got = dict(zip(names, torch.autograd.grad([y, final], [d[k] for k in names], [dy, dfinal])))
    held = {k: d[k].detach().clamp(min=-125 * 0.6931471805599453) for k in ("gate", "input_gate")}
    want, bound = ref.gated_scan(d["x"], held["gate"], d.get("decay"), held["input_gate"], d["initial_state"], None, dy, dfinal)
    if decay:
        r, i = (torch.sigmoid(ref.double(held[k])) for k in ("gate", "input_gate"))
        dec = ref.double(d["decay"]).clamp(max=0)
        a, w = torch.exp(dec * r), torch.sqrt(-torch.expm1(2 * dec * r))
        lam, size = ref.double(dfinal).abs(), torch.zeros_like(r)
        for t in reversed(range(T)):
            size[t] = ref.double(dy)[t].abs() + lam
            lam = a[t] * size[t]
        lost = torch.where(w * w < 1e-23, size * w * i, 0.0)
        u = ref.double(d["x"]).abs()
        bound["dx"] += lost
        bound["dinput_gate"] += lost * u
        bound["dgate"] += lost * u / 2
        over = torch.where(dec != 0, (lost * u / 2).sum((0, 1)) / -dec, 0.0)
        bound["ddecay"] += over
        keep = torch.arange(D) % 8 != 1
        got["decay"], want["ddecay"], bound["ddecay"] = (v[keep.to(v.device)] for v in (got["decay"], want["ddecay"], bound["ddecay"]))
    for k in names:
        ref.check(got[k], want[NAMES[k]], bound[NAMES[k]], NAMES[k])
