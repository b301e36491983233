"""Projections whose sums lie beyond their type's range but not beyond float32's: every slope has reached 0 or 1 there, however the
sum is kept for the backward pass."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
# the slope at sums so far above and so far below zero
ENDS = {"relu": (1, 0), "silu": (1, 0), "gelu": (1, 0), "tanh": (0, 0), "sigmoid": (0, 0)}
ACTS = {"relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": lambda p: 0.5 * p * torch.erfc(-p / math.sqrt(2)),
        "tanh": torch.tanh, "sigmoid": torch.sigmoid}


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("out", [None, F16, F32], ids=["no residual", "residual", "fp32 residual"])
@pytest.mark.parametrize("act", list(ENDS))
# few rows; tiles of whole words and of odd ones; parts of K; pairs
@pytest.mark.parametrize("M,C,H", [(8, 16, 16), (20, 16, 19), (40, 16, 16), (300, 16, 24), (300, 16, 19), (40, 2048, 72), (40, 2048, 67),
                                   (2304, 1024, 2048)])
def test_finite_sums_beyond_the_types_range(M, C, H, act, out, dtype):
    """Column 0 and 1: from the products, 256 x 281.25 = 72000 (in float16 only); others: from a float32 bias."""
    from haste_b200 import ssm
    out = None if out is None else dtype if out == F16 else F32
    most = torch.finfo(dtype).max
    far = [65519.0, 65520.0, 70000.0, 1e6, 1e30] if dtype == F16 else [3.39e38, 3.396e38, 3.4e38]
    v = torch.zeros(H, device="cuda")
    v[2:2 + len(far)], v[8:8 + len(far)] = torch.tensor(far, device="cuda"), -torch.tensor(far, device="cuda")
    v[14:16] = torch.tensor([0.5, -3.0], device="cuda")
    x, w = torch.zeros(M, C, device="cuda", dtype=dtype), torch.zeros(H, C, device="cuda", dtype=dtype)
    x[:, 0] = 256
    p = v.double()
    if dtype == F16:
        w[0, 0], w[1, 0] = 281.25, -281.25
        p[0], p[1] = 72000, -72000
    residual = None if out is None else torch.full((M, H), 2.0, device="cuda", dtype=out)
    leaf = [t.requires_grad_() for t in (x, w, v)]
    y = ssm.fused_linear(*leaf, activation=act, residual=residual)
    want = ACTS[act](p) + (0 if out is None else 2)
    beyond = want.abs() > (torch.finfo(y.dtype).max if y.dtype != F32 else math.inf)
    half = torch.finfo(y.dtype).eps / 2
    off = (y.detach().double() - want).abs()
    assert (off <= (half + 30 * 2.0 ** -24) * (want.abs() + 2))[:, ~beyond].all()
    big = y[:, beyond].double()  # rounded to an infinity, or, next to the border, to the largest value
    assert ((big == math.copysign(math.inf, 1)) | (big == most)).all() and (y.dtype == F32 or not beyond.any() or big.isinf().any())

    # 1/64 times slopes of 0 and 1: exact, and so are their sums
    dx, dw, db = torch.autograd.grad(y, leaf, torch.full_like(y, 1 / 64))
    ends = p.abs() > 60000
    slope = torch.where(p > 0, ENDS[act][0], ENDS[act][1])
    assert torch.equal(db.double()[ends], slope.double()[ends] * M / 64)
    assert torch.equal(dw[ends][:, 0].double(), slope.double()[ends] * M * 4) and not dw[:, 1:].any()
    assert torch.equal(dx[:, 0].double(), (slope.double() * w[:, 0].double() / 64).sum().expand(M)) and not dx[:, 1:].any()
    q = p[~ends].clone().requires_grad_()
    (d,) = torch.autograd.grad(ACTS[act](q).sum(), q)
    # a slope of the sum in 16 bits, and the gradient of the sum in 16 bits
    assert ((db.double()[~ends] - d * M / 64).abs() <= M / 64 * 4 * torch.finfo(dtype).eps).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("act", list(ENDS))
@pytest.mark.parametrize("M", [8, 40, 300])
def test_infinite_sums_have_the_slopes_limits(M, act, dtype):
    from haste_b200 import ssm
    v = torch.tensor([math.inf, -math.inf, math.nan, 0.0] * 4, device="cuda", requires_grad=True)
    x, w = torch.zeros(M, 16, device="cuda", dtype=dtype), torch.zeros(16, 16, device="cuda", dtype=dtype)
    y = ssm.fused_linear(x, w, v, activation=act)
    (db,) = torch.autograd.grad(y, v, torch.ones_like(y))
    assert (db[0::4] == M * ENDS[act][0]).all() and (db[1::4] == M * ENDS[act][1]).all() and db[2::4].isnan().all()
