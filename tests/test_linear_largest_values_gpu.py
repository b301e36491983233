"""float32 projections of values next to float32's largest, which bfloat16 rounds to infinity."""
import pytest
import torch

pytestmark = pytest.mark.gpu

MOST = torch.finfo(torch.float32).max


# few rows; tiles; parts of K; pairs
@pytest.mark.parametrize("M,C,H", [(3, 40, 24), (9, 40, 24), (40, 1024, 65), (300, 33, 40), (2304, 1024, 2048)])
def test_largest_values(M, C, H):
    """Each row of x and of the weight has one value that is not zero, in the same place: every product is a result, forward and
    backward."""
    from haste_b200 import ssm
    g = torch.Generator(device="cuda").manual_seed(M)
    big = torch.tensor([MOST, -MOST, 3.397e38, 3.39e38, 1e38, 1.0], device="cuda")
    x, w = torch.zeros(M, C, device="cuda"), torch.zeros(H, C, device="cuda")
    x[:, 7] = big[torch.arange(M, device="cuda") % 6]
    w[:, 7] = torch.rand(H, generator=g, device="cuda") * 1e-30
    w[H // 2, 7], x[0, 7] = MOST, 1.0
    x.requires_grad_(), w.requires_grad_()
    y = ssm.fused_linear(x, w)
    want = x.double() @ w.double().t()
    fits = want.abs() <= MOST
    # three planes of eight bits: the products that are left out are 3 x 2^-24 of the result at most, the last sum is cut off (2^-23)
    # and added up (2^-24)
    bound = 8 * 2.0 ** -24
    assert y[fits].isfinite().all() and ((y.double() - want).abs() <= bound * want.abs())[fits].all()
    dy = torch.zeros(M, H, device="cuda")
    dy[0, H // 2] = 1.0
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    assert dx.isfinite().all() and (dx[0, 7].double() - MOST).abs() <= bound * MOST and dx.count_nonzero() == 1
    assert dw.isfinite().all() and (dw[H // 2, 7].double() - 1).abs() <= bound and dw.count_nonzero() == 1
