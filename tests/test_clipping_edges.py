"""Gradient clipping: what a call takes and refuses, without a GPU, and the same on one."""
import ctypes

import pytest
import torch


class Gradient(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("out", ctypes.c_void_p), ("numel", ctypes.c_longlong), ("dtype", ctypes.c_int), ("out_dtype", ctypes.c_int)]


LAYOUTS = [lambda: (torch.ones(4, 1), torch.empty(1, 4).t()), lambda: (torch.ones(1, 5, 3), torch.empty(5, 1, 3).transpose(0, 1)),
           lambda: (torch.ones(3, 1, 2).transpose(0, 1), torch.empty(1, 3, 2)), lambda: (torch.ones(6, 2).t()[None], torch.empty(6, 2).t()[None])]


@pytest.mark.parametrize("make", LAYOUTS)
def test_axes_of_one_element_have_any_stride(make):
    """(The check behind the one of strides is what refuses tensors that are not on a GPU.)"""
    from haste_b200 import gradients
    g, out = make()
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        gradients.clip_gradients([g], 1.0, out=[out])


@pytest.mark.gpu
@pytest.mark.parametrize("make", LAYOUTS)
def test_axes_of_one_element_on_a_gpu(make):
    from haste_b200 import gradients
    g, out = make()
    dev = [torch.empty_strided(t.shape, t.stride(), device="cuda").copy_(t) for t in (g, out)]
    norm = gradients.clip_gradients([dev[0]], 0.5, out=[dev[1]])
    want = dev[0] * (0.5 / (norm + 1e-6))
    # six roundings: the norm, its sum, the division and the product here, the factor and the product there
    assert torch.allclose(dev[1], want, rtol=6 * 2.0 ** -24, atol=0)


def test_another_type_in_place_is_refused():
    """Through the C ABI: elements of another type do not lie where the gradient's do."""
    from haste_b200 import _C
    L = _C.lib()
    memory = (ctypes.c_char * 64)()
    at = ctypes.addressof(memory) + -ctypes.addressof(memory) % 16
    for dtype, out_dtype in ((0, 1), (1, 0), (1, 2), (2, 1)):
        g = Gradient(at, at, 4, dtype, out_dtype)
        assert L.haste_b200_clip_gradients(ctypes.byref(g), 1, 1.0, at, at, None) == 1
        assert b"own type" in L.haste_b200_last_error()


@pytest.mark.gpu
def test_a_parameter_listed_twice_counts_once_for_its_norm_too():
    """3e38 is finite; twice its square has a root beyond float32."""
    import haste_b200
    p = torch.nn.Parameter(torch.zeros(1, device="cuda"))
    p.grad = torch.full((1,), 3e38, device="cuda")
    norm = haste_b200.clip_grad_norm_([p, p], 1.0, error_if_nonfinite=True)
    assert norm.item() == p.grad.new_tensor(3e38).item() and abs(p.grad.item() - 1) < 1e-6


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_zeros_of_either_sign_beside_values_whose_squares_vanish(dtype):
    from haste_b200 import gradients
    zeros = torch.zeros(70001, device="cuda", dtype=dtype)
    zeros[::2] *= -1
    assert gradients.grad_norm([zeros, zeros[:3]]).item() == 0
    small = torch.finfo(dtype).smallest_normal
    some = zeros.clone()
    some[4321], some[70000], some[1] = small, -small, small
    want = small * 3 ** 0.5
    assert abs(gradients.grad_norm([zeros, some, zeros]).item() - want) <= 2.0 ** -24 * want + 2.0 ** -149
