"""Operators of a gated linear recurrence block without a GPU: the float64 reference of the GPU tests against
differences, and the refusals of wrong calls."""
import pytest
import torch

import gated_reference as ref


def _rand(*shape, g, scale=1.0):
    return torch.randn(*shape, generator=g, dtype=torch.float64) * scale


@pytest.mark.parametrize("decay,inner", [(False, False), (False, True), (True, False), (True, True)])
def test_gated_scan_reference_against_differences(decay, inner):
    """Central differences with a step of 1e-5: off by about 1e-10 |third derivative| + 1e-16 / 1e-5."""
    g = torch.Generator().manual_seed(1)
    T, N, D = 6, 2, 3
    v = dict(x=_rand(T, N, D, g=g), gate=_rand(T, N, D, g=g), state=_rand(N, D, g=g))
    if decay:
        v["decay"] = -_rand(D, g=g).abs() - 0.1
    if inner:
        v["input_gate"] = _rand(T, N, D, g=g)
    lengths = torch.tensor([6, 4])
    wy, wf = _rand(T, N, D, g=g), _rand(N, D, g=g)
    full, _ = ref.gated_scan(**v, lengths=lengths, dy=wy, dfinal=wf)
    for k in v:
        flat = v[k].flatten()
        for i in range(0, flat.numel(), max(1, flat.numel() // 8)):
            vals = []
            for sign in (1, -1):
                moved = flat.clone()
                moved[i] += sign * 1e-5
                out, _ = ref.gated_scan(**(v | {k: moved.reshape(v[k].shape)}), lengths=lengths)
                vals.append(((out["y"] * wy).sum() + (out["final"] * wf).sum()).item())
            assert abs((vals[0] - vals[1]) / 2e-5 - full["d" + k].flatten()[i].item()) < 1e-6, (k, i)


def test_a_result_beyond_its_bound_is_noticed():
    want = torch.tensor([1.0, 2.0], dtype=torch.float64)
    ref.check(torch.tensor([1.0, 2.0 + 1e-6]), want, want * 1e-6, "y")
    for wrong in (2.0 + 3e-6, float("nan"), float("inf")):
        with pytest.raises(AssertionError):
            ref.check(torch.tensor([1.0, wrong]), want, want * 1e-6, "y")


def z(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("change,error,says", [
    (dict(x=z(5, 4)), ValueError, "3 dimensions"),
    (dict(x=z(5, 2, 4, dtype=torch.float64)), TypeError, "float32, bfloat16 and float16"),
    (dict(gate=z(5, 2, 3)), ValueError, "gate must be"),
    (dict(gate=z(5, 2, 4, dtype=torch.bfloat16)), TypeError, "gate must be"),
    (dict(decay=z(5)), ValueError, "decay must be"),
    (dict(input_gate=z(5, 1, 4)), ValueError, "input_gate must be"),
    (dict(input_gate=z(5, 2, 4, dtype=torch.float16)), TypeError, "input_gate must be"),
    (dict(initial_state=z(2, 4, 1)), ValueError, "state must be"),
    (dict(initial_state=z(2, 4, dtype=torch.bfloat16)), TypeError, "state must be"),
    (dict(lengths=torch.zeros(3, dtype=torch.long)), ValueError, "lengths must be"),
    (dict(lengths=torch.zeros(2)), TypeError, "lengths must be"),
    (dict(), RuntimeError, "CUDA tensor"),
])
def test_gated_scan_refuses(change, error, says):
    from haste_b200 import ssm
    with pytest.raises(error, match=says):
        ssm.gated_scan(**(dict(x=z(5, 2, 4), gate=z(5, 2, 4), decay=z(4)) | change))


def test_gated_scan_step_refuses():
    from haste_b200 import ssm
    with pytest.raises(ValueError, match="2 dimensions"):
        ssm.gated_scan_step(z(1, 2, 4), z(1, 2, 4), z(2, 4))
    with pytest.raises(ValueError, match="state must be"):
        ssm.gated_scan_step(z(2, 4), z(2, 4), z(2, 5))
    with pytest.raises(ValueError, match="out_state"):
        ssm.gated_scan_step(z(2, 4).requires_grad_(), z(2, 4), z(2, 4), out_state=z(2, 4))


@pytest.mark.parametrize("change,error,says", [
    (dict(x=torch.tensor(1.0)), ValueError, "a dimension at least"),
    (dict(x=z(5, 2, 4, dtype=torch.float64)), TypeError, "float32, bfloat16 and float16"),
    (dict(weight=z(6)), ValueError, "2 dimensions"),
    (dict(weight=z(6, 5)), ValueError, "weight must be"),
    (dict(weight=z(0, 4)), ValueError, "weight must have"),
    (dict(weight=z(1 << 20, 4)), ValueError, "weight must have"),
    (dict(x=z(5, 2, 0), weight=z(6, 0)), ValueError, "weight must have"),
    (dict(weight=z(6, 4, dtype=torch.bfloat16)), TypeError, "weight must be"),
    (dict(bias=z(4)), ValueError, "bias must be"),
    (dict(bias=z(6, dtype=torch.float16)), TypeError, "bias must be"),
    (dict(activation="swish"), ValueError, "activation must be one of"),
    (dict(), RuntimeError, "CUDA tensor"),
])
def test_fused_linear_refuses(change, error, says):
    from haste_b200 import ssm
    with pytest.raises(error, match=says):
        ssm.fused_linear(**(dict(x=z(5, 2, 4), weight=z(6, 4), bias=z(6)) | change))


@pytest.mark.parametrize("args,error,says", [
    (([z(4, 4)[:, ::2]], 1.0), ValueError, "one range of memory"),
    (([z(4, dtype=torch.float64)], 1.0), TypeError, "float32, bfloat16 and float16"),
    (([z(4).to_sparse()], 1.0), ValueError, "sparse"),
    (([z(4)], -1.0), ValueError, "max_norm"),
    (([z(4)], 1.0, [z(5)]), ValueError, "shapes"),
    (([z(4, 5)], 1.0, [z(5, 4).t()]), ValueError, "lie in memory"),
    (([z(4)], 1.0, [z(4), z(4)]), ValueError, "as many"),
    (([z(4)], 1.0), RuntimeError, "CUDA tensor"),
])
def test_clip_gradients_refuses(args, error, says):
    from haste_b200 import gradients
    with pytest.raises(error, match=says):
        gradients.clip_gradients(*args)


def test_no_gradients_have_a_norm_of_zero():
    import haste_b200
    from haste_b200 import gradients
    assert gradients.grad_norm([None]).item() == 0 and gradients.clip_gradients([], 1.0).item() == 0
    assert haste_b200.clip_grad_norm_(torch.nn.Parameter(z(3)), 1.0).item() == 0


def test_entry_points_refuse_bad_blocks():
    """Through the C ABI: arguments are checked before anything touches a device."""
    import ctypes
    from haste_b200 import _C
    L = _C.lib()
    for name in ("gated_scan_forward", "gated_scan_backward", "linear_forward", "linear_backward"):
        call = getattr(L, f"haste_b200_{name}")
        assert call(None, None) == 1
        assert b"null pointer" in L.haste_b200_last_error()
        whole = (ctypes.c_char * 4096)()
        ctypes.memmove(whole, (ctypes.c_int * 1)(7), 4)  # an unknown dtype
        assert call(whole, None) == 1
        assert b"dtype" in L.haste_b200_last_error()
