"""State space operators without a GPU: the float64 reference of the GPU tests against automatic
differentiation and finite differences, and the refusals of wrong calls."""
import pytest
import torch

import state_space_reference as ref


def _rand(*shape, g, scale=1.0):
    return torch.randn(*shape, generator=g, dtype=torch.float64) * scale


def _conv_inputs(T=6, N=2, D=3, W=4):
    g = torch.Generator().manual_seed(1)
    return dict(x=_rand(T, N, D, g=g), weight=_rand(D, W, g=g), bias=_rand(D, g=g), state=_rand(N, W - 1, D, g=g))


def _scan_inputs(T=5, N=2, D=4, S=3, G=2):
    g = torch.Generator().manual_seed(2)
    return dict(x=_rand(T, N, D, g=g), dt=_rand(T, N, D, g=g), A=-_rand(D, S, g=g).abs(), B=_rand(T, N, G, S, g=g),
                C=_rand(T, N, G, S, g=g), D=_rand(D, g=g), z=_rand(T, N, D, g=g), dt_bias=_rand(D, g=g),
                state=_rand(N, D, S, g=g))


def _norm_inputs(T=2, N=2, H=5):
    g = torch.Generator().manual_seed(3)
    return dict(x=_rand(T, N, H, g=g), weight=_rand(H, g=g), bias=_rand(H, g=g), gate=_rand(T, N, H, g=g),
                residual=_rand(T, N, H, g=g), scale=_rand(H, g=g))


def _objective(out, weights):
    return sum((out[k] * w).sum() for k, w in weights.items())


@pytest.mark.parametrize("op,make,call,outputs,grads", [
    ("conv", _conv_inputs, lambda v, **k: ref.conv(**v, lengths=[6, 2], use_silu=True, **k),
     ("y", "final"), {"x": "dx", "weight": "dweight", "bias": "dbias", "state": "dstate"}),
    ("scan", _scan_inputs, lambda v, **k: ref.scan(**v, lengths=torch.tensor([5, 3]), **k), ("y", "final"),
     {"x": "dx", "dt": "ddt", "A": "dA", "B": "dB", "C": "dC", "D": "dD", "z": "dz", "dt_bias": "ddt_bias", "state": "dstate"}),
    ("norm", _norm_inputs, lambda v, **k: ref.norm(**v, kind="layer", **k), ("y", "r"),
     {"x": "dx", "weight": "dweight", "bias": "dbias", "gate": "dgate", "residual": "dresidual", "scale": "dscale"}),
])
def test_reference_gradients_against_differences(op, make, call, outputs, grads):
    """Central differences of the reference's outputs: step 1e-5, so off by about 1e-10 |third derivative| + 1e-16 / 1e-5."""
    v = make()
    g = torch.Generator().manual_seed(9)
    out, _, _ = call(v)
    w = {k: torch.randn(out[k].shape, generator=g, dtype=torch.float64) for k in outputs}
    names = {"y": "dy", "final": "dfinal", "r": "dr"}
    full, _, _ = call(v, **{names[k]: w[k] for k in outputs})
    for k, name in grads.items():
        flat = v[k].flatten()
        for i in range(0, flat.numel(), max(1, flat.numel() // 6)):
            vals = []
            for sign in (1, -1):
                moved = flat.clone()
                moved[i] += sign * 1e-5
                vals.append(_objective(call(v | {k: moved.reshape(v[k].shape)})[0], w))
            assert abs((vals[0] - vals[1]).item() / 2e-5 - full[name].flatten()[i].item()) < 1e-6, (op, k, i)


def test_a_result_off_by_more_than_its_roundings_is_noticed():
    want = torch.tensor([1.0, 2.0], dtype=torch.float64)
    ref.check(torch.tensor([1.0, 2.0 + 2e-6]), want, want, 32, "y")
    with pytest.raises(AssertionError):
        ref.check(torch.tensor([1.0, 2.0 + 2e-5]), want, want, 32, "y")
    with pytest.raises(AssertionError):
        ref.check(torch.tensor([1.0, float("nan")]), want, want, 32, "y")


def z(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("change,error,says", [
    (dict(x=z(5, 4)), ValueError, "three|3 dimensions"),
    (dict(x=z(5, 2, 4, dtype=torch.float64)), TypeError, "float32, bfloat16 and float16"),
    (dict(weight=z(4, 5)), ValueError, "2, 3 or 4 taps"),
    (dict(weight=z(4, 1)), ValueError, "2, 3 or 4 taps"),
    (dict(weight=z(3, 4)), ValueError, "weight must be"),
    (dict(weight=z(4, 4, dtype=torch.bfloat16)), TypeError, "weight must be"),
    (dict(bias=z(5)), ValueError, "bias must be"),
    (dict(bias=z(4, dtype=torch.bfloat16)), TypeError, "bias must be"),
    (dict(initial_state=z(2, 4, 4)), ValueError, "state must be"),
    (dict(initial_state=z(2, 3, 4, dtype=torch.float16)), TypeError, "state must be"),
    (dict(lengths=torch.zeros(3, dtype=torch.long)), ValueError, "lengths must be"),
    (dict(lengths=torch.zeros(2)), TypeError, "lengths must be"),
    (dict(), RuntimeError, "CUDA tensor"),
])
def test_causal_conv1d_refuses(change, error, says):
    from haste_b200 import ssm
    args = dict(x=z(5, 2, 4), weight=z(4, 4), bias=z(4)) | change
    with pytest.raises(error, match=says):
        ssm.causal_conv1d(**args)


@pytest.mark.parametrize("change,error,says", [
    (dict(x=z(5, 4)), ValueError, "3 dimensions"),
    (dict(dt=z(5, 2, 3)), ValueError, "dt must be"),
    (dict(dt=z(5, 2, 4, dtype=torch.bfloat16)), TypeError, "dt must be"),
    (dict(A=z(4, 129)), ValueError, "1 to 128 states"),
    (dict(A=z(4, 0)), ValueError, "1 to 128 states"),
    (dict(A=z(3, 8)), ValueError, "A must be"),
    (dict(B=z(5, 2, 3, 8), C=z(5, 2, 3, 8)), ValueError, "divide the channels"),
    (dict(C=z(5, 2, 7)), ValueError, "C must be"),
    (dict(B=z(5, 2, 8, dtype=torch.float16)), TypeError, "B must be"),
    (dict(D=z(8)), ValueError, "D must be"),
    (dict(z=z(5, 2, 8)), ValueError, "z must be"),
    (dict(dt_bias=z(2)), ValueError, "dt_bias must be"),
    (dict(initial_state=z(2, 4, 4)), ValueError, "state must be"),
    (dict(initial_state=z(2, 4, 8, dtype=torch.bfloat16)), TypeError, "state must be"),
    (dict(lengths=torch.zeros(1, dtype=torch.long)), ValueError, "lengths must be"),
    (dict(), RuntimeError, "CUDA tensor"),
])
def test_selective_scan_refuses(change, error, says):
    from haste_b200 import ssm
    args = dict(x=z(5, 2, 4), dt=z(5, 2, 4), A=z(4, 8), B=z(5, 2, 8), C=z(5, 2, 8)) | change
    with pytest.raises(error, match=says):
        ssm.selective_scan(**args)


@pytest.mark.parametrize("change,error,says", [
    (dict(x=z(5, 2, 8193), weight=z(8193)), ValueError, "1 to 8192"),
    (dict(weight=z(5)), ValueError, "weight must be"),
    (dict(bias=z(5)), ValueError, "bias must be"),
    (dict(gate=z(5, 2, 5)), ValueError, "gate must be"),
    (dict(residual=z(5, 1, 4)), ValueError, "residual must be"),
    (dict(residual=z(5, 2, 4, dtype=torch.bfloat16)), TypeError, "residual must be"),
    (dict(scale=z(4)), ValueError, "needs a residual"),
    (dict(kind="group"), ValueError, "'rms' or 'layer'"),
    (dict(eps=-1.0), ValueError, "eps"),
    (dict(), RuntimeError, "CUDA tensor"),
])
def test_fused_norm_refuses(change, error, says):
    from haste_b200 import ssm
    with pytest.raises(error, match=says):
        ssm.fused_norm(**(dict(x=z(5, 2, 4), weight=z(4)) | change))


def test_steps_refuse():
    from haste_b200 import ssm
    with pytest.raises(ValueError, match="2 dimensions"):
        ssm.causal_conv1d_step(z(1, 2, 4), z(2, 3, 4), z(4, 4))
    with pytest.raises(ValueError, match="state must be"):
        ssm.causal_conv1d_step(z(2, 4), z(2, 4, 4), z(4, 4))
    with pytest.raises(ValueError, match="2 dimensions"):
        ssm.selective_scan_step(z(1, 2, 4), z(2, 4), z(4, 8), z(2, 8), z(2, 8), z(2, 4, 8))
    with pytest.raises(ValueError, match="out_state"):
        ssm.causal_conv1d_step(z(2, 4), z(2, 3, 4), z(4, 4).requires_grad_(), out_state=z(2, 3, 4))


def test_entry_points_refuse_bad_blocks():
    """Through the C ABI: arguments are checked before anything touches a device."""
    import ctypes
    from haste_b200 import _C
    L = _C.lib()
    for op in ("causal_conv1d", "selective_scan", "fused_norm"):
        for direction in ("forward", "backward"):
            call = getattr(L, f"haste_b200_{op}_{direction}")
            assert call(None, None) == 1
            assert b"null pointer" in L.haste_b200_last_error()
            block = (ctypes.c_int * 4)(7)  # an unknown dtype
            whole = (ctypes.c_char * 4096)()
            ctypes.memmove(whole, block, 16)
            assert call(whole, None) == 1
            assert b"dtype" in L.haste_b200_last_error()
