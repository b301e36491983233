"""The gated linear recurrence's backward pass over no rows through the C ABI: the decay's gradient is a sum of nothing."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu


class Sequence(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("t_stride", ctypes.c_longlong), ("n_stride", ctypes.c_longlong)]


class Scan(ctypes.Structure):
    _fields_ = [*((k, ctypes.c_int) for k in ("dtype", "T", "N", "D")), *((k, Sequence) for k in ("x", "gate", "input_gate", "y")),
                *((k, ctypes.c_void_p) for k in ("decay", "state", "final_state", "lengths", "checkpoints")),
                *((k, Sequence) for k in ("dy", "dx", "dgate", "dinput_gate")),
                *((k, ctypes.c_void_p) for k in ("dfinal_state", "ddecay", "dstate", "scratch"))]


@pytest.mark.parametrize("T,N,D", [(5, 0, 7), (0, 0, 7), (0, 2, 7)])
def test_the_gradient_of_the_decay_is_written(T, N, D):
    from haste_b200 import _C
    L = _C.lib()
    decay, ddecay = torch.full((D,), -1.0, device="cuda"), torch.full((D,), 7.0, device="cuda")
    a = Scan(T=T, N=N, D=D, decay=decay.data_ptr(), ddecay=ddecay.data_ptr())
    scratch = torch.empty(max(2, L.haste_b200_gated_scan_scratch(ctypes.byref(a), 1)), device="cuda")
    a.scratch = scratch.data_ptr()
    assert L.haste_b200_gated_scan_backward(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == 0, L.haste_b200_last_error()
    assert not ddecay.any()
