"""Projections through the C ABI whose residual is the result's own buffer, as the header allows."""
import ctypes

import pytest
import torch

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


class Linear(ctypes.Structure):
    _fields_ = [*((k, ctypes.c_int) for k in ("dtype", "param_dtype", "out_dtype", "activation", "M", "C", "H")),
                *((k, ctypes.c_void_p) for k in ("x", "weight", "bias", "residual")), ("x_ld", ctypes.c_longlong),
                ("residual_ld", ctypes.c_longlong), ("y", ctypes.c_void_p), ("y_ld", ctypes.c_longlong), ("pre", ctypes.c_void_p),
                ("dy", ctypes.c_void_p), ("dy_ld", ctypes.c_longlong), ("dx", ctypes.c_void_p), ("dx_ld", ctypes.c_longlong),
                ("dweight", ctypes.c_void_p), ("dbias", ctypes.c_void_p), ("scratch", ctypes.c_void_p)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,out", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
# few rows; tiles of whole words, of single elements, rows that start on 16 bytes but not on a line; parts of K; pairs
@pytest.mark.parametrize("M,C,H,ld", [(5, 256, 64, 64), (32, 512, 40, 41), (64, 64, 256, 256), (300, 128, 200, 208), (300, 128, 130, 131),
                                      (40, 2048, 72, 72), (2304, 1024, 2048, 2056), (9000, 64, 264, 272)])
def test_residual_in_the_results_place(M, C, H, ld, dtype, out):
    from haste_b200 import _C
    L = _C.lib()
    code = {F32: 0, BF16: 1, F16: 2}
    g = torch.Generator(device="cuda").manual_seed(M + H)
    x, w = (torch.randn(*s, generator=g, device="cuda").to(dtype) for s in ((M, C), (H, C)))
    r = torch.randn(M, ld, generator=g, device="cuda").to(out)
    results = []
    for place in (torch.full_like(r, 7.0), r.clone()):
        residual = r if place[0, 0] == 7 else place
        a = Linear(dtype=code[dtype], param_dtype=code[dtype], out_dtype=code[out], activation=2, M=M, C=C, H=H, x=x.data_ptr(), x_ld=C,
                   weight=w.data_ptr(), residual=residual.data_ptr(), residual_ld=ld, y=place.data_ptr(), y_ld=ld)
        scratch = torch.empty(max(1, L.haste_b200_linear_scratch(ctypes.byref(a), 0)), dtype=torch.uint8, device="cuda")
        a.scratch = scratch.data_ptr()
        stream = torch.cuda.current_stream().cuda_stream
        assert L.haste_b200_linear_forward(ctypes.byref(a), stream) == 0, L.haste_b200_last_error()
        results.append(place)
    assert torch.equal(results[0][:, :H], results[1][:, :H])
    assert torch.equal(results[1][:, H:], r[:, H:]) and (results[0][:, H:] == 7).all()


def test_other_rows_in_the_results_place_are_refused():
    """(Arguments are checked before anything touches a device.)"""
    from haste_b200 import _C
    L = _C.lib()
    memory = (ctypes.c_char * 4096)()
    at = ctypes.addressof(memory) + -ctypes.addressof(memory) % 256
    a = Linear(M=3, C=4, H=4, x=at, x_ld=4, weight=at, residual=at + 1024, residual_ld=8, y=at + 1024, y_ld=4, scratch=at + 2048)
    assert L.haste_b200_linear_forward(ctypes.byref(a), None) == 1
    assert b"in y's place" in L.haste_b200_last_error()
