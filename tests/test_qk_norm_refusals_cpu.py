"""No-GPU check of pa_qk_norm_bwd: a weight gradient that would not be written is refused."""
import ctypes as C

import pytest

from paraattention_b200 import _lib as L
from paraattention_b200 import build_ext


@pytest.mark.parametrize("gone", ["weight", "x"])
def test_a_weight_gradient_without_a_weight_is_refused(gone):
    build_ext.build()
    lib = L.load()
    buf = (C.c_uint8 * 256)()
    addr = (C.addressof(buf) + 15) // 16 * 16
    a = L.QkNormArgs()
    for i in range(2):
        a.x[i] = a.y[i] = a.dy[i] = a.weight[i] = a.dweight[i] = addr
        for s in (a.x_stride, a.y_stride, a.dy_stride):
            s[i][:] = (640, 128, 64)
    a.heads[:] = (2, 1)
    a.batch, a.rows, a.head_dim, a.eps, a.interleaved = 1, 5, 64, 1e-6, 1
    assert lib.pa_qk_norm_bwd(C.byref(a), None) == L.PA_EINVAL and b"workspace" in lib.pa_last_error()
    getattr(a, gone)[1] = None
    assert lib.pa_qk_norm_bwd(C.byref(a), None) == L.PA_EINVAL and b"dweight[1]" in lib.pa_last_error()
    a.dweight[1] = None
    assert lib.pa_qk_norm_bwd(C.byref(a), None) == L.PA_EINVAL and b"workspace" in lib.pa_last_error()
