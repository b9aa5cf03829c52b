"""Rows in four bits: sizes whose bytes do not fit 64 bits are refused before anything is copied or launched."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    import vectorstorekit_b200 as vsk
    d = vsk.CUDAComputeDevice(0)
    yield d
    d.close()


@pytest.mark.parametrize("n,dim,code_stride,scale_stride", [
    (1 << 33, 64, 1 << 31, 2),              # the codes reach over 2^64 bytes
    (3, 64, (1 << 63) - 1, 2),
    (1 << 33, 64, 32, 1 << 30),             # twice the scales
    (5, 64, 32, (1 << 62) + 1),
    (1 << 40, 1 << 24, 1 << 23, 1 << 19)])  # the values
def test_sizes_beyond_64_bits_are_refused(dev, n, dim, code_stride, scale_stride):
    import torch
    from vectorstorekit_b200 import _lib
    codes, scales, out = np.zeros((3, 32), np.uint8), np.ones((3, 2), np.float16), np.full((3, 64), 7.0, np.float32)
    r = _lib.Q4Rows(codes.ctypes.data, scales.ctypes.data, None, code_stride, scale_stride, n, dim, 32)
    assert dev._lib.vsk_q4_decode(dev._h, C.byref(r), C.c_void_p(out.ctypes.data)) == 4 and np.all(out == 7.0)
    on = [torch.from_numpy(a).cuda() for a in (codes, scales, out)]
    torch.cuda.synchronize()
    r = _lib.Q4Rows(on[0].data_ptr(), on[1].data_ptr(), None, code_stride, scale_stride, n, dim, 32)
    assert dev._lib.vsk_q4_decode_dev(dev._h, C.byref(r), C.c_void_p(on[2].data_ptr())) == 4 and bool((on[2] == 7.0).all())
    assert dev._lib.vsk_q4_product_dev(dev._h, C.byref(r), C.c_void_p(on[2].data_ptr()), 0, 1, dim, C.c_void_p(on[2].data_ptr()), 0, n) == 4
    if dim > 64:
        assert dev._lib.vsk_q4_encode(dev._h, C.c_void_p(out.ctypes.data), n, dim, 32, 1, C.c_void_p(codes.ctypes.data), code_stride,
                                      C.c_void_p(scales.ctypes.data), None) == 4
    # one row lies at no distance from another
    r = _lib.Q4Rows(codes.ctypes.data, scales.ctypes.data, None, 1 << 62, 1 << 62, 1, 64, 32)
    assert dev._lib.vsk_q4_decode(dev._h, C.byref(r), C.c_void_p(out.ctypes.data)) == 0 and np.all(out[0] == -8.0) and np.all(out[1:] == 7.0)
