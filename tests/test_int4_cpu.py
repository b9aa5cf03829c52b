"""Rows in four bits without a device: what the Python layer refuses, and the plain form the GPU tests compare with."""
import ctypes as C
import types

import numpy as np
import pytest

import int4_plain as plain


def _quantizer(group=64, symmetric=True):
    import vectorstorekit_b200 as vsk
    return vsk.Int4Quantizer(types.SimpleNamespace(_lib=None, device=0), group, symmetric)


def test_refusals_before_any_device_call():
    import torch
    import vectorstorekit_b200 as vsk
    for group in (0, 16, 48, 256):
        with pytest.raises(vsk.UnsupportedOperation):
            _quantizer(group)
    q = _quantizer()
    x = torch.zeros((2, 64))
    codes, scales = torch.zeros((3, 32), dtype=torch.uint8), torch.zeros((3, 1), dtype=torch.float16)
    with pytest.raises(vsk.InvalidInput):
        q.product(x, codes, scales)                       # host tensors
    with pytest.raises(vsk.EmptyInput):
        q.quantizeBatch(np.zeros((0, 4), np.float32))
    with pytest.raises(vsk.DimensionMismatch):
        q.quantizeBatch(np.zeros((4, 0), np.float32))
    with pytest.raises(vsk.DimensionMismatch):
        q.quantizeBatch(np.zeros(4, np.float32))
    c, s = np.zeros((3, 32), np.uint8), np.zeros((3, 1), np.float16)
    with pytest.raises(vsk.DimensionMismatch):
        q.dequantizeBatch(c, s, None, 62)
    with pytest.raises(vsk.DimensionMismatch):
        q.dequantizeBatch(c, s[:2], None, 64)
    with pytest.raises(vsk.DimensionMismatch):
        q.dequantizeBatch(c, s, None, 0)
    with pytest.raises(vsk.InvalidInput):
        q.dequantizeBatch(c, s, s, 64)
    with pytest.raises(vsk.InvalidInput):
        _quantizer(64, False).dequantizeBatch(c, s, None, 64)
    with pytest.raises(vsk.EmptyInput):
        q.dequantizeBatch(c[:0], s[:0], None, 64)


def test_entry_points_without_a_context():
    from vectorstorekit_b200 import _lib, build
    build.build_library()
    lib = _lib.load()
    r = _lib.Q4Rows()
    assert lib.vsk_q4_encode(None, None, 1, 1, 32, 1, None, 1, None, None) == 7
    assert lib.vsk_q4_encode_dev(None, None, 0, 1, 1, 1, 32, 1, None, 1, None, None) == 7
    assert lib.vsk_q4_decode(None, C.byref(r), None) == 7
    assert lib.vsk_q4_decode_dev(None, C.byref(r), None) == 7
    assert lib.vsk_q4_product_dev(None, C.byref(r), None, 0, 1, 1, None, 0, 1) == 7


@pytest.mark.parametrize("symmetric", [True, False])
def test_the_plain_codec_is_within_half_a_step(symmetric):
    """|value - x| is at most half a step of the group, plus what rounding the scale and the middle moves (a relative 2^-11 each)."""
    x = np.random.default_rng(2).standard_normal((50, 100)).astype(np.float32)
    codes, scales, middles = plain.encode(x, 32, symmetric)
    s = np.repeat(scales.astype(np.float64), 32, 1)[:, :100]
    slack = 8 * 2.0 ** -11 * s + (0 if symmetric else 2.0 ** -11 * np.abs(np.repeat(middles.astype(np.float64), 32, 1)[:, :100]))
    assert np.all(np.abs(plain.values(codes, scales, middles, 32) - x) <= s / 2 + slack)
    assert codes.min() >= 0 and codes.max() <= 15
    assert plain.pack(codes[:, :3])[0, 1] >> 4 == 8
