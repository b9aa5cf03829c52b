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


def test_cpp_quantiser_refuses_codes_of_other_sizes(tmp_path):
    """Rows whose vectors do not have the size that the call states are not read behind their ends: no device is asked."""
    import os
    import subprocess
    from vectorstorekit_b200 import build
    build.build_library()
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    source, exe = tmp_path / "sizes.cpp", str(tmp_path / "sizes")
    source.write_text('''
#include "vectorstorekit_b200/host/vsk.hpp"
template <typename E, typename F> int refused(F f) { try { f(); } catch (const E&) { return 0; } return 1; }
int main() {
  vsk::Int4Quantizer symmetric(nullptr, 32), other(nullptr, 32, false);
  vsk::Int4Quantizer::Rows r;
  r.codes.resize(2 * 20);
  r.scales.resize(2 * 2);
  int bad = refused<vsk::DimensionMismatch>([&] { symmetric.dequantizeBatch(r, 3, 40); });   // a row too few
  bad += refused<vsk::DimensionMismatch>([&] { symmetric.dequantizeBatch(r, 2, 65); });      // too many columns
  bad += refused<vsk::DimensionMismatch>([&] { other.dequantizeBatch(r, 2, 40); });          // no middles
  bad += refused<vsk::EmptyInput>([&] { symmetric.dequantizeBatch(r, 0, 40); });
  r.middles.resize(2 * 2);
  return bad + refused<vsk::DimensionMismatch>([&] { symmetric.dequantizeBatch(r, 2, 40); });
}
''')
    subprocess.run(["g++", "-std=c++17", "-pthread", "-I", root, str(source), "-o", exe, "-L", os.path.join(root, "vectorstorekit_b200"),
                    "-lvsk_cuda", "-Wl,-rpath," + os.path.join(root, "vectorstorekit_b200")], check=True)
    assert subprocess.run([exe]).returncode == 0
