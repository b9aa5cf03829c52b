"""Rows in four bits with a scale per group of columns: the quantiser and the products of vectors with such rows.

``Int4Quantizer`` stands beside ``ScalarQuantizer`` (int8, one scale per column or per matrix;
``Quantization/ScalarQuantizer.swift:129-164``).  The format is stated in ``include/vsk_cuda.h``.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _lib
from .engine import (CUDAComputeDevice, DimensionMismatch, EmptyInput, InvalidInput, UnsupportedOperation, _device_pointers, _dtype_id,
                     _host, _is_dev, _ptr, _row_stride, _rows_2d)

try:  # torch is plumbing for device memory only
    import torch
except Exception:  # pragma: no cover
    torch = None


class Int4Quantizer:
    """Rows in four bits: two codes a byte and one fp16 scale per ``groupSize`` columns of a row (32, 64 or 128).

    ``symmetric=True``: a value is ``scale * (code - 8)``.  ``symmetric=False``: ``scale * (code - 8) + middle``, for groups whose
    values do not lie around zero.  There is nothing to train: a group's scale comes from its own values."""

    def __init__(self, dev: CUDAComputeDevice, groupSize: int = 64, symmetric: bool = True):
        if groupSize not in (32, 64, 128):
            raise UnsupportedOperation(f"groups of {groupSize} columns are not supported (32, 64 or 128)")
        self.dev, self._lib = dev, dev._lib
        self.groupSize, self.symmetric = int(groupSize), bool(symmetric)

    def _groups(self, dim: int) -> int:
        return -(-dim // self.groupSize)

    def quantizeBatch(self, vectors):
        """Finite rows ``[n][dim]`` -> ``(codes, scales, middles)``: ``[n][ceil(dim / 2)]`` bytes, ``[n][groups]`` fp16 and the same
        or None.  CUDA tensors of float32, float16 or bfloat16 give CUDA tensors, whose code rows begin at 16-byte boundaries; host
        arrays are taken as float32 and give host arrays."""
        if len(vectors) == 0:
            raise EmptyInput("no rows")
        if len(vectors.shape) != 2 or vectors.shape[1] == 0:
            raise DimensionMismatch("rows must be a matrix with at least one column")
        n, dim = (int(v) for v in vectors.shape)
        width, groups, sym = (dim + 1) // 2, self._groups(dim), 1 if self.symmetric else 0
        if _is_dev(vectors):
            x = _rows_2d(vectors, "rows")
            kind = _dtype_id(x.dtype)
            codes = torch.empty((n, -(-width // 16) * 16), dtype=torch.uint8, device=x.device)[:, :width]
            scales = torch.empty((n, groups), dtype=torch.float16, device=x.device)
            middles = None if self.symmetric else torch.empty_like(scales)
            px, pc, ps, pm = _device_pointers(self.dev, x, codes, scales, middles)
            self.dev.check(self._lib.vsk_q4_encode_dev(self.dev._h, px, kind, n, dim, _row_stride(x), self.groupSize, sym, pc,
                                                       _row_stride(codes), ps, pm))
            return codes, scales, middles
        x = _host(vectors, np.float32)
        codes = np.empty((n, width), np.uint8)
        scales = np.empty((n, groups), np.float16)
        middles = None if self.symmetric else np.empty((n, groups), np.float16)
        self.dev.check(self._lib.vsk_q4_encode(self.dev._h, _ptr(x), n, dim, self.groupSize, sym, _ptr(codes), width, _ptr(scales),
                                               _ptr(middles)))
        return codes, scales, middles

    def _descriptor(self, n, dim, pointers, code_stride, scale_stride):
        return _lib.Q4Rows(*pointers, code_stride, scale_stride, n, dim, self.groupSize)

    def _check(self, codes, scales, middles, dim):
        if dim <= 0:
            raise DimensionMismatch("dimension must be positive")
        if self.symmetric != (middles is None):
            raise InvalidInput("a symmetric quantiser has no middles, the other one has")
        shape = codes.shape
        if len(shape) != 2 or shape[1] != (dim + 1) // 2:
            raise DimensionMismatch(f"expected {(dim + 1) // 2} bytes of codes per row for {dim} columns, got {tuple(shape)}")
        if shape[0] == 0:
            raise EmptyInput("no rows")
        want = (shape[0], self._groups(dim))
        for name, t in (("scales", scales), ("middles", middles)):
            if t is not None and t.shape != want:
                raise DimensionMismatch(f"expected {name} of shape {want}, got {tuple(t.shape)}")

    def _device_rows(self, codes, scales, middles, dim):
        """Codes and scales in device memory, checked, with contiguous rows and the strides of the two -> (codes, scales, middles, strides)"""
        self._check(codes, scales, middles, dim)
        for name, t, want in (("codes", codes, torch.uint8), ("scales", scales, torch.float16), ("middles", middles, torch.float16)):
            if t is not None and (not _is_dev(t) or t.dtype != want):
                raise InvalidInput(f"{name} must be a CUDA tensor of {want}")
        codes, scales = _rows_2d(codes, "codes"), _rows_2d(scales, "scales")
        per_scales = _row_stride(scales)
        if middles is not None:
            middles = _rows_2d(middles, "middles")
            if _row_stride(middles) != per_scales:
                scales, middles = scales.contiguous(), middles.contiguous()
                per_scales = _row_stride(scales)
        return codes, scales, middles, (_row_stride(codes), per_scales)

    def dequantizeBatch(self, codes, scales, middles, dimensions: int):
        """The fp32 values ``[n][dimensions]`` that the codes stand for."""
        dim = int(dimensions)
        if _is_dev(codes):
            codes, scales, middles, strides = self._device_rows(codes, scales, middles, dim)
            out = torch.empty((codes.shape[0], dim), dtype=torch.float32, device=codes.device)
            *p, po = _device_pointers(self.dev, codes, scales, middles, out)
            r = self._descriptor(codes.shape[0], dim, p, *strides)
            self.dev.check(self._lib.vsk_q4_decode_dev(self.dev._h, C.byref(r), po))
            return out
        codes, scales = _host(codes, np.uint8), _host(scales, np.float16)
        middles = None if middles is None else _host(middles, np.float16)
        self._check(codes, scales, middles, dim)
        out = np.empty((codes.shape[0], dim), np.float32)
        p = [None if a is None else a.ctypes.data for a in (codes, scales, middles)]
        r = self._descriptor(codes.shape[0], dim, p, codes.shape[1], scales.shape[1])
        self.dev.check(self._lib.vsk_q4_decode(self.dev._h, C.byref(r), _ptr(out)))
        return out

    def product(self, x, codes, scales, middles=None, out_dtype=None):
        """``[queries][n]`` products of vectors ``x [queries][dim]`` with all rows: the logits of an output head, a projection of
        tokens, or the scores of queries against a store (``DistanceMetric.dotProduct`` is their negative).  Sums in fp32, rounded
        once to ``out_dtype`` (float32, float16 or bfloat16; default: x's type).  fp32 vectors, and up to four 16-bit ones, are taken to
        2^-31 of their largest element, others exactly; the order of the sums depends on the numbers of rows and vectors.  CUDA tensors;
        no gradient flows."""
        if not _is_dev(x):
            raise InvalidInput("product takes CUDA tensors")
        if x.dim() != 2:
            raise DimensionMismatch("x must be a matrix of one vector per row")
        nq, dim = x.shape
        if nq == 0:
            raise EmptyInput("no vectors")
        codes, scales, middles, strides = self._device_rows(codes, scales, middles, dim)
        x = _rows_2d(x, "x")
        out_dtype = out_dtype or x.dtype
        kind, out_kind, n = _dtype_id(x.dtype), _dtype_id(out_dtype), codes.shape[0]
        y = torch.empty((nq, n), dtype=out_dtype, device=x.device)
        *p, px, py = _device_pointers(self.dev, codes, scales, middles, x, y)
        r = self._descriptor(n, dim, p, *strides)
        self.dev.check(self._lib.vsk_q4_product_dev(self.dev._h, C.byref(r), px, kind, nq, _row_stride(x), py, out_kind, n))
        return y
