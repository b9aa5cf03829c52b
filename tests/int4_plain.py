"""Rows in four bits from their definition, in 64 bits (numpy): what the codec and the products are compared with."""
import numpy as np


def encode(rows, group, symmetric):
    """-> codes [n][dim] (0 .. 15), scales fp16 [n][groups], middles fp16 or None"""
    x = np.asarray(rows).astype(np.float64)
    n, dim = x.shape
    groups = -(-dim // group)
    codes = np.empty((n, dim), np.int64)
    scales, middles = np.empty((n, groups), np.float16), np.empty((n, groups), np.float16)
    for g in range(groups):
        v = x[:, g * group:(g + 1) * group]
        lo, hi = v.min(1), v.max(1)
        s = np.maximum(hi, -lo) / 7.0 if symmetric else (hi - lo) / 15.0
        s = np.minimum(s.astype(np.float32), np.float32(65504)).astype(np.float16)
        m = np.zeros(n, np.float16) if symmetric else \
            np.clip((lo + 8.0 * s.astype(np.float64)).astype(np.float32), -65504, 65504).astype(np.float16)
        with np.errstate(divide="ignore", invalid="ignore"):
            u = np.where(s[:, None] > 0, (v - m.astype(np.float64)[:, None]) / s.astype(np.float64)[:, None], 0.0)
        codes[:, g * group:(g + 1) * group] = np.clip(np.rint(u) + 8, 0, 15)
        scales[:, g], middles[:, g] = s, m
    return codes, scales, None if symmetric else middles


def pack(codes):
    n, dim = codes.shape
    if dim % 2:
        codes = np.concatenate([codes, np.full((n, 1), 8, codes.dtype)], 1)
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).astype(np.uint8)


def values(codes, scales, middles, group):
    """What codes 0 .. 15 stand for, in 64 bits (exact)."""
    dim = codes.shape[1]
    out = (codes - 8.0) * np.repeat(scales.astype(np.float64), group, 1)[:, :dim]
    return out if middles is None else out + np.repeat(middles.astype(np.float64), group, 1)[:, :dim]


# half a step of a type, relative to the value, and its smallest step's half (the error of a number below the normal range)
HALF = {"f32": (2.0 ** -24, 2.0 ** -150), "f16": (2.0 ** -11, 2.0 ** -25), "bf16": (2.0 ** -8, 2.0 ** -134)}


def product_bound(codes, scales, middles, group, x, y, out):
    """How far a product in fp32 sums may be from the exact y.  A group's sum is a chain of at most `group` additions per part of x,
    the groups one multiply-add each (two with middles), the parts and the shares of eight warps a dozen more; the sums of x over a group
    chain `group` additions too.  Each addition loses at most 2^-23 (a unit that cuts off rather than rounds) of a partial sum, and no partial
    sum is larger than the sum of the magnitudes.  A vector may be held in whole numbers of 2^-30 of its largest element (31 bits): half of
    that per element.  Then one rounding to the result's type."""
    dim = codes.shape[1]
    mag = np.abs(codes - 8.0) * np.repeat(np.abs(scales.astype(np.float64)), group, 1)[:, :dim]
    if middles is not None:
        mag = mag + np.repeat(np.abs(middles.astype(np.float64)), group, 1)[:, :dim]
    steps = 2 * group + 2 * scales.shape[1] + 16
    x = np.abs(x.astype(np.float64))
    sums, grid = x @ mag.T, 2.0 ** -31 * np.max(x, axis=1, keepdims=True) * np.sum(mag, axis=1)
    rel, tiny = HALF[out]
    return (steps * 2.0 ** -23 * sums + grid) * (1 + rel) + rel * np.abs(y) + tiny
