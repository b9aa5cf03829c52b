"""Products with rows in four bits: many vectors, and vectors that are not finite."""
import numpy as np
import pytest

import int4_plain as plain
from test_gpu_int4 import _case, _compare, _run, _t

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    import vectorstorekit_b200 as vsk
    d = vsk.CUDAComputeDevice(0)
    yield d
    d.close()


# their preparation takes launches of at most 65 535 vectors: one vector in a second launch, many, and three launches
@pytest.mark.parametrize("n,nq", [(40, 65_536), (40, 65_600), (5, 70_000), (130, 131_100)])
@pytest.mark.parametrize("kind,symmetric,group", [("f16", False, 32), ("bf16", True, 64), ("bf16", False, 128)])
def test_products_of_more_vectors_than_a_launch_prepares(dev, n, nq, kind, symmetric, group):
    import torch
    rng = np.random.default_rng(n + nq + group)
    dim = 64
    codes, scales, middles = _case(rng, n, dim, group, symmetric)
    x = torch.from_numpy(rng.standard_normal((nq, dim)).astype(np.float32)).to(_t(kind))
    for code_pad in (0, 1):       # rows at 16-byte places, and others
        got = _run(dev, codes, scales, middles, group, x, "f32", code_pad=code_pad)
        _compare(got, codes, scales, middles, group, x, "f32")


def _by_definition(codes, scales, middles, group, x):
    """sum of value(row, column) x(column) with 64-bit infinities and NaN as they come"""
    with np.errstate(invalid="ignore"):
        return np.einsum("qrd->qr", x.double().numpy()[:, None, :] * plain.values(codes, scales, middles, group)[None])


# up to four vectors, the warp form, the tiles (rows enough; vectors enough)
@pytest.mark.parametrize("n,nq", [(40, 4), (40, 5), (40, 9), (33, 16), (40, 33), (18_944, 17), (40, 4_800)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("symmetric", [True, False])
def test_infinities_and_nan_answer_as_the_definition_however_many_vectors(dev, n, nq, group, kind, symmetric):
    """The codes of the infinite columns take every value, middles are smaller and larger than s (c - 8) there: also where s (c - 8) + m
    has the other sign than s (c - 8), and where it is 0."""
    import torch
    rng = np.random.default_rng(group + nq)
    dim = 72
    codes, scales, middles = _case(rng, n, dim, group, symmetric)
    codes[:, 5] = np.arange(n) % 16
    codes[:, 71] = np.arange(n) // 2 % 16
    if not symmetric:
        scales[:] = (2.0 ** rng.integers(-3, 1, scales.shape)).astype(np.float16)
        middles[:] = (scales * rng.choice([-8.0, -3.0, 0.0, 0.5, 2.0, 100.0], scales.shape)).astype(np.float16)
    x = torch.from_numpy(rng.standard_normal((nq, dim)).astype(np.float32)).to(_t(kind))
    clean = x.clone()
    inf = float("inf")
    for q, places in {1: {5: inf}, 2: {71: -inf}, 3: {40: float("nan")}, nq - 1: {5: -inf, 71: -inf}, nq // 2 + 1: {5: inf, 71: -inf}}.items():
        for column, value in places.items():
            x[q, column] = value
    touched = ~torch.isfinite(x).all(1).numpy()
    code_pad = -((dim + 1) // 2) % 16
    for out in {"f32", kind}:
        got = _run(dev, codes, scales, middles, group, x, out, code_pad=code_pad)
        want = _by_definition(codes, scales, middles, group, x[torch.from_numpy(touched)])
        assert not np.isfinite(want).any()
        assert np.array_equal(got[touched], want.astype(np.float32), equal_nan=True)
        # the others are what they are without them
        assert np.array_equal(got[~touched], _run(dev, codes, scales, middles, group, clean, out, code_pad=code_pad)[~touched])
        _compare(got[~touched], codes, scales, middles, group, clean[torch.from_numpy(~touched)], out)
