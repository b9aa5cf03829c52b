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
