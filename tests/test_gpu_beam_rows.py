"""A beam search's selection over rows that are copies of one another: at whatever address a row lies, its totals are the same bits, so
beams with equal rows and scores tie, and the lowest comes first."""
import numpy as np
import pytest

import beam_plain as plain

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def engine():
    import vectorstorekit_b200 as vsk
    d = vsk.CUDAComputeDevice(0)
    yield vsk.CUDAAccelerationEngine(d)
    d.close()


def _t(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


@pytest.mark.parametrize("vocab", [301, 1027, 5001, 33_335])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_equal_rows_tie_whatever_their_addresses(engine, vocab, dtype):
    """Eight beams hold the same row, one behind the other without gaps: an odd row puts them at every place within 16 bytes."""
    import torch
    for seed in range(6):
        rng = np.random.default_rng(vocab + seed)
        row = torch.from_numpy(3 * rng.standard_normal((2, 1, vocab)).astype(np.float32)).to(_t(dtype))
        x = row.repeat(1, 8, 1)
        scores = np.repeat(-rng.uniform(0, 20, (2, 1)), 8, 1).astype(np.float32)
        for k in (8, 30, 128):
            _, beams, tokens = engine.selectBeams(x.cuda(), torch.from_numpy(scores).cuda(), k)
            want = plain.choose(plain.totals(x.float().numpy(), scores, None, 0, True), k)
            assert np.array_equal(beams.cpu().numpy(), want // vocab) and np.array_equal(tokens.cpu().numpy(), want % vocab), (seed, k)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("normalize", [True, False])
def test_totals_do_not_depend_on_the_address(engine, dtype, normalize):
    import torch
    rng = np.random.default_rng(8)
    for batch, beams, vocab, k in ((3, 4, 5001, 9), (1, 1, 8000, 64), (2, 3, 40_000, 128), (2, 2, 1024, 7), (1, 3, 1023, 20)):
        x = torch.from_numpy(3 * rng.standard_normal((batch, beams, vocab)).astype(np.float32)).to(_t(dtype)).cuda()
        x[torch.from_numpy(rng.random(x.shape) < 0.3).cuda()] = float("-inf")
        scores = torch.from_numpy(-rng.uniform(0, 20, (batch, beams)).astype(np.float32)).cuda()
        first = engine.selectBeams(x, scores, k, normalize=normalize)
        plain.compare([g.cpu().numpy() for g in first], x.float().cpu().numpy(), scores.cpu().numpy(), None, 0, normalize)
        for pad in (1, 8):
            wide = torch.full((batch, beams, vocab + pad), float("nan"), dtype=x.dtype, device="cuda")
            for at in range(0, pad + 1):
                wide[:] = float("nan")
                wide[:, :, at:at + vocab] = x
                got = engine.selectBeams(wide[:, :, at:at + vocab], scores, k, normalize=normalize)
                assert all(torch.equal(a, b) for a, b in zip(first, got)), (vocab, pad, at)


def test_an_end_token_outside_the_vocabulary_is_refused_however_large(engine):
    import torch
    import vectorstorekit_b200 as vsk
    x, scores, finished = torch.zeros((1, 2, 100), device="cuda"), torch.zeros((1, 2), device="cuda"), torch.ones((1, 2), dtype=torch.bool, device="cuda")
    for end in (100, -1, 2 ** 64 + 3, -2 ** 64 + 3, 2 ** 200):
        with pytest.raises(vsk.InvalidInput):
            engine.selectBeams(x, scores, 2, finished=finished, end_token=end)
        assert engine.selectBeams(x, scores, 2, end_token=end)[2].tolist() == [[0, 1]]      # nobody has finished
    assert engine.selectBeams(x, scores, 2, finished=finished, end_token=99)[2].tolist() == [[99, 99]]
