"""Rows in four bits and a beam search's step over arrays whose places do not fit 32 bits: what lies behind them equals a call on that part
alone.  Batches of more entries than a launch's third axis has."""
import numpy as np
import pytest

import beam_plain as plain

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def engine():
    import torch
    import vectorstorekit_b200 as vsk
    d = vsk.CUDAComputeDevice(0)
    yield vsk.CUDAAccelerationEngine(d)
    d.close()
    torch.cuda.empty_cache()


def test_encoding_and_decoding(engine):
    import torch
    import vectorstorekit_b200 as vsk
    n, dim = 5_400_001, 402                                     # 2.2 billion elements
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty((n, dim), dtype=torch.float16, device="cuda")
    for at in range(0, n, 1 << 20):
        x[at:at + (1 << 20)].normal_(generator=gen)
    q = vsk.Int4Quantizer(engine.dev, 32, False)
    held = q.quantizeBatch(x)
    values = q.dequantizeBatch(*held, dim)                      # 8.7 GB
    for part in (slice(0, 3000), slice(n - 3000, n), slice(n // 2, n // 2 + 3000)):
        alone = q.quantizeBatch(x[part].clone())
        assert all(torch.equal(a[part], b) for a, b in zip(held, alone))
        assert torch.equal(values[part], q.dequantizeBatch(*alone, dim))


@pytest.mark.parametrize("nq,kind", [(1, "float32"), (6, "float16"), (20, "bfloat16")])
def test_products(engine, nq, kind):
    import torch
    import vectorstorekit_b200 as vsk
    n, dim = 36_000_001, 256                                    # 4.6 GB of codes
    gen = torch.Generator(device="cuda").manual_seed(2)
    codes = torch.randint(0, 256, (n, dim // 2), dtype=torch.uint8, device="cuda", generator=gen)
    scales = torch.rand((n, dim // 128), device="cuda", generator=gen).half()
    x = torch.randn((nq, dim), device="cuda", generator=gen).to(getattr(torch, kind))
    q = vsk.Int4Quantizer(engine.dev, 128)
    y = q.product(x, codes, scales, out_dtype=torch.float32)
    values = torch.zeros((256, 2), dtype=torch.float64, device="cuda")
    values[:, 0], values[:, 1] = torch.arange(256, device="cuda") % 16 - 8, torch.arange(256, device="cuda") // 16 - 8
    for part in (slice(0, 5000), slice(n - 5000, n), slice(33_554_432 - 100, 33_554_432 + 100)):
        w = values[codes[part].long()].view(-1, dim) * scales[part].double().repeat_interleave(128, 1)
        want = x.double() @ w.T
        # chains of at most 128 + 2 x 2 + 16 fp32 additions per group's share, and 31 bits of each vector's elements (int4_plain.product_bound)
        bound = (2 * 128 + 2 * 2 + 16) * 2.0 ** -23 * (x.double().abs() @ w.abs().T) + 2.0 ** -31 * x.double().abs().amax(1, keepdim=True) * w.abs().sum(1)
        assert bool(((y[:, part].double() - want).abs() <= bound * (1 + 2.0 ** -24) + 2.0 ** -24 * want.abs()).all())


@pytest.mark.parametrize("off", [0, 1])
def test_selection(engine, off):
    import torch
    vocab, beams = 1_200_000_000 + off, 2                       # 2.4 billion logits
    x = torch.zeros((1, beams, vocab), dtype=torch.float16, device="cuda")
    scores = torch.tensor([[0.0, -0.5]], device="cuda")
    places = [(0, 0, 5.0), (0, vocab - 1, 7.0), (1, vocab - 1, 7.0), (1, 1_073_741_824, 6.0), (1, 947_483_648 - off, 9.0), (0, 1_073_741_823, 6.5)]
    for j, v, value in places:
        x[0, j, v] = value
    best = sorted(((value + float(scores[0, j]), -j, -v) for j, v, value in places), reverse=True)
    s, b, t = engine.selectBeams(x, scores, 8, normalize=False)
    want = [(total, -j, -v) for total, j, v in best] + [(0.0, 0, 1), (0.0, 0, 2)]
    assert list(zip(s[0].tolist(), b[0].tolist(), t[0].tolist())) == want
    s, b, t = engine.selectBeams(x, scores, 6)
    assert list(zip(b[0].tolist(), t[0].tolist())) == [w[1:] for w in want[:6]]
    lse = [np.log(vocab - len(p) + np.sum(np.exp(p))) for p in ([value for j, _, value in places if j == i] for i in range(beams))]
    assert np.allclose(s[0].tolist(), [w[0] - lse[w[1]] for w in want[:6]], rtol=0, atol=2 * plain.LSE)


@pytest.mark.parametrize("in_place", [True, False])
def test_reordering(engine, in_place):
    import torch
    steps, width = 4_500_001, 66
    t = torch.empty((4, 2, steps, width), dtype=torch.float16, device="cuda")      # 4.8 GB
    for i in range(4):
        for h in range(2):
            t[i, h] = (torch.arange(steps, device="cuda") % 1000)[:, None] + 2000 * h
            t[i, h, :, 0] = i
    parents = torch.tensor([[2, 1, -1, 0]], device="cuda")
    lengths = torch.tensor([steps - 7], device="cuda")
    out = None if in_place else [torch.full_like(t, -1.0)]
    got, = engine.reorderStates([t], parents, lengths=lengths, time_axis=2, out=out)
    for i, p in enumerate((2, 1, -1, 0)):
        for h in range(2):
            for at in (0, 1, steps // 2, steps - 8):
                row = got[i, h, at]
                if p < 0:
                    assert float(row[0]) == (i if in_place else -1)
                else:
                    assert float(row[0]) == p and bool((row[1:] == at % 1000 + 2000 * h).all())
            assert float(got[i, h, steps - 7, 0]) == (i if in_place else -1) and float(got[i, h, steps - 1, 0]) == (i if in_place else -1)
            if p >= 0:
                assert bool((got[i, h, :steps - 7, 0] == p).all())


def test_batches_of_more_than_a_launch_s_third_axis(engine):
    import torch
    batch, vocab, k = 66_000, 2_051, 3
    x = torch.randn((batch, 1, vocab), device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)).half()
    scores = torch.zeros((batch, 1), device="cuda")
    all_of = engine.selectBeams(x, scores, k)
    for part in (slice(0, 40), slice(65_500, 65_600), slice(batch - 40, batch)):
        got = engine.selectBeams(x[part], scores[part], k)
        assert all(torch.equal(a[part], b) for a, b in zip(all_of, got))
        plain.compare([g.cpu().numpy() for g in got], x[part].float().cpu().numpy(), scores[part].cpu().numpy(), None, 0, True)
