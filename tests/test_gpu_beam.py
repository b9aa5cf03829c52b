"""A beam search's step: selection against the 64-bit definition (beam_plain), states against indexing, and both together with
an output head in four bits."""
import ctypes as C

import numpy as np
import pytest

import beam_plain as plain
import int4_plain

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


def _check(engine, logits, scores, k, normalize=True, finished=None, end=0):
    """logits, finished: torch on the host or the device (their layout is kept)."""
    import torch
    got = engine.selectBeams(logits.cuda(), torch.from_numpy(scores.astype(np.float32)).cuda(), k, normalize=normalize,
                             finished=None if finished is None else finished.cuda(), end_token=end)
    assert [g.dtype for g in got] == [torch.float32, torch.int64, torch.int64]
    plain.compare([g.cpu().numpy() for g in got], logits.float().cpu().numpy(), scores.astype(np.float32),
                  None if finished is None else finished.cpu().numpy(), end, normalize)
    return got


SHAPES = [(1, 1, 1, 1), (1, 1, 5, 8), (2, 3, 7, 4), (3, 64, 64, 128), (1, 4, 1023, 5), (2, 4, 1024, 8), (2, 4, 1025, 8), (3, 5, 5001, 10),
          (1, 1, 100_000, 100), (2, 8, 32_768, 16), (1, 64, 3001, 128), (300, 2, 40, 3), (1, 2, 300_001, 1), (5, 1, 4096, 128), (5, 1, 4097, 64),
          (40, 33, 129, 33)]


@pytest.mark.parametrize("batch,beams,vocab,k", SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("normalize", [True, False])
def test_selection(engine, batch, beams, vocab, k, dtype, normalize):
    import torch
    rng = np.random.default_rng(vocab + 3 * beams + k)
    x = torch.from_numpy(rng.standard_normal((batch, beams, vocab)).astype(np.float32) * 3).to(_t(dtype))
    scores = -rng.uniform(0, 20, (batch, beams))
    _check(engine, x, scores, k, normalize)
    # forbidden tokens, finished and dead beams, rows without a token
    x[torch.from_numpy(rng.random(x.shape) < 0.5)] = float("-inf")
    x[0, 0] = float("-inf")
    finished = torch.from_numpy(rng.random((batch, beams)) < 0.3)
    scores[rng.random(scores.shape) < 0.2] = -np.inf
    _check(engine, x, scores, k, normalize, finished, vocab - 1)


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("vocab", [90, 20_000])
def test_ties_go_to_the_lowest_beam_and_token(engine, normalize, vocab):
    """All logits equal; beams that are copies of one another; zeros of both signs; logits of few values."""
    import torch
    rng = np.random.default_rng(1)
    for k in (1, 7, 128):
        for value in (0.0, -7.25, torch.finfo(torch.float32).min):
            got = _check(engine, torch.full((2, 5, vocab), value), np.zeros((2, 5)), k, normalize)
            assert got[1].cpu().tolist() == [[i // vocab for i in range(k)]] * 2 and got[2].cpu().tolist() == [[i % vocab for i in range(k)]] * 2
        zeros = torch.zeros((1, 3, vocab))
        zeros[:, :, ::2] = -0.0
        assert _check(engine, zeros, np.zeros((1, 3)), k, normalize)[2].cpu().tolist()[0] == [i % vocab for i in range(k)]
        row = torch.from_numpy(rng.integers(-3, 3, (4, 1, vocab)).astype(np.float32))
        _check(engine, row.expand(4, 6, vocab), np.zeros((4, 6)), k, normalize)
        _check(engine, row.expand(4, 6, vocab).half(), np.repeat(-np.arange(3.0), 2)[None].repeat(4, 0), k, normalize)


@pytest.mark.parametrize("vocab", [50, 7000])
def test_infinities_and_nan(engine, vocab):
    import torch
    rng = np.random.default_rng(2)
    x = torch.from_numpy(rng.standard_normal((2, 6, vocab)).astype(np.float32))
    x[0, 0, 3], x[0, 1, vocab - 1], x[0, 2, :], x[0, 3, 5] = float("nan"), float("inf"), float("nan"), float("-inf")
    x[1, 0, 1:] = float("-inf")
    x[1, 1] = float("-inf")
    x[1, 2, ::2] = torch.finfo(torch.float32).min
    scores = np.array([[0, -1, -2, -3, np.nan, np.inf], [0, 0, 0, -np.inf, -2, -3.0]])
    for normalize in (True, False):
        for k in (1, 20, 128):
            _check(engine, x, scores, k, normalize)
    # nothing at all to choose from
    s, b, t = engine.selectBeams(torch.full((1, 2, vocab), float("-inf"), device="cuda"), torch.zeros((1, 2), device="cuda"), 3)
    assert bool(torch.isneginf(s).all()) and bool((b == -1).all()) and bool((t == -1).all())


def test_finished_beams_offer_one_candidate_and_their_logits_are_not_read(engine):
    import torch
    x = torch.randn((2, 3, 9000))
    x[0, 1] = float("nan")
    finished = torch.tensor([[False, True, False], [True, True, True]])
    for end in (0, 17, 8999):
        got = _check(engine, x, np.array([[-3.0, -0.5, -4.0], [-1.0, -1.0, -2.0]]), 4, True, finished, end)
        assert got[1][0, 0] == 1 and got[2][0, 0] == end and got[0][0, 0] == -0.5
        assert got[1][1].tolist() == [0, 1, 2, -1] and got[2][1].tolist() == [end, end, end, -1]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_rows_inside_wider_ones_and_shared_rows(engine, dtype):
    import torch
    rng = np.random.default_rng(4)
    for vocab, pad in ((1023, 1), (5001, 3), (60, 7)):
        wide = torch.from_numpy(rng.standard_normal((3, 4, vocab + pad)).astype(np.float32)).to(_t(dtype)).cuda()
        for first in range(0, pad + 1):
            view = wide[:, :, first:first + vocab]
            _check(engine, view, rng.standard_normal((3, 4)), 9)
        _check(engine, wide[:, :1, pad:].expand(3, 4, vocab), rng.standard_normal((3, 4)), 9)     # all beams share a row
        _check(engine, wide[:1, :, :vocab].expand(3, 4, vocab), rng.standard_normal((3, 4)), 9)
        _check(engine, wide[:, :, :vocab].transpose(0, 1), rng.standard_normal((4, 3)), 9)


def test_more_good_candidates_in_few_shares_than_a_list_orders(engine):
    """Candidates at places that few threads look at: the second stage (5 of 512 places of every piece), the first (120 of 512
    pieces), and the small form."""
    import torch
    rng = np.random.default_rng(5)
    x = torch.full((1, 1, 200_000), float("-inf"))
    at = np.arange(200_000)
    at = at[at % 512 < 5]
    x[0, 0, at] = torch.from_numpy(rng.standard_normal(at.size).astype(np.float32))
    for normalize in (True, False):
        _check(engine, x, np.zeros((1, 1)), 128, normalize)
        _check(engine, torch.where(x > -1e9, 1.0, x), np.zeros((1, 1)), 128, normalize)
    vocab = 75 * 1024
    pieces = -(-(vocab + 3) // 1024)
    x = torch.from_numpy(rng.standard_normal((1, 64, vocab)).astype(np.float32))
    for j in range(64):
        for p in range(pieces):
            if (j * pieces + p) % 512 >= 120:
                x[0, j, p * 1024:(p + 1) * 1024] = float("-inf")
    _check(engine, x, rng.standard_normal((1, 64)), 128)
    x = torch.full((1, 1, 4096), float("-inf"))
    x[0, 0, ::2] = 1.0
    _check(engine, x, np.zeros((1, 1)), 100)


def test_selection_is_the_top_k_of_each_row_with_one_beam(engine):
    import torch
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn((7, 1, 123_457), device="cuda", generator=g)
    s, b, t = engine.selectBeams(x, torch.zeros((7, 1), device="cuda"), 100, normalize=False)
    v, i = torch.topk(x[:, 0], 100, dim=1)
    assert torch.equal(s, v) and torch.equal(torch.gather(x[:, 0], 1, t), v) and bool((b == 0).all())


# ---- states ---------------------------------------------------------------------------------------------------------------------

def _moved(t, o, parents, lengths, axis):
    """What reorderStates makes of result o from state t (host tensors), by indexing."""
    b, w = parents.shape
    new = o.clone()
    for i in range(b):
        for j in range(w):
            p = int(parents[i, j])
            if p < 0:
                continue
            if lengths is None or axis is None:
                new[i * w + j] = t[i * w + p]
            else:
                n = max(0, min(int(lengths[i]), t.shape[axis]))
                take = [slice(None)] * (t.dim() - 1)
                take[axis - 1] = slice(0, n)
                new[i * w + j][tuple(take)] = t[i * w + p][tuple(take)]
    return new


def _state(gen, shape, dtype):
    import torch
    if dtype in (torch.int64, torch.uint8, torch.bool):
        return torch.randint(0, 2 if dtype == torch.bool else 100, shape, generator=gen).to(dtype)
    return torch.randn(shape, generator=gen).to(dtype)


@pytest.mark.parametrize("beams", [1, 2, 3, 8, 9, 16, 17, 32, 33, 64])
@pytest.mark.parametrize("in_place", [True, False])
def test_reordering(engine, beams, in_place):
    import torch
    gen = torch.Generator().manual_seed(beams)
    batch = 3
    rows = batch * beams
    shapes = [((rows, 2, 19, 33), torch.float16, 2), ((rows, 50), torch.int64, 1), ((rows, 7), torch.uint8, None), ((rows, 3, 8, 64), torch.bfloat16, 2),
              ((rows,), torch.float32, None), ((rows, 5, 3), torch.float16, 1), ((rows, 4, 1025), torch.float32, 2), ((rows, 1), torch.bool, 1)]
    for parents in (torch.randint(-1, beams, (batch, beams), generator=gen), torch.stack([torch.randperm(beams, generator=gen) for _ in range(batch)]),
                    torch.arange(beams).expand(batch, beams), torch.full((batch, beams), -1), torch.arange(beams).roll(1).expand(batch, beams)):
        for lengths in (None, torch.tensor([0, 6, 10 ** 6]), torch.tensor([-4, 1, 19])):
            states = [_state(gen, s, d) for s, d, _ in shapes]
            results = states if in_place else [_state(gen, s, d) for s, d, _ in shapes]
            want = [_moved(t, o, parents, lengths, x[2]) for t, o, x in zip(states, results, shapes)]
            dev = [t.cuda() for t in states]
            out = None if in_place else [t.cuda() for t in results]
            got = engine.reorderStates(dev, parents.cuda(), lengths=None if lengths is None else lengths.cuda(),
                                       time_axis=[x[2] for x in shapes], out=out)
            for g, e, d in zip(got, want, dev if in_place else out):
                assert g is d and torch.equal(g.cpu(), e)
            if not in_place:
                assert all(torch.equal(d.cpu(), t) for d, t in zip(dev, states))


def test_reordering_many_states_and_rows_inside_wider_ones(engine):
    import torch
    gen = torch.Generator().manual_seed(77)
    parents = torch.randint(0, 4, (5, 4), generator=gen)
    lengths = torch.randint(0, 12, (5,), generator=gen)
    packed = torch.randn((20, 2, 3, 11, 16), generator=gen).cuda()               # keys and values side by side
    before = packed.cpu()
    many = [torch.randn((20, 3, 11, 16), generator=gen).cuda() for _ in range(70)]
    many_before = [t.cpu() for t in many]
    heads_first = torch.randn((3, 20, 11, 16), generator=gen).cuda()             # rows between heads
    hf_before = heads_first.cpu()
    engine.reorderStates([packed[:, 0], packed[:, 1], heads_first.transpose(0, 1)] + many, parents.cuda(), lengths=lengths.cuda(), time_axis=2)
    for k in range(2):
        assert torch.equal(packed[:, k].cpu(), _moved(before[:, k], before[:, k], parents, lengths, 2))
    assert torch.equal(heads_first.transpose(0, 1).cpu(), _moved(hf_before.transpose(0, 1), hf_before.transpose(0, 1), parents, lengths, 2))
    for t, o in zip(many, many_before):
        assert torch.equal(t.cpu(), _moved(o, o, parents, lengths, 2))


def test_a_bad_parent_leaves_its_batch_entry_alone(engine):
    import torch
    import vectorstorekit_b200 as vsk
    for bad in (4, -2, 2 ** 40):
        t = torch.arange(8 * 300).view(8, 300).cuda()
        was = t.clone()
        parents = torch.tensor([[1, 0, 3, 2], [1, bad, 0, 0]]).cuda()
        with pytest.raises(vsk.InvalidInput):
            engine.reorderStates([t], parents)
        assert torch.equal(t[4:], was[4:]) and torch.equal(t[:4], was[:4][parents[0]])
    parents[1, 1] = 2
    engine.reorderStates([t], parents)               # the next call is not touched by it


def test_beam_refusals(engine):
    import torch
    import vectorstorekit_b200 as vsk
    x, s = torch.randn((2, 3, 100), device="cuda"), torch.zeros((2, 3), device="cuda")
    bad = [(vsk.InvalidInput, dict(logits=x.cpu())), (vsk.DimensionMismatch, dict(logits=x[0])), (vsk.UnsupportedOperation, dict(logits=x.double())),
           (vsk.EmptyInput, dict(logits=x[:, :, :0])), (vsk.DimensionMismatch, dict(scores=s[:1])), (vsk.InvalidInput, dict(scores=s.half())),
           (vsk.InvalidInput, dict(scores=s.cpu())), (vsk.InvalidInput, dict(k=0)), (vsk.InvalidInput, dict(k=129)),
           (vsk.DimensionMismatch, dict(finished=torch.zeros((2, 2), dtype=torch.bool, device="cuda"))),
           (vsk.InvalidInput, dict(finished=s)), (vsk.InvalidInput, dict(finished=s.bool(), end_token=100)),
           (vsk.InvalidInput, dict(finished=s.bool(), end_token=-1)), (vsk.InvalidInput, dict(logits=x[:, :1].expand(2, 65, 100), scores=torch.zeros((2, 65), device="cuda")))]
    for error, kw in bad:
        a = dict(logits=x, scores=s, k=4)
        a.update(kw)
        with pytest.raises(error):
            engine.selectBeams(**a)
    t, p = torch.zeros((6, 5, 8), device="cuda"), torch.zeros((2, 3), dtype=torch.int64, device="cuda")
    n = torch.zeros(2, dtype=torch.int64, device="cuda")
    bad = [(vsk.EmptyInput, dict(states=[])), (vsk.InvalidInput, dict(states=[t.cpu()])), (vsk.DimensionMismatch, dict(states=[t[:5]])),
           (vsk.InvalidInput, dict(parents=p.int())), (vsk.InvalidInput, dict(parents=p.cpu())), (vsk.InvalidInput, dict(lengths=n[:1], time_axis=1)),
           (vsk.InvalidInput, dict(lengths=n.int(), time_axis=1)), (vsk.InvalidInput, dict(lengths=n, time_axis=0)),
           (vsk.InvalidInput, dict(lengths=n, time_axis=3)), (vsk.DimensionMismatch, dict(out=[])), (vsk.DimensionMismatch, dict(out=[t.half()])),
           (vsk.InvalidInput, dict(states=[t, t])), (vsk.InvalidInput, dict(states=[t, t + 1], out=[t + 2, t])),
           (vsk.InvalidInput, dict(states=[t.transpose(1, 2)], lengths=n, time_axis=1)),
           (vsk.InvalidBufferSize, dict(states=[torch.zeros((1, 40), device="cuda").expand(6, 40)])),
           (vsk.InvalidInput, dict(states=[torch.zeros((65, 2), device="cuda")], parents=torch.zeros((1, 65), dtype=torch.int64, device="cuda")))]
    for error, kw in bad:
        a = dict(states=[t], parents=p)
        a.update(kw)
        with pytest.raises(error):
            engine.reorderStates(**a)


def test_a_refused_state_leaves_the_others_of_its_call_alone(engine):
    """A state of more parts than a launch has blocks (2^31, of one byte), beside one that could move: nothing moves."""
    import torch
    from vectorstorekit_b200 import _lib
    a = torch.arange(2 * 64, dtype=torch.uint8, device="cuda").reshape(2, 64)
    before, other = a.clone(), torch.zeros(64, dtype=torch.uint8, device="cuda")
    parents = torch.tensor([[1, 0]], device="cuda")
    good = _lib.STATE.pack(a.data_ptr(), a.data_ptr(), 64, 64, 0, 0, 1, 1, 64, 0, 0)
    call = lambda states, p: engine._lib.vsk_reorder_states_dev(engine.dev._h, b"".join(states), len(states), 1, 2, C.c_void_p(p), None)
    large = _lib.STATE.pack(other.data_ptr(), other.data_ptr(), 1, 1, 1, 1, 1 << 31, 1, 1, 0, 0)
    assert call([good, large], parents.data_ptr()) == 4 and call([good], parents.data_ptr() + 4) == 7
    assert call([good], a.data_ptr() + 16) == 7   # parents in the state
    assert torch.equal(a, before)
    assert call([good], parents.data_ptr()) == 0
    assert torch.equal(a, before.flip(0))


def test_two_contexts_at_once_and_a_stream_of_the_callers(engine):
    """Workspaces belong to a context: steps of two threads do not disturb each other.  Inputs still being made on another stream are waited for."""
    import threading

    import torch
    import vectorstorekit_b200 as vsk
    gen = torch.Generator().manual_seed(5)
    inputs = []
    for vocab, dim, w in ((5003, 320, 4), (2000, 1030, 6)):
        rows, x = torch.randn((vocab, dim), generator=gen).cuda(), torch.randn((w, dim), generator=gen).half().cuda()
        inputs.append((rows, x, torch.randn((1, w), generator=gen).cuda(), torch.randn((w, 3, 50, 8), generator=gen).cuda()))

    def step(e, rows, x, scores, state):
        q = vsk.Int4Quantizer(e.dev, 64)
        logits = q.product(x, *q.quantizeBatch(rows), out_dtype=torch.float32)
        got = e.selectBeams(logits[None], scores, x.shape[0])
        out = [torch.empty_like(state)]
        e.reorderStates([state], got[1], out=out)
        return [logits, *got, *out]

    want = [step(engine, *i) for i in inputs]
    other = vsk.CUDAAccelerationEngine(vsk.CUDAComputeDevice(0))
    wrong, done = [], []

    def repeat(e, i):
        torch.cuda.set_device(0)
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                fresh = [t.clone() for t in inputs[i]]   # (made on this thread's stream)
                wrong.extend(j for j, (a, b) in enumerate(zip(step(e, *fresh), want[i])) if not torch.equal(a, b))
                done.append(i)

    threads = [threading.Thread(target=repeat, args=a) for a in ((engine, 0), (other, 1))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    other.dev.close()
    assert wrong == [] and len(done) == 40


def test_a_beam_search_with_an_output_head_in_four_bits(engine):
    """Head -> selection -> states, six steps, beams that finish on the way: the same sequences as in 64 bits."""
    import torch
    import vectorstorekit_b200 as vsk
    rng = np.random.default_rng(21)
    batch, beams, vocab, dim, end, steps = 3, 5, 5003, 200, 11, 6
    head = vsk.Int4Quantizer(engine.dev, 32, False)
    w = rng.standard_normal((vocab, dim)).astype(np.float32) * 0.3
    w[end] += 0.05
    codes, scales, middles = head.quantizeBatch(torch.from_numpy(w).cuda())
    w64 = int4_plain.values(*int4_plain.encode(w, 32, False), 32)
    embed = rng.standard_normal((vocab, dim)).astype(np.float32)
    h = rng.standard_normal((batch * beams, dim)).astype(np.float32)
    h = np.repeat(h[::beams], beams, 0)                       # one prompt per batch entry: its beams begin as copies
    first = np.full((batch, beams), -np.inf, np.float32)
    first[:, 0] = 0
    hd, ed = torch.from_numpy(h).cuda(), torch.from_numpy(embed).cuda()
    history = torch.full((batch * beams, steps), -1, dtype=torch.int64, device="cuda")
    scores, finished = torch.from_numpy(first).cuda(), torch.zeros((batch, beams), dtype=torch.bool, device="cuda")
    h64, hist64, s64, f64 = h.astype(np.float64), np.full((batch * beams, steps), -1), first.astype(np.float64), np.zeros((batch, beams), bool)
    for step in range(steps):
        logits = head.product(hd, codes, scales, middles).view(batch, beams, vocab)
        scores, parents, tokens = engine.selectBeams(logits, scores, beams, finished=finished, end_token=end)
        engine.reorderStates([hd, history], parents, lengths=torch.full((batch,), step, device="cuda"), time_axis=[None, 1])
        history[:, step] = tokens.view(-1)
        finished = torch.gather(finished, 1, parents.clamp(min=0)) | (tokens == end)
        hd = 0.5 * hd + ed[tokens.clamp(min=0).view(-1)]
        # the same in 64 bits
        total = plain.totals((h64 @ w64.T).reshape(batch, beams, vocab), s64, f64, end, True)
        at = plain.choose(total, beams)
        par, tok = at // vocab, at % vocab
        s64 = np.take_along_axis(total, at, 1)
        rows = (np.arange(batch)[:, None] * beams + par).reshape(-1)
        h64, hist64 = h64[rows], hist64[rows]
        hist64[:, step] = tok.reshape(-1)
        f64 = np.take_along_axis(f64, par, 1) | (tok == end)
        h64 = 0.5 * h64 + embed.astype(np.float64)[tok.reshape(-1)]
    assert np.array_equal(history.cpu().numpy(), hist64)
    # six normalised steps on logits of magnitude below 64: fp32 sums of 200 terms and the sums of exponentials
    assert np.allclose(scores.cpu().numpy(), s64, rtol=0, atol=6 * (plain.LSE + 2 * 300 * 2.0 ** -23 * 64))
