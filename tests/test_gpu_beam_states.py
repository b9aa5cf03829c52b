"""States that share memory: those that lie between one another move, those that overlap are refused and nothing moves."""
import pytest

from test_gpu_beam import _moved

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def engine():
    import vectorstorekit_b200 as vsk
    d = vsk.CUDAComputeDevice(0)
    yield vsk.CUDAAccelerationEngine(d)
    d.close()


def test_states_that_overlap_are_refused(engine):
    import torch
    import vectorstorekit_b200 as vsk
    room = torch.arange(4000, device="cuda").float()
    was = room.clone()
    parents = torch.tensor([[1, 0, 2], [2, 2, 0]], device="cuda")
    lengths = torch.tensor([3, 4], device="cuda")
    at = lambda first, *shape: room[first:first + torch.Size(shape).numel()].view(shape)
    strided = lambda first, shape, stride: torch.as_strided(room, shape, stride, first)
    later = at(1000, 6, 5, 8)
    bad = [(vsk.InvalidInput, dict(states=[at(0, 6, 40)], out=[at(40, 6, 40)])),            # a row further on
           (vsk.InvalidInput, dict(states=[at(0, 6, 40)], out=[at(239, 6, 40)])),           # by one element
           (vsk.InvalidInput, dict(states=[later, at(0, 6, 40)], out=[at(2000, 6, 5, 8), at(1100, 6, 40)])),   # another state's source
           (vsk.InvalidInput, dict(states=[at(0, 6, 40), later], out=[at(2000, 6, 40), at(2200, 6, 5, 8)])),   # two results
           (vsk.InvalidInput, dict(states=[at(0, 6, 40), at(200, 6, 40)])),                  # two in place
           (vsk.InvalidInput, dict(states=[strided(0, (6, 3, 8), (80, 16, 1)), strided(7, (6, 3, 8), (80, 16, 1))])),
           (vsk.InvalidInput, dict(states=[strided(0, (6, 3, 8), (80, 16, 1)), strided(60, (6, 2, 8), (100, 9, 1))])),   # other strides
           (vsk.InvalidBufferSize, dict(states=[strided(0, (6, 3, 8), (16, 24, 1))])),       # parts of one row in another row
           (vsk.InvalidBufferSize, dict(states=[later], out=[strided(0, (6, 5, 8), (20, 8, 1))]))]
    for error, kw in bad:
        with pytest.raises(error):
            engine.reorderStates(parents=parents, **kw)
        assert torch.equal(room, was)
    with pytest.raises(vsk.InvalidInput):
        engine.reorderStates([at(0, 6, 5, 8), at(100, 6, 5, 8)], parents, lengths=lengths, time_axis=1)
    assert torch.equal(room, was)


@pytest.mark.parametrize("in_place", [True, False])
def test_states_between_one_another_move(engine, in_place):
    """Caches of several layers in one block: keys and values of other widths in a row, heads before rows, halves of a time axis; the
    same source into two results."""
    import torch
    gen = torch.Generator().manual_seed(3)
    batch, beams, layers, heads, steps = 2, 3, 3, 4, 6
    rows = batch * beams
    parents = torch.randint(-1, beams, (batch, beams), generator=gen)
    lengths = torch.tensor([steps, 2])

    def views(t):
        row, behind = t["rows"], t["heads"]
        found = []
        for i in range(layers):
            layer = row[:, i]
            found += [layer[:, :heads * steps * 16].view(rows, heads, steps, 16), layer[:, heads * steps * 16:].view(rows, heads, steps, 8)]
        found += [behind[i].transpose(0, 1) for i in range(layers)]
        found += [t["halves"][:, :, :, :5], t["halves"][:, :, :, 5:]]
        found += [torch.as_strided(t["teeth"], (rows, heads, steps, 4), (steps * 8, rows * steps * 8, 4, 1))]
        return found

    def made():
        return {"rows": torch.randn((rows, layers, heads * steps * 24), generator=gen), "heads": torch.randn((layers, heads, rows, steps, 16), generator=gen),
                "halves": torch.randn((rows, heads, 2, 10), generator=gen).contiguous(), "teeth": torch.randn((heads, rows, steps * 8), generator=gen)}

    src = made()
    dst = src if in_place else made()
    axes = [2] * (3 * layers) + [None, None, 2]
    want = [_moved(t, o, parents, lengths if axis else None, axis) for t, o, axis in zip(views(src), views(dst), axes)]
    on = {k: v.cuda() for k, v in src.items()}
    to = on if in_place else {k: v.cuda() for k, v in dst.items()}
    engine.reorderStates(views(on), parents.cuda(), lengths=lengths.cuda(), time_axis=axes, out=None if in_place else views(to))
    assert all(torch.equal(g.cpu(), w) for g, w in zip(views(to), want))
    if not in_place:
        assert all(torch.equal(on[k].cpu(), src[k]) for k in src)
        one = torch.randn((rows, 50), generator=gen).cuda()
        two = [torch.zeros_like(one), torch.zeros_like(one)]
        engine.reorderStates([one, one], parents.cuda(), out=two)
        assert torch.equal(two[0], two[1]) and torch.equal(two[0].cpu(), _moved(one.cpu(), torch.zeros_like(one).cpu(), parents, None, None))
