"""A beam search's step without a device: the row layouts of states, entry points without a context, and the plain form."""
import numpy as np
import pytest

import beam_plain as plain


def test_entry_points_without_a_context():
    from vectorstorekit_b200 import _lib, build
    build.build_library()
    lib = _lib.load()
    assert lib.vsk_beam_select_dev(None, None, 0, 1, 1, 1, 1, 1, None, None, 0, 1, 1, None, None, None) == 7
    assert _lib.STATE.size == 80 and lib.vsk_reorder_states_dev(None, bytes(80), 1, 1, 1, None, None) == 7


def test_row_layouts():
    """(outer parts, elements of one, steps, elements of a step, distances of parts)"""
    import torch
    import vectorstorekit_b200 as vsk
    from vectorstorekit_b200.engine import _row_parts
    t = torch.empty((6, 4, 10, 8))
    assert _row_parts(t, t, 2) == (4, 80, 10, 8, 80, 80)
    assert _row_parts(t, t, 1) == (1, 320, 4, 80, 0, 0)
    assert _row_parts(t, t, None) == (1, 320, 1, 320, 0, 0)
    wide = torch.empty((6, 4, 12, 8))[:, :, :10]
    assert _row_parts(t, wide, 2) == (4, 80, 10, 8, 80, 96)
    assert _row_parts(wide, wide, None) == (4, 80, 1, 80, 96, 96)
    assert _row_parts(torch.empty(6), torch.empty(6), None) == (1, 1, 1, 1, 0, 0)
    assert _row_parts(t[:, 1], t[:, 1], 1) == (1, 80, 10, 8, 0, 0)
    for bad in (t.transpose(1, 2), t[:, :, :, :4], torch.empty((6, 3, 4, 2, 10, 8))[:, :, :2].transpose(1, 2)):
        axis = 2 if bad.dim() == 4 else 4
        with pytest.raises(vsk.InvalidInput):
            _row_parts(bad, bad, axis)


def test_refusals_before_any_device_call():
    import types

    import torch
    import vectorstorekit_b200 as vsk
    e = vsk.CUDAAccelerationEngine(types.SimpleNamespace(_lib=None, device=0))
    with pytest.raises(vsk.InvalidInput):
        e.selectBeams(torch.zeros((1, 1, 4)), torch.zeros((1, 1)), 1)
    with pytest.raises(vsk.EmptyInput):
        e.reorderStates([], torch.zeros((1, 1), dtype=torch.int64))
    with pytest.raises(vsk.InvalidInput):
        e.reorderStates([torch.zeros((1, 1))], torch.zeros((1, 1), dtype=torch.int64))


def test_the_plain_selection_on_numbers_worked_out_by_hand():
    x = np.log(np.array([[[1.0, 2.0, 1.0], [4.0, 2.0, 2.0]]]))
    total = plain.totals(x, np.zeros((1, 2)), None, 0, True)
    assert np.allclose(np.exp(total), [[0.25, 0.5, 0.25, 0.5, 0.25, 0.25]])
    assert plain.choose(np.round(total, 12), 4).tolist() == [[1, 3, 0, 2]]
    done = np.array([[True, False]])
    total = plain.totals(x, np.array([[np.log(0.75), 0.0]]), done, 2, True)
    assert plain.choose(np.round(total, 12), 6).tolist() == [[2, 3, 4, 5, -1, -1]]
