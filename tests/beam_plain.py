"""A beam search's selection from its definition, in 64 bits (numpy), and the comparison the tests use."""
import numpy as np

# Two totals of different beams that lie nearer than this may change places: a row's log-sum-exp from fp32 terms.  A term exp(d),
# d = x - max <= 0, is off by |d| 3 2^-24 (the difference, the product with log2 e, the constant) and 2^-22 (the function), relative; weighted
# with the terms themselves |d| averages below ln(vocab) < 20; sums of 32 terms and trees of 15 steps add 64 roundings at most.
LSE = (20 * 3 + 4 + 64) * 2.0 ** -24


def totals(logits, scores, finished, end, normalize):
    """[batch][beams * vocab] in 64 bits, -inf where there is no candidate"""
    x = logits.astype(np.float64)
    b, w, v = x.shape
    live = np.isfinite(scores)
    out = np.full(x.shape, -np.inf)
    for i in range(b):
        for j in range(w):
            if not live[i, j]:
                continue
            if finished is not None and finished[i, j]:
                out[i, j, end] = scores[i, j]
                continue
            row = x[i, j]
            if normalize:
                top = row.max()
                if not np.isfinite(top):      # nothing but -inf, a +inf, a NaN
                    continue
                row = row - (top + np.log(np.exp(row - top).sum()))
            out[i, j] = np.where(np.isnan(row), -np.inf, float(scores[i, j]) + row)
    return out.reshape(b, w * v)


def choose(total, k):
    """-> (places [batch][k], -1 where there is none); equal totals by the lowest place"""
    out = np.full((total.shape[0], k), -1, np.int64)
    for i, row in enumerate(total):
        order = np.argsort(-row, kind="stable")[:k]
        order = order[row[order] > -np.inf]
        out[i, :order.size] = order
    return out


def compare(got, logits, scores, finished, end, normalize):
    gs, gb, gt = (np.asarray(a) for a in got)
    v, k = logits.shape[2], gs.shape[1]
    total = totals(logits, scores, finished, end, normalize)
    want = choose(total, k)
    at = np.where(gb < 0, -1, gb * v + gt)
    assert np.array_equal(gb < 0, gt < 0) and np.array_equal(at < 0, want < 0)
    assert np.all(np.isneginf(gs[at < 0]))
    r, c = np.nonzero(at >= 0)
    mine, theirs = total[r, at[r, c]], total[r, want[r, c]]
    other = at[r, c] != want[r, c]
    # a different place only among different beams, with totals that near
    slack = LSE if normalize else 0.0
    assert np.all(np.abs(mine - theirs)[other] <= 2 * slack) and np.all(gb[r, c][other] != (want // v)[r, c][other])
    for row in at:
        assert np.unique(row[row >= 0]).size == (row >= 0).sum()
    both_inf = np.isinf(mine)
    assert np.array_equal(gs[r, c][both_inf], mine[both_inf].astype(np.float32))
    off = np.abs(gs[r, c][~both_inf] - mine[~both_inf])
    assert np.all(off <= slack + 2.0 ** -24 * (np.abs(mine[~both_inf]) + slack) + 2.0 ** -149), off.max()
    assert np.all(gs[:, :-1] >= gs[:, 1:])
    return int(other.sum())
