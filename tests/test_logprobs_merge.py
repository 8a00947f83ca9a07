"""The merge of slices' log probabilities (host) where a slice has no distribution."""
import numpy as np
import pytest


def merge(fnx, lse, ent, lp, top, ids):
    """Slices' results, [slice][row]...; (lse, entropy, lp, top_lp, top_i) of the whole."""
    a = [np.ascontiguousarray(x, np.int32 if i == 4 else np.float32) for i, x in enumerate((lse, ent, lp, top, ids))]
    out = [np.full(x.shape[1:], -7, x.dtype) for x in a]
    fnx.call("fnx_logprobs_merge", *(x.ctypes.data for x in a), a[0].shape[0], a[0].shape[1], a[2].shape[2], a[3].shape[2], *(x.ctypes.data for x in out))
    return out


def _slice(x, v0, tok, k):
    """What a slice of a row of logits gives, from the definition in 64 bits."""
    x = np.asarray(x, np.float64)
    m = x.max()
    lse = m + np.log(np.exp(x - m).sum())
    order = np.argsort(-x, kind="stable")[:k]
    lp = [x[t - v0] - lse if 0 <= t - v0 < len(x) else -np.inf for t in tok]
    return lse, -(np.exp(x - lse) * (x - lse)).sum(), lp, x[order] - lse, order + v0


@pytest.mark.parametrize("where", [0, 1, 2])
def test_a_slice_without_a_distribution_takes_the_row_with_it(fnx, where):
    """Wherever the slice lies, the row is what the whole row's is: NaNs, no ids; the row after it is untouched."""
    nan, k, tok = np.nan, 3, [1, 9]
    good = [_slice(x, v0, tok, k) for x, v0 in (([1.0, 2, 3, 4], 0), ([5.0, 0, 1], 4), ([2.0, 2.5, 7, 1], 7))]
    bad = [(nan, nan, [nan if v <= t < e else -np.inf for t in tok], [nan] * k, [-1] * k) for v, e in ((0, 4), (4, 7), (7, 11))]
    rows = [[bad[i] if i == where else g for i, g in enumerate(good)], good]
    lse, ent, lp, top, ids = merge(fnx, *([[rows[t][i][f] for t in range(2)] for i in range(3)] for f in range(5)))
    assert np.isnan(lse[0]) and np.isnan(ent[0]) and np.isnan(lp[0]).all() and np.isnan(top[0]).all()
    assert ids[0].tolist() == [-1] * k
    whole = _slice([1, 2, 3, 4, 5, 0, 1, 2, 2.5, 7, 1], 0, tok, k)
    assert ids[1].tolist() == whole[4].tolist() and np.allclose(top[1], whole[3], rtol=0, atol=2.0 ** -20) and np.allclose(lp[1], whole[2], rtol=0, atol=2.0 ** -20)


@pytest.mark.parametrize("base", [0.0, 40.0, 5000.0, -3e7, float(np.finfo(np.float32).min), 3e38])
def test_the_size_of_the_logits_costs_nothing(fnx, base):
    """Two slices of the same weight: the whole's entropy and log probabilities come from differences of the slices' lse, never from a
    difference of sums that hold it.  Roundings: the slices' values are exact in 32 bits here, the results are rounded once (2^-24 of at
    most 8).  The order of two slices' alternatives is that of their logits in 32 bits, so one may come for the other where they
    differ by less than 2^-23 of those."""
    k, tok, ln = 2, [0, 3], np.log
    lse = [[base], [base]]   # two slices of the same weight: e^lse each
    ent, own = [[1.25], [0.5]], [[[-0.75, -np.inf]], [[-np.inf, -0.125]]]
    top, ids = [[[-0.75, -1.5]], [[-0.125, -2.5]]], [[[0, 1]], [[3, 2]]]
    got = merge(fnx, lse, ent, own, top, ids)
    want_lse = np.float64(np.float32(base)) + ln(2)
    assert abs(got[0][0] - want_lse) <= 2.0 ** -24 * abs(want_lse) + 1e-7
    assert abs(got[1][0] - (0.875 + ln(2))) <= 2.0 ** -20
    assert np.allclose(got[2][0], [-0.75 - ln(2), -0.125 - ln(2)], rtol=0, atol=2.0 ** -20)
    near = 2.0 ** -20 + 2.0 ** -23 * abs(base)
    assert (np.abs(got[3][0] - [-0.125 - ln(2), -0.75 - ln(2)]) <= near).all() and got[3][0][1] <= got[3][0][0] <= 0
    if near < 0.5:   # (else the logits may all be alike in 32 bits, and lower ids come first)
        assert got[4][0].tolist() == [3, 0]


def test_a_certain_token_is_never_above_0(fnx):
    """The merged log probability of a token that has everything: lists in order, nothing positive."""
    rng = np.random.default_rng(1)
    for _ in range(300):
        x = rng.standard_normal(12)
        x[rng.integers(12)] += rng.uniform(8, 60)
        x += rng.choice([0.0, 30.0, 1000.0])
        x = x.astype(np.float32).astype(np.float64)
        tok, k = [int(x.argmax()), 2], 3
        rows = [_slice(x[a:b], a, tok, k) for a, b in ((0, 5), (5, 12))]
        got = merge(fnx, *([[r[f]] for r in rows] for f in range(5)))
        assert (got[2] <= 0).all() and (got[3] <= 0).all() and (np.diff(got[3][0]) <= 0).all() and got[1][0] >= 0
