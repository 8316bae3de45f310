"""The long row of pages_long.py tells a right merge of its pieces from wrong ones (on the CPU, in 64 bits)."""
import numpy as np
import pytest

import pages_long as L
import pages_ref as R


@pytest.mark.parametrize("t", [R.F16, R.Q8_0], ids=["f16", "q8"])
@pytest.mark.parametrize("hd", [32, 160])
def test_wrong_merges_are_seen(t, hd):
    row = L.LongRow(np.random.default_rng(hd), t, hd)
    m, l, o = row.parts()
    assert len(m) > L.BATCH and (m[:L.BATCH].max(0) != m[L.BATCH:].max(0)).all()
    want, tol = row.want(m, l, o)
    whole = np.exp(row.held["k"] - row.held["k"].max(0))
    assert (np.abs((whole.T @ row.held["v"]) / whole.sum(0)[:, None] - want) < 1e-9 * tol / R.S.F32).all()
    for what, out in row.wrong(m, l, o):
        assert (np.abs(out - want).max(1) > 4 * tol.max(1)).all(), (what, np.abs(out - want).max(1), tol.max(1))
