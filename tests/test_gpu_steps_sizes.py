"""Steps of several tokens over the f16 KV cache at sizes of their own: more ranges of slots than a wave has lanes.
Against the formulas in 64 bits (steps_ref.py)."""
import numpy as np
import pytest

import steps_ref as R
from test_gpu_kernels import mem  # noqa: F401 (fixture)
from test_gpu_steps import Step, close

pytestmark = pytest.mark.gpu


def check_chunk(s, see, **terms):
    """One call with a mass against the oracle: out, the mass of the slots in use, everything else as it was."""
    ref = {k: terms[k] for k in ("cap", "slopes") if k in terms}
    want, w, tol, wtol = s.want(see, **ref)
    total = s.past + s.n
    mass0 = np.random.default_rng(9).random((s.layers, s.nkh, s.max_ctx)).astype(np.float32)
    close(s.chunk(mass=mass0, **terms), want, tol)
    add, off = R.mass(w, wtol, s.nkh)
    exp = mass0.astype(np.float64)
    exp[s.layer, :, :total] += add
    full = np.zeros_like(exp)
    full[s.layer, :, :total] = off + 2 * R.F32 * exp[s.layer, :, :total]
    close(s.dev.download(s.pm, mass0.shape, np.float32).astype(np.float64), exp, full)


@pytest.mark.parametrize("n,past,nqh,nkh,hd", [
    (1, 10000, 4, 1, 64), (1, 16383, 16, 1, 128), (2, 16382, 6, 2, 40), (1, 20500, 2, 2, 96), (1, 40000, 3, 1, 32),
    (3, 16381, 16, 2, 64), (20, 9000, 2, 1, 128), (1, 9000, 2, 1, 250), (5, 10000, 4, 1, 256)])
def test_more_ranges_than_lanes(dev, mem, n, past, nqh, nkh, hd):
    """65 to 128 ranges of slots a row, and contexts whose ranges are longer for the limit of 128."""
    s = Step(np.random.default_rng(past), mem, dev, n, past, nqh, nkh, hd, layer=0, out_pad=3)
    check_chunk(s, R.sees_chunk(n, past), cap=12.0)
