"""Values of the operators for steps of several tokens that need no device: what vbs_gfx950_rope_axes refuses of theta
(checked on the host before a device is looked at; nothing is launched), and the tanh of capped scores."""
import os
import re

import numpy as np
import pytest

import vbs_gfx950 as V
from test_steps_refusals import ROPE, refused


@pytest.mark.parametrize("theta", [4.7e-7, 1e-30, 1e-45])
def test_thetas_whose_angles_pass_64_bits(theta):
    """Below 2^-21 the last pairs of far positions turn by more than 2^52: their angles are no numbers to 64 bits."""
    lib = V.DeviceLib()
    refused(lib, lib.rope_axes, {**ROPE, "theta": theta}, "theta")


def test_the_tanh_polynomial():
    """The coefficients of csrc/vbs_attn_rows.h against tanh on |x| < 0.8: 1.3e-8 of the value in exact arithmetic; in f32
    the last step rounds (one half step), x^2 p (at most 0.18 of the factor) loses three, and the fit a quarter: two
    half steps in all."""
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "verum-bespoke-singularity_amd", "csrc")
    with open(os.path.join(at, "vbs_attn_rows.h")) as f:
        body = re.search(r"float tanh_poly\(float x\) \{(.*?)\n\}", f.read(), re.S).group(1)
    coef = [np.float32(c) for c in re.findall(r"(-?0\.\d+)f", body)]
    assert len(coef) == 6
    x = np.linspace(1e-4, 0.8, 400001).astype(np.float32)
    want = np.tanh(x.astype(np.float64))

    def poly(t):
        fma = lambda a, b, c: (a.astype(np.float64) * b.astype(np.float64) + np.float64(c)).astype(t)  # noqa: E731
        y = x.astype(t)
        z = (y * y).astype(t)
        p = np.full(x.shape, coef[0], t)
        for c in coef[1:]:
            p = fma(p, z, c)
        return fma(y, (z * p).astype(t), y.astype(np.float64))
    assert np.abs(poly(np.float64) / want - 1).max() <= 1.3e-8
    assert np.abs(poly(np.float32) / want - 1).max() <= 2 * 2.0 ** -24
