"""What vbs_gfx950_rope_axes refuses of theta, checked on the host before a device is looked at (nothing is launched)."""
import pytest

import vbs_gfx950 as V
from test_steps_refusals import ROPE, refused


@pytest.mark.parametrize("theta", [4.7e-7, 1e-30, 1e-45])
def test_thetas_whose_angles_pass_64_bits(theta):
    """Below 2^-21 the last pairs of far positions turn by more than 2^52: their angles are no numbers to 64 bits."""
    lib = V.DeviceLib()
    refused(lib, lib.rope_axes, {**ROPE, "theta": theta}, "theta")
