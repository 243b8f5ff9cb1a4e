"""Microscaled rows without a GPU: calls that have to be refused before anything is launched."""
import ctypes as C

import numpy as np
import pytest

from lidar_ai_solution_amd import capi


@pytest.mark.parametrize("shape, at, where", [((4, 3, 3, 3, 64), (1, 2, 0, 1, 40), "channel 1, kernel offset 19, input channels 32 to 63"),
                                              ((40, 1, 1, 1, 5), (39, 0, 0, 0, 4), "channel 39, kernel offset 0, input channels 0 to 4"),
                                              ((16, 1, 3, 1, 160), (0, 0, 1, 0, 159), "channel 0, kernel offset 1, input channels 128 to 159")])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_convolution_refuses_weights_that_are_not_finite(shape, at, where, bad):
    """A block that is not finite would make a NaN of rows without a neighbour at its offset, too."""
    w = np.ones(shape, np.float16)
    w[at] = bad
    assert not capi.lib().scn_conv_create(w.ctypes.data_as(C.c_void_p), capi.i5(*shape), None, None, capi.PRECISION_MXFP4)
    text = capi.lib().scn_last_error().decode()
    assert "finite" in text and where in text
