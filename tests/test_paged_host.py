"""Host side of the paged-serving operators: the axis of each rotary pair."""
import numpy as np


def test_axis_maps(lq8_lib):
    R = lq8_lib.Rotary
    assert R.blocks([2, 3, 1]).tolist() == [0, 0, 1, 1, 1, 2]
    assert R.cyclic([2, 2, 2]).tolist() == [0, 1, 2, 0, 1, 2]
    a = R.cyclic([24, 20, 20])
    assert a[:60].tolist() == [0, 1, 2] * 20 and not a[60:].any()
    assert np.bincount(a).tolist() == [24, 20, 20]
    assert R.cyclic([3, 1]).tolist() == [0, 1, 0, 0]
