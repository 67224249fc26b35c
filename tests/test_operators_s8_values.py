"""Values that Python gives as int8."""
import numpy as np
import pytest

from cldnn_amd import ops


@pytest.mark.parametrize("kind", [np.float32, np.float64, list])
def test_values_are_rounded_to_int8(kind):
    values = [0.0, 0.4, 0.5, 1.5, 2.5, -0.5, -1.5, 1.7, -1.7, 126.6, 127.4, 127.6, 300.0, -128.4, -128.6, -1e30, 1e30, np.inf, -np.inf, np.nan]
    want = [0, 0, 0, 2, 2, 0, -2, 2, -2, 127, 127, 127, 127, -128, -128, -128, 127, 127, -128, 0]
    got = ops.to_type(values if kind is list else np.array(values, kind), "s8")
    assert got.dtype == np.int8 and got.tolist() == want


def test_whole_numbers_are_held_to_int8():
    for kind in (np.int16, np.int32, np.int64, np.uint8):
        assert ops.to_type(np.array([0, 1, 127, 128, 255], kind), "s8").tolist() == [0, 1, 127, 127, 127]
    every = np.arange(-128, 128, dtype=np.int8)
    assert np.array_equal(ops.to_type(every, "s8"), every) and np.array_equal(ops.to_type(every.reshape(16, 16).T, "s8"), every.reshape(16, 16).T)
