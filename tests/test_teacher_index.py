"""A teacher's class indices on their way into a session (no device: a session is asked for last)."""
import numpy as np
import pytest

import catboost_rs_b200 as cb


@pytest.mark.parametrize("bad", [np.array([[1 << 32]]), np.array([[(1 << 32) + 1]]), np.array([[-(1 << 32)]]),
                                 np.array([[1 << 63]], dtype=np.uint64), np.array([[0.5]]), np.array([[np.nan]]),
                                 np.array([[1e20]])])
def test_indices_that_are_no_classes_are_refused(bad):
    with pytest.raises(cb.CbGpuError, match="whole number"):
        cb.B200MultiRuntime().set_teacher(bad, np.zeros((1, 1)))


@pytest.mark.parametrize("good", [np.array([[2]]), np.array([[-1]]), np.array([[2.0]]), np.array([[3]], dtype=np.uint8),
                                  [[1]]])
def test_whole_numbers_of_any_type_are_taken(good):
    with pytest.raises(cb.CbGpuError, match="no session"):
        cb.B200MultiRuntime().set_teacher(good, np.zeros((1, 1)))
