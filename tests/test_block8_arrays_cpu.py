"""CPU suite: what Block8 takes for a pattern."""
import numpy as np
import pytest

from alphasparse_b200 import block8, capi


@pytest.mark.parametrize("ptr,col", [
    ([0, 1, 1], [0.7]), ([0, 1.5, 1], [0]), (np.array([0.0, 0.5, 1.0]), [0]), ([0, 1, np.nan], [0]), ([0, 1, 1], [float("inf")]), ([0, 1, 1], ["0"]), ([0, 1, 1], np.array([0], dtype=object)),
])
def test_arrays_that_are_no_whole_numbers_are_refused(ptr, col):
    with pytest.raises(ValueError):
        block8.Block8(None, 200, 200, ptr, col)


@pytest.mark.parametrize("ptr,col", [
    ([0, 1, 1], [0]), (np.array([0, 1, 1], dtype=np.uint8), np.array([1], dtype=np.int16)), ([0, 0, 0], []), (np.array([0, 1, 2], dtype=np.uint64), (0, 1)), (range(3), range(2)), (np.array([0.0, 1.0, 1.0]), np.array([1.0])),
])
def test_all_kinds_of_whole_numbers_are_taken(ptr, col):
    """Up to the context, which is looked at last (a closed one here)."""
    ctx = object.__new__(capi.Context)
    ctx._h = block8.C.c_void_p()
    with pytest.raises(capi.AspError) as e:
        block8.Block8(ctx, 200, 200, ptr, col)
    assert "ctx is NULL" in str(e.value)
