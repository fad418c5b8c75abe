"""Workspace sizes of the row operators: for what the calls take, and refused for
what they refuse."""

import pytest

import numba_mlir_b200 as nm


@pytest.mark.parametrize("count,groups", [(-1, 3), (2**31, 3), (2**63 - 1, 3), (5, -3), (5, 2**31 - 1), (5, 2**62), (5, 2**63 - 1)])
def test_group_rows(runtime_lib, count, groups):
    assert runtime_lib._mlir_ciface_nmb_group_rows_workspace(count, groups) == 0
    with pytest.raises(ValueError, match="must be in"):
        nm.group_rows_workspace(count, groups)


@pytest.mark.parametrize("count,rows,cols", [(-1, 3, 3), (2**31, 3, 3), (5, -3, 3), (5, 2**31 - 1, 3), (5, 2**62, 3),
                                             (5, 3, -1), (5, 3, 2**31)])
def test_take_rows_grad(runtime_lib, count, rows, cols):
    assert runtime_lib._mlir_ciface_nmb_take_rows_grad_workspace(count, rows, cols, 0) == 0
    with pytest.raises(ValueError, match="must be in"):
        nm.take_rows_grad_workspace(count, rows, cols)


def test_the_largest_sizes_are_answered(runtime_lib):
    # two buffers of keys and two of entries at least
    assert nm.group_rows_workspace(2**31 - 1, 2**31 - 2) >= 4 * 4 * (2**31 - 1)
    # order, keys and those
    assert nm.take_rows_grad_workspace(2**31 - 1, 2**31 - 2, 1) >= 6 * 4 * (2**31 - 1)
    assert nm.take_rows_grad_workspace(0, 0, 0) == 0
