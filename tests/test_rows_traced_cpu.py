"""The row operators inside traced functions, as far as that goes without a
device: what they record and what they refuse."""

import numpy as np
import pytest

import numba_mlir_b200 as nm
from numba_mlir_b200.lazy import fake_array

F, I = np.float32, np.int32


def _calls(queue=None, workspace=None):
    """Every routine on the traced arrays (x, y, ids, order, place, offsets)."""
    q = {} if queue is None else {"queue": queue}
    w = {} if workspace is None else {"workspace": workspace}
    plan = lambda a: nm.RowGroups(*a[3:])  # noqa: E731
    return {
        "take_rows": lambda *a: nm.take_rows(a[0], a[2], **q),
        "take_rows_grad": lambda *a: nm.take_rows_grad(a[1], a[4], 3, **q, **w),
        "group_rows": lambda *a: nm.group_rows(a[2], 3, **q, **w).place,
        "dispatch_rows": lambda *a: nm.dispatch_rows(a[0], a[2], 3, **q)[0],
        "dispatch_rows_grad": lambda *a: nm.dispatch_rows_grad(a[1], plan(a), **q),
        "combine_rows": lambda *a: nm.combine_rows(a[1], plan(a), **q),
        "combine_rows_grad": lambda *a: nm.combine_rows_grad(a[0], a[1], plan(a), **q)[1],
    }


def _arrays(which):
    shapes = [((5, 8), F), ((10, 8), F), ((5, 2), I), ((10,), I), ((5, 2), I), ((4,), I)]
    if which == "take_rows_grad":
        shapes[1] = ((5, 2, 8), F)
    return [fake_array(s, d) for s, d in shapes]


@pytest.mark.parametrize("which", sorted(_calls()))
def test_a_call_is_a_step_of_the_plan(which):
    trace, plan = nm.njit(_calls()[which]).trace_dry(*_arrays(which))
    assert plan is not None and [s[0] for s in trace.steps if s[0] != "alloc"][0] == "rows"


@pytest.mark.parametrize("which", sorted(_calls()))
def test_queue_is_refused(which):
    with pytest.raises(ValueError, match="queue"):
        nm.njit(_calls(queue=object())[which]).trace_dry(*_arrays(which))


@pytest.mark.parametrize("which", ["take_rows_grad", "group_rows"])
def test_workspace_is_refused(which):
    with pytest.raises(ValueError, match="workspace"):
        nm.njit(_calls(workspace=fake_array((4096,), np.uint8))[which]).trace_dry(*_arrays(which))
