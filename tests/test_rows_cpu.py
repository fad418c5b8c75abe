"""What the row operators refuse, checked before anything reaches a device: the
argument checks of numba_mlir_b200.rows and those of the C entries."""

import ctypes

import numpy as np
import pytest

import numba_mlir_b200 as nm
from numba_mlir_b200 import rows, runtime
from numba_mlir_b200.device_array import DeviceArray, _Foreign
from numba_mlir_b200.lazy import fake_array


class _Queue:
    """Stands in for a queue: every call of the library is refused (null handle)."""

    def __init__(self, device=0, stream=5):
        self.device, self.stream, self.handle, self.waits = device, stream, None, []

    def wait_stream(self, s):
        self.waits.append(s)


Q = _Queue()


def arr(shape, dtype=np.float32, queue=Q, strides=None, ptr=None):
    if ptr is None:
        ptr = fake_array(shape, dtype).ptr
    return DeviceArray(_Foreign(None, ptr, 1 << 30, queue), shape, dtype, strides)


def test_argument_checks(runtime_lib):
    t, ids = arr((5, 8)), arr((3,), np.int32)
    cases = [
        (TypeError, lambda: nm.take_rows(np.zeros((5, 8)), ids)),
        (TypeError, lambda: nm.take_rows(t, arr((3,), np.float32))),
        (TypeError, lambda: nm.take_rows(t, arr((3,), np.int16))),
        (TypeError, lambda: nm.take_rows(arr((5, 8), np.int32), ids, out=arr((3, 8)))),
        (ValueError, lambda: nm.take_rows(arr((8,)), ids, out=arr((3, 8)))),
        (ValueError, lambda: nm.take_rows(arr((5, 8), strides=(64, 8)), ids, out=arr((3, 8)))),
        (ValueError, lambda: nm.take_rows(arr((5, 8), strides=(34, 4)), ids, out=arr((3, 8)))),
        (ValueError, lambda: nm.take_rows(t, arr((3,), np.int32, strides=(8,)), out=arr((3, 8)))),
        (ValueError, lambda: nm.take_rows(t, ids, out=arr((3, 9)))),
        (TypeError, lambda: nm.take_rows(t, ids, out=arr((3, 8), np.float64))),
        (TypeError, lambda: nm.take_rows(arr((5, 8), np.float16), ids, out=arr((3, 8), nm.bfloat16))),
        (ValueError, lambda: nm.take_rows(t, ids, out=arr((3, 8), ptr=t.ptr + 32))),
        (ValueError, lambda: nm.take_rows(t, arr((3,), np.int32, _Queue(1)), out=arr((3, 8)))),
        (ValueError, lambda: nm.take_rows_grad(arr((3, 8)), ids)),
        (ValueError, lambda: nm.take_rows_grad(arr((4, 8)), ids, out=arr((5, 8)))),
        (ValueError, lambda: nm.take_rows_grad(arr((3, 8)), ids, 6, out=arr((5, 8)))),
        (ValueError, lambda: nm.take_rows_grad(arr((3, 8)), ids, 5, accumulate=True)),
        (ValueError, lambda: nm.group_rows(ids, -1)),
        (ValueError, lambda: nm.group_rows(ids, 2, plan=nm.RowGroups(arr((4,), np.int32), arr((3,), np.int32), arr((3,), np.int32)))),
        (TypeError, lambda: nm.group_rows(ids, 2, plan=nm.RowGroups(arr((3,), np.int64), arr((3,), np.int32), arr((3,), np.int32)))),
        (ValueError, lambda: nm.dispatch_rows(t, ids, 2, out=arr((5, 8)))),
        (ValueError, lambda: nm.dispatch_rows(t, arr((5,), np.int32))),
        (TypeError, lambda: nm.dispatch_rows(t, arr((5,), np.int32), 2, out=arr((5, 8), np.float16))),
        (TypeError, lambda: nm.take_rows_grad_workspace(3, 4, 5, np.int32)),
    ]
    for i, (kind, call) in enumerate(cases):
        with pytest.raises(kind):
            call()
            pytest.fail(f"case {i} was accepted")
    with pytest.raises(runtime.GpuRuntimeError, match="null"):
        nm.take_rows(t, ids, out=arr((3, 8)))  # all in order: reaches the library, which has no queue here


def test_leading_axes():
    view = lambda *a, **k: rows._row_view(rows._operand(arr(*a, **k), "x"), "x")  # noqa: E731
    assert view((4, 3, 8)) == (12, 8, 8)
    assert view((4, 3, 8), strides=(192, 64, 4)) == (12, 8, 16)
    assert view((4, 1, 8), strides=(64, 4000, 4)) == (4, 8, 16)
    assert view((8,)) == (1, 8, 8)
    assert view((3, 0, 8)) == (0, 8, 8)
    assert view((3, 8), strides=(-64, 4)) == (3, 8, -16)
    with pytest.raises(ValueError):
        view((4, 3, 8), strides=(256, 64, 4))
    with pytest.raises(ValueError):
        view(())


def test_columns_of_one_buffer_are_apart():
    op = lambda a: rows._operand(a, "a")  # noqa: E731
    left = arr((6, 8), strides=(64, 4))
    right = arr((6, 8), strides=(64, 4), ptr=left.ptr + 32)
    rows._no_overlap([op(left)], [op(right)])
    rows._no_overlap([op(right)], [op(left)])
    for off in (0, 4, 28, 36, 60):
        with pytest.raises(ValueError):
            rows._no_overlap([op(left)], [op(arr((6, 8), strides=(64, 4), ptr=left.ptr + off))])
    with pytest.raises(ValueError):  # rows one further down
        rows._no_overlap([op(left)], [op(arr((2, 8), strides=(64, 4), ptr=left.ptr + 64))])


def test_streams_are_ordered_both_ways():
    a, b = _Queue(stream=5), _Queue(stream=7)
    on = rows._On(None, [rows._operand(arr((2, 2), queue=a), "x"), rows._operand(arr((2, 2), queue=b), "y"),
                         rows._operand(arr((2, 2), queue=b), "z")])
    assert on.queue is a and a.waits == [7] and b.waits == []
    on.done(0)
    assert b.waits == [5]
    c = _Queue(stream=0)
    on = rows._On(c, [rows._operand(arr((2, 2), queue=a), "x")])
    assert c.waits == [5]
    on.done(0)
    assert a.waits[-1] == 1  # the legacy default stream by its name in the array interface


def _rows(ptr, r, c, stride=None, kind=0):
    return ctypes.byref(rows._Rows(ptr, r, c, c if stride is None else stride, kind, 0))


def _index(ptr, n, nbytes=4):
    return ctypes.byref(rows._Index(ptr, n, nbytes, 0))


def test_c_entries_refuse(runtime_lib):
    """Refusals come before the queue is looked at; nothing is enqueued."""
    lib = runtime_lib
    A, B, C = 0x10000, 0x20000, 0x30000
    take = lib._mlir_ciface_nmb_take_rows_device
    grad = lib._mlir_ciface_nmb_take_rows_grad_device
    group = lib._mlir_ciface_nmb_group_rows_device
    disp = lib._mlir_ciface_nmb_dispatch_rows_device
    comb = lib._mlir_ciface_nmb_combine_rows_device
    cgrad = lib._mlir_ciface_nmb_combine_rows_grad_device

    def refused(match, fn, *args):
        assert fn(None, *args) != 0
        with pytest.raises(runtime.GpuRuntimeError, match=match):
            runtime.check()

    refused("null", take, None, _index(B, 3), 1.0, _rows(C, 3, 8))
    refused("unknown element type", take, _rows(A, 5, 8, kind=4), _index(B, 3), 1.0, _rows(C, 3, 8))
    refused("aligned", take, _rows(A + 2, 5, 8), _index(B, 3), 1.0, _rows(C, 3, 8))
    refused("aligned", take, _rows(0, 5, 8), _index(B, 3), 1.0, _rows(C, 3, 8))
    refused("impossible", take, _rows(A, -1, 8), _index(B, 3), 1.0, _rows(C, 3, 8))
    refused("overlap", take, _rows(A, 5, 8), _index(B, 3), 1.0, _rows(C, 3, 8, 7))
    refused("indices", take, _rows(A, 5, 8), _index(B, 3, 2), 1.0, _rows(C, 3, 8))
    refused("indices", take, _rows(A, 5, 8), _index(B + 4, 3, 8), 1.0, _rows(C, 3, 8))
    refused("2\\^31", take, _rows(A, 5, 8), _index(B, 2**31), 1.0, _rows(C, 2**31, 8))
    refused("rows for", take, _rows(A, 5, 8), _index(B, 3), 1.0, _rows(C, 4, 8))
    refused("elements", take, _rows(A, 5, 9), _index(B, 3), 1.0, _rows(C, 3, 8))
    refused("16 bits", take, _rows(A, 5, 8, kind=1), _index(B, 3), 1.0, _rows(C, 3, 8))
    refused("null\\) queue", take, _rows(A, 5, 8), _index(B, 3), 1.0, _rows(C, 3, 8))
    assert take(None, _rows(A, 5, 8), _index(0, 0), 1.0, _rows(0, 0, 8)) == 0  # nothing to do
    refused("rows for", grad, _rows(A, 4, 8), _index(B, 3), 1.0, _rows(C, 5, 8), 0, None, 0)
    refused("range|rows", grad, _rows(A, 3, 1), _index(B, 3), 1.0, _rows(C, 2**31 - 1, 1), 0, None, 0)
    refused("groups", group, _index(B, 3), -1, C, C, C, None, 0)
    refused("groups", group, _index(B, 3), 2**31 - 1, C, C, C, None, 0)
    refused("null result", group, _index(B, 3), 4, None, C, C, None, 0)
    sdisp = lib._mlir_ciface_nmb_sort_dispatch_rows_device
    refused("for 5 tokens", sdisp, _rows(A, 5, 8), _index(B, 9), 4, C, C, C, None, 0, _rows(C, 10, 8))
    refused("for 5 tokens", sdisp, _rows(A, 5, 8), _index(B, 10), 4, C, C, C, None, 0, _rows(C, 9, 8))
    refused("for 0 tokens", sdisp, _rows(A, 0, 8), _index(B, 1), 4, C, C, C, None, 0, _rows(C, 9, 8))
    refused("groups", sdisp, _rows(A, 5, 8), _index(B, 10), -1, C, C, C, None, 0, _rows(C, 10, 8))
    refused("null result", sdisp, _rows(A, 5, 8), _index(B, 10), 4, C, None, C, None, 0, _rows(C, 10, 8))
    refused("different types", disp, _rows(A, 5, 8), 2, B, B, _rows(C, 10, 8, kind=2))
    refused("below 2", disp, _rows(A, 2**30, 8), 2, B, B, _rows(C, 2**31 - 1, 8))
    refused("null positions", disp, _rows(A, 5, 8), 2, None, B, _rows(C, 10, 8))
    refused("null positions", comb, _rows(A, 10, 8), 2, B, None, None, 0, _rows(C, 5, 8))
    refused("weights", comb, _rows(A, 10, 8), 2, B, B, A + 2, 0, _rows(C, 5, 8))
    refused("weights", comb, _rows(A, 10, 8), 2, B, B, A, 7, _rows(C, 5, 8))
    refused("different types", cgrad, _rows(A, 5, 8), _rows(B, 10, 8, kind=3), 2, B, B, None, 0, _rows(C, 10, 8), C)


def test_workspace_sizes_grow(runtime_lib):
    assert nm.group_rows_workspace(0, 5) == 0
    small, large = nm.take_rows_grad_workspace(100, 1000, 64), nm.take_rows_grad_workspace(10**6, 1000, 64)
    assert 0 < small < large < 64 * 10**6
    assert nm.group_rows_workspace(2**31 - 1, 2**31 - 2) > 2**34
