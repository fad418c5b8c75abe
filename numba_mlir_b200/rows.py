"""Rows picked, grouped and added by index: embedding lookups and their
gradients, tokens sorted by expert and back.

What a program writes as `a[m]`, `a[m] += b` and `argsort` on rows
(numba_mlir/numba_mlir/mlir/tests/test_numpy.py: test_getitem_offset), as
routines with the scale or the weights and the conversion to the result's type
inside.  They take device arrays or anything else that exports
`__cuda_array_interface__`, run asynchronously on a queue, and can be called
inside `njit` functions, whose recorded plans replay them (there on the queue of
the function's call, without `queue` and `workspace` of their own; a number of
rows or groups that is an argument of the function has it traced anew).  A
kernel whose wait for its own copies runs out (the bound is far above the time
of a copy) leaves what it had not written yet as it was; `Queue.check_status` of
the queue that the call ran on raises then (`torch_queue` names the queue of
torch's tensors).

    out            = take_rows(table, ids, scale)
    dtable         = take_rows_grad(dout, ids, rows, scale)
    xs, plan       = dispatch_rows(x, expert_ids, experts)
    y              = combine_rows(ys, plan, weights)
    dys, dweights  = combine_rows_grad(dy, ys, plan, weights)
    dx             = dispatch_rows_grad(dxs, plan)

Types: rows are float32, float64, float16 or bfloat16 (`bfloat16`, the two-byte
type "V2" under which torch and ml_dtypes export it); indices are int32 or
int64.  Sums run in float32 (float64 for float64 rows) in an order that does not
depend on the run, and are rounded once.  The last axis of a row operand has
unit stride; the axes before it may be strided as long as they can be walked
with one stride.  An index outside its range (negative ones included: padding,
dropped choices) picks nothing: its row is zero, it adds nothing, its gradient
is zero.
"""

import ctypes
import sys
from typing import Any, NamedTuple

import numpy as np

from . import lazy
from . import runtime as _rt
from .device_array import DeviceArray, as_device_array, empty

bfloat16 = np.dtype("V2")

_FLOATS = {"<f4": 0, "<f8": 1, "<f2": 2, "<V2": 3, "|V2": 3}
_INTS = {"<i4": 4, "<i8": 8}
_FLOAT_OF = {0: np.dtype(np.float32), 1: np.dtype(np.float64), 2: np.dtype(np.float16), 3: bfloat16}
_SIZE = (4, 8, 2, 2)


class RowGroups(NamedTuple):
    """Entries sorted by group, as `group_rows` leaves them: int32 arrays
    `order` (entry at each sorted position), `place` (position of each entry, in
    the shape of the ids: the inverse of `order`) and `offsets` (groups + 1
    values: where each group begins; the last one is the number of entries
    inside the range, which is where the entries outside it begin)."""

    order: Any
    place: Any
    offsets: Any


class _Rows(ctypes.Structure):
    """GPUXRows of include/numba_mlir_gpu_runtime_cuda.h."""

    _fields_ = [("data", ctypes.c_void_p), ("rows", ctypes.c_int64), ("cols", ctypes.c_int64),
                ("stride", ctypes.c_int64), ("type", ctypes.c_int32), ("reserved", ctypes.c_int32)]


class _Index(ctypes.Structure):
    """GPUXIndex of include/numba_mlir_gpu_runtime_cuda.h."""

    _fields_ = [("data", ctypes.c_void_p), ("count", ctypes.c_int64), ("bytes", ctypes.c_int32),
                ("reserved", ctypes.c_int32)]


# --------------------------------------------------------------- operands ---
class _Operand:
    """One array argument: address, shape, strides in elements, element type
    (`kind`: a float code, or None; `index`: bytes of an integer, or 0)."""

    __slots__ = ("obj", "ptr", "shape", "strides", "kind", "index", "item", "queue", "device")


_torch_types = {}


def _torch_type(dtype):
    """(float code, index bytes, item size) of a torch dtype; the table is
    filled when a torch tensor is first seen."""
    if not _torch_types:
        t = sys.modules["torch"]
        _torch_types.update({t.float32: (0, 0, 4), t.float64: (1, 0, 8), t.float16: (2, 0, 2),
                             t.bfloat16: (3, 0, 2), t.int32: (None, 4, 4), t.int64: (None, 8, 8)})
        _fast_torch()
    return _torch_types.get(dtype)


def _torch_raw_stream(device):
    """Handle of torch's current stream of a device."""
    return sys.modules["torch"].cuda.current_stream(device).cuda_stream


_native = None
_native_types = {np.dtype(t): (-1 if k > 3 else k, 0 if k <= 3 else k, np.dtype(t).itemsize)
                 for t, k in list(_FLOATS.items()) + list(_INTS.items())}


def _fast():
    """The native call path (csrc/fastcall/rows_call.h), bound on first use."""
    global _native
    fast, lib = _rt.fastcall(), _rt.load()
    entries = ("take_rows", "take_rows_grad", "group_rows", "dispatch_rows", "combine_rows", "combine_rows_grad",
               "sort_dispatch_rows")
    fast.rows_init(tuple(ctypes.cast(getattr(lib, f"_mlir_ciface_nmb_{e}_device"), ctypes.c_void_p).value
                         for e in entries), _native_types, DeviceArray)
    _native = fast
    return fast


def _fast_torch():
    """Lets the native path take torch's tensors, from the first one on."""
    torch = sys.modules["torch"]
    _native_types.update({t: (-1 if k is None else k, i, n) for t, (k, i, n) in _torch_types.items()})
    (_native or _fast()).rows_torch(torch.Tensor, getattr(torch._C, "_cuda_getCurrentRawStream", _torch_raw_stream))


def _operand(obj, name):
    """The array argument `obj`.  Tensors of torch are read through their own
    attributes, which costs a fifth of building the interface's dict and names
    the device; the rules are the interface's (no tensors that require a
    gradient, CUDA only)."""
    op = _Operand()
    op.obj = obj
    if type(obj) is not DeviceArray and "torch" in sys.modules and isinstance(obj, sys.modules["torch"].Tensor):
        known = _torch_type(obj.dtype)
        if known is not None and obj.is_cuda:
            if obj.requires_grad:
                raise RuntimeError(f"{name}: a tensor that requires a gradient; use tensor.detach()")
            if known[0] is not None and obj.is_neg():  # its memory holds the values with the other sign
                raise RuntimeError(f"{name}: a tensor with the negative bit set; use tensor.resolve_neg()")
            op.kind, op.index, op.item = known
            op.ptr, op.shape, op.strides = obj.data_ptr(), tuple(obj.shape), obj.stride()
            op.queue, op.device = None, obj.device.index
            return op
    if isinstance(obj, DeviceArray):
        arr = obj
    elif hasattr(obj, "__cuda_array_interface__"):
        arr = op.obj = as_device_array(obj)
    else:
        raise TypeError(f"{name} must be a device array (or export __cuda_array_interface__), not {type(obj).__name__}")
    dt = arr.dtype
    op.item = dt.itemsize
    op.kind = _FLOATS.get(dt.str) if dt.names is None else None
    op.index = _INTS.get(dt.str, 0)
    if any(s % op.item for s in arr.strides):
        raise ValueError(f"{name}: strides that are not multiples of the element size")
    op.ptr, op.shape, op.strides = arr.ptr, arr.shape, tuple(s // op.item for s in arr.strides)
    op.queue, op.device = arr.queue, arr.queue.device
    return op


def _size(shape):
    n = 1
    for s in shape:
        n *= s
    return n


def _contiguous(op):
    """Whether the elements lie one behind the other in C order."""
    step = 1
    for n, st in zip(reversed(op.shape), reversed(op.strides)):
        if n == 0:
            return True
        if n != 1 and st != step:
            return False
        step *= n
    return True


def _row_view(op, name):
    """(rows, columns, elements between rows) of an array of rows."""
    shape, strides = op.shape, op.strides
    if op.kind is None:
        raise TypeError(f"{name} must hold float32, float64, float16 or bfloat16")
    nd = len(shape)
    if nd == 0:
        raise ValueError(f"{name} must have at least one axis")
    cols = shape[-1]
    if cols > 1 and strides[-1] != 1:
        raise ValueError(f"{name}: the last axis must have unit stride")
    if nd == 2:
        return shape[0], cols, strides[0] if shape[0] > 1 else cols
    rows, step = _size(shape[:-1]), cols
    if rows > 1:
        # the leading axes, from the innermost that has more than one index
        step, span = None, None
        for n, st in zip(reversed(shape[:-1]), reversed(strides[:-1])):
            if n == 1:
                continue
            if step is None:
                step, span = st, st * n
            elif st != span:
                raise ValueError(f"{name}: the axes before the last cannot be walked with one stride")
            else:
                span = st * n
    return rows, cols, step


def _rows_arg(op, name):
    rows, cols, stride = _row_view(op, name)
    return _Rows(op.ptr, rows, cols, stride, op.kind, 0)


def _index_arg(op, name):
    if not op.index:
        raise TypeError(f"{name} must hold int32 or int64")
    if not _contiguous(op):
        raise ValueError(f"{name} must be C-contiguous")
    return _Index(op.ptr, _size(op.shape), op.index, 0)


def _int32_arg(op, name, count=None):
    """Address of a contiguous int32 array (of `count` elements)."""
    if op.index != 4:
        raise TypeError(f"{name} must hold int32")
    if not _contiguous(op) or (count is not None and _size(op.shape) != count):
        raise ValueError(f"{name} must be C-contiguous" + (f" and hold {count} values" if count is not None else ""))
    return op.ptr


def _weights_arg(op, name, shape):
    if op.kind is None:
        raise TypeError(f"{name} must hold floating-point values")
    if op.shape != tuple(shape) or not _contiguous(op):
        raise ValueError(f"{name} must be C-contiguous and have the shape of the plan's place, {tuple(shape)}")
    return op.ptr


def _range(op):
    lo = hi = op.ptr
    for n, st in zip(op.shape, op.strides):
        if n == 0:
            return 0, 0
        if st >= 0:
            hi += (n - 1) * st * op.item
        else:
            lo += (n - 1) * st * op.item
    return lo, hi + op.item


def _apart(a, b):
    """Two sets of rows in one buffer that are different columns of it."""
    if len(a.shape) != 2 or len(b.shape) != 2:
        return False
    step = a.strides[0] * a.item
    if step <= 0 or step != b.strides[0] * b.item:
        return False
    gap = (b.ptr - a.ptr) % step
    return a.shape[1] * a.item <= gap and gap + b.shape[1] * b.item <= step


def _no_overlap(results, operands):
    """Results are written while operands are read: they must not share memory."""
    every = results + operands
    ranges = [_range(o) for o in every]
    for i in range(len(results)):
        lo, hi = ranges[i]
        for j in range(i + 1, len(every)):
            if lo < ranges[j][1] and ranges[j][0] < hi and not _apart(every[i], every[j]):
                raise ValueError("a result shares memory with another argument")


# ------------------------------------------------------------------ queue ---
_stream_queues = {}


def _torch_stream(device):
    """Queue over torch's current stream of the device, made once per stream."""
    stream = _torch_raw_stream(device)
    q = _stream_queues.get((device, stream))
    if q is None:
        with sys.modules["torch"].cuda.device(device):
            q = _stream_queues[(device, stream)] = _rt.Queue.from_stream(stream)
    return q


def torch_queue(device=None):
    """The queue that the row operators run on when all of their arrays are
    torch's: one over torch's current stream of the device (torch's current one
    by default).  Its `check_status` synchronises and raises if a kernel of theirs
    gave up on a wait."""
    torch = sys.modules.get("torch")
    if torch is None:
        raise RuntimeError("torch is not in use")
    if device is None:
        index = torch.cuda.current_device()
    elif isinstance(device, int):
        index = device
    else:
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError(f"{device} is not a CUDA device")
        index = torch.cuda.current_device() if device.index is None else device.index
    return _torch_stream(index)


def _raw_stream(q):
    raw = q.__dict__.get("_raw_stream")
    if raw is None:
        raw = q.__dict__["_raw_stream"] = int(q.stream)
    return raw


class _On:
    """The queue a call runs on, ordered with the streams its arrays belong to.

    The queue is the caller's choice, or that of the first device array, or
    torch's current stream when all arrays are torch's.  Where an array belongs
    to another stream of the device (a device array to its own queue, a torch
    tensor to torch's current stream), the call's work is ordered after what
    that stream has been given so far and that stream after the call's work, so
    memory may be freed or reused there at once."""

    __slots__ = ("queue", "others")

    def __init__(self, queue, operands):
        if queue is None:
            for op in operands:
                if op.queue is not None:
                    queue = op.queue
                    break
            else:
                queue = _torch_stream(operands[0].device)
        self.queue = queue
        mine, others, torch_seen = _raw_stream(queue), None, False
        for op in operands:
            if op.device != queue.device:
                raise ValueError(f"Device arrays have different devices: {sorted({op.device, queue.device})}")
            q = op.queue
            if q is queue:
                continue
            if q is None:
                if torch_seen:
                    continue
                torch_seen = True
                if _torch_raw_stream(op.device) == mine:
                    continue
                q = _torch_stream(op.device)
            if _raw_stream(q) != mine:
                others = others or []
                if q not in others:
                    others.append(q)
        self.others = others
        if others:
            for q in others:
                queue.wait_stream(_named(_raw_stream(q)))

    def done(self, failed):
        if self.others:
            for q in self.others:
                q.wait_stream(_named(_raw_stream(self.queue)))
        if failed:
            _rt.check()
            raise _rt.GpuRuntimeError("a row operation failed")


def _named(raw):
    """The stream handle as the array interface names it (1: legacy default)."""
    return raw or 1


def _result(queue, shape, kind):
    return empty(shape, _FLOAT_OF[kind], queue=queue)


def _workspace(workspace, name):
    """(address, bytes, operand) of a caller's workspace: a contiguous device
    array of any type."""
    if workspace is None:
        return None, 0, None
    op = _Operand()
    op.obj, op.item, op.strides = workspace, 1, (1,)
    if type(workspace) is not DeviceArray and "torch" in sys.modules and isinstance(
            workspace, sys.modules["torch"].Tensor) and workspace.is_cuda:
        if not workspace.is_contiguous():
            raise ValueError(f"{name} must be C-contiguous")
        op.ptr, op.shape = workspace.data_ptr(), (workspace.numel() * workspace.element_size(),)
        op.queue, op.device = None, workspace.get_device()
    else:
        arr = as_device_array(workspace)
        if not arr.is_c_contiguous:
            raise ValueError(f"{name} must be C-contiguous")
        op.ptr, op.shape, op.queue, op.device = arr.ptr, (arr.nbytes,), arr.queue, arr.queue.device
    return op.ptr, op.shape[0], op


_ref = ctypes.byref


def _default(first):
    """The queue of a call whose arrays are like `first` (None: not known)."""
    if type(first) is DeviceArray:
        return first._buf.queue
    if "torch" in sys.modules and isinstance(first, sys.modules["torch"].Tensor) and first.is_cuda:
        return _torch_stream(first.get_device())
    return None


def _failed():
    """The native path reached the library and that refused or failed."""
    _rt.check()
    raise _rt.GpuRuntimeError("a row operation failed")


# ---------------------------------------------------------------- routines ---
def take_rows(table, ids, scale=1.0, out=None, queue=None):
    """`scale * table[ids]`: out[i..., :] = scale * table[ids[i...], :] for a
    table (R, D) and ids of any shape; zero rows for ids outside [0, R).  `out`
    has the table's type, or one of the two is float32 and the other 16 bits
    wide; the product is rounded once, to that type."""
    if lazy.current_trace() is not None:
        _traced(queue)
        return _trace_take(table, ids, scale, out)
    if out is not None:
        done = (_native or _fast()).rows_take(queue or _default(table), table, ids, scale, out)
        if done:
            return out if done == 1 else _failed()
    t, i = _operand(table, "table"), _operand(ids, "ids")
    o = _operand(out, "out") if out is not None else None
    on = _On(queue, (t, i) if o is None else (t, i, o))
    index = _index_arg(i, "ids")
    if len(t.shape) != 2:
        raise ValueError("table must have two axes")
    shape = i.shape + (t.shape[1],)
    src = _rows_arg(t, "table")
    if o is None:
        out = _result(on.queue, shape, t.kind)
        o = _operand(out, "out")
    elif o.shape != shape:
        raise ValueError(f"out has shape {o.shape}, the rows {shape}")
    dst = _rows_arg(o, "out")
    _check_pair(t, o, "table")
    _no_overlap([o], [t, i])
    on.done(_rt.load()._mlir_ciface_nmb_take_rows_device(on.queue.handle, _ref(src), _ref(index), float(scale),
                                                         _ref(dst)))
    return out


def take_rows_grad(dout, ids, rows=None, scale=1.0, out=None, accumulate=False, workspace=None, queue=None):
    """The gradient of `take_rows` with respect to the table: out[v, :] = scale *
    sum of dout[i..., :] over ids[i...] == v, in the order of i.  `rows` is the
    number of rows of the table (that of `out` when it is given), `out` may be
    float32 for a 16-bit dout and the other way round.  `accumulate=True` adds
    to `out` and touches only the rows that an id names.  `workspace`: a device
    array of at least `take_rows_grad_workspace(...)` bytes; without one the call
    takes memory from the stream-ordered pool."""
    if lazy.current_trace() is not None:
        _traced(queue, workspace)
        return _trace_take_grad(dout, ids, rows, scale, out, accumulate)
    if out is not None and rows is None and workspace is None:
        done = (_native or _fast()).rows_take_grad(queue or _default(dout), dout, ids, scale, out, bool(accumulate))
        if done:
            return out if done == 1 else _failed()
    d, i = _operand(dout, "dout"), _operand(ids, "ids")
    o = _operand(out, "out") if out is not None else None
    ws, ws_bytes, w = _workspace(workspace, "workspace")
    on = _On(queue, [x for x in (d, i, o, w) if x is not None])
    index = _index_arg(i, "ids")
    if d.shape[:-1] != i.shape:
        raise ValueError(f"dout has shape {d.shape} for ids of shape {i.shape}")
    src = _rows_arg(d, "dout")
    if o is None:
        if accumulate:
            raise ValueError("accumulate needs out")
        if rows is None:
            raise ValueError("the number of rows of the table is needed: rows or out")
        out = _result(on.queue, (int(rows), d.shape[-1]), d.kind)
        o = _operand(out, "out")
    elif len(o.shape) != 2 or o.shape[1] != d.shape[-1] or (rows is not None and o.shape[0] != rows):
        raise ValueError(f"out has shape {o.shape}, the gradient ({o.shape[0] if rows is None else rows}, {d.shape[-1]})")
    dst = _rows_arg(o, "out")
    _check_pair(d, o, "dout")
    _no_overlap([o] if w is None else [o, w], [d, i])
    on.done(_rt.load()._mlir_ciface_nmb_take_rows_grad_device(
        on.queue.handle, _ref(src), _ref(index), float(scale), _ref(dst), int(bool(accumulate)), ws, ws_bytes))
    return out


def take_rows_grad_workspace(count, rows, cols, dtype=np.float32):
    """Bytes of workspace of `take_rows_grad` for `count` ids, a table of `rows`
    rows of `cols` elements and a dout of `dtype`."""
    kind = _FLOATS.get(np.dtype(dtype).str)
    if kind is None:
        raise TypeError(f"rows of {dtype} are not supported")
    _sizes(count=(count, 2**31), rows=(rows, 2**31 - 1), cols=(cols, 2**31))
    return int(_rt.load()._mlir_ciface_nmb_take_rows_grad_workspace(int(count), int(rows), int(cols), kind))


def _sizes(**sizes):
    for name, (value, end) in sizes.items():
        if not 0 <= value < end:
            raise ValueError(f"{name} = {value}: must be in 0 .. {end - 1}")


def group_rows_workspace(count, groups):
    """Bytes of workspace of `group_rows` for `count` ids."""
    _sizes(count=(count, 2**31), groups=(groups, 2**31 - 1))
    return int(_rt.load()._mlir_ciface_nmb_group_rows_workspace(int(count), int(groups)))


def group_rows(ids, groups, plan=None, workspace=None, queue=None):
    """Sorts the entries of `ids` (any shape) by group, `groups` groups, keeping
    their order within a group; entries outside [0, groups) come last.  Returns
    RowGroups, written into the arrays of `plan` when one is given."""
    if lazy.current_trace() is not None:
        _traced(queue, workspace)
        return _trace_group(ids, groups, plan)
    if plan is not None and workspace is None:
        done = (_native or _fast()).rows_group(queue or _default(ids), ids, groups, plan)
        if done:
            return RowGroups(*plan) if done == 1 else _failed()
    i = _operand(ids, "ids")
    results = [_operand(x, n) for x, n in zip(plan, RowGroups._fields)] if plan is not None else []
    ws, ws_bytes, w = _workspace(workspace, "workspace")
    on = _On(queue, [i] + results + ([w] if w is not None else []))
    index, groups = _index_arg(i, "ids"), int(groups)
    if groups < 0:
        raise ValueError("a negative number of groups")
    if plan is None:
        plan = _new_plan(on.queue, i.shape, groups)
        results = [_operand(x, n) for x, n in zip(plan, RowGroups._fields)]
    order, place, offsets = _whole_plan(results, index.count, groups)
    _no_overlap(results if w is None else results + [w], [i])
    on.done(_rt.load()._mlir_ciface_nmb_group_rows_device(on.queue.handle, _ref(index), groups, order, place, offsets,
                                                          ws, ws_bytes))
    return RowGroups(*plan)


def _new_plan(queue, shape, groups):
    new = lambda s: empty(s, np.int32, queue=queue)  # noqa: E731
    return RowGroups(new((_size(shape),)), new(shape), new((groups + 1,)))


def _whole_plan(results, count, groups):
    """Addresses of order, place and offsets of a plan that is to be written."""
    return (_int32_arg(results[0], "order", count), _int32_arg(results[1], "place", count),
            _int32_arg(results[2], "offsets", groups + 1))


def dispatch_rows(x, ids, groups=None, out=None, plan=None, queue=None):
    """Tokens sorted by expert: every token t of x (T, D) is copied to the places
    of its choices ids[t] ((T, k) or (T,) experts below `groups`), experts
    ascending and tokens in order within one.  Returns (xs, plan) with xs
    (T * k, D) and the RowGroups of the ids; rows of xs behind the last kept
    choice (plan.offsets[-1]) are zero.  `out` may have more rows, which are left
    as they are; `plan` holds arrays to write the RowGroups into.  A RowGroups in
    the place of `ids` is used as it is."""
    if lazy.current_trace() is not None:
        _traced(queue)
        return _trace_dispatch(x, ids, groups, out, plan)
    sorted_already = isinstance(ids, RowGroups)
    if out is not None and (plan is None if sorted_already else plan is not None):
        known, entries = (ids, None) if sorted_already else (plan, ids)
        done = (groups is None) == sorted_already and (_native or _fast()).rows_dispatch(
            queue or _default(x), x, entries, groups, known, out)
        if done:
            return (out, known if type(known) is RowGroups else RowGroups(*known)) if done == 1 else _failed()
    r = _operand(x, "x")
    if sorted_already:
        if groups is not None or plan is not None:
            raise ValueError("groups and plan are for ids that are not sorted yet")
        plan = ids
    elif groups is None:
        raise ValueError("the number of groups is needed")
    results = [_operand(a, n) for a, n in zip(plan, RowGroups._fields)] if plan is not None else []
    o = _operand(out, "out") if out is not None else None
    i = None if sorted_already else _operand(ids, "ids")
    on = _On(queue, [a for a in (r, i, o) if a is not None] + results)
    entries = results[1].shape if sorted_already else i.shape
    k = _choices(r, entries, "x")
    src = _rows_arg(r, "x")
    shape = (r.shape[0] * k, r.shape[1])
    if o is None:
        out = _result(on.queue, shape, r.kind)
        o = _operand(out, "out")
    elif len(o.shape) != 2 or o.shape[1] != shape[1] or o.shape[0] < shape[0]:
        raise ValueError(f"out has shape {o.shape}, the rows {shape}")
    if o.kind != r.kind:
        raise TypeError("out must have the type of x")
    dst = _rows_arg(o, "out")
    if not sorted_already:
        index, groups = _index_arg(i, "ids"), int(groups)
        if groups < 0:
            raise ValueError("a negative number of groups")
        if plan is None:
            plan = _new_plan(on.queue, i.shape, groups)
            results = [_operand(a, n) for a, n in zip(plan, RowGroups._fields)]
        order, place, offsets = _whole_plan(results, index.count, groups)
        _no_overlap([o] + results, [r, i])
        on.done(_rt.load()._mlir_ciface_nmb_sort_dispatch_rows_device(
            on.queue.handle, _ref(src), _ref(index), groups, order, place, offsets, None, 0, _ref(dst)))
        return out, RowGroups(*plan)
    _no_overlap([o], [r] + results)
    place, kept = _plan_args(results)
    on.done(_rt.load()._mlir_ciface_nmb_dispatch_rows_device(on.queue.handle, _ref(src), k, place, kept, _ref(dst)))
    return out, plan


def _choices(rows, entries, name):
    """Choices per token of entries (T,) or (T, k) over rows (T, D)."""
    if len(rows.shape) != 2:
        raise ValueError(f"{name} must have two axes")
    if len(entries) not in (1, 2) or entries[0] != rows.shape[0]:
        raise ValueError(f"{rows.shape[0]} tokens with choices of shape {entries}")
    return entries[1] if len(entries) == 2 else 1


def _plan_args(results):
    """(address of place, address of the number of kept entries)."""
    place = _int32_arg(results[1], "place")
    offsets = _int32_arg(results[2], "offsets")
    n = _size(results[2].shape)
    if n < 1:
        raise ValueError("offsets must hold at least one value")
    return place, offsets + 4 * (n - 1)


def combine_rows(ys, plan, weights=None, out=None, queue=None):
    """The experts' rows back at their tokens: out[t, :] = sum over j of
    weights[t, j] * ys[plan.place[t, j], :], choices that were dropped left out.
    `weights` has the shape of plan.place (ones when it is None) and any
    floating-point type; `out` (T, D) has the type of ys."""
    if lazy.current_trace() is not None:
        _traced(queue)
        return _trace_combine(ys, plan, weights, out)
    return _combine(ys, plan, weights, out, queue, "ys")


def _combine(ys, plan, weights, out, queue, name):
    if out is not None:
        done = (_native or _fast()).rows_combine(queue or _default(ys), ys, plan, weights, out)
        if done:
            return out if done == 1 else _failed()
    y = _operand(ys, name)
    results = [_operand(plan[1], "place"), _operand(plan[2], "offsets")]
    w = _operand(weights, "weights") if weights is not None else None
    o = _operand(out, "out") if out is not None else None
    on = _On(queue, [a for a in (y, w, o) if a is not None] + results)
    entries = results[0].shape
    if len(y.shape) != 2 or len(entries) not in (1, 2):
        raise ValueError(f"{name} must have two axes, place one or two")
    k = entries[1] if len(entries) == 2 else 1
    shape = (entries[0], y.shape[1])
    src = _rows_arg(y, name)
    if o is None:
        out = _result(on.queue, shape, y.kind)
        o = _operand(out, "out")
    elif o.shape != shape:
        raise ValueError(f"out has shape {o.shape}, the tokens {shape}")
    if o.kind != y.kind:
        raise TypeError(f"out must have the type of {name}")
    dst = _rows_arg(o, "out")
    wp, wt = (_weights_arg(w, "weights", entries), w.kind) if w is not None else (None, 0)
    place, kept = _plan_args([None] + results)
    _no_overlap([o], [y] + results + ([w] if w is not None else []))
    on.done(_rt.load()._mlir_ciface_nmb_combine_rows_device(on.queue.handle, _ref(src), k, place, kept, wp, wt,
                                                            _ref(dst)))
    return out


def dispatch_rows_grad(dxs, plan, out=None, queue=None):
    """The gradient of `dispatch_rows` with respect to x: the sum of the rows at
    a token's places, out[t, :] = sum over j of dxs[plan.place[t, j], :]."""
    if lazy.current_trace() is not None:
        _traced(queue)
        return _trace_combine(dxs, plan, None, out)
    return _combine(dxs, plan, None, out, queue, "dxs")


def combine_rows_grad(dout, ys, plan, weights=None, out=None, dweights=None, queue=None):
    """The gradients of `combine_rows` for the incoming gradient dout (T, D):
    dys[plan.place[t, j], :] = weights[t, j] * dout[t, :] and dweights[t, j] =
    dout[t, :] . ys[plan.place[t, j], :]; both zero for dropped choices.
    Returns (dys, dweights), written into `out` and `dweights` when given;
    dweights has the type of the weights (float32 when they are None)."""
    if lazy.current_trace() is not None:
        _traced(queue)
        return _trace_combine_grad(dout, ys, plan, weights, out, dweights)
    if out is not None and dweights is not None:
        done = (_native or _fast()).rows_combine_grad(queue or _default(dout), dout, ys, plan, weights, out, dweights)
        if done:
            return (out, dweights) if done == 1 else _failed()
    d, y = _operand(dout, "dout"), _operand(ys, "ys")
    results = [_operand(plan[1], "place"), _operand(plan[2], "offsets")]
    w = _operand(weights, "weights") if weights is not None else None
    o = _operand(out, "out") if out is not None else None
    dw = _operand(dweights, "dweights") if dweights is not None else None
    on = _On(queue, [a for a in (d, y, w, o, dw) if a is not None] + results)
    entries = results[0].shape
    k = _choices(d, entries, "dout")
    if len(y.shape) != 2 or y.shape != (d.shape[0] * k, d.shape[1]):
        raise ValueError(f"ys has shape {y.shape} for {d.shape[0]} tokens with {k} choices of width {d.shape[1]}")
    if o is None:
        out = _result(on.queue, y.shape, y.kind)
        o = _operand(out, "out")
    elif o.shape != y.shape:
        raise ValueError(f"out has shape {o.shape}, ys {y.shape}")
    if not y.kind == d.kind == o.kind:
        raise TypeError("dout, ys and out must have one type")
    wt = w.kind if w is not None else 0
    if dw is None:
        dweights = _result(on.queue, entries, wt)
        dw = _operand(dweights, "dweights")
    elif dw.kind != wt:
        raise TypeError("dweights must have the type of the weights (float32 without weights)")
    wp = _weights_arg(w, "weights", entries) if w is not None else None
    dwp = _weights_arg(dw, "dweights", entries)
    a, b, c = _rows_arg(d, "dout"), _rows_arg(y, "ys"), _rows_arg(o, "out")
    place, kept = _plan_args([None] + results)
    _no_overlap([o, dw], [d, y] + results + ([w] if w is not None else []))
    on.done(_rt.load()._mlir_ciface_nmb_combine_rows_grad_device(
        on.queue.handle, _ref(a), _ref(b), k, place, kept, wp, wt, _ref(c), dwp))
    return out, dweights


def _check_pair(a, b, name):
    if a.kind != b.kind and (1 in (a.kind, b.kind) or 0 not in (a.kind, b.kind)):
        raise TypeError(f"out must have the type of {name}, or one of them float32 and the other 16 bits wide")


# ------------------------------------------------- inside a traced function ---
# A routine called while an `njit` function is traced runs at once on the arrays
# of the trace and is a step of the recorded plan, like a reduction or a product.
def _step(routine, arrays, consts, results):
    """Runs `routine(**arrays, **consts, **results)` inside the active trace.
    `results`: name -> (shape, dtype) of a new array or an existing one to write;
    returns the results' arrays, in order."""
    trace = lazy.current_trace()

    slots = {name: ("slot", trace.materialize(a)) for name, a in arrays.items() if a is not None}
    outs = {}
    for name, r in results.items():
        if isinstance(r, tuple):
            outs[name] = trace.add_tmp_slot(*r)
        else:
            if r.node.kind != "leaf":
                raise TypeError(f"{name} must be an array, not an expression")
            outs[name] = trace.materialize(r)
            trace.before_direct_write(outs[name])
        slots[name] = ("slot", outs[name])
    trace.flush()
    for name, c in consts.items():
        if isinstance(c, lazy.LazyArray):
            # a scalar argument of the call is read anew by every replay; one
            # computed from arguments keeps the call from being replayed
            c = ("arg", c.node.value) if c.node.kind == "arg" else ("const", c._escape())
        else:
            c = ("const", c)
        slots[name] = c
    step = ("rows", routine, tuple(slots.items()))
    trace.steps.append(step)
    if not trace.dry:
        with lazy._TraceScope(None):
            run_step(step, trace.arrays.__getitem__, trace.args)
    return [trace.leaf(s) for s in outs.values()]


def run_step(step, get, args):
    """Runs a recorded step: `get` gives the array of a slot, `args` are the call's."""
    _tag, routine, params = step
    kwargs = {name: get(v) if how == "slot" else args[v] if how == "arg" else v for name, (how, v) in params}
    routine(**kwargs)


def _traced(queue, workspace=None):
    """Inside a traced function the queue is that of the function's call, in every
    replay anew, and workspaces come from the pool."""
    if queue is not None or workspace is not None:
        raise ValueError("queue and workspace cannot be given inside a traced function: its steps run on the queue "
                         "of its call and take workspaces from the pool")


def _lift(a):
    """An array argument as an array of the active trace.  One that is not an
    argument of the traced function is captured: such a call is not replayed."""
    if a is None or isinstance(a, lazy.LazyArray):
        return a
    if not isinstance(a, DeviceArray):
        if not hasattr(a, "__cuda_array_interface__"):
            raise TypeError(f"an array is needed, not {type(a).__name__}")
        a = as_device_array(a)
    trace = lazy.current_trace()
    return lazy.LazyArray(trace, lazy._as_node(trace, a))


def _row_type(a):
    dt = np.dtype(a.dtype)
    if dt.names is not None or dt.str not in _FLOATS:
        raise TypeError("rows must hold float32, float64, float16 or bfloat16")
    return dt


def _trace_take(table, ids, scale, out):
    table, ids, out = _lift(table), _lift(ids), _lift(out)
    shape = tuple(ids.shape) + (table.shape[-1],)
    (res,) = _step(take_rows, {"table": table, "ids": ids}, {"scale": scale},
                   {"out": out if out is not None else (shape, _row_type(table))})
    return res


def _trace_take_grad(dout, ids, rows, scale, out, accumulate):
    dout, ids, out = _lift(dout), _lift(ids), _lift(out)
    if out is None and rows is None:
        raise ValueError("the number of rows of the table is needed: rows or out")
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs out")
        out = ((int(rows), dout.shape[-1]), _row_type(dout))
    elif rows is not None and tuple(out.shape)[0] != int(rows):
        raise ValueError(f"out has {out.shape[0]} rows, not {int(rows)}")
    (res,) = _step(take_rows_grad, {"dout": dout, "ids": ids}, {"scale": scale, "accumulate": bool(accumulate)},
                   {"out": out})
    return res


def _run_group(ids, order, place, offsets, groups):
    group_rows(ids, groups, plan=RowGroups(order, place, offsets))


def _trace_group(ids, groups, plan):
    ids, plan, groups = _lift(ids), None if plan is None else tuple(map(_lift, plan)), int(groups)
    if plan is None:
        i32 = np.dtype(np.int32)
        plan = ((_size(ids.shape),), i32), (tuple(ids.shape), i32), ((groups + 1,), i32)
    res = _step(_run_group, {"ids": ids}, {"groups": groups}, dict(zip(RowGroups._fields, plan)))
    return RowGroups(*res)


def _run_dispatch(x, place, offsets, out):
    dispatch_rows(x, RowGroups(place, place, offsets), out=out)


def _trace_dispatch(x, ids, groups, out, plan):
    x, out = _lift(x), _lift(out)
    if isinstance(ids, RowGroups):
        if groups is not None or plan is not None:
            raise ValueError("groups and plan are for ids that are not sorted yet")
        plan = RowGroups(*map(_lift, ids))
    else:
        if groups is None:
            raise ValueError("the number of groups is needed")
        plan = _trace_group(ids, groups, plan)
    shape = (_size(plan.place.shape), x.shape[-1])
    (res,) = _step(_run_dispatch, {"x": x, "place": plan.place, "offsets": plan.offsets}, {},
                   {"out": out if out is not None else (shape, _row_type(x))})
    return res, plan


def _run_combine(ys, place, offsets, out, weights=None):
    combine_rows(ys, RowGroups(place, place, offsets), weights, out=out)


def _trace_combine(ys, plan, weights, out):
    ys, weights, out, plan = _lift(ys), _lift(weights), _lift(out), (None, _lift(plan[1]), _lift(plan[2]))
    shape = (plan[1].shape[0], ys.shape[-1])
    (res,) = _step(_run_combine, {"ys": ys, "place": plan[1], "offsets": plan[2], "weights": weights}, {},
                   {"out": out if out is not None else (shape, _row_type(ys))})
    return res


def _run_combine_grad(dout, ys, place, offsets, out, dweights, weights=None):
    combine_rows_grad(dout, ys, RowGroups(place, place, offsets), weights, out=out, dweights=dweights)


def _trace_combine_grad(dout, ys, plan, weights, out, dweights):
    dout, ys, weights, out, dweights = map(_lift, (dout, ys, weights, out, dweights))
    plan = (None, _lift(plan[1]), _lift(plan[2]))
    wt = _row_type(weights) if weights is not None else np.dtype(np.float32)
    return tuple(_step(
        _run_combine_grad,
        {"dout": dout, "ys": ys, "place": plan[1], "offsets": plan[2], "weights": weights}, {},
        {"out": out if out is not None else (tuple(ys.shape), _row_type(ys)),
         "dweights": dweights if dweights is not None else (tuple(plan[1].shape), wt)}))
