"""The row operators' kernels that fetch rows by bulk copies, on every type, both
conversions, both alignments, padding, joined sums and results inside larger
arrays.  A call is known to take those kernels when it reports waits that were
told to run out at once.  Tolerances as in test_rows_gpu."""

import numpy as np
import pytest

from test_rows_gpu import (TYPES, assert_near, bits_of, dev, dtype_of, grad_bound, host_values, plan_of, route,
                           rows_on_device, unit, values_of)
from test_rows_waits_gpu import no_patience

pytestmark = pytest.mark.gpu

PAIRS = [(t, t) for t in TYPES] + [("float32", "float16"), ("float32", "bfloat16"), ("float16", "float32"), ("bfloat16", "float32")]


def by_bulk_copies(queue, lib, call):
    """Whether the call's kernel waits for bulk copies (its results are not written)."""
    from numba_mlir_b200.runtime import GpuRuntimeError

    queue.check_status()
    with no_patience(lib):
        call()
        try:
            queue.check_status()
        except GpuRuntimeError:
            return True
    return False


def inside(shape, name, queue, rows=3, left=0, right=0, fill=-7.5):
    """(the array around, a part of it): `rows` rows more on either end, `left`
    and `right` columns more."""
    whole = dev(bits_of(np.full((shape[0] + 2 * rows, shape[1] + left + right), fill), name), queue)
    return whole, whole[rows:rows + shape[0], left:left + shape[1]]


def around(whole, shape, name, rows=3, left=0, fill=-7.5):
    """The part's values, after checking that everything around it still holds `fill`."""
    got = values_of(whole.copy_to_host(), name)
    part = got[rows:rows + shape[0], left:left + shape[1]].copy()
    got[rows:rows + shape[0], left:left + shape[1]] = fill
    assert (got == fill).all()
    return part


# ------------------------------------------------------------------- take ---
# (ids, width, columns beside the table, beside the result): widths off the words by
# odd numbers, by 8 and by 4 bytes, in one slab and in several, tables whose first and
# last word belong to them in part; aligned ones with several rows a block and a rest
TAKE = [(1100, 1027, 0, 0), (700, 5001, 1, 0), (1101, 1004, 0, 3), (1099, 1030, 3, 0), (540, 2048, 1, 0), (530, 2049, 0, 7),
        (8203, 520, 0, 0), (2101, 4104, 8, 0), (4105, 1032, 0, 16)]


@pytest.mark.parametrize("name,to", PAIRS)
@pytest.mark.parametrize("n,dim,pad,out_pad", TAKE)
def test_take_rows(queue, runtime_lib, name, to, n, dim, pad, out_pad):
    import numba_mlir_b200 as nm

    rng = np.random.default_rng(n + dim)
    rows = 61
    table, t = rows_on_device(rng.standard_normal((rows, dim)), name, pad)
    ids = rng.integers(-2, rows + 2, n)
    ids[:4], ids[-3:] = (0, rows - 1, -1, rows), (rows - 1, 0, rows - 1)
    ids = ids.astype(np.int64 if n % 2 else np.int32)
    whole, out = inside((n, dim), to, queue, right=out_pad)
    call = lambda: nm.take_rows(table, dev(ids), 1.7, out=out)  # noqa: E731
    assert by_bulk_copies(queue, runtime_lib, call)
    call()
    kept = (ids >= 0) & (ids < rows)
    want = np.where(kept[:, None], t[np.where(kept, ids, 0)], 0.0) * 1.7
    assert_near(around(whole, (n, dim), to), want, 2 * unit(name) * np.abs(want), to)


# -------------------------------------------------------------- gradient ---
def frequent(rng, n, rows):
    """Ids of which two come up often (their runs are joined from many chunks), a
    tenth outside."""
    ids = np.where(rng.random(n) < 0.7, rng.integers(0, 2, n) * (rows - 1), rng.integers(0, rows, n))
    return np.where(rng.random(n) < 0.1, rng.choice([-1, rows], n), ids)


def sum_bound(d, ids, rows, scale, name):
    want, bound = grad_bound(d, ids, rows, scale, unit(name))
    return want, bound * (2 if name == "float64" else 1)  # the float64 reference rounds as much itself


@pytest.mark.parametrize("name,to", PAIRS)
@pytest.mark.parametrize("n,dim,pad", [(5000, 1024, 0), (3000, 1027, 0), (5001, 1032, 3), (900, 4104, 0), (1500, 2050, 0),
                                       (4500, 512, 0), (300, 5001, 2)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_take_rows_grad(queue, runtime_lib, name, to, n, dim, pad, accumulate):
    import numba_mlir_b200 as nm

    rng = np.random.default_rng(n + dim)
    rows = 150
    ids = frequent(rng, n, rows // 2).astype(np.int32 if n % 2 else np.int64)  # the upper half has none
    dout, d = rows_on_device(rng.standard_normal((n, dim)), name, pad)
    host = rng.standard_normal((rows, dim))
    host[rows // 2 + 1:] = np.nan  # not even read when added to; overwritten when not
    out, old = rows_on_device(host, to)
    call = lambda o: nm.take_rows_grad(dout, dev(ids), out=o, scale=1.5, accumulate=accumulate)  # noqa: E731
    spare, _ = rows_on_device(np.zeros((rows, dim)), to)
    wide = dim * dtype_of(name).itemsize >= 1024
    assert by_bulk_copies(queue, runtime_lib, lambda: call(spare)) == wide
    again = dev(out.copy_to_host())
    call(out)
    got = host_values(out, to)
    want, bound = sum_bound(d, ids, rows, 1.5, name)
    if accumulate:
        assert np.isnan(got[rows // 2 + 1:]).all()
        got, want, bound, old = (a[:rows // 2 + 1] for a in (got, want, bound, old))
        bound = bound + unit(name) * (np.abs(want) + np.abs(old))
        want = want + old
    assert_near(got, want, bound, to)
    call(again)
    assert again.copy_to_host().tobytes() == out.copy_to_host().tobytes()


# (ids, rows, width, columns to the left and to the right of the result)
WITHIN = [(900, 700, 520, 8, 8), (900, 700, 520, 1, 0), (900, 30000, 520, 0, 4), (5000, 700, 520, 2, 2), (5000, 3000, 40, 0, 8),
          (900, 3000, 40, 4, 4), (900, 3000, 41, 3, 2), (5000, 700, 1023, 0, 1), (1, 900, 64, 0, 64), (0, 500, 40, 3, 5),
          (9000, 30000, 6, 1, 1), (700, 900, 1030, 2, 6)]


@pytest.mark.parametrize("name,to", PAIRS)
@pytest.mark.parametrize("n,rows,dim,left,right", WITHIN)
@pytest.mark.parametrize("accumulate", [False, True])
def test_a_gradient_inside_a_larger_array(queue, name, to, n, rows, dim, left, right, accumulate):
    import numba_mlir_b200 as nm

    rng = np.random.default_rng(n + rows + dim)
    ids = frequent(rng, n, rows)
    dout, d = rows_on_device(rng.standard_normal((n, dim)), name)
    whole, out = inside((rows, dim), to, queue, left=left, right=right)
    di = dev(ids.astype(np.int32)) if n else nm.empty((0,), np.int32, queue=queue)
    nm.take_rows_grad(dout, di, out=out, scale=1.5, accumulate=accumulate)
    got = around(whole, (rows, dim), to, left=left)
    want, bound = sum_bound(d, ids, rows, 1.5, name)
    if accumulate:
        bound = bound + unit(name) * (np.abs(want) + 7.5)
        want = want - 7.5
    assert_near(got, want, bound, to)


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("dim", [40, 1024, 1023])
def test_rows_in_reverse(queue, dim, accumulate):
    """Negative strides: a table, its ids' rows and a gradient read and written from
    the last row up."""
    import numba_mlir_b200 as nm

    rng = np.random.default_rng(dim)
    t = rng.standard_normal((50, dim)).astype(np.float32)
    ids = rng.integers(-1, 51, 5000).astype(np.int32)
    kept = (ids >= 0) & (ids < 50)
    want = np.where(kept[:, None], t[::-1][np.where(kept, ids, 0)], 0)
    assert np.array_equal(nm.take_rows(dev(t)[::-1], dev(ids)).copy_to_host(), want)
    d = rng.integers(-8, 9, (5000, dim)).astype(np.float32)  # whole numbers: exact sums
    whole, out = inside((50, dim), "float32", queue, left=2, right=1)
    nm.take_rows_grad(dev(d)[::-1], dev(ids), out=out[::-1], accumulate=accumulate)
    got = around(whole, (50, dim), "float32", left=2)
    grad = np.zeros((50, dim))
    np.add.at(grad, ids[kept], d[::-1][kept])
    assert np.array_equal(got[::-1], grad + (-7.5 if accumulate else 0.0))


# --------------------------------------------------------------- dispatch ---
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("tokens,k,groups,dim,left,right", [(40, 3, 9, 2047, 0, 1), (700, 8, 20, 1030, 2, 2), (900, 6, 2000, 64, 8, 8),
                                                            (33, 2, 5, 1024, 0, 16), (4096, 1, 8, 24, 1, 0), (4100, 1, 8, 24, 4, 4)])
def test_dispatch_inside_a_larger_array(queue, name, tokens, k, groups, dim, left, right):
    import numba_mlir_b200 as nm

    rng = np.random.default_rng(tokens + dim)
    x, v = rows_on_device(rng.standard_normal((tokens, dim)), name, 1)
    ids = route(tokens, k, groups, rng)
    order, place, offsets = plan_of(ids, groups)
    want = v[order // k]
    want[offsets[-1]:] = 0.0
    n = tokens * k
    whole, out = inside((n + 2, dim), name, queue, left=left, right=right)
    _, plan = nm.dispatch_rows(x, dev(ids), groups, out=out)
    got = around(whole, (n + 2, dim), name, left=left)
    assert np.array_equal(got[:n], want) and (got[n:] == -7.5).all()
    for a, b in zip(plan, (order, place, offsets)):
        assert np.array_equal(a.copy_to_host(), b)
    whole, out = inside((n + 2, dim), name, queue, left=left, right=right)
    nm.dispatch_rows(x, plan, out=out)
    got = around(whole, (n + 2, dim), name, left=left)
    assert np.array_equal(got[:n], want) and (got[n:] == -7.5).all()


# ------------------------------------------------------- traced, together ---
@pytest.mark.parametrize("name", ["float16", "bfloat16"])
def test_rows_of_16_bits_inside_njit(queue, name):
    """Traced functions move 16-bit rows, convert them on the way in and out, and
    replay; arithmetic on them is refused there."""
    import numba_mlir_b200 as nm

    @nm.njit(parallel=True)
    def step(table, tok, ids, w, x, grad):
        nm.take_rows(table, tok, np.float32(2), out=x)     # float32 rows of a 16-bit table
        x[:] = x * np.float32(0.5)
        rows = nm.take_rows(table, tok)
        xs, plan = nm.dispatch_rows(rows, ids, 5)
        y = nm.combine_rows(xs, plan, w)
        nm.take_rows_grad(y, tok, out=grad)
        return xs, y

    rng = np.random.default_rng(2)
    for _ in range(2):  # the second call replays the recorded plan
        table, t = rows_on_device(rng.integers(-8, 9, (30, 24)), name)  # whole numbers: exact
        tok = rng.integers(0, 30, 60).astype(np.int32)
        ids = route(60, 2, 5, rng, 0.0)
        x, grad = nm.empty((60, 24), np.float32, queue=queue), nm.empty((30, 24), np.float32, queue=queue)
        xs, y = step(table, dev(tok), dev(ids), dev(np.ones((60, 2), np.float32)), x, grad)
        order = plan_of(ids, 5)[0]
        assert np.array_equal(x.copy_to_host(), t[tok])
        assert np.array_equal(host_values(xs, name), t[tok][order // 2])
        assert np.array_equal(host_values(y, name), 2 * t[tok])
        want = np.zeros((30, 24))
        np.add.at(want, tok, 2 * t[tok])
        assert np.array_equal(grad.copy_to_host(), want)
    assert len(step._plans) == 1

    @nm.njit(parallel=True)
    def halves(table, tok):
        return nm.take_rows(table, tok) * np.float32(0.5)

    with pytest.raises(Exception):
        halves(table, dev(tok))


def test_two_threads_at_once(queue):
    """Calls of two threads, each on a queue of its own, with results to allocate
    and without."""
    import threading

    import numba_mlir_b200 as nm

    rng = np.random.default_rng(0)
    failed = []

    def work(seed):
        try:
            q = nm.runtime.Queue("cuda:0")
            rng = np.random.default_rng(seed)
            t = rng.integers(-8, 9, (300, 520)).astype(np.float32)
            table, grad = dev(t, q), nm.empty((300, 520), np.float32, queue=q)
            for i in range(30):
                ids = rng.integers(-1, 301, 5000 if i % 2 else 700).astype(np.int32)
                kept = (ids >= 0) & (ids < 300)
                picked = nm.take_rows(table, dev(ids, q))
                nm.take_rows_grad(picked, dev(ids, q), out=grad)
                want = t * np.bincount(ids[kept], minlength=300)[:, None].astype(np.float32)
                assert np.array_equal(grad.copy_to_host(), want)
        except BaseException as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(int(s),)) for s in rng.integers(0, 2**31, 3)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not failed, failed[0]


@pytest.mark.parametrize("tokens,k,one", [(4, 8, True), (512, 8, True), (1024, 4, True), (2048, 1, True), (2048, 2, False),
                                          (4096, 1, False), (1025, 4, False), (100, 64, False)])
def test_dispatch_in_one_launch(queue, tokens, k, one):
    """Sort and copy are one launch where every token's block can look at all
    entries: up to 4096 of them, and up to 2^22 tokens x entries."""
    import numba_mlir_b200 as nm

    rng = np.random.default_rng(tokens)
    x = rng.standard_normal((tokens, 16)).astype(np.float32)
    ids = route(tokens, k, 80, rng)
    out, plan = nm.dispatch_rows(dev(x), dev(ids), 80)
    before = nm.runtime.launch_count()
    nm.dispatch_rows(dev(x), dev(ids), 80, out=out, plan=plan)
    assert (nm.runtime.launch_count() - before == 1) == one
    order, place, offsets = plan_of(ids, 80)
    assert np.array_equal(out.copy_to_host()[:offsets[-1]], x[order // k][:offsets[-1]])
    for a, b in zip(plan, (order, place, offsets)):
        assert np.array_equal(a.copy_to_host(), b)


@pytest.mark.parametrize("tokens,k,one", [(1, 64, True), (60, 64, True), (1, 65, False), (1, 1000, False), (4, 1000, False)])
def test_many_choices_are_sorted_apart(queue, tokens, k, one):
    """A token's block looks for up to 64 choices."""
    import numba_mlir_b200 as nm

    rng = np.random.default_rng(k)
    x = rng.standard_normal((tokens, 24)).astype(np.float32)
    ids = route(tokens, k, 1000, rng)
    out, plan = nm.dispatch_rows(dev(x), dev(ids), 1000)
    before = nm.runtime.launch_count()
    nm.dispatch_rows(dev(x), dev(ids), 1000, out=out, plan=plan)
    assert (nm.runtime.launch_count() - before == 1) == one
    order, place, offsets = plan_of(ids, 1000)
    assert np.array_equal(out.copy_to_host()[:offsets[-1]], x[order // k][:offsets[-1]])
    for a, b in zip(plan, (order, place, offsets)):
        assert np.array_equal(a.copy_to_host(), b)


def test_a_lazily_negated_tensor_is_refused(queue):
    """torch keeps the sign of such a view beside its memory."""
    import torch

    import numba_mlir_b200 as nm

    ids = torch.zeros(3, dtype=torch.int32, device="cuda")
    table = torch.complex(torch.ones(4, 1, device="cuda"), torch.ones(4, 1, device="cuda")).conj().imag
    assert table.is_neg() and table.shape == (4, 1)
    out = torch.empty(3, 1, device="cuda")
    for call in (lambda: nm.take_rows(table, ids, out=out), lambda: nm.take_rows(table, ids)):
        with pytest.raises(RuntimeError, match="resolve_neg"):
            call()
    nm.take_rows(table.resolve_neg(), ids, out=out)
    assert out.tolist() == [[-1.0]] * 3
