"""The row operators (numba_mlir_b200.rows) against their definitions in
float64: embedding lookup and its gradient, tokens sorted by expert and back,
the gradients of both.

Tolerances count roundings.  With u the unit roundoff of float32 (2^-24; 2^-53
for float64 rows) a sum of n products in any order is off by at most
(n + 1) u sum|terms|, the scale's product by u, the rounding to the result's
type by eps / 2 of the value (or half its smallest subnormal)."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TYPES = ("float32", "float64", "float16", "bfloat16")
HALF_ULP = {"float32": 2.0**-24, "float64": 2.0**-53, "float16": 2.0**-11, "bfloat16": 2.0**-8}
HALF_TINY = {"float32": 2.0**-150, "float64": 0.0, "float16": 2.0**-25, "bfloat16": 2.0**-134}


def unit(name):
    return 2.0**-53 if name == "float64" else 2.0**-24


def bits_of(x, name):
    """float64 values rounded to the named type, as the array to upload."""
    if name != "bfloat16":
        return np.asarray(x, np.float64).astype(name)
    w = np.asarray(x, np.float32).view(np.uint32)
    nan = np.isnan(np.asarray(x, np.float32))
    r = ((w + 0x7FFF + ((w >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(nan, np.uint16(0x7FC0), r).astype(np.uint16).view("V2")


def values_of(a, name):
    """The values that an array of the named type holds, in float64."""
    if name != "bfloat16":
        return a.astype(np.float64)
    return (np.ascontiguousarray(a).view(np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def dev(a, queue=None):
    from numba_mlir_b200 import from_host

    return from_host(a, queue=queue)


def rows_on_device(x, name, pad=0):
    """(device array, its values): rows of a buffer that is `pad` columns wider."""
    full = np.concatenate([x, np.full(x.shape[:-1] + (pad,), 7.0)], axis=-1) if pad else x
    host = bits_of(full, name)
    d = dev(host)
    return (d[..., :x.shape[-1]] if pad else d), values_of(host, name)[..., :x.shape[-1]]


def dtype_of(name):
    import numba_mlir_b200 as nm

    return nm.bfloat16 if name == "bfloat16" else np.dtype(name)


def host_values(d, name):
    return values_of(d.copy_to_host(), name)


def assert_near(got, want, bound, name):
    slack = bound + (np.abs(want) + bound) * HALF_ULP[name] + HALF_TINY[name]
    bad = ~(np.abs(got - want) <= slack)
    assert not bad.any(), f"{bad.sum()} of {bad.size} outside, worst {np.nanmax(np.abs(got - want) - slack)}"


def plan_of(ids, groups):
    """order, place, offsets by their definition."""
    flat = ids.reshape(-1).astype(np.int64)
    key = np.where((flat >= 0) & (flat < groups), flat, groups)
    order = np.argsort(key, kind="stable")
    place = np.empty_like(order)
    place[order] = np.arange(len(order))
    offsets = np.array([(key < g).sum() for g in range(groups + 1)]) if groups < 3000 else \
        np.searchsorted(key[order], np.arange(groups + 1))
    return order, place.reshape(ids.shape), offsets


def plan_on_device(ids, groups):
    import numba_mlir_b200 as nm

    order, place, offsets = plan_of(ids, groups)
    return nm.RowGroups(*(dev(a.astype(np.int32)) for a in (order, place, offsets)))


# ------------------------------------------------------------------- take ---
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rows,dim,shape,pad", [(60, 2047, (33,), 0), (60, 259, (33,), 3), (60, 514, (4,), 1), (60, 33, (70,), 0), (1, 1, (1,), 0), (7, 3, (5,), 0), (50, 64, (4, 9), 8), (33, 1000, (77,), 0),
                                                (100, 4096, (3,), 0), (20, 1025, (16,), 3), (300, 130, (2, 3, 11), 2)])
def test_take_rows(queue, name, rows, dim, shape, pad):
    import numba_mlir_b200 as nm

    rng = np.random.default_rng(rows * dim)
    table, t = rows_on_device(rng.standard_normal((rows, dim)), name, pad)
    ids = rng.integers(-2, rows + 2, shape).astype(np.int64 if dim % 2 else np.int32)
    out = nm.take_rows(table, dev(ids), 1.7)
    assert out.shape == shape + (dim,) and out.dtype == dtype_of(name)
    inside = (ids >= 0) & (ids < rows)
    want = np.where(inside[..., None], t[np.where(inside, ids, 0)], 0.0) * 1.7
    # the scale is a float32 (float64) number: 1.7 is off by u, the product by u
    assert_near(host_values(out, name), want, 2 * unit(name) * np.abs(want), name)


@pytest.mark.parametrize("name,to", [("float32", "float16"), ("float32", "bfloat16"), ("float16", "float32"),
                                     ("bfloat16", "float32")])
@pytest.mark.parametrize("dim", [8, 36, 129])
def test_take_rows_and_gradient_convert(queue, name, to, dim):
    import numba_mlir_b200 as nm

    rng = np.random.default_rng(dim)
    table, t = rows_on_device(rng.standard_normal((11, dim)), name)
    ids = rng.integers(0, 11, 40).astype(np.int32)
    out = nm.empty((40, dim), dtype_of(to), queue=queue)
    assert nm.take_rows(table, dev(ids), 0.5, out=out) is out
    assert_near(host_values(out, to), t[ids] * 0.5, 0.0, to)  # a power of two: only the last rounding
    dout, d = rows_on_device(rng.standard_normal((40, dim)), name)
    grad = nm.empty((11, dim), dtype_of(to), queue=queue)
    nm.take_rows_grad(dout, dev(ids), scale=0.5, out=grad)
    want, mag = np.zeros((11, dim)), np.zeros((11, dim))
    np.add.at(want, ids, d * 0.5)
    np.add.at(mag, ids, np.abs(d) * 0.5)
    assert_near(host_values(grad, to), want, 41 * 2.0**-24 * mag, to)


def test_take_rows_specials(queue):
    """Values pass through as they are, rows that are not picked are not read."""
    import numba_mlir_b200 as nm

    t = np.ones((4, 5), np.float32)
    t[0], t[1, 2], t[3] = np.nan, np.inf, -np.inf
    out = nm.take_rows(dev(t), dev(np.array([2, 1, -1, 4, 2**31 - 1, -2**31], np.int32)), 1.0).copy_to_host()
    assert np.array_equal(out[0], t[2]) and np.array_equal(out[1], t[1]) and not out[2:].any()
    far = nm.take_rows(dev(t), dev(np.array([2**40 + 1, -2**63, 2**63 - 1, 1], np.int64))).copy_to_host()
    assert not far[:3].any() and np.array_equal(far[3], t[1])
    half = nm.take_rows(dev(np.full((1, 3), 60000.0, np.float16)), dev(np.zeros(1, np.int32)), 2.0)
    assert np.isinf(half.copy_to_host()).all()  # past the largest half


def test_take_rows_empty(queue):
    import numba_mlir_b200 as nm

    ids = dev(np.array([0, 3], np.int32))
    assert nm.take_rows(nm.empty((0, 4), np.float32, queue=queue), ids).copy_to_host().tolist() == [[0.0] * 4] * 2
    assert nm.take_rows(nm.empty((5, 0), np.float32, queue=queue), ids).shape == (2, 0)
    assert nm.take_rows(dev(np.ones((5, 3), np.float32)), nm.empty((0,), np.int64, queue=queue)).shape == (0, 3)
    g = nm.take_rows_grad(nm.empty((0, 3), np.float32, queue=queue), nm.empty((0,), np.int64, queue=queue), 4)
    assert g.copy_to_host().tolist() == [[0.0] * 3] * 4
    assert nm.take_rows_grad(nm.empty((2, 3), np.float32, queue=queue), ids, 0).shape == (0, 3)
    assert nm.take_rows_grad(nm.empty((2, 0), np.float32, queue=queue), ids, 4).shape == (4, 0)


# -------------------------------------------------------------- gradient ---
def grad_bound(d, ids, rows, scale, u):
    want, mag, n = np.zeros((rows, d.shape[-1])), np.zeros((rows, d.shape[-1])), np.zeros((rows, 1))
    inside = (ids >= 0) & (ids < rows)
    np.add.at(want, ids[inside], d[inside] * scale)
    np.add.at(mag, ids[inside], np.abs(d[inside] * scale))
    np.add.at(n, ids[inside], 1.0)
    return want, (n + 2) * u * mag


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("n,rows,dim,pad,kind", [
    (1, 1, 1, 0, "any"), (5, 3, 7, 0, "any"), (77, 1000, 64, 8, "any"), (300, 20, 130, 2, "any"), (31, 40, 4096, 0, "any"),
    (257, 9, 33, 0, "one"), (1000, 5, 24, 0, "one"), (1000, 300, 1001, 0, "few"), (2500, 70000, 16, 0, "few"),
    (300, 20, 131, 2, "any"), (700, 9, 1023, 0, "few"), (900, 400, 66, 1, "any"), (4000, 3, 35, 0, "any"), (2100, 4000, 263, 5, "any"), (9000, 50, 8, 0, "any"), (20000, 3000, 12, 0, "few"), (9001, 2000000, 1, 0, "any"), (640, 100, 48, 0, "none")])
def test_take_rows_grad(queue, name, n, rows, dim, pad, kind):
    import numba_mlir_b200 as nm

    if name == "float64" and n * rows > 10**9:
        pytest.skip("covered by the other types")
    rng = np.random.default_rng(n + rows + dim)
    if kind == "any":
        ids = rng.integers(-1, rows + 1, n)
    elif kind == "few":  # a few rows take most of the entries
        ids = np.where(rng.random(n) < 0.6, rng.integers(0, min(rows, 3), n), rng.integers(0, rows, n))
    elif kind == "one":
        ids = np.full(n, rows // 2)
    else:
        ids = np.where(rng.random(n) < 0.5, -1, rows)
    ids = ids.astype(np.int32 if n % 2 else np.int64)
    dout, d = rows_on_device(rng.standard_normal((n, dim)), name, pad)
    out = nm.take_rows_grad(dout, dev(ids), rows, 1.5)
    assert out.shape == (rows, dim)
    want, bound = grad_bound(d, ids, rows, 1.5, unit(name))
    assert_near(host_values(out, name), want, bound, name)
    again = nm.take_rows_grad(dout, dev(ids), rows, 1.5)
    assert out.copy_to_host().tobytes() == again.copy_to_host().tobytes()


@pytest.mark.parametrize("name", ["float32", "bfloat16"])
@pytest.mark.parametrize("n,rows,dim", [(40, 100, 36), (3000, 100, 36), (9000, 12000, 8)])
def test_take_rows_grad_accumulates(queue, name, n, rows, dim):
    import numba_mlir_b200 as nm

    rng = np.random.default_rng(n)
    ids = rng.integers(-1, rows // 2, n).astype(np.int32)
    dout, d = rows_on_device(rng.standard_normal((n, dim)), name)
    old = rng.standard_normal((rows, dim)).astype(np.float32)
    old[rows // 2:] = np.nan  # rows without an entry: not even read
    out = dev(old)
    nm.take_rows_grad(dout, dev(ids), out=out, accumulate=True, scale=0.25)
    got = out.copy_to_host()
    assert got[rows // 2:].tobytes() == old[rows // 2:].tobytes()
    want, bound = grad_bound(d, ids, rows, 0.25, 2.0**-24)
    keep = slice(0, rows // 2)
    assert_near(got[keep].astype(np.float64), want[keep] + old[keep],
                bound[keep] + 2.0**-24 * (np.abs(want[keep]) + np.abs(old[keep])), "float32")


def test_take_rows_grad_by_differences(queue):
    """The table moved along a direction moves <g, take(table)> by <gradient, direction>."""
    import numba_mlir_b200 as nm

    rng = np.random.default_rng(3)
    table, step = rng.standard_normal((13, 20)), rng.standard_normal((13, 20))
    g = rng.standard_normal((4, 9, 20))
    ids = rng.integers(-1, 14, (4, 9))
    grad = nm.take_rows_grad(dev(g), dev(ids), 13, 1.25).copy_to_host()
    h = 2.0**-10
    up, lo = (nm.take_rows(dev(table + s * h * step), dev(ids), 1.25).copy_to_host() for s in (1, -1))
    # linear in the table: the quotient is off by the roundings of the two lookups alone
    assert abs((g * (up - lo)).sum() / (2 * h) - (grad * step).sum()) < 1e-9 * np.abs(g).sum()


def test_offsets_past_32_bits(queue):
    """Rows whose elements begin past 2^31 and 2^32 bytes."""
    import numba_mlir_b200 as nm

    rows, dim = 270001, 8192
    table = nm.zeros((rows, dim), np.float16, queue=queue)
    rng = np.random.default_rng(0)
    at = np.array([0, 131071, 131072, 262143, 262144, rows - 1])
    marks = rng.standard_normal((6, dim)).astype(np.float16)
    for r, m in zip(at, marks):
        table[int(r)].copy_from_host(m)
    ids = dev(at[::-1].copy())
    assert np.array_equal(nm.take_rows(table, ids).copy_to_host(), marks[::-1])
    # the gradient into the same table: every other row becomes zero
    rest = dev(np.array([5, 262145, rows - 2], np.int64))
    nm.take_rows_grad(dev(np.concatenate([marks, marks])), dev(np.concatenate([at, at])), out=table, scale=0.5)
    assert np.array_equal(nm.take_rows(table, ids).copy_to_host(), marks[::-1])
    assert not nm.take_rows(table, rest).copy_to_host().any()


# ------------------------------------------------------------------ group ---
@pytest.mark.parametrize("n,groups", [(1, 1), (8, 64), (31, 2), (33, 5), (1000, 8), (8191, 256), (8192, 1023), (8193, 1023),
                                      (4096, 1024), (20000, 128), (70001, 511), (12289, 5000), (300, 100000),
                                      (9000, 2**31 - 2), (50, 2**31 - 2), (200000, 16),
                                      (1025, 7), (2049, 2000), (40000, 130000), (131072, 128), (131071, 3), (131073, 128), (150000, 4000),
                                      (4095, 1023), (4096, 1024), (4097, 5), (127, 9), (128, 1), (129, 70000), (400000, 64), (1300000, 300), (1300000, 5000)])
@pytest.mark.parametrize("kind", ["any", "one"])
def test_group_rows(queue, n, groups, kind):
    import numba_mlir_b200 as nm

    big = groups > 10**6  # the offsets would be 8 GB: the order through the gradient's tests, here a smaller range
    groups = min(groups, 10**6) if big else groups
    rng = np.random.default_rng(n + groups)
    ids = (rng.integers(-1, groups + 1, n) if kind == "any" else np.full(n, groups - 1)).astype(np.int64 if n % 2 else np.int32)
    plan = nm.group_rows(dev(ids), groups)
    order, place, offsets = plan_of(ids, groups)
    assert np.array_equal(plan.order.copy_to_host(), order)
    assert np.array_equal(plan.place.copy_to_host(), place)
    assert np.array_equal(plan.offsets.copy_to_host(), offsets)


def test_group_rows_edges(queue):
    import numba_mlir_b200 as nm

    none = nm.group_rows(nm.empty((0, 4), np.int32, queue=queue), 3)
    assert none.order.shape == (0,) and none.place.shape == (0, 4) and none.offsets.copy_to_host().tolist() == [0] * 4
    out = nm.group_rows(dev(np.array([1, 0, -5], np.int32)), 0)  # no groups: everything is outside
    assert out.order.copy_to_host().tolist() == [0, 1, 2] and out.offsets.copy_to_host().tolist() == [0]
    wide = nm.group_rows(dev(np.array([2**32, 1, -2**32 + 1, 0], np.int64)), 2)  # 64-bit ids are not cut
    assert wide.order.copy_to_host().tolist() == [3, 1, 0, 2] and wide.offsets.copy_to_host().tolist() == [0, 1, 2]


# --------------------------------------------------------------- dispatch ---
ROUTES = [(1, 1, 1, 1, 0), (4, 8, 64, 2048, 0), (33, 3, 17, 1001, 0), (100, 2, 8, 40, 8), (3000, 6, 60, 24, 0),
          (257, 10, 300, 7, 1), (2000, 8, 128, 130, 2), (1, 8, 1024, 16, 0), (3, 2, 1025, 5, 0), (512, 8, 1000, 9, 0), (585, 7, 64, 33, 0), (40, 5, 9, 2047, 0), (1000, 6, 20, 262, 3), (90, 9, 20, 263, 1)]


def route(tokens, k, groups, rng, drop=0.1):
    ids = np.argsort(rng.random((tokens, max(groups, k))), axis=1)[:, :k]
    return np.where(rng.random((tokens, k)) < drop, -1, ids).astype(np.int32)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("tokens,k,groups,dim,pad", ROUTES)
def test_dispatch_rows(queue, name, tokens, k, groups, dim, pad):
    import numba_mlir_b200 as nm

    rng = np.random.default_rng(tokens + dim)
    x, v = rows_on_device(rng.standard_normal((tokens, dim)), name, pad)
    ids = route(tokens, k, groups, rng)
    xs, plan = nm.dispatch_rows(x, dev(ids), groups)
    order, place, offsets = plan_of(ids, groups)
    assert np.array_equal(plan.order.copy_to_host(), order) and np.array_equal(plan.place.copy_to_host(), place)
    assert np.array_equal(plan.offsets.copy_to_host(), offsets)
    want = v[order // k]
    want[offsets[-1]:] = 0.0
    assert np.array_equal(host_values(xs, name), want)
    # the same plan again, into a larger buffer whose other rows stay
    marked = np.full((tokens * k + 3, dim), 3.0)
    out, _ = rows_on_device(marked, name)
    nm.dispatch_rows(x, plan, out=out)
    got = host_values(out, name)
    assert np.array_equal(got[:tokens * k], want) and (got[tokens * k:] == 3.0).all()


# ---------------------------------------------------------------- combine ---
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("tokens,k,groups,dim,pad", ROUTES + [(6, 32, 40, 1024, 0), (3, 33, 40, 1024, 0), (9, 5, 7, 8192, 8)])
def test_combine_rows(queue, name, tokens, k, groups, dim, pad):
    import numba_mlir_b200 as nm

    rng = np.random.default_rng(tokens + dim)
    ids = route(tokens, k, groups, rng)
    plan = plan_on_device(ids, groups)
    order, place, offsets = plan_of(ids, groups)
    raw = rng.standard_normal((tokens * k, dim))
    raw[offsets[-1]:] = np.nan  # rows of dropped choices hold anything
    ys, y = rows_on_device(raw, name, pad)
    w = rng.random((tokens, k)).astype(np.float32)
    kept = place < offsets[-1]
    picked = np.where(kept[..., None], y[place], 0.0)
    u = unit(name)
    for weights, dw in ((w, dev(w)), (np.ones_like(w), None)):
        terms = picked * weights[..., None].astype(np.float64)
        out = nm.combine_rows(ys, plan, dw)
        assert out.shape == (tokens, dim)
        assert_near(host_values(out, name), terms.sum(1), (k + 1) * u * np.abs(terms).sum(1), name)
    back = nm.dispatch_rows_grad(ys, plan)
    assert back.copy_to_host().tobytes() == out.copy_to_host().tobytes()


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("tokens,k,groups,dim,pad", ROUTES + [(5, 40, 50, 96, 0), (6, 32, 40, 1024, 0), (3, 33, 40, 1024, 0), (9, 5, 7, 8192, 8)])
def test_combine_rows_grad(queue, name, tokens, k, groups, dim, pad):
    import numba_mlir_b200 as nm

    rng = np.random.default_rng(tokens + dim)
    ids = route(tokens, k, groups, rng)
    plan = plan_on_device(ids, groups)
    order, place, offsets = plan_of(ids, groups)
    raw = rng.standard_normal((tokens * k, dim))
    raw[offsets[-1]:] = np.nan
    ys, y = rows_on_device(raw, name, pad)
    dout, d = rows_on_device(rng.standard_normal((tokens, dim)), name, pad)
    w = rng.random((tokens, k)).astype(np.float32)
    dys, dw = nm.combine_rows_grad(dout, ys, plan, dev(w))
    kept = place < offsets[-1]
    want = np.zeros((tokens * k, dim))
    want[place] = np.where(kept[..., None], w[..., None].astype(np.float64) * d[:, None], 0.0)
    u = unit(name)
    assert_near(host_values(dys, name), want, u * np.abs(want), name)
    terms = np.where(kept[..., None], y[place], 0.0) * d[:, None]
    assert dw.dtype == np.float32
    assert_near(dw.copy_to_host().astype(np.float64), terms.sum(-1), (dim + 1) * u * np.abs(terms).sum(-1), "float32")


# Narrow rows of many tokens: two or four tokens share a block, the last block has
# fewer; widths on both sides of where the bulk copies begin.
SHARED = [(2371, 2, 16, 400, 0), (2369, 1, 5, 520, 8), (1187, 3, 16, 264, 0), (2371, 8, 9, 256, 0), (2370, 2, 16, 99, 0),
          (1187, 4, 9, 48, 1), (2371, 2, 16, 47, 0), (2371, 5, 9, 515, 0), (2375, 9, 10, 128, 0), (1186, 12, 13, 72, 1)]


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("tokens,k,groups,dim,pad", SHARED)
def test_tokens_that_share_a_block(queue, name, tokens, k, groups, dim, pad):
    test_combine_rows(queue, name, tokens, k, groups, dim, pad)
    test_combine_rows_grad(queue, name, tokens, k, groups, dim, pad)


@pytest.mark.parametrize("tokens,k,dim", [(2371, 2, 512), (2371, 2, 515), (2370, 3, 264), (1187, 1, 99), (2371, 2, 64)])
def test_memory_around_the_results_is_left_alone(queue, tokens, k, dim):
    """Results are parts of larger arrays whose other rows and columns keep what
    they hold, bit for bit, also behind the last token of a shared block."""
    import numba_mlir_b200 as nm

    rng = np.random.default_rng(tokens + dim)
    ids = route(tokens, k, 9, rng)
    plan = plan_on_device(ids, 9)
    ys = dev(rng.standard_normal((tokens * k, dim)).astype(np.float32))
    dout = dev(rng.standard_normal((tokens, dim)).astype(np.float32))
    w = dev(rng.random((tokens, k)).astype(np.float32))
    whole = {n: dev(np.full((rows + 7, dim + 9), -7.5, np.float32)) for n, rows in (("out", tokens), ("dys", tokens * k))}
    dwhole = dev(np.full((tokens + 7, k), -7.5, np.float32))
    parts = {"out": whole["out"][3:3 + tokens, 5:5 + dim], "dys": whole["dys"][3:3 + tokens * k, 5:5 + dim]}
    nm.combine_rows(ys, plan, w, out=parts["out"])
    nm.combine_rows_grad(dout, ys, plan, w, out=parts["dys"], dweights=dwhole[3:3 + tokens])
    for n, rows in (("out", tokens), ("dys", tokens * k)):
        got = whole[n].copy_to_host()
        inside = got[3:3 + rows, 5:5 + dim].copy()
        assert not (inside == -7.5).any()
        got[3:3 + rows, 5:5 + dim] = -7.5
        assert (got == -7.5).all()
    got = dwhole.copy_to_host()
    assert (got[:3] == -7.5).all() and (got[3 + tokens:] == -7.5).all() and not (got[3:3 + tokens] == -7.5).any()
    # the same call once more gives the same bits (one with another alignment may add in another order)
    again = nm.combine_rows_grad(dout, ys, plan, w, out=parts["dys"])[1].copy_to_host()
    assert again.tobytes() == got[3:3 + tokens].tobytes()


@pytest.mark.parametrize("wname", ["float16", "bfloat16", "float64"])
def test_weights_of_other_types(queue, wname):
    import numba_mlir_b200 as nm

    rng = np.random.default_rng(1)
    ids = route(50, 3, 9, rng, 0.0)
    plan = plan_on_device(ids, 9)
    _, place, _ = plan_of(ids, 9)
    ys, y = rows_on_device(rng.standard_normal((150, 17)), "float32")
    dout, d = rows_on_device(rng.standard_normal((50, 17)), "float32")
    weights, w = rows_on_device(rng.random((50, 3)), wname)
    terms = y[place] * w[..., None]
    u = 2.0**-24
    # float64 weights are rounded to float32 first: one more u
    assert_near(host_values(nm.combine_rows(ys, plan, weights), "float32"), terms.sum(1), 5 * u * np.abs(terms).sum(1),
                "float32")
    dys, dw = nm.combine_rows_grad(dout, ys, plan, weights)
    assert dw.dtype == dtype_of(wname)
    dots = y[place] * d[:, None]
    got = host_values(dw, wname)
    bound = 18 * u * np.abs(dots).sum(-1)
    assert_near(got, dots.sum(-1), bound, wname)


def test_routing_gradients_by_differences(queue):
    """<g, combine(dispatch(x), w)> moves with x and w as the gradients say."""
    import numba_mlir_b200 as nm

    rng = np.random.default_rng(5)
    tokens, k, groups, dim = 40, 3, 7, 12
    ids = route(tokens, k, groups, rng, 0.2)
    x, g = rng.standard_normal((tokens, dim)), rng.standard_normal((tokens, dim))
    w = rng.random((tokens, k))
    factor = rng.standard_normal((tokens * k, 1))  # what the experts do to their rows

    def forward(x, w):
        xs, plan = nm.dispatch_rows(dev(x), dev(ids), groups)
        ys = dev(xs.copy_to_host() * factor)
        return nm.combine_rows(ys, plan, dev(w)).copy_to_host(), ys, plan

    _, ys, plan = forward(x, w)
    dys, dw = nm.combine_rows_grad(dev(g), ys, plan, dev(w))
    dx = nm.dispatch_rows_grad(dev(dys.copy_to_host() * factor), plan).copy_to_host()
    h = 2.0**-12
    for grad, which in ((dx, 0), (dw.copy_to_host(), 1)):
        step = rng.standard_normal(grad.shape)
        ends = []
        for s in (1, -1):
            moved = (x + s * h * step, w) if which == 0 else (x, w + s * h * step)
            ends.append((forward(*moved)[0] * g).sum())
        # linear in each: off by the roundings of two sums of 40 x 12 terms of order 10
        assert abs((ends[0] - ends[1]) / (2 * h) - (grad * step).sum()) < 1e-7


# ------------------------------------------------- together, queues, graphs ---
@pytest.mark.parametrize("name", ["float32", "bfloat16"])
def test_a_training_step_end_to_end(queue, name):
    """Lookup, experts that scale their rows by their number, the way back, and
    all gradients down to the table, as a program runs them."""
    import numba_mlir_b200 as nm

    rng = np.random.default_rng(11)
    tokens, vocab, dim, k, groups = 700, 90, 64, 2, 4
    tok = np.where(rng.random(tokens) < 0.1, -1, rng.integers(0, vocab, tokens)).astype(np.int64)
    ids = route(tokens, k, groups, rng, 0.05)
    w = rng.random((tokens, k)).astype(np.float32)
    table, t = rows_on_device(np.round(rng.standard_normal((vocab, dim)) * 8) / 8, name)  # few bits: most of it is exact
    dy, g = rows_on_device(np.round(rng.standard_normal((tokens, dim)) * 8) / 8, name)
    x = nm.take_rows(table, dev(tok), 2.0)
    xs, plan = nm.dispatch_rows(x, dev(ids), groups)
    y = nm.combine_rows(xs, plan, dev(w))
    dxs, dw = nm.combine_rows_grad(dy, xs, plan, dev(w))
    dx = nm.dispatch_rows_grad(dxs, plan)
    dtable = nm.take_rows_grad(dx, dev(tok), vocab, 2.0)

    kept, live = ids >= 0, (tok >= 0)[:, None]
    xv = np.where(live, 2.0 * t[np.maximum(tok, 0)], 0.0)
    wk = np.where(kept, w, 0.0).astype(np.float64)
    assert_near(host_values(y, name), xv * wk.sum(1, keepdims=True), 3 * 2.0**-24 * np.abs(xv) * wk.sum(1, keepdims=True), name)
    dots = (xv * g).sum(1, keepdims=True) * kept
    assert_near(dw.copy_to_host().astype(np.float64), dots, 65 * 2.0**-24 * (np.abs(xv * g).sum(1, keepdims=True) * kept),
                "float32")
    want, mag = np.zeros((vocab, dim)), np.zeros((vocab, dim))
    each = 2.0 * g * wk.sum(1, keepdims=True)
    size = 2.0 * np.abs(g) * wk.sum(1, keepdims=True)
    np.add.at(want, tok[tok >= 0], each[tok >= 0])
    np.add.at(mag, tok[tok >= 0], size[tok >= 0])
    # two roundings to the type on the way (dxs, dx), float32 sums
    assert_near(host_values(dtable, name), want, (2.1 * HALF_ULP[name] + 40 * 2.0**-24) * mag, name)


def test_inside_njit(queue):
    import numba_mlir_b200 as nm

    @nm.njit(parallel=True)
    def step(table, tok, ids, w, scale, dy):
        x = nm.take_rows(table, tok, scale)
        x = x * np.float32(2) + np.float32(1)
        xs, plan = nm.dispatch_rows(x, ids, 5)
        ys = xs * np.float32(0.5)
        y = nm.combine_rows(ys, plan, w)
        dys, dw = nm.combine_rows_grad(dy, ys, plan, w)
        dx = nm.dispatch_rows_grad(dys * np.float32(0.5), plan)
        return y, dw, nm.take_rows_grad(dx * np.float32(2), tok, 30, scale)

    rng = np.random.default_rng(2)
    for scale in (np.float32(1.5), np.float32(-0.25)):  # the second call replays the recorded plan
        table = rng.standard_normal((30, 24)).astype(np.float32)
        tok = rng.integers(-1, 31, 60).astype(np.int32)
        ids = route(60, 2, 5, rng)
        w, dy = rng.random((60, 2)).astype(np.float32), rng.standard_normal((60, 24)).astype(np.float32)
        y, dw, dt = step(*(dev(a) for a in (table, tok, ids, w)), scale, dev(dy))
        inside = (tok >= 0) & (tok < 30)
        x = np.where(inside[:, None], table.astype(np.float64)[np.where(inside, tok, 0)] * float(scale), 0.0) * 2 + 1
        kept = ids >= 0
        wk = np.where(kept, w, 0.0).sum(1, keepdims=True)
        np.testing.assert_allclose(y.copy_to_host(), x * 0.5 * wk, rtol=1e-5, atol=1e-6)
        np.testing.assert_allclose(dw.copy_to_host(), (x * 0.5 * dy).sum(1, keepdims=True) * kept, rtol=1e-4, atol=1e-4)
        want = np.zeros((30, 24))
        np.add.at(want, tok[inside], (dy * wk * 0.5 * 2 * float(scale))[inside])
        np.testing.assert_allclose(dt.copy_to_host(), want, rtol=1e-4, atol=1e-5)
    assert len(step._plans) == 1


def test_inside_njit_orders_with_stores(queue):
    """Arrays written by the traced function are read, and read arrays are
    written, in program order."""
    import numba_mlir_b200 as nm

    @nm.njit(parallel=True)
    def f(table, ids, out):
        before = table + np.float32(1)     # not evaluated yet
        table[:] = table * np.float32(2)
        nm.take_rows(table, ids, np.float32(1), out=out)
        nm.take_rows_grad(out, ids, out=table)
        return before

    t = np.arange(12, dtype=np.float32).reshape(4, 3)
    ids = np.array([3, 0, 3], np.int32)
    for _ in range(2):
        table, out = dev(t), dev(np.zeros((3, 3), np.float32))
        before = f(table, dev(ids), out).copy_to_host()
        assert np.array_equal(before, t + 1) and np.array_equal(out.copy_to_host(), 2 * t[ids])
        want = np.zeros_like(t)
        np.add.at(want, ids, 2 * t[ids])
        assert np.array_equal(table.copy_to_host(), want)


@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("n", [200, 20000])
def test_two_graphs_share_nothing(queue, given, n):
    """Calls recorded into graphs, with workspaces of their own and without."""
    import numba_mlir_b200 as nm

    rng = np.random.default_rng(n)
    rows, dim = 300, 16
    qs = [nm.runtime.Queue("cuda:0") for _ in range(2)]
    made = []
    for q in qs:
        ids = rng.integers(-1, rows, n).astype(np.int32)
        d = rng.standard_normal((n, dim)).astype(np.float32)
        di, dd = dev(ids, q), dev(d, q)
        out = nm.empty((rows, dim), np.float32, queue=q)
        xs, plan = nm.dispatch_rows(dd, di, rows)
        ws = nm.empty((nm.take_rows_grad_workspace(n, rows, dim),), np.uint8, queue=q) if given else None
        q.synchronize()
        q.graph_begin()
        nm.take_rows_grad(dd, di, out=out, workspace=ws)
        nm.dispatch_rows(dd, di, rows, out=xs, plan=plan)
        made.append((q, q.graph_end(), di, dd, out, xs, plan))
    for _ in range(2):
        for q, g, di, dd, out, xs, plan in made:  # new inputs, both graphs in flight at once
            di.copy_from_host(rng.integers(-1, rows, n).astype(np.int32))
            dd.copy_from_host(rng.standard_normal((n, dim)).astype(np.float32))
        for _ in range(3):
            for q, g, *_rest in made:
                q.graph_launch(g)
        for q, g, di, dd, out, xs, plan in made:
            q.synchronize()
            ids, d = di.copy_to_host(), dd.copy_to_host()
            want, bound = grad_bound(d.astype(np.float64), ids, rows, 1.0, 2.0**-24)
            assert_near(out.copy_to_host().astype(np.float64), want, bound, "float32")
            order, place, offsets = plan_of(ids, rows)
            got = xs.copy_to_host()
            assert np.array_equal(got[:offsets[-1]], d[order[:offsets[-1]]]) and not got[offsets[-1]:].any()
    for q, g, *_rest in made:
        q.graph_destroy(g)


def test_arrays_of_another_queue(queue):
    """Arrays that belong to other streams are read after those streams' work
    and may be overwritten there right after the call."""
    import numba_mlir_b200 as nm

    a, b = nm.runtime.Queue("cuda:0"), nm.runtime.Queue("cuda:0")
    rng = np.random.default_rng(0)
    t = rng.standard_normal((2000, 4096)).astype(np.float32)
    ids = rng.integers(0, 2000, 3000).astype(np.int32)
    for _ in range(3):
        table = nm.zeros(t.shape, np.float32, queue=a)
        src = dev(t, a)
        a.synchronize()
        a.memcpy(table.ptr, src.ptr, table.nbytes)           # not waited for
        out = nm.take_rows(table, dev(ids, b), queue=b)
        a.memset(table.ptr, 0, table.nbytes)                 # right behind the call
        assert np.array_equal(out.copy_to_host(), t[ids])


def test_torch_tensors(queue):
    """Tensors of torch run on torch's current stream, whichever it is."""
    import torch

    import numba_mlir_b200 as nm

    ids = torch.randint(-1, 500, (64, 2), device="cuda")
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        with torch.cuda.stream(stream):
            table = torch.randn(500, 257, device="cuda").bfloat16()
            out = torch.empty(64, 2, 257, dtype=torch.bfloat16, device="cuda")
            nm.take_rows(table, ids, 2.0, out=out)
            want = torch.where((ids >= 0)[..., None], table[ids.clamp(min=0)] * 2.0, 0.0)
            assert torch.equal(out, want)
            grad = torch.empty(500, 257, dtype=torch.float32, device="cuda")
            nm.take_rows_grad(out, ids, out=grad)
            ref = torch.zeros(501, 257, dtype=torch.float64, device="cuda")
            ref.index_add_(0, torch.where(ids >= 0, ids, 500).reshape(-1), out.reshape(-1, 257).double())
            assert torch.allclose(grad.double(), ref[:500], rtol=1e-5, atol=1e-5)
            # a queue of its own beside torch's stream
            q = nm.runtime.Queue("cuda:0")
            nm.take_rows(table, ids, 1.0, out=out, queue=q)
            assert torch.equal(out, torch.where((ids >= 0)[..., None], table[ids.clamp(min=0)], 0.0))
    with pytest.raises(RuntimeError, match="requires a gradient"):
        nm.take_rows(torch.randn(4, 4, device="cuda", requires_grad=True), ids)
    with pytest.raises(TypeError):
        nm.take_rows(torch.randn(4, 4), ids)


def test_torch_graph_with_workspaces(queue):
    """Calls recorded by torch on a stream of its own, with torch's workspaces
    and without, replay on new inputs."""
    import torch

    import numba_mlir_b200 as nm

    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        ids = torch.randint(-1, 400, (6000,), device="cuda", dtype=torch.int32)
        d = torch.randn(6000, 520, device="cuda")
        grads = [torch.empty(400, 520, device="cuda") for _ in range(2)]
        plan = nm.RowGroups(torch.empty_like(ids), torch.empty_like(ids), torch.empty(401, dtype=torch.int32, device="cuda"))
        ws = torch.empty(nm.take_rows_grad_workspace(6000, 400, 520), dtype=torch.uint8, device="cuda")
        ws2 = torch.empty(nm.group_rows_workspace(6000, 400), dtype=torch.uint8, device="cuda")

        def calls():
            nm.take_rows_grad(d, ids, out=grads[0], workspace=ws)
            nm.take_rows_grad(d, ids, out=grads[1])
            nm.group_rows(ids, 400, plan=plan, workspace=ws2)

        calls()
        st.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            calls()
        for seed in (1, 2):
            ids.copy_(torch.randint(-1, 400, (6000,), device="cuda", dtype=torch.int32))
            d.normal_()
            g.replay()
            st.synchronize()
            want, bound = grad_bound(d.double().cpu().numpy(), ids.cpu().numpy(), 400, 1.0, 2.0**-24)
            for got in grads:
                assert_near(got.double().cpu().numpy(), want, bound, "float32")
            order, place, offsets = plan_of(ids.cpu().numpy(), 400)
            for got, ref in zip(plan, (order, place, offsets)):
                assert np.array_equal(got.cpu().numpy(), ref)
        del g


def test_refusals(queue):
    import numba_mlir_b200 as nm

    f = lambda *s: nm.zeros(s, np.float32, queue=queue)  # noqa: E731
    i = lambda *s: nm.zeros(s, np.int32, queue=queue)  # noqa: E731
    t = f(5, 8)
    with pytest.raises(TypeError):
        nm.take_rows(t, f(3))
    with pytest.raises(TypeError):
        nm.take_rows(nm.zeros((5, 8), np.int32, queue=queue), i(3))
    with pytest.raises(TypeError):
        nm.take_rows(np.zeros((5, 8), np.float32), i(3))
    with pytest.raises(ValueError, match="unit stride"):
        nm.take_rows(t[:, ::2], i(3))
    with pytest.raises(ValueError, match="contiguous"):
        nm.take_rows(t, i(6)[::2])
    with pytest.raises(ValueError, match="shape"):
        nm.take_rows(t, i(3), out=f(4, 8))
    with pytest.raises(TypeError, match="type"):
        nm.take_rows(t, i(3), out=nm.zeros((3, 8), np.float64, queue=queue))
    with pytest.raises(ValueError, match="shares memory"):
        nm.take_rows(t, i(3), out=t[1:4])
    with pytest.raises(nm.runtime.GpuRuntimeError, match="overlap"):
        flat = nm.device_array.DeviceArray(t._buf, (3, 8), np.float32, (4, 4))
        nm.take_rows(f(5, 8), i(3), out=flat)
    with pytest.raises(ValueError, match="one stride"):
        nm.take_rows_grad(f(4, 4, 8)[:, :3], i(4, 3), 5)
    with pytest.raises(ValueError, match="number of rows"):
        nm.take_rows_grad(f(3, 8), i(3))
    with pytest.raises(ValueError, match="accumulate"):
        nm.take_rows_grad(f(3, 8), i(3), 5, accumulate=True)
    with pytest.raises(nm.runtime.GpuRuntimeError, match="workspace"):
        nm.take_rows_grad(f(3, 8), i(3), 5, workspace=nm.empty((16,), np.uint8, queue=queue))
    with pytest.raises(ValueError, match="negative"):
        nm.group_rows(i(3), -1)
    with pytest.raises(ValueError, match="groups"):
        nm.dispatch_rows(t, i(5))
    with pytest.raises(ValueError, match="choices"):
        nm.dispatch_rows(t, i(4, 2), 3)
    plan = nm.group_rows(i(5, 2), 3)
    with pytest.raises(ValueError):
        nm.combine_rows(f(10, 8), plan, f(5, 3))
    with pytest.raises(ValueError, match="ys has shape"):
        nm.combine_rows_grad(f(5, 8), f(9, 8), plan)
    with pytest.raises(TypeError, match="one type"):
        nm.combine_rows_grad(f(5, 8), nm.zeros((10, 8), np.float16, queue=queue), plan)
    with pytest.raises(TypeError, match="int32"):
        nm.combine_rows(f(10, 8), nm.RowGroups(plan.order, nm.zeros((5, 2), np.int64, queue=queue), plan.offsets))
    nm.runtime.check()  # nothing left behind
    # different columns of one buffer do not share memory
    both = f(6, 16)
    assert nm.take_rows(both[:, :8], i(6), out=both[:, 8:]).shape == (6, 8)


def test_positions_outside_are_left_out(queue):
    """A plan that does not fit its rows reads and writes nothing outside them."""
    import numba_mlir_b200 as nm

    place = dev(np.array([[0, 7], [-3, 2**31 - 1]], np.int32))
    plan = nm.RowGroups(place, place, dev(np.array([2**31 - 1], np.int32)))
    ys = dev(np.arange(12, dtype=np.float32).reshape(4, 3))
    assert nm.combine_rows(ys, plan).copy_to_host().tolist() == [[0.0, 1.0, 2.0], [0.0] * 3]
    out = dev(np.full((4, 3), 9.0, np.float32))
    nm.dispatch_rows(dev(np.ones((2, 3), np.float32)), plan, out=out)
    assert out.copy_to_host().tolist() == [[1.0] * 3] + [[9.0] * 3] * 3
    dys, dw = nm.combine_rows_grad(dev(np.ones((2, 3), np.float32)), ys, plan, out=out)
    assert dw.copy_to_host().tolist() == [[3.0, 0.0], [0.0, 0.0]]
    assert dys.copy_to_host().tolist() == [[1.0] * 3] + [[9.0] * 3] * 3


@pytest.mark.parametrize("source", ["device", "torch"])
def test_native_path_takes_ordinary_calls(queue, source):
    """The native call path answers 1 for calls in order, 0 for the others, and
    writes what the Python path writes."""
    import torch

    import numba_mlir_b200 as nm
    from numba_mlir_b200 import rows

    rng = np.random.default_rng(4)
    ids = rng.integers(-1, 9, (50, 2)).astype(np.int32)
    host = {"table": rng.standard_normal((9, 24)).astype(np.float32), "ids": ids, "x": rng.standard_normal((50, 24)).astype(np.float32),
            "w": rng.random((50, 2)).astype(np.float32)}
    if source == "torch":
        put = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
        new = lambda shape, dt=np.float32: torch.zeros(shape, dtype=torch.float32 if dt == np.float32 else torch.int32, device="cuda")  # noqa: E731
        get = lambda t: t.cpu().numpy()  # noqa: E731
        q = rows._torch_stream(0)
        nm.take_rows(put(host["table"]), put(ids), out=new((50, 2, 24)))  # the first tensor binds
    else:
        put, get, q = dev, (lambda t: t.copy_to_host()), queue
        new = lambda shape, dt=np.float32: nm.zeros(shape, dt, queue=queue)  # noqa: E731
        nm.take_rows(put(host["table"]), put(ids), out=new((50, 2, 24)))
    rows._raw_stream(q)
    fast = rows._fast()
    table, i, x, w = (put(host[n]) for n in ("table", "ids", "x", "w"))
    picked, grad = new((50, 2, 24)), new((9, 24))
    plan = nm.RowGroups(new((100,), np.int32), new((50, 2), np.int32), new((10,), np.int32))
    xs, y, dys, dw = new((100, 24)), new((50, 24)), new((100, 24)), new((50, 2))
    assert fast.rows_take(q, table, i, 1.5, picked) == 1
    assert fast.rows_take_grad(q, picked, i, 1.5, grad, False) == 1
    assert fast.rows_group(q, i, 9, plan) == 1
    assert fast.rows_dispatch(q, x, None, None, plan, xs) == 1
    assert fast.rows_dispatch(q, x, i, 9, plan, xs) == 1
    assert fast.rows_combine(q, xs, plan, w, y) == 1
    assert fast.rows_combine(q, xs, plan, None, y) == 1
    assert fast.rows_combine(q, xs, plan, w, y) == 1
    assert fast.rows_combine_grad(q, x, xs, plan, w, dys, dw) == 1
    d = {n: dev(a) for n, a in host.items()}
    picked2 = nm.take_rows(d["table"], d["ids"], 1.5)
    grad2 = nm.take_rows_grad(picked2, d["ids"], 9, 1.5)
    xs2, plan2 = nm.dispatch_rows(d["x"], d["ids"], 9)
    y2 = nm.combine_rows(xs2, plan2, d["w"])
    dys2, dw2 = nm.combine_rows_grad(d["x"], xs2, plan2, d["w"])
    for a, b in ((picked, picked2), (grad, grad2), (xs, xs2), (y, y2), (dys, dys2), (dw, dw2), *zip(plan, plan2)):
        assert get(a).tobytes() == b.copy_to_host().tobytes()
    # out of order: another queue, a wrong shape, type or overlap, a missing result
    other = nm.runtime.Queue("cuda:0")
    rows._raw_stream(other)
    assert fast.rows_take(other, table, i, 1.5, picked) == 0
    assert fast.rows_take(q, table, i, 1.5, xs) == 0
    assert fast.rows_take(q, table, w, 1.5, picked) == 0
    assert fast.rows_take(q, table, i, "x", picked) == 0
    assert fast.rows_take(q, table, i, 1.5, None) == 0
    assert fast.rows_take(q, host["table"], i, 1.5, picked) == 0
    assert fast.rows_dispatch(q, xs[:50], None, None, plan, xs) == 0
    assert fast.rows_combine(q, xs, plan, w[:40], y) == 0
    assert fast.rows_combine(q, xs, (1, 2), w, y) == 0
    assert fast.rows_combine_grad(q, x, xs[:90], plan, w, dys, dw) == 0


def test_arrays_captured_by_a_traced_function(queue):
    """A routine called inside a traced function on arrays that are not its
    arguments runs in every call, not only in the traced one."""
    import numba_mlir_b200 as nm

    table, ids, out = dev(np.ones((4, 3), np.float32)), dev(np.array([1, 2], np.int32)), nm.zeros((2, 3), np.float32, queue=queue)

    @nm.njit(parallel=True)
    def f(a):
        nm.take_rows(table, ids, 2.0, out=out)
        return a + np.float32(1)

    for v in (1.0, 5.0):
        table.copy_from_host(np.full((4, 3), v, np.float32))
        f(dev(np.zeros(3, np.float32)))
        assert (out.copy_to_host() == 2 * v).all()
