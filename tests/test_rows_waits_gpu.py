"""Waits of the row operators' kernels that run out: the kernels are told to give
up at once (their own copies arrive all the same and are waited for), so nothing
hangs.  What a block gave up on is not written, and the queue reports it."""

import contextlib

import numpy as np
import pytest

from test_rows_gpu import bits_of, dev, plan_on_device, route, values_of

pytestmark = pytest.mark.gpu


@contextlib.contextmanager
def no_patience(lib):
    lib.gpuxTestRowWaitSpins(0)
    try:
        yield
    finally:
        lib.gpuxTestRowWaitSpins(2**32 - 1)


def marked(shape, name, queue):
    return dev(bits_of(np.full(shape, 7.0), name), queue)


def runs_out(q, lib, call, results):
    """`call` gives up: the status says so once, `results` (arrays full of 7) are
    left as they are."""
    from numba_mlir_b200.runtime import GpuRuntimeError

    with no_patience(lib):
        call()
        with pytest.raises(GpuRuntimeError, match="timed out"):
            q.check_status()
    for d, name in results:
        assert (values_of(d.copy_to_host(), name) == 7.0).all()
    call()
    q.check_status()
    for d, name in results:
        assert not (values_of(d.copy_to_host(), name) == 7.0).any()


@pytest.mark.parametrize("dim", [4096, 2047])
@pytest.mark.parametrize("name", ["float32", "bfloat16"])
def test_take_rows(runtime_lib, name, dim):
    import numba_mlir_b200 as nm

    q = nm.runtime.Queue("cuda:0")
    n = 1100 if name == "bfloat16" else 600  # enough bytes for the bulk copies
    rng = np.random.default_rng(dim)
    table = dev(bits_of(rng.standard_normal((50, dim)), name), q)
    ids = dev(rng.integers(0, 50, n).astype(np.int32), q)
    out = marked((n, dim), name, q)
    runs_out(q, runtime_lib, lambda: nm.take_rows(table, ids, 0.5, out=out), [(out, name)])


@pytest.mark.parametrize("dim", [1024, 1023])
@pytest.mark.parametrize("n", [300, 5000])
@pytest.mark.parametrize("ids_kind", ["one", "any"])
def test_take_rows_grad(runtime_lib, ids_kind, n, dim):
    """Rows that a block gave up on hold what they held (zero in a fresh gradient,
    their old values where it is added to): never a part of a sum."""
    import numba_mlir_b200 as nm
    from numba_mlir_b200.runtime import GpuRuntimeError

    q = nm.runtime.Queue("cuda:0")
    rng = np.random.default_rng(n + dim)
    ids = np.full(n, 3) if ids_kind == "one" else rng.integers(0, 40, n)
    d = np.ones((n, dim), np.float32)
    dout, di = dev(d, q), dev(ids.astype(np.int32), q)
    grad, added = marked((40, dim), "float32", q), marked((40, dim), "float32", q)
    with no_patience(runtime_lib):
        nm.take_rows_grad(dout, di, out=grad)
        with pytest.raises(GpuRuntimeError, match="timed out"):
            q.check_status()
        nm.take_rows_grad(dout, di, out=added, accumulate=True)
        with pytest.raises(GpuRuntimeError, match="timed out"):
            q.check_status()
    assert np.isin(grad.copy_to_host(), (0.0, 7.0)).all()
    assert (added.copy_to_host() == 7.0).all()
    nm.take_rows_grad(dout, di, out=grad)
    nm.take_rows_grad(dout, di, out=added, accumulate=True)
    q.check_status()
    counts = np.bincount(ids, minlength=40)[:, None]  # whole numbers: exact
    assert (grad.copy_to_host() == counts).all() and (added.copy_to_host() == counts + 7).all()


@pytest.mark.parametrize("tokens,k,dim", [(40, 3, 2047), (5, 2, 5001)])
def test_dispatch_rows(runtime_lib, tokens, k, dim):
    import numba_mlir_b200 as nm

    q = nm.runtime.Queue("cuda:0")
    rng = np.random.default_rng(dim)
    x = dev(rng.standard_normal((tokens, dim)).astype(np.float32), q)
    plan = nm.group_rows(dev(route(tokens, k, 9, rng, 0.0), q), 9)
    out = marked((tokens * k, dim), "float32", q)
    runs_out(q, runtime_lib, lambda: nm.dispatch_rows(x, plan, out=out), [(out, "float32")])


@pytest.mark.parametrize("name", ["float32", "float16"])
@pytest.mark.parametrize("tokens,k,dim", [(40, 8, 2048), (40, 8, 2047), (2371, 2, 520), (2371, 2, 515), (3, 32, 1024)])
def test_combine_rows_and_gradient(runtime_lib, name, tokens, k, dim):
    import numba_mlir_b200 as nm

    q = nm.runtime.Queue("cuda:0")
    rng = np.random.default_rng(dim)
    plan = nm.RowGroups(*(dev(a.copy_to_host(), q) for a in plan_on_device(route(tokens, k, 40, rng, 0.0), 40)))
    ys = dev(bits_of(rng.random((tokens * k, dim)), name), q)
    dout = dev(bits_of(rng.random((tokens, dim)) * 0.01, name), q)
    w = dev(rng.random((tokens, k)).astype(np.float32), q)
    out, dys = marked((tokens, dim), name, q), marked((tokens * k, dim), name, q)
    dw = marked((tokens, k), "float32", q)
    # ys < 1 and weights < 1: no sum of up to 5 of them is 7; more choices are scaled down
    scaled = dev(w.copy_to_host() * np.float32(0.1), q)
    runs_out(q, runtime_lib, lambda: nm.combine_rows(ys, plan, scaled, out=out), [(out, name)])
    # dout < 0.01: dys < 0.01; a product of rows that hits 7 exactly: not for these seeds, and checked below
    from numba_mlir_b200.runtime import GpuRuntimeError

    with no_patience(runtime_lib):
        nm.combine_rows_grad(dout, ys, plan, w, out=dys, dweights=dw)
        with pytest.raises(GpuRuntimeError, match="timed out"):
            q.check_status()
    assert (values_of(dys.copy_to_host(), name) == 7.0).all() and (dw.copy_to_host() == 7.0).all()
    nm.combine_rows_grad(dout, ys, plan, w, out=dys, dweights=dw)
    q.check_status()
    assert (values_of(dys.copy_to_host(), name) < 0.01 + 1e-3).all()
    want = (values_of(ys.copy_to_host(), name)[plan.place.copy_to_host()] * values_of(dout.copy_to_host(), name)[:, None]).sum(-1)
    assert np.abs(dw.copy_to_host() - want).max() <= (dim + 2) * 2.0**-24 * want.max()


def test_a_graph_of_the_first_call_reports_too(runtime_lib):
    """A queue whose first call is recorded into a graph: the replays report waits
    that ran out, each anew, and the word is the queue's own afterwards."""
    import numba_mlir_b200 as nm
    from numba_mlir_b200.runtime import GpuRuntimeError

    q = nm.runtime.Queue("cuda:0")
    rng = np.random.default_rng(0)
    table, ids = dev(rng.standard_normal((50, 4096)).astype(np.float32), q), dev(rng.integers(0, 50, 600).astype(np.int32), q)
    out = marked((600, 4096), "float32", q)
    q.synchronize()
    with no_patience(runtime_lib):
        q.graph_begin()
        nm.take_rows(table, ids, out=out)
        g = q.graph_end()
    for _ in range(2):
        q.graph_launch(g)
        with pytest.raises(GpuRuntimeError, match="timed out"):
            q.check_status()
    assert (out.copy_to_host() == 7.0).all()
    q.graph_destroy(g)
    nm.take_rows(table, ids, out=out)
    q.check_status()
    assert np.array_equal(out.copy_to_host(), table.copy_to_host()[ids.copy_to_host()])


def test_calls_on_torch_tensors_report_to_a_queue_that_can_be_asked(runtime_lib):
    import torch

    import numba_mlir_b200 as nm
    from numba_mlir_b200.runtime import GpuRuntimeError

    table = torch.randn(50, 4096, device="cuda")
    ids = torch.randint(0, 50, (600,), device="cuda")
    out = torch.full((600, 4096), 7.0, device="cuda")
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            q = nm.torch_queue()
            assert q is nm.torch_queue("cuda") and q is nm.torch_queue(table.device) and q is nm.torch_queue(0)
            assert q.stream == stream.cuda_stream
            out.fill_(7.0)
            with no_patience(runtime_lib):
                nm.take_rows(table, ids, out=out)
                with pytest.raises(GpuRuntimeError, match="timed out"):
                    q.check_status()
            assert bool((out == 7.0).all())
            nm.take_rows(table, ids, out=out)
            q.check_status()
            assert torch.equal(out, table[ids])
    with pytest.raises(ValueError):
        nm.torch_queue("cpu")


def test_a_first_call_recorded_by_torch_reports_too(runtime_lib):
    """The same under torch's recording, which forbids other threads and streams
    more than the queue's own does."""
    import torch

    import numba_mlir_b200 as nm
    from numba_mlir_b200.runtime import GpuRuntimeError

    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        table, ids = torch.randn(50, 4096, device="cuda"), torch.randint(0, 50, (600,), device="cuda")
        out = torch.full((600, 4096), 7.0, device="cuda")
        q = nm.runtime.Queue.from_stream(st.cuda_stream)
        st.synchronize()
        g = torch.cuda.CUDAGraph()
        with no_patience(runtime_lib), torch.cuda.graph(g, stream=st):
            nm.take_rows(table, ids, out=out, queue=q)
        g.replay()
        with pytest.raises(GpuRuntimeError, match="timed out"):
            q.check_status()
        assert bool((out == 7.0).all())
        patient = torch.cuda.CUDAGraph()
        with torch.cuda.graph(patient, stream=st):
            nm.take_rows(table, ids, out=out, queue=q)
        patient.replay()
        q.check_status()
        assert torch.equal(out, table[ids])
        del g, patient
