"""Calls of the routed and the 4-bit linears that a program makes and a single
call in a quiet process does not show (-m gpu): several host threads, captured
modules, uploads beside queued work, the sizes at which the kernels' rings,
clusters and accumulators come round."""
import ctypes as C
import threading

import numpy as np
import pytest

from tests.gpu_util import device_error, np_dtype, to_device, to_host32

pytestmark = pytest.mark.gpu


def _in_threads(*calls):
    """Every call in a thread of its own, started together."""
    errors, gate = [], threading.Barrier(len(calls))

    def run(fn):
        try:
            gate.wait(30)
            fn()
        except BaseException as e:  # noqa: BLE001 - reported below
            errors.append(e)

    threads = [threading.Thread(target=run, args=(fn,)) for fn in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert not errors and not any(t.is_alive() for t in threads), errors


def test_gathered_batches_of_two_threads(gpu, ops):
    """Two threads on the default stream, each with gathered batches of its own
    that go through the stream's workspace, the second's larger at times: the
    bits of the same calls made one by one."""
    rng = np.random.default_rng(5)
    X, K, N, T = 4, 64, 1024, 300
    gw, _ = to_device(ops, rng.standard_normal((X, N, K), dtype=np.float32), "bf16")
    jobs = []
    for M in (2100, 2400, 4300):
        gx, _ = to_device(ops, rng.standard_normal((T, K), dtype=np.float32), "bf16")
        rows = ops.gputensor_from_numpy(rng.integers(0, T, M).astype(np.int32))
        off = ops.gputensor_from_numpy(np.array([0, M // 3, M // 2, M - 7, M], np.int32))
        want = to_host32(ops, ops.dev_grouped_linear(gx, gw, off, rows=rows))
        jobs.append((gx, off, rows, want))

    def loop(which):
        for i in range(40):
            gx, off, rows, want = jobs[which[i % len(which)]]
            assert np.array_equal(to_host32(ops, ops.dev_grouped_linear(gx, gw, off, rows=rows)), want)

    _in_threads(lambda: loop([0]), lambda: loop([1, 2]))
    assert device_error(0) == 0


@pytest.fixture
def own_stream(gpu, ops):
    """The engine's launches on a non-blocking stream, which the uploads of the
    legacy stream do not wait for by themselves."""
    from scaffolding_b200 import engine as E
    s = ops.CudaStream(0)
    E.set_stream(0, s.cuda_stream)
    yield s
    s.synchronize()
    E.set_stream(0, None)


def test_upload_beside_an_unpacked_weight(ops, own_stream):
    """Uploads of tensors of the unpacked weight's size right after 4-bit
    linears of many rows, whose products are still queued."""
    rng = np.random.default_rng(9)
    N, K, M = 1024, 2048, 4000
    gw, _ = to_device(ops, rng.standard_normal((N, K), dtype=np.float32), "bf16")
    w4 = ops.dev_quantize_w4(gw, 64, True)
    gx, _ = to_device(ops, rng.standard_normal((M, K), dtype=np.float32), "bf16")
    want = to_host32(ops, ops.dev_linear_w4(gx, w4))
    other = np.full((N, K), 3, np_dtype("bf16"))
    for _ in range(20):
        ys = [ops.dev_linear_w4(gx, w4) for _ in range(3)]
        up = ops.gputensor_from_numpy(other)
        for y in ys:
            assert np.array_equal(to_host32(ops, y), want)
        del up
    assert device_error(0) == 0


def test_upload_beside_dropped_intermediates(ops, own_stream):
    """Uploads of the size of an intermediate that queued linears still read."""
    rng = np.random.default_rng(19)
    M, K = 4096, 1024
    gw, _ = to_device(ops, rng.standard_normal((K, K), dtype=np.float32) / np.float32(32), "bf16")
    gx, _ = to_device(ops, rng.standard_normal((M, K), dtype=np.float32), "bf16")
    chain = lambda: ops.dev_linear_forward(ops.dev_linear_forward(gx, gw), gw)  # noqa: E731
    want = to_host32(ops, chain())
    other = np.full((M, K), 3, np_dtype("bf16"))
    for _ in range(20):
        ys = [chain() for _ in range(3)]
        up = ops.gputensor_from_numpy(other)
        for y in ys:
            assert np.array_equal(to_host32(ops, y), want)
        del up


class Capture:
    """``with Capture(ops) as g:`` captures the engine's calls on a stream of
    its own; ``g.launch()`` replays them there (or on ``stream``)."""

    def __init__(self, ops, stream=None):
        self.stream = stream or ops.CudaStream(0)

    def __enter__(self):
        from scaffolding_b200 import engine as E
        E.set_stream(0, self.stream.cuda_stream)
        E.check(E.lib.sf_graph_begin(C.c_void_p(self.stream.cuda_stream)), "begin")
        return self

    def __exit__(self, kind, *exc):
        from scaffolding_b200 import engine as E
        self.exe = C.c_void_p()
        st = E.lib.sf_graph_end(C.c_void_p(self.stream.cuda_stream), C.byref(self.exe))
        E.set_stream(0, None)
        if kind is None:
            E.check(st, "end")

    def launch(self, stream=None):
        from scaffolding_b200 import engine as E
        E.check(E.lib.sf_graph_launch(self.exe, C.c_void_p((stream or self.stream).cuda_stream)), "launch")

    def destroy(self):
        from scaffolding_b200 import engine as E
        E.check(E.lib.sf_graph_destroy(self.exe), "destroy")


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_captured_workspaces(gpu, ops, dt):
    """Two graphs captured on one stream, whose products keep sums or operand
    panels in a workspace, replayed side by side and beside direct calls of the
    stream with a larger one."""
    from oracle import oracle as O
    from scaffolding_b200 import engine as E
    rng = np.random.default_rng(23)
    K, N = 4096, 256
    gw, w = to_device(ops, rng.standard_normal((N, K), dtype=np.float32) / np.float32(64), dt)
    xs = [to_device(ops, rng.standard_normal((M, K), dtype=np.float32), dt) for M in (64, 64, 256)]
    s1, s2 = ops.CudaStream(0), ops.CudaStream(0)
    graphs, ys = [], []
    for gx, _ in xs[:2]:
        with Capture(ops, s1) as g:
            ys.append(ops.dev_linear_forward(gx, gw))
        graphs.append(g)
    assert len(E._captured) >= 2
    E.set_stream(0, s1.cuda_stream)
    try:
        for _ in range(10):
            graphs[0].launch(s1)
            graphs[1].launch(s2)
            big = ops.dev_linear_forward(xs[2][0], gw)
        ops.empty_cache()
        for g, s in zip(graphs, (s2, s1)):
            g.launch(s)
        ops.device_synchronize()
    finally:
        E.set_stream(0, None)
    for y, (_, x) in zip(ys + [big], xs):
        ref = x.astype(np.float64) @ w.astype(np.float64).T
        # 2 K operations of the sum, the output's rounding, 3xTF32 for fp32
        tol = 2.0 ** -22 * K * (np.abs(x).astype(np.float64) @ np.abs(w).T) + 2.0 ** -8 * (dt == "bf16") * np.abs(ref)
        assert (np.abs(to_host32(ops, y) - ref) <= tol).all()
    for g in graphs:
        g.destroy()
    E.release_workspaces(captured=True)
    assert device_error(0) == 0


@pytest.mark.parametrize("T", [3, 300])
def test_captured_moe_layer(gpu, ops, T):
    """A captured nn.MoE replayed after direct calls, uploads and allocations
    of the sizes of everything between its steps: the bits of the direct call,
    and nothing of what was allocated since is written."""
    from scaffolding_b200 import engine as E
    from scaffolding_b200 import nn
    rng = np.random.default_rng(T)
    dim, hidden, X, k = 64, 96, 12, 3
    bf = np_dtype("bf16")
    m = nn.MoE(dim, hidden, X, k, device=0, dtype=bf, rng=rng)
    gx, _ = to_device(ops, rng.standard_normal((T, dim), dtype=np.float32), "bf16")
    out = ops._alloc((T, dim), bf, 0)
    want = to_host32(ops, m(gx, gx))
    with Capture(ops) as g:
        m(gx, gx, out=out)
    X1 = X + 1
    guards = [ops.gputensor_from_numpy(np.full(n, 77, np.uint8))
              for n in (T * X * 4, T * k * 4, T * k * 4, X1 * 4, T * k * hidden * 2, T * k * dim * 2) for _ in range(3)]
    other, _ = to_device(ops, rng.standard_normal((T, dim), dtype=np.float32), "bf16")
    for _ in range(3):
        m(other)
        g.launch()
        g.stream.synchronize()
        assert np.array_equal(to_host32(ops, out), want)
    for t in guards:
        assert (ops.gputensor_to_numpy(t) == 77).all()
    g.destroy()
    E.release_workspaces(captured=True)
    assert device_error(0) == 0


def test_moe_layers_of_two_threads(gpu, ops):
    """Two layers in two threads on the default stream: the bits of the same
    calls made one by one."""
    from scaffolding_b200 import nn
    rng = np.random.default_rng(2)
    bf = np_dtype("bf16")
    jobs = []
    for T in (40, 700):
        m = nn.MoE(64, 96, 12, 3, device=0, dtype=bf, rng=rng)
        gx, _ = to_device(ops, rng.standard_normal((T, 64), dtype=np.float32), "bf16")
        jobs.append((m, gx, to_host32(ops, m(gx))))

    def loop(m, gx, want):
        for _ in range(60):
            assert np.array_equal(to_host32(ops, m(gx)), want)

    _in_threads(*[lambda j=j: loop(*j) for j in jobs])
    assert device_error(0) == 0
