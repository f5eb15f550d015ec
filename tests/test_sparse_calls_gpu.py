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


# ───────────── sizes at which rings, clusters and accumulators come round ─────────────
# The expected launch is worked out from the sizes by the rules of the dispatch: rows
# per group choose the tile, tiles and k-blocks the cluster.

SMS = 148


def grouped_plan(X, M, K, N, gate):
    """(rows of a tile, CTAs that share one, most tiles, k-blocks)."""
    few = M <= 16 * X
    bn = (32 if gate else 64) if few else (128 if gate else 256)
    most, kb = (M // bn + min(X, M)) * -(-N // 128), -(-K // 64)
    splits = 1
    while few and splits < 8 and kb >= 8 * splits and most * splits * 2 <= (
            SMS if splits == 1 else SMS * 3 // 4 if splits == 2 else SMS // 3):
        splits *= 2
    return bn, splits, most, kb


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("X,M,K,N,act,gather,splits", [
    (8, 2, 512, 300, "none", 1, 2),        # eight k-blocks, three weight blocks
    (2, 5, 520, 2000, "silu", None, 2),    # 9 = 5 + 4 k-blocks, the last of 8 columns
    (1, 1, 1024, 128, "none", None, 4),    # one tile
    (3, 40, 1096, 500, "gelu_tanh", 7, 4), # 18 k-blocks in shares of 5: 3 for the last
    (4, 9, 2048, 100, "none", 9, 8),
    (1, 16, 2112, 500, "silu", None, 8),   # 33 k-blocks in shares of 5: none for the last rank
    (2, 31, 4104, 260, "none", 3, 8),      # 65 in shares of 9
    (1, 1, 512, 1000, "silu_gate", 1, 2),
    (2, 20, 1032, 300, "silu_gate", None, 4),
    (1, 13, 2112, 140, "silu_gate", 13, 8),
    (2, 30, 2104, 20, "silu_gate", 8, 8),
])
def test_grouped_clusters(gpu, ops, dt, X, M, K, N, act, gather, splits):
    """A tile's k-blocks shared by two, four and eight CTAs: uneven shares, a
    rank without any, K no multiple of 64."""
    from tests.test_moe_gpu import assert_within, run_grouped
    assert grouped_plan(X, M, K, N, act == "silu_gate")[1] == splits
    rng = np.random.default_rng(K + N)
    for bias in (False, True):
        assert_within(*run_grouped(ops, rng, dt, X, M, K, N, act, bias, gather), f"{X} {M} {K} {N} {act}")
    assert device_error(0) == 0


@pytest.mark.parametrize("X,M,K,N,act,gather,bn", [
    (64, 256, 640, 1000, "silu_gate", 40, 32),     # narrow gated: 10 k-blocks in a ring of five
    (64, 700, 576, 1100, "none", None, 64),        # narrow: 9 in a ring of eight
    (64, 1000, 704, 1100, "gelu_tanh", 300, 64),
    (3, 900, 712, 4000, "silu_gate", 100, 128),    # gated: 12 in a ring of four
    (2, 700, 328, 9000, "silu_gate", None, 128),
    (3, 2000, 584, 4000, "silu", None, 256),       # wide
    (2, 1500, 456, 5000, "gelu_tanh", 80, 256),
])
def test_grouped_many_tiles(gpu, ops, X, M, K, N, act, gather, bn):
    """More tiles than SMs, so that a CTA runs several: the accumulators take
    turns, the ring wraps within and across tiles, an epilogue overlaps the next
    tile's products."""
    from tests.test_moe_gpu import assert_within, run_grouped
    tile, splits, most, kb = grouped_plan(X, M, K, N, act == "silu_gate")
    real = (M // tile) * -(-N // 128)
    assert (tile, splits) == (bn, 1) and max(real, X // 2 * -(-N // 128)) > 1.2 * SMS and kb > 4
    rng = np.random.default_rng(M + K)
    for dt in ("bf16", "f16"):
        assert_within(*run_grouped(ops, rng, dt, X, M, K, N, act, True, gather), f"{X} {M} {K} {N} {act} {dt}")
    assert device_error(0) == 0


def test_grouped_long_group_in_narrow_tiles(gpu, ops):
    """Every row in one of many groups: the mean says narrow tiles, the group
    is cut into many of them."""
    from tests.test_moe_gpu import assert_within, run_grouped
    rng = np.random.default_rng(31)
    for act, N in (("none", 1200), ("silu_gate", 600)):
        offsets = np.zeros(65, np.int32)
        offsets[38:] = 997
        assert_within(*run_grouped(ops, rng, "bf16", 64, 997, 520, N, act, True, 50, offsets=offsets))
    assert device_error(0) == 0


_FIRST_IN_CAPTURE = """
import ctypes as C, numpy as np, sys
from scaffolding_b200 import _cuda_ops as ops, engine as E
bf = E.bfloat16
rng = np.random.default_rng(0)
N, K, M = 16392, 4064, {M}
q = rng.integers(0, 16, (N, K)).astype(np.uint8)
s = np.full((N, 32), 2.0 ** -8, np.float32).astype(bf)
w4 = ops.W4Weight.from_arrays(q, s, None, 128, 0)
x = rng.integers(-3, 4, (M, K)).astype(np.float32)
gx = ops.gputensor_from_numpy(x.astype(bf), 0)
out = ops._alloc((M, N), np.float32, 0)
st = ops.CudaStream(0)
E.set_stream(0, st.cuda_stream)
E.check(E.lib.sf_graph_begin(C.c_void_p(st.cuda_stream)), "begin")
ops.dev_linear_w4(gx, w4, out=out)
exe = C.c_void_p()
E.check(E.lib.sf_graph_end(C.c_void_p(st.cuda_stream), C.byref(exe)), "end")
for _ in range(2):
    E.check(E.lib.sf_graph_launch(exe, C.c_void_p(st.cuda_stream)), "launch")
st.synchronize()
y = ops.gputensor_to_numpy(out)
# whole numbers below 2^24 over a power of two: every sum is exact
ref = (x.astype(np.float64) @ (q.astype(np.float64) - 8).T) / 256
assert np.array_equal(y, ref), np.abs(y - ref).max()
assert E.device_error_status(0) == 0
print("exact")
"""


@pytest.mark.parametrize("M", [1, 16, 40])
def test_first_call_of_a_process_in_a_capture(gpu, M):
    """The first 4-bit linear of a process is captured: the opt-in to shared
    memory and the question of how many clusters fit come inside the capture."""
    import subprocess
    import sys

    from tests.conftest import ROOT
    r = subprocess.run([sys.executable, "-c", _FIRST_IN_CAPTURE.format(M=M)], cwd=ROOT, capture_output=True,
                       text=True, timeout=300)
    assert r.returncode == 0 and "exact" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]


@pytest.mark.parametrize("dt,sdt", [("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("N,K,group", [(33, 300, 32), (64, 512, 128), (7, 200, 64)])
def test_quantised_values(gpu, ops, dt, sdt, zeros, N, K, group):
    """Scale, zero point and every 4-bit value of the stored weight: those of
    the definition, from the stored scale on.  Quotients are divided in fp32 on
    both sides; where one lies within 2^-20 of a tie either neighbour is right
    (fp32 rounding of a quotient below 16: 2^-21)."""
    rng = np.random.default_rng(N + K)
    w = rng.standard_normal((N, K), dtype=np.float32)
    w[0, :group] = 0
    w[1, :group] = np.abs(w[1, :group])   # a range without negative values
    w[2, :group] = -np.abs(w[2, :group])
    gw, w = to_device(ops, w, dt)
    w4 = ops.dev_quantize_w4(gw, group, zeros, np_dtype(sdt))
    words = ops.gputensor_to_numpy(w4.packed)
    q = np.zeros((N, words.shape[1] * 8), np.int64)
    for t in range(4):
        for j in range(4):
            for i, c in enumerate((0, 2, 4, 6, 1, 3, 5, 7)):
                q[:, 32 * j + 8 * t + c::128] = (words[:, 4 * t + j::16] >> np.uint32(4 * i)) & 15
    s = to_host32(ops, w4.scales).astype(np.float64).T
    z = to_host32(ops, w4.zeros).T if zeros else np.full(s.shape, 8.0)
    for g in range(s.shape[1]):
        cols = slice(g * group, min(K, (g + 1) * group))
        v = w[:, cols].astype(np.float64)
        lo, hi = np.minimum(v.min(1), 0), np.maximum(v.max(1), 0)
        exact = (hi - lo) / 15 if zeros else np.maximum(hi, -lo) / 7
        # one rounding of the difference, one of the quotient, one to the scale's type
        step = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}[sdt]
        assert (np.abs(s[:, g] - exact) <= (step + 2.0 ** -22) * exact + 2.0 ** -25).all()
        live = s[:, g] > 0
        some = np.where(live, s[:, g], 1.0)
        if zeros:
            ideal = np.where(live, -lo / some, 0.0)
            clear = np.abs(ideal - np.floor(ideal) - 0.5) > 2.0 ** -20
            assert np.array_equal(z[clear, g], np.clip(np.rint(ideal), 0, 15)[clear])
            assert (np.abs(z[:, g] - ideal) <= 0.5 + 2.0 ** -20).all() and (z[:, g] == np.rint(z[:, g])).all()
        ideal = np.where(live[:, None], v / some[:, None], 0.0)
        clear = np.abs(ideal - np.floor(ideal) - 0.5) > 2.0 ** -20
        want = np.clip(np.rint(ideal) + z[:, g, None], 0, 15)
        assert np.array_equal(q[:, cols][clear], want[clear])
        assert (np.abs(q[:, cols] - want) <= 1).all()
        assert (q[~live][:, cols] == z[~live, g, None]).all()


def test_first_call_of_a_thread(gpu, ops):
    """A host thread whose first use of the device is a launch into kept
    buffers: the driver has no context on it yet."""
    from scaffolding_b200._lib import check, lib
    rng = np.random.default_rng(3)
    x = {M: to_device(ops, rng.standard_normal((M, 256), dtype=np.float32), "bf16")[0] for M in (4, 40)}
    gw, _ = to_device(ops, rng.standard_normal((128, 256), dtype=np.float32), "bf16")
    g3 = ops.dev_reshape(gw, (1, 128, 256))
    w4 = ops.dev_quantize_w4(gw, 64)
    sw, _ = to_device(ops, rng.standard_normal((16384, 4096), dtype=np.float32), "bf16")
    sx, _ = to_device(ops, rng.standard_normal((2, 4096), dtype=np.float32), "bf16")
    big = ops.dev_quantize_w4(sw, 128)
    off = ops.gputensor_from_numpy(np.array([0, 40], np.int32))

    def noalloc(out):
        check(lib.sf_linear_skinny_noalloc(40, 128, 256, x[40].ptr, 256, gw.ptr, 256, None, 0, out.ptr, 128, 2, 2,
                                           0, None), "sf_linear_skinny_noalloc")

    calls = [((40, 128), lambda out: ops.dev_grouped_linear(x[40], g3, off, out=out)),
             ((40, 128), lambda out: ops.dev_linear_w4(x[40], w4, out=out)),
             ((4, 128), lambda out: ops.dev_linear_w4(x[4], w4, out=out)),
             ((2, 16384), lambda out: ops.dev_linear_w4(sx, big, out=out)),
             ((40, 128), lambda out: ops.dev_linear_forward(x[40], gw, out=out)),
             ((40, 128), noalloc)]
    for shape, call in calls:
        want, got = (ops.gputensor_from_numpy(np.full(shape, v).astype(np_dtype("bf16"))) for v in (1, 2))
        call(want)
        _in_threads(lambda: call(got))
        assert np.array_equal(to_host32(ops, got), to_host32(ops, want))
    assert device_error(0) == 0


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_quantised_non_finite_weights(gpu, ops, zeros, bad):
    """A NaN or infinite weight makes its group NaN, and the outputs of its row,
    as it does in a plain linear; it is not turned into a number."""
    rng = np.random.default_rng(6)
    w = rng.standard_normal((20, 256), dtype=np.float32)
    w[3, 70] = bad
    w[9, 128:192] = bad
    gw, w = to_device(ops, w, "bf16")
    w4 = ops.dev_quantize_w4(gw, 64, zeros)
    back = to_host32(ops, ops.dev_dequantize_w4(w4))
    nan = np.zeros(w.shape, bool)
    nan[3, 64:128] = nan[9, 128:192] = True
    assert np.array_equal(np.isnan(back), nan) and np.isfinite(back[~nan]).all()
    for M in (1, 40):
        gx, _ = to_device(ops, rng.standard_normal((M, 256), dtype=np.float32), "bf16")
        y = to_host32(ops, ops.dev_linear_w4(gx, w4))
        assert np.array_equal(np.isnan(y), np.broadcast_to(nan.any(1), y.shape))
    assert device_error(0) == 0


@pytest.mark.parametrize("act", ["none", "silu_gate"])
def test_captured_gather_of_a_long_batch(gpu, ops, act):
    """A captured batch gathers its rows as it reads them, a direct one copies
    them first: the same bits."""
    rng = np.random.default_rng(41)
    X, M, K, N, T = 5, 2600, 264, 1030, 700
    wide = 2 * N if act == "silu_gate" else N
    gx, _ = to_device(ops, rng.standard_normal((T, K), dtype=np.float32), "bf16")
    gw, _ = to_device(ops, rng.standard_normal((X, wide, K), dtype=np.float32) / np.float32(16), "bf16")
    rows = ops.gputensor_from_numpy(rng.integers(-1, T + 1, M).astype(np.int32))
    off = ops.gputensor_from_numpy(np.array([0, 700, 700, 1500, 2590, M], np.int32))
    want = to_host32(ops, ops.dev_grouped_linear(gx, gw, off, activation=act, rows=rows))
    out = ops._alloc((M, N), np_dtype("bf16"), 0)
    with Capture(ops) as g:
        ops.dev_grouped_linear(gx, gw, off, activation=act, rows=rows, out=out)
    for _ in range(2):
        g.launch()
    g.stream.synchronize()
    assert np.array_equal(to_host32(ops, out), want)
    g.destroy()
    assert device_error(0) == 0


@pytest.mark.parametrize("M", [300, 70000])
def test_grouped_most_groups(gpu, ops, M):
    """4096 groups, most of them empty or of a few rows, in narrow and in wide
    tiles; their bounds take the most shared memory there can be."""
    from tests.test_moe_gpu import assert_within, run_grouped
    rng = np.random.default_rng(M)
    counts = np.bincount(np.minimum(rng.geometric(1 / 300, M) - 1, 4095), minlength=4096)
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    for act in ("none", "silu_gate"):
        for gather in (None, 90):
            assert_within(*run_grouped(ops, rng, "bf16", 4096, M, 72, 20, act, True, gather, offsets=offsets))
    assert device_error(0) == 0


def test_combine_without_rows(gpu, ops):
    """No expert rows at all: the residual alone, or zeros."""
    rng = np.random.default_rng(0)
    gr, res = to_device(ops, rng.standard_normal((6, 40), dtype=np.float32), "bf16")
    y = ops._alloc((0, 40), np_dtype("bf16"), 0)
    s = ops.gputensor_from_numpy(np.array([[0, -1]] * 6, np.int32))
    w = ops.gputensor_from_numpy(np.ones((6, 2), np.float32))
    assert np.array_equal(to_host32(ops, ops.dev_moe_combine(y, s, w, gr)), res)
    assert not to_host32(ops, ops.dev_moe_combine(y, s, w)).any()
