"""4-bit linears on the device (-m gpu): sf_linear_w4, sf_quantize_w4 and
sf_dequantize_w4 behind dev_linear_w4 / dev_quantize_w4 / nn.Linear4, against
plain implementations in 64 bits.

Tolerances as in test_moe_gpu: the output's half step, and K + K / group fp32
operations of a sum of |x| scale (|q - 8| + |zero - 8|), which bounds every
term that a kernel forms whether it subtracts the zero before or after the sum."""
import numpy as np
import pytest

from oracle import oracle as O
from tests.gpu_util import device_error, np_dtype, to_device, to_host32

pytestmark = pytest.mark.gpu

U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}
TINY = {"bf16": 2.0 ** -134, "f16": 2.0 ** -25, "f32": 2.0 ** -149}


def plain_act(v, act):
    if act == "silu":
        return v / (1 + np.exp(-v))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + np.tanh(np.sqrt(2 / np.pi) * (v + 0.044715 * v ** 3)))
    return v


def weight(ops, rng, N, K, group, dt, zeros):
    """(W4Weight, W, bound on what enters the sums) with awkward values: zero
    points at both ends, a zero and a large scale."""
    G = -(-K // group)
    q = rng.integers(0, 16, (N, K)).astype(np.uint8)
    s = O.round_to((rng.random((N, G), dtype=np.float32) + np.float32(0.1)) / np.float32(8 * np.sqrt(K)), dt)
    s[0, 0] = 0.0
    s[-1, -1] = O.round_to(np.float32([3.0]), dt)[0]
    z = rng.integers(0, 16, (N, G)).astype(np.float32) if zeros else None
    w4 = ops.W4Weight.from_arrays(q, s.astype(np_dtype(dt)), z.astype(np_dtype(dt)) if zeros else None,
                                  group=group, device_id=0)
    col = np.arange(K) // group
    zc = z[:, col].astype(np.float64) if zeros else 8.0
    sc = s[:, col].astype(np.float64)
    return w4, sc * (q - zc), sc * (np.abs(q - 8.0) + np.abs(zc - 8.0))


def run(ops, rng, dt, M, N, K, group, zeros, act="none", bias=False, odt=None):
    odt = odt or dt
    w4, w, wabs = weight(ops, rng, N, K, group, dt, zeros)
    gx, x = to_device(ops, rng.standard_normal((M, K), dtype=np.float32), dt)
    gb = b = None
    if bias:
        gb, b = to_device(ops, rng.standard_normal(N, dtype=np.float32), dt)
    y = to_host32(ops, ops.dev_linear_w4(gx, w4, gb, act, out_dtype=np_dtype(odt))).astype(np.float64)
    v = x.astype(np.float64) @ w.T + (0 if b is None else b)
    off = (K + 2 * (K // group) + 8) * 2.0 ** -23 * (np.abs(x.astype(np.float64)) @ wabs.T) + 2.0 ** -24 * np.abs(v)
    ref = plain_act(v, act)
    tol = 1.13 * off + (0 if act == "none" else 2.0 ** -18 * (np.abs(ref) + np.abs(v)))
    tol = tol + U[odt] * (np.abs(ref) + tol) + TINY[odt]
    assert np.isfinite(y).all()
    worst = np.max(np.abs(y - ref) - tol)
    assert worst <= 0, f"{worst:.3e} beyond the bound, at most {np.max(np.abs(y - ref)):.3e} off"


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,N,K", [(1, 1, 8), (1, 64, 128), (1, 300, 1000), (2, 129, 384), (3, 16, 2048),
                                   (5, 100, 136), (8, 257, 512), (9, 96, 640), (17, 77, 1288), (33, 40, 256),
                                   (64, 130, 512), (64, 515, 1024)])
def test_linear(gpu, ops, dt, group, M, N, K):
    rng = np.random.default_rng(M * 1000 + N + K + group)
    for zeros in (False, True):
        run(ops, rng, dt, M, N, K, group, zeros)
    assert device_error(0) == 0


@pytest.mark.parametrize("K", [1, 31, 33, 127, 129, 1001])
@pytest.mark.parametrize("M", [1, 6, 40])
def test_linear_odd_widths(gpu, ops, K, M):
    """x rows that do not start on 16-byte boundaries, groups cut short."""
    rng = np.random.default_rng(K)
    run(ops, rng, "bf16", M, 50, K, 32, True, "silu", True)
    run(ops, rng, "f16", M, 50, K, 128, False)


@pytest.mark.parametrize("act", ["none", "silu", "gelu_tanh"])
@pytest.mark.parametrize("dt,odt", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32")])
def test_linear_bias_and_activation(gpu, ops, act, dt, odt):
    rng = np.random.default_rng(2)
    for M, N, K, group in [(1, 200, 512, 128), (7, 75, 264, 32), (48, 140, 384, 64)]:
        run(ops, rng, dt, M, N, K, group, True, act, True, odt)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_linear_wide(gpu, ops, dt):
    """Long rows and many of them: every CTA and split of the stream is used."""
    rng = np.random.default_rng(6)
    run(ops, rng, dt, 4, 3001, 4096, 128, True)
    run(ops, rng, dt, 64, 700, 4224, 64, False)


@pytest.mark.parametrize("dt,group,zeros", [("bf16", 128, False), ("f16", 32, True), ("bf16", 64, True)])
@pytest.mark.parametrize("M", [1, 5, 16])
def test_linear_streamed(gpu, ops, dt, group, zeros, M):
    """Sizes of the streaming kernel (4096 blocks of 128 x 128 and more, up to
    16 rows): a last tile of 8 rows, a last block cut short, clusters of four."""
    rng = np.random.default_rng(M)
    run(ops, rng, dt, M, 16392, 4064, group, zeros, "silu", True)
    assert device_error(0) == 0


@pytest.mark.parametrize("N,K", [(5000, 6880), (8900, 3840), (11008, 3104), (12700, 2720), (16392, 2080),
                                 (22000, 1568), (37888, 1024), (41000, 864)])
def test_linear_streamed_clusters(gpu, ops, N, K):
    """Rows and columns whose clusters are of each size from eight down to one;
    nine rows of x, whose sums the CTAs share out unevenly."""
    rng = np.random.default_rng(N)
    run(ops, rng, "bf16", 9, N, K, 128, True)
    run(ops, rng, "f16", 16, N, K, 32, False, "silu", True)
    assert device_error(0) == 0


@pytest.mark.parametrize("M", [1, 9])
def test_linear_large_values(gpu, ops, M):
    """x at the edge of fp16's range: group sums stay in fp32."""
    rng = np.random.default_rng(1)
    w4, w, _ = weight(ops, rng, 64, 256, 64, "f16", True)
    x = np.full((M, 256), 60000, np.float32)
    x[:, ::2] = -60000
    gx, x = to_device(ops, x, "f16")
    y = to_host32(ops, ops.dev_linear_w4(gx, w4, out_dtype=np.float32)).astype(np.float64)
    ref = x.astype(np.float64) @ w.T
    np.testing.assert_allclose(y, ref, rtol=0, atol=float(2.0 ** -14 * (np.abs(x) @ np.abs(w).T).max()))


def test_linear_infinities_stay_in_their_row(gpu, ops):
    rng = np.random.default_rng(12)
    w4, w, _ = weight(ops, rng, 40, 256, 128, "bf16", False)
    x = rng.standard_normal((6, 256)).astype(np.float32)
    x[2, 7], x[4, 9] = np.inf, np.nan
    gx, x = to_device(ops, x, "bf16")
    y = to_host32(ops, ops.dev_linear_w4(gx, w4))
    assert np.isnan(y[4]).all() and not np.isfinite(y[2]).any()
    assert np.isfinite(y[[0, 1, 3, 5]]).all()


def test_many_rows_dequantise(gpu, ops):
    """More than 64 rows: the product of the rounded weights."""
    rng = np.random.default_rng(7)
    w4, w, _ = weight(ops, rng, 130, 512, 64, "bf16", True)
    gw = ops.dev_dequantize_w4(w4)
    assert np.array_equal(to_host32(ops, gw), O.round_to(w.astype(np.float32), "bf16"))
    gx, x = to_device(ops, rng.standard_normal((2, 100, 512), dtype=np.float32), "bf16")
    y = ops.dev_linear_w4(gx, w4, activation="silu")
    assert y.shape == (2, 100, 130)
    z = ops.dev_linear_forward(gx, gw, activation="silu")
    assert np.array_equal(to_host32(ops, y), to_host32(ops, z))


def test_many_rows_captured(gpu, ops):
    """In a capture more than 64 rows run 64 at a time, with no memory of the
    call's own in the graph; the replay gives the same bits as those calls."""
    import ctypes as C

    from scaffolding_b200 import engine as E
    from scaffolding_b200._lib import check, lib
    rng = np.random.default_rng(17)
    w4, w, _ = weight(ops, rng, 100, 256, 64, "bf16", True)
    gx, x = to_device(ops, rng.standard_normal((150, 256), dtype=np.float32), "bf16")
    out = ops._alloc((150, 100), np_dtype("bf16"), 0)
    parts = []
    for m0 in (0, 64, 128):
        px, _ = to_device(ops, x[m0:m0 + 64], "bf16")
        parts.append(to_host32(ops, ops.dev_linear_w4(px, w4, activation="silu")))
    s = ops.CudaStream(0)
    E.set_stream(0, s.cuda_stream)
    try:
        check(lib.sf_graph_begin(C.c_void_p(s.cuda_stream)), "begin")
        assert E.stream_capturing(s.cuda_stream)
        ops.dev_linear_w4(gx, w4, activation="silu", out=out)
        exe = C.c_void_p()
        check(lib.sf_graph_end(C.c_void_p(s.cuda_stream), C.byref(exe)), "end")
    finally:
        E.set_stream(0, None)
    assert not E.stream_capturing(s.cuda_stream) and not E.stream_capturing(None)
    for _ in range(2):
        check(lib.sf_graph_launch(exe, C.c_void_p(s.cuda_stream)), "launch")
    s.synchronize()
    assert np.array_equal(to_host32(ops, out), np.concatenate(parts))
    check(lib.sf_graph_destroy(exe), "destroy")


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("N,K", [(1, 1), (5, 200), (64, 384)])
def test_quantise(gpu, ops, dt, group, N, K):
    """The stored values are those of the definition, bit for bit where the
    quotient is not within fp32 rounding of a tie, and no weight is off by
    more than half a step (and the rounding of the scale's type)."""
    rng = np.random.default_rng(N + K)
    gw, w = to_device(ops, rng.standard_normal((N, K), dtype=np.float32), dt)
    sdt = "bf16" if dt == "f32" else dt
    for zeros in (False, True):
        w4 = ops.dev_quantize_w4(gw, group, zeros, np_dtype(sdt))
        back = to_host32(ops, ops.dev_dequantize_w4(w4, np.float32)).astype(np.float64)
        s = to_host32(ops, w4.scales).astype(np.float64).T
        G = s.shape[1]
        for g in range(G):
            cols = slice(g * group, min(K, (g + 1) * group))
            lo, hi = np.minimum(w[:, cols].min(1), 0), np.maximum(w[:, cols].max(1), 0)
            want = (hi - lo) / 15 if zeros else np.maximum(hi, -lo) / 7
            np.testing.assert_allclose(s[:, g], want, rtol=U[sdt] + 2.0 ** -22)
            # the rounded scale may cut the range short by 15 roundings of it
            step = s[:, g, None]
            assert (np.abs(back[:, cols] - w[:, cols]) <= step * (0.5 + 2.0 ** -20 + 15 * U[sdt] * 2)).all()


def test_linear4_module(gpu, ops):
    from scaffolding_b200 import nn
    rng = np.random.default_rng(3)
    lin = nn.Linear(256, 96, device=0, rng=rng)
    m = nn.Linear4.from_linear(lin, group=64, zeros=True, dtype=np_dtype("bf16"))
    gx, x = to_device(ops, rng.standard_normal((3, 2, 256), dtype=np.float32), "bf16")
    y = to_host32(ops, m(gx, "silu")).astype(np.float64)
    w = to_host32(ops, ops.dev_dequantize_w4(m.weight, np.float32)).astype(np.float64)
    v = x.astype(np.float64) @ w.T + to_host32(ops, m.bias)
    tol = 2.0 ** -8 * np.abs(plain_act(v, "silu")) + 300 * 2.0 ** -22 * (np.abs(x) @ np.abs(w).T + 1)
    assert (np.abs(y - plain_act(v, "silu")) <= tol).all()
