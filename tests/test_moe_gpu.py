"""Routed layers on the device (-m gpu): sf_moe_route, sf_gemm_grouped and
sf_moe_combine behind dev_moe_route / dev_grouped_linear / dev_moe_combine and
nn.MoE, against plain implementations in 64 bits.

Tolerances.  u is the largest relative rounding of the output type (half a
step: 2^-8 bf16, 2^-11 fp16, 2^-24 fp32).  A sum of n products in fp32 is off
by at most n * 2^-23 * sum |products| (2^-24 for each IEEE addition; twice
that for the tensor core, which truncates where it aligns the addends)."""
import ctypes as C

import numpy as np
import pytest

from tests.gpu_util import device_error, np_dtype, to_device, to_host32

pytestmark = pytest.mark.gpu

U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}
TINY = {"bf16": 2.0 ** -134, "f16": 2.0 ** -25, "f32": 2.0 ** -149}  # half the least subnormal


# ───────────────────────────── router ─────────────────────────────

def plain_route(z, k, renormalize):
    """experts, weights, offsets, rows, slots from fp32 logits, in 64 bits."""
    z = np.where(np.isnan(z), -np.inf, z.astype(np.float64))
    T, X = z.shape
    experts = np.argsort(-z, axis=1, kind="stable")[:, :k]
    picked = np.take_along_axis(z, experts, 1)
    weights = np.zeros((T, k))
    for t in range(T):
        top = picked[t, 0]
        over = picked[t] if renormalize else z[t]
        if top == -np.inf:
            continue
        e = lambda v: np.exp(np.subtract(v, top, out=np.zeros_like(v), where=v != top))  # noqa: E731
        weights[t] = e(picked[t]) / e(over).sum()
    flat = experts.reshape(-1)
    order = np.argsort(flat, kind="stable")
    slots = np.empty(T * k, np.int64)
    slots[order] = np.arange(T * k)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat, minlength=X))])
    return experts, weights, offsets, order // k, slots.reshape(T, k)


def check_route(ops, r, z, k, renormalize):
    get = ops.gputensor_to_numpy
    experts, weights, offsets, rows, slots = plain_route(z, k, renormalize)
    np.testing.assert_array_equal(get(r.experts), experts)
    np.testing.assert_array_equal(get(r.offsets), offsets)
    np.testing.assert_array_equal(get(r.rows), rows)
    np.testing.assert_array_equal(get(r.slots), slots)
    # exp(z - top): the difference is rounded (2^-24 |z - top|), expf is good
    # to 2 ulp; the sum takes at most 37 roundings (32 in a lane, 5 across),
    # the quotient one; numerator and sum both carry the first two.
    finite = z[np.isfinite(z)]
    spread = float(finite.max() - finite.min()) if finite.size else 0.0
    tol = 2.0 ** -24 * (2 * min(spread, 104.0) + 48)
    np.testing.assert_allclose(get(r.weights), weights, rtol=tol, atol=2.0 ** -126)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,X,k", [(1, 8, 2), (1, 1, 1), (7, 3, 3), (64, 64, 4), (255, 31, 5),
                                   (256, 128, 8), (257, 33, 1), (1000, 256, 8), (300, 1000, 32), (256, 1024, 32), (200, 300, 16),
                                   (17776, 60, 2), (40000, 16, 4)])
def test_route(gpu, ops, dt, T, X, k):
    rng = np.random.default_rng(T + X)
    gz, z = to_device(ops, rng.standard_normal((T, X), dtype=np.float32) * np.float32(2), dt)
    for renorm in (True, False):
        check_route(ops, ops.dev_moe_route(gz, k, renormalize=renorm), z, k, renorm)
    assert device_error(0) == 0


@pytest.mark.parametrize("T", [5, 600])
def test_route_ties_infinities_nan(gpu, ops, T):
    """Equal logits go to the lowest expert (+0 and -0 are equal), a masked
    (-inf) or NaN expert is chosen last with weight 0, a row with nothing
    but those has weights 0, +inf takes everything."""
    rng = np.random.default_rng(0)
    z = rng.integers(-2, 3, (T, 40)).astype(np.float32)
    z[0] = 0.0
    z[0, ::2] = -0.0
    z[1] = -np.inf
    z[1, 39] = 1.0
    z[2] = -np.inf
    z[2, 3] = np.nan
    z[3, 5:7] = np.inf
    z[4] = np.finfo(np.float32).min
    z[4, 20] = np.nan
    gz = ops.gputensor_from_numpy(z)
    for renorm in (True, False):
        check_route(ops, ops.dev_moe_route(gz, 4, renormalize=renorm), z, 4, renorm)


def test_route_all_to_one_expert_and_no_tokens(gpu, ops):
    z = np.zeros((3000, 20), np.float32)
    z[:, 7] = 1
    gz = ops.gputensor_from_numpy(z)
    check_route(ops, ops.dev_moe_route(gz, 1), z, 1, True)
    empty = ops.GpuTensor(ops.CudaBuffer(0, 0, 0, False), (0, 20), np.float32, 0)
    r = ops.dev_moe_route(empty, 2)
    np.testing.assert_array_equal(ops.gputensor_to_numpy(r.offsets), np.zeros(21, np.int32))


def test_route_into_kept_buffers(gpu, ops):
    """out= is written in place, its scratch grows with a longer batch of the
    same shape family, and the same inputs give the same bits."""
    rng = np.random.default_rng(3)
    z = rng.standard_normal((900, 24), dtype=np.float32)
    gz = ops.gputensor_from_numpy(z)
    r = ops.dev_moe_route(gz, 3)
    ptrs = [getattr(r, n).ptr for n in ("experts", "weights", "offsets", "rows", "slots")]
    first = ops.gputensor_to_numpy(r.weights).copy()
    assert ops.dev_moe_route(gz, 3, out=r) is r
    assert ptrs == [getattr(r, n).ptr for n in ("experts", "weights", "offsets", "rows", "slots")]
    assert np.array_equal(first, ops.gputensor_to_numpy(r.weights))
    check_route(ops, r, z, 3, True)


# ───────────────────────────── grouped products ─────────────────────────────

def silu(v):
    return v / (1 + np.exp(-v))


def plain_act(v, act):
    if act == "silu":
        return silu(v)
    if act == "gelu_tanh":
        return 0.5 * v * (1 + np.tanh(np.sqrt(2 / np.pi) * (v + 0.044715 * v ** 3)))
    return v


def plain_grouped(x, w, offsets, bias, act, rows, odt):
    """(result, allowed error) in 64 bits; rows in no group are NaN."""
    M = len(rows) if rows is not None else len(x)
    x, w = x.astype(np.float64), w.astype(np.float64)
    wide = w.shape[1]
    N = wide // 2 if act == "silu_gate" else wide
    y = np.full((M, N), np.nan)
    tol = np.zeros((M, N))
    K = x.shape[1]
    for g in range(len(w)):
        lo, hi = int(offsets[g]), int(offsets[g + 1])
        if hi == lo:
            continue
        src = x[lo:hi] if rows is None else np.stack(
            [x[r] if 0 <= r < len(x) else np.zeros(K) for r in rows[lo:hi]])
        v = src @ w[g].T
        off = (K + 1) * 2.0 ** -23 * (np.abs(src) @ np.abs(w[g]).T)
        if bias is not None:
            v = v + bias[g].astype(np.float64)
            off += 2.0 ** -24 * np.abs(v)
        if act == "silu_gate":
            gt, up = v[:, :N], v[:, N:]
            y[lo:hi] = silu(gt) * up
            tol[lo:hi] = 1.1 * off[:, :N] * (np.abs(up) + off[:, N:]) + np.abs(silu(gt)) * off[:, N:]
        else:
            y[lo:hi] = plain_act(v, act)
            tol[lo:hi] = 1.13 * off  # the largest slope of SiLU and GELU
        if act != "none":
            # expf / tanhf (fp32 results) within a few units of 2^-23; the
            # fast forms of 16-bit results within 2^-18, argument included
            rel = 2.0 ** -20 if odt == "f32" else 2.0 ** -18
            tol[lo:hi] += rel * (np.abs(y[lo:hi]) + np.abs(v[:, :N]) *
                                 (np.abs(v[:, N:]) if act == "silu_gate" else 1.0))
    return y, tol + U[odt] * (np.abs(y) + tol) + TINY[odt]


def groups_of(rng, M, X, empty=()):
    p = rng.random(X) + 0.05
    p[list(empty)] = 0
    counts = rng.multinomial(M, p / p.sum())
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


def run_grouped(ops, rng, dt, X, M, K, N, act="none", bias=False, gather=None, offsets=None,
                rows=None, odt=None):
    odt = odt or dt
    wide = 2 * N if act == "silu_gate" else N
    gx, x = to_device(ops, rng.standard_normal((gather or M, K), dtype=np.float32), dt)
    gw, w = to_device(ops, rng.uniform(-1, 1, (X, wide, K)).astype(np.float32) * np.float32(1 / np.sqrt(K)), dt)
    gb = b = None
    if bias:
        gb, b = to_device(ops, rng.standard_normal((X, wide), dtype=np.float32) * np.float32(0.5), dt)
    if offsets is None:
        offsets = groups_of(rng, M, X, empty=(0, X - 1) if X > 3 else ())
    if gather and rows is None:
        rows = rng.integers(0, gather, M).astype(np.int32)
    gr = ops.gputensor_from_numpy(rows) if rows is not None else None
    y = ops.dev_grouped_linear(gx, gw, ops.gputensor_from_numpy(offsets), gb, act, rows=gr,
                               out_dtype=np_dtype(odt))
    ref, tol = plain_grouped(x, w, offsets, b, act, rows, odt)
    return to_host32(ops, y).astype(np.float64), ref, tol


def assert_within(y, ref, tol, what=""):
    assert np.isfinite(y).all(), f"{what}: non-finite output"
    worst = np.max(np.abs(y - ref) - tol)
    assert worst <= 0, f"{what}: {worst:.3e} beyond the bound, at most {np.max(np.abs(y - ref)):.3e} off"


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("X,M,K,N", [(1, 1, 8, 1), (4, 1, 64, 128), (8, 3, 128, 130), (5, 40, 72, 100),
                                     (3, 257, 200, 129), (16, 333, 136, 257), (2, 700, 328, 384),
                                     (64, 200, 64, 96), (300, 900, 64, 40)])
def test_grouped(gpu, ops, dt, X, M, K, N):
    rng = np.random.default_rng(X * 1000 + M)
    for gather in (None, max(1, M // 2)):
        assert_within(*run_grouped(ops, rng, dt, X, M, K, N, gather=gather), f"{dt} {X} {M} {K} {N} {gather}")
    assert device_error(0) == 0


@pytest.mark.parametrize("act", ["silu", "gelu_tanh", "silu_gate"])
@pytest.mark.parametrize("dt,odt", [("bf16", "bf16"), ("f16", "f32"), ("f32", "f32")])
def test_grouped_bias_and_activation(gpu, ops, act, dt, odt):
    rng = np.random.default_rng(5)
    for X, M, K, N, gather in [(6, 50, 64, 200, 20), (4, 300, 192, 67, None), (9, 20, 136, 258, 5)]:
        assert_within(*run_grouped(ops, rng, dt, X, M, K, N, act, True, gather, odt=odt),
                      f"{act} {dt}->{odt} {X} {M}")
    assert device_error(0) == 0


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("K", [1, 7, 33, 65, 100])
def test_grouped_widths_tma_cannot_describe(gpu, ops, dt, K):
    rng = np.random.default_rng(K)
    assert_within(*run_grouped(ops, rng, dt, 5, 130, K, 70, "silu_gate", True, 60), f"K={K}")


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_grouped_every_row_in_one_group_and_long_groups(gpu, ops, dt):
    rng = np.random.default_rng(9)
    for X, M, at in [(5, 600, 0), (5, 600, 4), (3, 1025, 1)]:
        offsets = np.zeros(X + 1, np.int32)
        offsets[at + 1:] = M
        assert_within(*run_grouped(ops, rng, dt, X, M, 256, 320, "gelu_tanh", True, offsets=offsets))


@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_grouped_rows_gathered_first(gpu, ops, dt):
    """Long batches copy their rows into grouped order first (outside a
    capture): the same bits as the rows given in that order, zeros for an
    index outside x, a width that ends inside a 16-byte vector."""
    from scaffolding_b200 import engine as E
    rng = np.random.default_rng(21)
    X, M, K, N, T = 6, 2500, 200, 1030, 900
    gx, x = to_device(ops, rng.standard_normal((T, K), dtype=np.float32), dt)
    gw, w = to_device(ops, rng.uniform(-1, 1, (X, N, K)).astype(np.float32) / np.float32(14), dt)
    rows = rng.integers(0, T, M).astype(np.int32)
    rows[[0, 77, 2499]] = [-1, T, 2 ** 31 - 1]
    offsets = groups_of(rng, M, X, empty=(2,))
    need = C.c_size_t()
    assert E.lib.sf_gemm_grouped_workspace_size(X, M, N, K, E.dtype_code(np_dtype(dt)), None, C.byref(need)) == 0
    assert need.value == M * K * 2
    go = ops.gputensor_from_numpy(offsets)
    y = to_host32(ops, ops.dev_grouped_linear(gx, gw, go, rows=ops.gputensor_from_numpy(rows)))
    ref, tol = plain_grouped(x, w, offsets, None, "none", rows, dt)
    assert_within(y.astype(np.float64), ref, tol)
    dense = np.stack([x[r] if 0 <= r < T else np.zeros(K, np.float32) for r in rows])
    gd, _ = to_device(ops, dense, dt)
    assert np.array_equal(y, to_host32(ops, ops.dev_grouped_linear(gd, gw, go)))
    assert device_error(0) == 0


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_grouped_rows_outside(gpu, ops, dt):
    """Rows in no group keep what they held, indices outside x read zeros and
    offsets outside 0..M are clamped."""
    rng = np.random.default_rng(4)
    X, M, K, N = 4, 200, 64, 96
    gx, x = to_device(ops, rng.standard_normal((50, K), dtype=np.float32), dt)
    gw, w = to_device(ops, rng.standard_normal((X, N, K), dtype=np.float32), dt)
    rows = rng.integers(0, 50, M).astype(np.int32)
    rows[[3, 60, 100, 130]] = [-1, 50, 2 ** 31 - 1, -2 ** 31]
    held = np.full((M, N), 7, np.float32)
    for raw, offsets in ([[10, 30, 30, 150, 180], [10, 30, 30, 150, 180]],
                         [[-5, 20, 70, 90, 5000], [0, 20, 70, 90, 200]]):
        out = ops.gputensor_from_numpy(held.astype(np_dtype(dt)))
        ops.dev_grouped_linear(gx, gw, ops.gputensor_from_numpy(np.array(raw, np.int32)),
                               rows=ops.gputensor_from_numpy(rows), out=out)
        y = to_host32(ops, out).astype(np.float64)
        ref, tol = plain_grouped(x, w, offsets, None, "none", rows, dt)
        inside = ~np.isnan(ref[:, 0])
        assert_within(y[inside], ref[inside], tol[inside])
        assert np.array_equal(y[~inside], held[~inside])
    assert device_error(0) == 0


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_grouped_strides_of_the_c_abi(gpu, ops, dt):
    """Leading dimensions and group strides wider than the matrices; what lies
    between the rows of C is not written."""
    from scaffolding_b200._lib import check, lib
    rng = np.random.default_rng(8)
    X, M, K, N, lda, ldb, ldc = 3, 150, 72, 100, 88, 80, 133
    bs = N * ldb + 160
    es = 4 if dt == "f32" else 2
    gx, x = to_device(ops, rng.standard_normal((M, lda), dtype=np.float32), dt)
    gw, w = to_device(ops, rng.standard_normal((X, bs), dtype=np.float32), dt)
    gb, b = to_device(ops, rng.standard_normal((X, N + 9), dtype=np.float32), dt)
    offsets = np.array([0, 20, 120, 150], np.int32)
    go = ops.gputensor_from_numpy(offsets)
    out = ops.gputensor_from_numpy(np.full((M, ldc), 3, np.float32).astype(np_dtype(dt)))
    from scaffolding_b200 import engine as E
    code = E.dtype_code(np_dtype(dt))
    check(lib.sf_gemm_grouped(X, M, N, K, C.c_void_p(gx.ptr), M, lda, None, C.c_void_p(go.ptr),
                              C.c_void_p(gw.ptr), ldb, bs, C.c_void_p(gb.ptr), code, N + 9,
                              C.c_void_p(out.ptr), ldc, code, code, 1, None, 0, None), "sf_gemm_grouped")
    y = to_host32(ops, out).astype(np.float64)
    dense = np.stack([w[g, :N * ldb].reshape(N, ldb)[:, :K] for g in range(X)])
    ref, tol = plain_grouped(x[:, :K], dense, offsets, b[:, :N], "silu", None, dt)
    assert_within(y[:, :N], ref, tol)
    assert (y[:, N:] == 3).all() and es


# ───────────────────────────── combine ─────────────────────────────

@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("T,k,C_", [(1, 1, 1), (5, 2, 7), (64, 4, 2048), (33, 3, 100), (1000, 2, 1920),
                                    (20, 8, 264), (3, 32, 48)])
def test_combine(gpu, ops, dt, T, k, C_):
    rng = np.random.default_rng(T * 10 + k)
    R = T * k
    gy, y = to_device(ops, rng.standard_normal((R, C_), dtype=np.float32), dt)
    gr, res = to_device(ops, rng.standard_normal((T, C_), dtype=np.float32), dt)
    slots = rng.permutation(R).reshape(T, k).astype(np.int32)
    slots.reshape(-1)[::5] = [[-1, R, 2 ** 31 - 1][i % 3] for i in range(len(slots.reshape(-1)[::5]))]
    w = rng.random((T, k), dtype=np.float32)
    gs, gw = ops.gputensor_from_numpy(slots), ops.gputensor_from_numpy(w)
    live = (slots >= 0) & (slots < R)
    part = np.where(live[:, :, None], w[:, :, None].astype(np.float64) *
                    y[np.where(live, slots, 0)].astype(np.float64), 0.0)
    for use in (False, True):
        ref = part.sum(1) + (res if use else 0.0)
        out = to_host32(ops, ops.dev_moe_combine(gy, gs, gw, gr if use else None)).astype(np.float64)
        # k fused multiply-adds onto the residual, then the output's rounding
        off = k * 2.0 ** -24 * (np.abs(part).sum(1) + np.abs(res if use else 0.0))
        assert_within(out, ref, off + U[dt] * (np.abs(ref) + off) + TINY[dt])
    in_place = ops.dev_moe_combine(gy, gs, gw, gr, out=gr)
    assert in_place is gr
    assert np.array_equal(to_host32(ops, gr), out.astype(np.float32))


# ───────────────────────────── together ─────────────────────────────

def plain_moe(x, layer_weights, k, act, renormalize, dt, residual=None):
    """nn.MoE in 64 bits, with the roundings of what it stores (the router's
    logits in fp32, the expert rows in the layer's type)."""
    router, up, down = layer_weights
    rnd = lambda v: v.astype(np.float32).astype(np_dtype(dt)).astype(np.float64)  # noqa: E731
    logits = (x.astype(np.float64) @ router.astype(np.float64).T)
    experts, weights, _, _, _ = plain_route(logits, k, renormalize)
    y = np.zeros_like(x, dtype=np.float64)
    mag = np.zeros_like(y)
    for t in range(len(x)):
        for j in range(k):
            v = up[experts[t, j]].astype(np.float64) @ x[t].astype(np.float64)
            n = len(v) // 2
            h = rnd(silu(v[:n]) * v[n:] if act == "silu_gate" else plain_act(v, act))
            d = down[experts[t, j]].astype(np.float64)
            y[t] += weights[t, j] * rnd(d @ h)
            mag[t] += weights[t, j] * (np.abs(d) @ np.abs(h))
    gap = np.sort(logits, axis=1)[:, ::-1]
    return y + (0 if residual is None else residual), mag, gap


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("act", ["silu_gate", "gelu_tanh"])
@pytest.mark.parametrize("T", [1, 50, 400])
def test_moe_layer(gpu, ops, dt, act, T):
    """Router linear, route, both grouped products and combine, as nn.MoE runs
    them."""
    from scaffolding_b200 import nn
    rng = np.random.default_rng(T)
    dim, hidden, X, k = 64, 96, 12, 3
    m = nn.MoE(dim, hidden, X, k, act, device=0, dtype=np_dtype(dt), rng=rng)
    gx, x = to_device(ops, rng.standard_normal((1, T, dim), dtype=np.float32), dt)
    gr, res = to_device(ops, rng.standard_normal((1, T, dim), dtype=np.float32), dt)
    y = to_host32(ops, m(gx, gr)).astype(np.float64)[0]
    ref, mag, gap = plain_moe(x[0], [to_host32(ops, w) for w in (m.router, m.up, m.down)], k, act,
                              True, dt, res[0])
    # Tokens whose k-th and next logit lie closer than the router's own error
    # (dim + 1 additions in fp32, 3xTF32 for fp32 inputs) may choose otherwise.
    clear = gap[:, k - 1] - gap[:, k] > 2.0 ** -14
    assert clear.mean() > 0.9
    # A stored expert row is a rounding (u) of a value that may differ by the
    # roundings of h (u per element, entering with |down| |h|) and by fp32
    # sums (hidden * 2^-23 of the same magnitude), so it may fall one step
    # (2 u) elsewhere; the weights differ by 2^-16 at most (logit errors).
    u = U[dt]
    tol = (4 * u + (hidden + dim) * 2.0 ** -22 + 2.0 ** -13 * (dt == "f32") + 2.0 ** -14) * mag
    tol += u * np.abs(ref) + TINY[dt]
    assert_within(y[clear], ref[clear], tol[clear], f"{dt} {act} {T}")
    assert device_error(0) == 0


def test_moe_layer_no_tokens_and_one_expert(gpu, ops):
    from scaffolding_b200 import nn
    rng = np.random.default_rng(0)
    m = nn.MoE(32, 48, 1, 1, "silu", device=0, dtype=np_dtype("bf16"), rng=rng)
    empty = ops._alloc((0, 32), np_dtype("bf16"), 0)
    assert m(empty).shape == (0, 32)
    gx, x = to_device(ops, rng.standard_normal((5, 32), dtype=np.float32), "bf16")
    up = ops.dev_linear_forward(gx, ops.dev_reshape(m.up, (48, 32)), activation="silu")
    ref = ops.dev_linear_forward(up, ops.dev_reshape(m.down, (32, 48)))
    y, r = to_host32(ops, m(gx)), to_host32(ops, ref)  # one expert: weight 1
    # the two products may round h, and then the sum, to neighbouring values
    assert (np.abs(y - r) <= 4 * U["bf16"] * (np.abs(r) + np.abs(to_host32(ops, up)).sum(1, keepdims=True) / 7)).all()


def test_decoder_feed_forward(gpu, ops):
    """The operators as a sparse layer runs them in decoding: a 4-bit
    projection, the routed experts with a residual, a 4-bit projection back,
    each stage against 64 bits on the stage's own input; the same through
    DataParallel on two shares of the one device."""
    from scaffolding_b200 import nn
    from scaffolding_b200.parallel import DataParallel
    rng = np.random.default_rng(8)
    dim, T = 256, 12
    bf = np_dtype("bf16")
    a = nn.Linear4.from_linear(nn.Linear(384, dim, device=0, rng=rng), 64, True, bf)
    moe = nn.MoE(dim, 128, 8, 2, device=0, dtype=bf, rng=rng)
    b = nn.Linear4.from_linear(nn.Linear(dim, 200, device=0, rng=rng), 128, False, bf)
    gx, x = to_device(ops, rng.standard_normal((T, 384), dtype=np.float32), "bf16")

    def linear4(m, v):
        w = to_host32(ops, ops.dev_dequantize_w4(m.weight, np.float32)).astype(np.float64)
        v = v.astype(np.float64)
        ref = v @ w.T + to_host32(ops, m.bias)
        # K + 2 K / group operations on terms of at most 15 |x| scale
        s = np.repeat(to_host32(ops, m.weight.scales).astype(np.float64).T, m.weight.group, 1)[:, :w.shape[1]]
        off = (w.shape[1] + 32) * 2.0 ** -23 * 15 * (np.abs(v) @ s.T) + 2.0 ** -24 * np.abs(ref)
        return ref, off + U["bf16"] * (np.abs(ref) + off)

    h = a(gx)
    ref, tol = linear4(a, x)
    assert_within(to_host32(ops, h).astype(np.float64), ref, tol)
    e = moe(h, h)
    hh = to_host32(ops, h)
    ref, mag, gap = plain_moe(hh, [to_host32(ops, w) for w in (moe.router, moe.up, moe.down)], 2, "silu_gate",
                              True, "bf16", hh)
    clear = gap[:, 1] - gap[:, 2] > 2.0 ** -14
    tol = (4 * U["bf16"] + 384 * 2.0 ** -22 + 2.0 ** -14) * mag + U["bf16"] * np.abs(ref)
    assert_within(to_host32(ops, e).astype(np.float64)[clear], ref[clear], tol[clear])
    y = b(e)
    ref, tol = linear4(b, to_host32(ops, e))
    assert_within(to_host32(ops, y).astype(np.float64), ref, tol)
    whole = to_host32(ops, nn.Sequential(a, moe, b)(gx))
    shares = to_host32(ops, DataParallel(nn.Sequential(a, moe, b), device_ids=[0, 0])(gx))
    assert whole.shape == shares.shape == (T, 200)
    assert np.abs(whole - shares).max() <= 2.0 ** -5 * np.abs(whole).max()
    assert device_error(0) == 0


def test_layer_captured_and_replayed(gpu, ops):
    """A captured layer replays on new inputs in the same buffers (the group
    sizes change between replays), while another stream runs another one."""
    from scaffolding_b200 import engine as E
    from scaffolding_b200._lib import check, lib
    rng = np.random.default_rng(11)
    T, k, X, K, N = 300, 2, 6, 128, 160
    gw, w = to_device(ops, rng.standard_normal((X, N, K), dtype=np.float32) / np.float32(12), "bf16")
    gx, _ = to_device(ops, np.zeros((T, K), np.float32), "bf16")
    gz = ops.gputensor_from_numpy(np.zeros((T, X), np.float32))
    out = ops._alloc((T * k, N), np_dtype("bf16"), 0)
    comb = ops._alloc((T, N), np_dtype("bf16"), 0)
    r = ops.dev_moe_route(gz, k)
    ops.device_synchronize()

    def layer():
        ops.dev_moe_route(gz, k, out=r)
        ops.dev_grouped_linear(gx, gw, r.offsets, rows=r.rows, out=out)
        ops.dev_moe_combine(out, r.slots, r.weights, out=comb)

    s = ops.CudaStream(0)
    E.set_stream(0, s.cuda_stream)
    try:
        layer()
        s.synchronize()
        check(lib.sf_graph_begin(C.c_void_p(s.cuda_stream)), "begin")
        layer()
        exe = C.c_void_p()
        check(lib.sf_graph_end(C.c_void_p(s.cuda_stream), C.byref(exe)), "end")
    finally:
        E.set_stream(0, None)
    for seed in (1, 2):
        g = np.random.default_rng(seed)
        x = g.standard_normal((T, K)).astype(np_dtype("bf16"))
        z = (g.standard_normal((T, X)) + seed * np.arange(X)).astype(np.float32)
        E.memcpy(gx.ptr, x.ctypes.data, x.nbytes, 0)
        E.memcpy(gz.ptr, z.ctypes.data, z.nbytes, 0)
        E.stream_sync(None)
        check(lib.sf_graph_launch(exe, C.c_void_p(s.cuda_stream)), "launch")
        other = ops.dev_moe_combine(*_layer_once(ops, gx, gz, gw, k))  # default stream, its own buffers
        s.synchronize()
        E.stream_sync(None)
        check_route(ops, r, z, k, True)
        _, _, offsets, rows, _ = plain_route(z, k, True)
        ref, tol = plain_grouped(x.astype(np.float32), w, offsets, None, "none", rows, "bf16")
        assert_within(to_host32(ops, out).astype(np.float64), ref, tol)
        assert np.array_equal(to_host32(ops, comb), to_host32(ops, other))
    check(lib.sf_graph_destroy(exe), "destroy")
    assert device_error(0) == 0


def _layer_once(ops, gx, gz, gw, k):
    r = ops.dev_moe_route(gz, k)
    return ops.dev_grouped_linear(gx, gw, r.offsets, rows=r.rows), r.slots, r.weights
