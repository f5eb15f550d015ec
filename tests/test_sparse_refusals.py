"""Refusals of the routed and the 4-bit linears, and the packed layout of
4-bit weights.  CPU only: every check precedes the first use of a device."""
import ctypes as C

import numpy as np
import pytest

I32, F32, F16 = np.int32, np.float32, np.float16


def _fake(ops, shape, dtype=F32, dev=0):
    return ops.GpuTensor(ops.CudaBuffer(0, 0, dev, False), shape, dtype, dev)


def test_route_refuses(ops):
    with pytest.raises(ValueError, match=r"\[tokens, experts\]"):
        ops.dev_moe_route(_fake(ops, (2, 3, 4)), 1)
    with pytest.raises(TypeError, match="unsupported dtype"):
        ops.dev_moe_route(_fake(ops, (4, 8), np.float64), 1)
    for k in (0, -1, 9):
        with pytest.raises(RuntimeError, match="top_k"):
            ops.dev_moe_route(_fake(ops, (4, 8)), k)
    with pytest.raises(RuntimeError, match="at most"):
        ops.dev_moe_route(_fake(ops, (4, 1025)), 2)
    with pytest.raises(RuntimeError, match="at most"):
        ops.dev_moe_route(_fake(ops, (4, 64)), 33)
    with pytest.raises(RuntimeError, match="2\\^31"):
        ops.dev_moe_route(_fake(ops, (1 << 30, 64)), 4)
    good = dict(experts=_fake(ops, (4, 2), I32), weights=_fake(ops, (4, 2)), offsets=_fake(ops, (9,), I32),
                rows=_fake(ops, (8,), I32), slots=_fake(ops, (4, 2), I32))
    for name, bad in [("experts", _fake(ops, (4, 3), I32)), ("weights", _fake(ops, (4, 2), F16)),
                      ("offsets", _fake(ops, (8,), I32)), ("rows", _fake(ops, (4, 2), I32)),
                      ("slots", _fake(ops, (4, 2), np.int64))]:
        with pytest.raises(ValueError, match=name):
            ops.dev_moe_route(_fake(ops, (4, 8)), 2, out=ops.MoeRoute(**{**good, name: bad}))
    with pytest.raises(ValueError, match="different devices"):
        ops.dev_moe_route(_fake(ops, (4, 8), dev=1), 2, out=ops.MoeRoute(**good))


def test_grouped_refuses(ops):
    x, w, off = _fake(ops, (10, 16)), _fake(ops, (3, 6, 16)), _fake(ops, (4,), I32)
    call = ops.dev_grouped_linear
    with pytest.raises(ValueError, match="shapes"):
        call(_fake(ops, (2, 5, 16)), w, off)
    with pytest.raises(ValueError, match="shape mismatch"):
        call(_fake(ops, (10, 15)), w, off)
    with pytest.raises(TypeError, match="share a dtype"):
        call(_fake(ops, (10, 16), F16), w, off)
    with pytest.raises(TypeError, match="int32"):
        call(x, w, _fake(ops, (4,), np.int64))
    with pytest.raises(ValueError, match="offsets"):
        call(x, w, _fake(ops, (3,), I32))
    with pytest.raises(ValueError, match="bias"):
        call(x, w, off, _fake(ops, (6,)))
    with pytest.raises(ValueError, match="activation"):
        call(x, w, off, activation="relu")
    with pytest.raises(ValueError, match="gate and value"):
        call(x, _fake(ops, (3, 7, 16)), off, activation="silu_gate")
    with pytest.raises(ValueError, match="rows"):
        call(x, w, off, rows=_fake(ops, (2, 2), I32))
    with pytest.raises(ValueError, match="out must be"):
        call(x, w, off, out=_fake(ops, (10, 5)))
    with pytest.raises(ValueError, match="different devices"):
        call(x, w, _fake(ops, (4,), I32, dev=1))


def test_gated_activation_is_the_grouped_products_only():
    from scaffolding_b200 import engine as E
    assert E.grouped_act_code("silu_gate") == 3 and E.grouped_act_code("silu") == E.act_code("silu")
    with pytest.raises(ValueError, match="activation"):
        E.act_code("silu_gate")


def test_combine_refuses(ops):
    y, s, w = _fake(ops, (8, 5)), _fake(ops, (4, 2), I32), _fake(ops, (4, 2))
    with pytest.raises(TypeError, match="int32"):
        ops.dev_moe_combine(y, _fake(ops, (4, 2)), w)
    with pytest.raises(ValueError, match="weights"):
        ops.dev_moe_combine(y, s, _fake(ops, (4, 2), F16))
    with pytest.raises(ValueError, match="residual"):
        ops.dev_moe_combine(y, s, w, _fake(ops, (4, 6)))
    with pytest.raises(ValueError, match="residual"):
        ops.dev_moe_combine(y, s, w, _fake(ops, (4, 5), F16))
    with pytest.raises(ValueError, match="out must be"):
        ops.dev_moe_combine(y, s, w, out=_fake(ops, (8, 5)))


def _w4(ops, N=6, K=200, group=64, dt=F16, dev=0):
    G = -(-K // group)
    return ops.W4Weight(_fake(ops, (N, 32), np.uint32, dev), _fake(ops, (G, N), dt, dev),
                        in_features=K, group=group)


def test_w4_refuses(ops):
    with pytest.raises(ValueError, match="group"):
        _w4(ops, group=48)
    with pytest.raises(ValueError, match="words"):
        _w4(ops, K=300)
    with pytest.raises(ValueError, match="scales"):
        ops.W4Weight(_fake(ops, (6, 32), np.uint32), _fake(ops, (6, 4), F16), in_features=200, group=64)
    with pytest.raises(ValueError, match="packed"):
        ops.W4Weight(_fake(ops, (6, 32), np.uint8), _fake(ops, (4, 6), F16), in_features=200, group=64)
    with pytest.raises(TypeError, match="zeros"):
        ops.W4Weight(_fake(ops, (6, 32), np.uint32), _fake(ops, (4, 6), F16), _fake(ops, (4, 6)),
                     in_features=200, group=64)
    w = _w4(ops)
    assert w.shape == (6, 200)
    with pytest.raises(TypeError, match="share a dtype"):
        ops.dev_linear_w4(_fake(ops, (1, 200)), w)
    with pytest.raises(TypeError, match="bf16 or fp16"):
        ops.dev_linear_w4(_fake(ops, (1, 200)), _w4(ops, dt=F32))
    with pytest.raises(ValueError, match="shape mismatch"):
        ops.dev_linear_w4(_fake(ops, (1, 201), F16), w)
    with pytest.raises(ValueError, match="bias"):
        ops.dev_linear_w4(_fake(ops, (1, 200), F16), w, _fake(ops, (5,), F16))
    with pytest.raises(ValueError, match="activation"):
        ops.dev_linear_w4(_fake(ops, (1, 200), F16), w, activation="silu_gate")
    with pytest.raises(ValueError, match="different devices"):
        ops.dev_linear_w4(_fake(ops, (1, 200), F16, dev=1), w)
    with pytest.raises(ValueError, match="group"):
        ops.dev_quantize_w4(_fake(ops, (4, 8), F16), group=16)


def test_result_buffers_apart(ops):
    """The result's buffer is not an input's (combine: not the rows')."""
    x, w, off = _fake(ops, (10, 16)), _fake(ops, (3, 16, 16)), _fake(ops, (4,), I32)
    with pytest.raises(ValueError, match="share memory"):
        ops.dev_grouped_linear(x, w, off, out=x)
    y = _fake(ops, (4, 5))
    with pytest.raises(ValueError, match="share memory"):
        ops.dev_moe_combine(y, _fake(ops, (4, 1), I32), _fake(ops, (4, 1)), out=y)
    h = _fake(ops, (6, 200), F16)
    with pytest.raises(ValueError, match="share memory"):
        ops.dev_linear_w4(h, _w4(ops, N=200, dt=F16, K=200), out=h)


def test_c_abi_refuses():
    from scaffolding_b200._lib import (SF_ERR_INVALID_ARGUMENT as BAD, SF_ERR_UNSUPPORTED as NO,
                                       SF_ERR_WORKSPACE, lib)
    p = C.c_void_p(4096)  # never read: the checks below come first
    odd = C.c_void_p(4100)
    sz = C.c_size_t()
    assert lib.sf_moe_route_workspace_size(100, 8, 2, C.byref(sz)) == 0 and sz.value == 0
    assert lib.sf_moe_route_workspace_size(1000, 8, 2, C.byref(sz)) == 0 and sz.value == 16 * 8 * 4
    assert lib.sf_moe_route(1000, 8, 2, p, 0, 8, 1, p, p, p, p, p, None, 0, None) == SF_ERR_WORKSPACE
    assert lib.sf_moe_route(10, 8, 2, p, 0, 7, 1, p, p, p, p, p, None, 0, None) == BAD
    assert lib.sf_moe_route(10, 8, 2, p, 5, 8, 1, p, p, p, p, p, None, 0, None) == BAD
    assert lib.sf_moe_route(10, 8, 2, None, 0, 8, 1, p, p, p, p, p, None, 0, None) == BAD
    assert lib.sf_moe_route(-1, 8, 2, p, 0, 8, 1, p, p, p, p, p, None, 0, None) == BAD

    def grouped(groups=2, M=4, N=8, K=8, a_rows=4, lda=8, rows=None, off=p, ldb=8, ldc=8, dt=2, act=0, A=p,
                b_stride=64):
        return lib.sf_gemm_grouped(groups, M, N, K, A, a_rows, lda, rows, off, p, ldb, b_stride, None, 0, 0, p,
                                   ldc, dt, dt, act, None, 0, None)

    assert grouped(M=-1) == BAD and grouped(act=4) == BAD and grouped(dt=3) == BAD
    assert grouped(off=None) == BAD and grouped(A=None) == BAD
    assert grouped(a_rows=3) == BAD and grouped(lda=7) == BAD and grouped(ldb=7) == BAD and grouped(ldc=7) == BAD
    assert grouped(groups=5000) == NO and grouped(M=1 << 31, a_rows=1 << 31) == NO
    assert grouped(M=(1 << 31) - 1, a_rows=(1 << 31) - 1) == NO and grouped(b_stride=-8) == BAD
    assert grouped(M=0) == 0 and grouped(groups=0) == 0 and grouped(N=0, ldc=0) == 0

    assert lib.sf_moe_combine(4, 8, 0, p, 8, 8, 2, p, p, None, 8, p, 8, None) == BAD
    assert lib.sf_moe_combine(4, 8, 2, p, 8, 7, 2, p, p, None, 8, p, 8, None) == BAD
    assert lib.sf_moe_combine(4, 8, 2, p, 8, 8, 2, None, p, None, 8, p, 8, None) == BAD
    assert lib.sf_moe_combine(0, 8, 2, p, 8, 8, 2, p, p, None, 8, p, 8, None) == 0

    def w4(M=1, N=8, K=128, ldx=128, packed=p, ldp=16, scales=p, lds=8, group=128, in_dt=2, act=0, ldy=8):
        return lib.sf_linear_w4(M, N, K, p, ldx, packed, ldp, scales, None, lds, group, None, 0, p, ldy,
                                in_dt, 2, act, None)

    assert w4(M=65) == NO and w4(group=16) == NO and w4(in_dt=0) == NO
    assert w4(M=-1) == BAD and w4(packed=odd) == BAD and w4(ldp=18) == BAD and w4(ldp=12) == BAD
    assert w4(K=0, ldx=0) == BAD and w4(lds=7) == BAD and w4(ldx=127) == BAD and w4(ldy=7) == BAD and w4(act=3) == BAD
    assert w4(scales=None) == BAD and w4(M=0) == 0
    assert lib.sf_quantize_w4(8, 128, None, 0, 128, 128, p, 16, p, None, 8, 2, None) == BAD
    assert lib.sf_dequantize_w4(8, 128, p, 16, p, None, 8, 128, 2, p, 2, 127, None) == BAD


def test_packed_layout(ops):
    """Nibble i of word 4 t + w of a block holds column 32 w + 8 t +
    (0, 2, 4, 6, 1, 3, 5, 7)[i]; columns past K hold 0."""
    rng = np.random.default_rng(0)
    q = rng.integers(0, 16, (3, 300)).astype(np.uint8)
    words = ops.pack_w4(q)
    assert words.shape == (3, 48) and words.dtype == np.uint32
    seen = np.zeros((3, 384), np.uint8)
    for b in range(3):
        for t in range(4):
            for w in range(4):
                for i, c in enumerate((0, 2, 4, 6, 1, 3, 5, 7)):
                    seen[:, 128 * b + 32 * w + 8 * t + c] = (words[:, 16 * b + 4 * t + w] >> (4 * i)) & 15
    assert np.array_equal(seen[:, :300], q) and not seen[:, 300:].any()
    with pytest.raises(ValueError, match="0..15"):
        ops.pack_w4(np.array([[16]]))


def test_moe_module_refuses():
    from scaffolding_b200 import nn
    with pytest.raises(ValueError, match="top_k"):
        nn.MoE(8, 8, 4, 5)
    with pytest.raises(ValueError, match="activation"):
        nn.MoE(8, 8, 4, 2, "relu")
