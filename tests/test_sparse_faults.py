"""Faults of the routed and the 4-bit linears that the host alone decides:
refused shapes, shared memory, the order of launches.  CPU only: the engine's
entry points are stood in for where a call would reach a device."""
import numpy as np
import pytest

I32, F32, F16 = np.int32, np.float32, np.float16


def _fake(ops, shape, dtype=F32, dev=0):
    return ops.GpuTensor(ops.CudaBuffer(0, 0, dev, False), shape, dtype, dev)


def _moe(ops, nn, dim=64, hidden=96, experts=4, top_k=2, dtype=F32):
    """An nn.MoE whose weights are placeholders."""
    m = nn.MoE.__new__(nn.MoE)
    m.dim, m.hidden, m.num_experts, m.top_k = dim, hidden, experts, top_k
    m.activation, m.renormalize = "silu_gate", True
    m.router = _fake(ops, (experts, dim), dtype)
    m.up = _fake(ops, (experts, 2 * hidden, dim), dtype)
    m.down = _fake(ops, (experts, dim, hidden), dtype)
    return m


def test_moe_refuses_another_width(ops):
    """A width of which the layer's is a divisor must not be cut into more
    tokens."""
    from scaffolding_b200 import nn
    m = _moe(ops, nn)
    for shape in ((4, 128), (2, 3, 640), (64, 1), (8, 32), (128,), ()):
        with pytest.raises(ValueError, match="width 64"):
            m(_fake(ops, shape))
