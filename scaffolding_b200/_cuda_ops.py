"""Drop-in replacement for the hot-path surface of ``scaffolding._cuda_ops``.

The reference's callers (``tensor.py:37``, ``nn/layers.py:12``,
``nn/functional.py:11``, ``nn/parallel.py:23``) import
``scaffolding._cuda_ops`` and call the names below; this module exports the
same names with the same signatures and argument meaning, backed by the
sm_100a engine (``libsf_engine.so``) instead of cuBLAS:

* ``GpuTensor`` / ``CudaBuffer`` and the NumPy transfer helpers
  (``_cuda_ops.pyx:307-341``, ``:807-875``);
* the matmul family ``dev_matmul``, ``dev_matmul_nt``, ``dev_batched_matmul``,
  ``dev_batched_matmul_nt``, ``dev_linear_forward`` (``_cuda_ops.pyx:1088-1302``)
  and the host-array ``cuda_*`` variants (``:2120-2230``, ``:2453-2471``);
* the glue the attention path uses: ``dev_muls``, ``dev_softmax``, ``dev_silu``,
  ``dev_gelu``, ``dev_reshape``, ``dev_unsqueeze``, ``dev_squeeze``;
* ``dev_layer_norm`` and the DiT blocks' adaptive norm ``dev_ada_layer_norm``
  (the bandwidth step in front of the QKV and FFN-up GEMMs);
* the linears of a sparse language-model layer: ``dev_moe_route``,
  ``dev_grouped_linear`` and ``dev_moe_combine``, and ``dev_linear_w4`` over
  4-bit weights (``W4Weight``, ``dev_quantize_w4``, ``dev_dequantize_w4``);
* runtime: devices, caching allocator, streams, events, peer access.

Differences from the reference, all deliberate:
* dtype-aware: bf16 (``ml_dtypes.bfloat16`` on the host) and fp16 tensors
  are computed as such with fp32 accumulation and returned in their own
  dtype; fp32 tensors behave exactly as before (fp32 in, fp32 out).  The
  reference read every buffer as ``float*`` (``_cuda_ops.pyx:1095-1102``).
* ``dev_linear_forward`` fuses bias and an optional activation into the GEMM
  epilogue (the reference launched SGEMM, then a bias kernel on the NULL
  stream, then the activation separately).
* ``dev_batched_matmul_nt`` is one launch (the reference looped over the
  batch on the host, ``_cuda_ops.pyx:1181-1187``).
* every op runs on the device that holds its inputs, and allocates there
  (the reference used the current device in ``dev_muls`` / ``dev_softmax``).
* ``gputensor_to_device`` copies ``numel * itemsize`` bytes (the reference
  assumed 4-byte elements, ``_cuda_ops.pyx:868-870``).

Operations outside the matmul path (RMS norm, cross-entropy, AdamW, ...)
raise ``NotImplementedError`` naming the op.
"""
from __future__ import annotations

import ctypes as C
import math

import numpy as np

from . import engine as E
from ._lib import (ACT_GELU_TANH, ACT_NONE, ACT_SILU, ACT_SILU_GATE, COPY_D2D, COPY_D2H, COPY_H2D,
                   DT_F32, FP32_ACCURATE, FP32_TF32, DeviceProps, check, lib)

bfloat16 = E.bfloat16


# ───────────────────────────── buffers / tensors ─────────────────────────────

class CudaBuffer(E.DeviceBuffer):
    """Device allocation from the engine's caching allocator
    (``_cuda_ops.pyx:307-341``)."""

    __slots__ = ()

    @property
    def data_ptr(self) -> int:
        return self.ptr

    @property
    def size(self) -> int:
        return self.nbytes

    def __reduce__(self):
        # Pickle the raw bytes (the reference pickled as float32 regardless
        # of the element type, _cuda_ops.pyx:333-341).
        arr = np.empty(self.nbytes, dtype=np.uint8)
        if self.ptr and self.nbytes:
            with E.on_device(self.device_id):
                E.memcpy(arr.ctypes.data, self.ptr, self.nbytes, COPY_D2H)
                E.stream_sync(None)
        return (_rebuild_cuda_buffer, (arr, self.device_id))


def _rebuild_cuda_buffer(arr: np.ndarray, device_id: int = 0):
    buf = _make_buffer(arr.nbytes, device_id)
    with E.on_device(device_id):
        stream = E.upload_stream(device_id)
        E.memcpy(buf.ptr, arr.ctypes.data, arr.nbytes, COPY_H2D, stream)
        E.stream_sync(stream)
    return buf


def _make_buffer(nbytes: int, device_id: int) -> CudaBuffer:
    p = C.c_void_p()
    check(lib.sf_malloc(int(device_id), int(nbytes), C.byref(p)), "sf_malloc")
    return CudaBuffer(p.value or 0, nbytes, device_id, True)


class GpuTensor:
    """GPU-resident tensor: CudaBuffer + shape + NumPy dtype + device id
    (``_cuda_ops.pyx:807-819``), contiguous row-major."""

    __slots__ = ("buffer", "shape", "dtype", "numel", "device_id")

    def __init__(self, buffer, shape: tuple, dtype, device_id: int = -1):
        self.buffer = buffer
        self.shape = tuple(int(s) for s in shape)
        self.dtype = np.dtype(dtype)
        self.device_id = device_id if device_id >= 0 else buffer.device_id
        n = 1
        for s in self.shape:
            n *= s
        self.numel = n

    @property
    def ptr(self) -> int:
        return self.buffer.ptr

    @property
    def ndim(self) -> int:
        return len(self.shape)

    def matmul(self, other: "GpuTensor", *, trans_b: bool = False, out_dtype=None) -> "GpuTensor":
        """``self @ other`` (``trans_b``: ``self @ other^T``, ``other`` in the
        ``nn.Linear`` weight layout).  2-D or batched, like ``sf.matmul`` /
        ``sf.matmul_nt`` (``tensor.py:1480-1539``)."""
        if self.ndim == 2 and other.ndim == 2:
            return _matmul2d(self, other, trans_b, out_dtype)
        return _batched(self, other, trans_b, out_dtype)

    def __matmul__(self, other: "GpuTensor") -> "GpuTensor":
        return self.matmul(other)

    def __repr__(self) -> str:
        return f"GpuTensor(shape={self.shape}, dtype={self.dtype}, device={self.device_id})"


def _alloc(shape, dtype, dev) -> GpuTensor:
    dt = np.dtype(dtype)
    n = int(np.prod(shape, dtype=np.int64)) if len(shape) else 1
    return GpuTensor(_make_buffer(n * dt.itemsize, dev), tuple(shape), dt, dev)


# ───────────────────────────── NumPy <-> GPU ─────────────────────────────

def gputensor_from_numpy(arr: np.ndarray, device_id: int = -1) -> GpuTensor:
    """Upload a NumPy array (``_cuda_ops.pyx:822-840``)."""
    flat = np.ascontiguousarray(arr)
    dev = device_id if device_id >= 0 else E.current_device()
    gt = _alloc(flat.shape, flat.dtype, dev)
    if flat.nbytes:
        with E.on_device(dev):
            stream = E.upload_stream(dev)
            E.memcpy(gt.ptr, flat.ctypes.data, flat.nbytes, COPY_H2D, stream)
            E.stream_sync(stream)
    return gt


def gputensor_to_numpy(gt: GpuTensor) -> np.ndarray:
    """Download a GpuTensor synchronously (``_cuda_ops.pyx:843-858``)."""
    out = np.empty(gt.shape, dtype=gt.dtype)
    if out.nbytes:
        with E.on_device(gt.device_id):
            stream = E.get_stream(gt.device_id)
            E.stream_sync(stream)
            E.memcpy(out.ctypes.data, gt.ptr, out.nbytes, COPY_D2H, stream)
            E.stream_sync(stream)
    return out


def gputensor_to_device(gt: GpuTensor, target_dev: int) -> GpuTensor:
    """Copy to another device (``_cuda_ops.pyx:861-875``), ``numel*itemsize`` bytes."""
    if gt.device_id == target_dev:
        return gt
    out = _alloc(gt.shape, gt.dtype, target_dev)
    nbytes = gt.numel * gt.dtype.itemsize
    if nbytes:
        with E.on_device(gt.device_id):
            E.stream_sync(E.get_stream(gt.device_id))
        with E.on_device(target_dev):
            stream = E.upload_stream(target_dev)
            check(lib.sf_memcpy_peer(C.c_void_p(out.ptr), int(target_dev), C.c_void_p(gt.ptr),
                                     int(gt.device_id), nbytes, stream), "sf_memcpy_peer")
            E.stream_sync(stream)
    return out


def gputensor_astype(gt: GpuTensor, dtype) -> GpuTensor:
    """Copy of ``gt`` converted to ``dtype`` on its device (fp32 / bf16 / fp16,
    round to nearest even), e.g. fp32 weights stored as bf16 after upload.
    New: the reference uploads fp32 only (``nn/layers.py:18-35``)."""
    dt = np.dtype(dtype)
    if dt == gt.dtype:
        return gt
    out = _alloc(gt.shape, dt, gt.device_id)
    if gt.numel:
        with E.on_device(gt.device_id):
            E.unary(gt.ptr, E.dtype_code(gt.dtype), out.ptr, E.dtype_code(dt), gt.numel, 1.0,
                    ACT_NONE, device=gt.device_id)
    return out


def numpy_to_gpu(arr: np.ndarray, stream=None):
    gt = gputensor_from_numpy(arr)
    return gt.buffer, arr.shape, arr.dtype


def gpu_to_numpy(buf: CudaBuffer, shape, dtype, stream=None) -> np.ndarray:
    return gputensor_to_numpy(GpuTensor(buf, tuple(shape), dtype, buf.device_id))


# ───────────────────────────── matmul family ─────────────────────────────

def _out_dtype(a: GpuTensor, out_dtype) -> np.dtype:
    return np.dtype(out_dtype) if out_dtype is not None else a.dtype


def _check_pair(a: GpuTensor, b: GpuTensor) -> None:
    if a.dtype != b.dtype:
        raise TypeError(f"matmul operands must share a dtype ({a.dtype} vs {b.dtype})")
    if a.device_id != b.device_id:
        raise ValueError(f"operands on different devices ({a.device_id} vs {b.device_id})")


def _matmul2d(a: GpuTensor, b: GpuTensor, trans_b: bool, out_dtype=None, epi=None) -> GpuTensor:
    _check_pair(a, b)
    M, K = a.shape
    if trans_b:
        N, Kb = b.shape
    else:
        Kb, N = b.shape
    if K != Kb:
        raise ValueError(f"matmul shape mismatch: {a.shape} x {b.shape}{'^T' if trans_b else ''}")
    odt = _out_dtype(a, out_dtype)
    dev = a.device_id
    c = _alloc((M, N), odt, dev)
    with E.on_device(dev):
        E.gemm(M, N, K, a.ptr, K, 0, b.ptr, K if trans_b else N, 1 if trans_b else 0,
               c.ptr, N, E.dtype_code(a.dtype), E.dtype_code(odt), epi=epi, device=dev)
    return c


def _batched(a: GpuTensor, b: GpuTensor, trans_b: bool, out_dtype=None, epi=None) -> GpuTensor:
    _check_pair(a, b)
    if a.ndim < 2 or b.ndim < 2:
        raise ValueError("batched matmul needs operands of rank >= 2")
    M, K = a.shape[-2:]
    if trans_b:
        N, Kb = b.shape[-2:]
    else:
        Kb, N = b.shape[-2:]
    if K != Kb:
        raise ValueError(f"matmul shape mismatch: {a.shape} x {b.shape}{'^T' if trans_b else ''}")
    lead = a.shape[:-2]
    batch = int(np.prod(lead, dtype=np.int64)) if lead else 1
    b_batch = int(np.prod(b.shape[:-2], dtype=np.int64)) if b.ndim > 2 else 1
    if b_batch not in (1, batch):
        raise ValueError(f"batch dims differ: {a.shape} vs {b.shape}")
    odt = _out_dtype(a, out_dtype)
    dev = a.device_id
    c = _alloc(lead + (M, N), odt, dev)
    ldb = K if trans_b else N
    with E.on_device(dev):
        if b.ndim == 2 or b_batch == 1:
            # Shared right operand: one GEMM over the stacked rows of A.
            E.gemm(batch * M, N, K, a.ptr, K, 0, b.ptr, ldb, 1 if trans_b else 0, c.ptr, N,
                   E.dtype_code(a.dtype), E.dtype_code(odt), epi=epi, device=dev)
        elif b_batch == batch:
            bt = E.make_batch(batch, 1, a=(M * K, 0), b=(N * K, 0), c=(M * N, 0))
            E.gemm(M, N, K, a.ptr, K, 0, b.ptr, ldb, 1 if trans_b else 0, c.ptr, N,
                   E.dtype_code(a.dtype), E.dtype_code(odt), epi=epi, batch=bt, device=dev)
        else:
            raise ValueError(f"batch dims differ: {a.shape} vs {b.shape}")
    return c


def dev_matmul(gt_a: GpuTensor, gt_b: GpuTensor) -> GpuTensor:
    """C = A @ B; A (M,K), B (K,N) (``_cuda_ops.pyx:1088-1102``)."""
    return _matmul2d(gt_a, gt_b, False)


def dev_matmul_nt(gt_a: GpuTensor, gt_b: GpuTensor) -> GpuTensor:
    """C = A @ B^T; A (M,K), B (N,K) (``_cuda_ops.pyx:1105-1119``)."""
    return _matmul2d(gt_a, gt_b, True)


def dev_batched_matmul(gt_a: GpuTensor, gt_b: GpuTensor) -> GpuTensor:
    """(..., M, K) @ (..., K, N) (``_cuda_ops.pyx:1122-1149``); B may also be
    2-D (shared across the batch)."""
    return _batched(gt_a, gt_b, False)


def dev_batched_matmul_nt(gt_a: GpuTensor, gt_b: GpuTensor) -> GpuTensor:
    """(..., M, K) @ (..., N, K)^T in one launch (``_cuda_ops.pyx:1152-1190``)."""
    return _batched(gt_a, gt_b, True)


def dev_linear_forward(gt_x: GpuTensor, gt_weight: GpuTensor, gt_bias: GpuTensor | None = None,
                       activation: str = "none", out_dtype=None, out: GpuTensor | None = None) -> GpuTensor:
    """y = act(x @ W^T + bias) with bias and activation fused into the GEMM
    epilogue (``_cuda_ops.pyx:1278-1302``; activation was a separate launch,
    ``nn/functional.py:37-40``).  ``out``: the result's buffer, which shares no
    memory with the operands."""
    _check_pair(gt_x, gt_weight)
    K = gt_x.shape[-1]
    M = int(np.prod(gt_x.shape[:-1], dtype=np.int64))
    N, Kw = gt_weight.shape
    if Kw != K:
        raise ValueError(f"linear shape mismatch: x {gt_x.shape}, W {gt_weight.shape}")
    _apart(out, gt_x, gt_weight, gt_bias)
    odt = _out_dtype(gt_x, out_dtype if out is None else out.dtype)
    dev = gt_x.device_id
    y = _result(out, gt_x.shape[:-1] + (N,), odt, dev, "out")
    bias_ptr, bias_dt = 0, DT_F32
    if gt_bias is not None:
        if gt_bias.numel != N:
            raise ValueError(f"bias has {gt_bias.numel} elements, expected {N}")
        bias_ptr, bias_dt = gt_bias.ptr, E.dtype_code(gt_bias.dtype)
    epi = E.make_epilogue(bias_ptr=bias_ptr, bias_dt=bias_dt, act=E.act_code(activation))
    with E.on_device(dev):
        E.gemm(M, N, K, gt_x.ptr, K, 0, gt_weight.ptr, K, 1, y.ptr, N,
               E.dtype_code(gt_x.dtype), E.dtype_code(odt), epi=epi, device=dev)
    return y


# ───────────────────────────── attention glue ─────────────────────────────

def _unary(gt: GpuTensor, alpha: float, act: int) -> GpuTensor:
    dev = gt.device_id
    out = _alloc(gt.shape, gt.dtype, dev)
    code = E.dtype_code(gt.dtype)
    with E.on_device(dev):
        E.unary(gt.ptr, code, out.ptr, code, gt.numel, alpha, act, device=dev)
    return out


def dev_muls(gt: GpuTensor, scalar: float) -> GpuTensor:
    """y = scalar * x (``_cuda_ops.pyx:990-998``)."""
    return _unary(gt, float(scalar), ACT_NONE)


def dev_silu(gt: GpuTensor) -> GpuTensor:
    """SiLU (``_cuda_ops.pyx:944-945``)."""
    return _unary(gt, 1.0, ACT_SILU)


def dev_gelu(gt: GpuTensor) -> GpuTensor:
    """GELU, tanh form (``_cuda_ops.pyx:947-948``)."""
    return _unary(gt, 1.0, ACT_GELU_TANH)


def dev_softmax(gt: GpuTensor, dim: int = -1) -> GpuTensor:
    """Softmax over the last dimension (``_cuda_ops.pyx:1016-1034``)."""
    nd = len(gt.shape)
    if nd == 0:
        raise ValueError("softmax of a 0-d tensor")
    if dim not in (-1, nd - 1):
        raise NotImplementedError("dev_softmax supports the last dimension only")
    cols = gt.shape[-1]
    rows = gt.numel // cols if cols else 0
    dev = gt.device_id
    out = _alloc(gt.shape, gt.dtype, dev)
    code = E.dtype_code(gt.dtype)
    with E.on_device(dev):
        E.softmax_rows(gt.ptr, code, cols, out.ptr, code, cols, rows, cols, 1.0, device=dev)
    return out


def _norm_launch(gt: GpuTensor, gamma, beta, eps: float, mod=None, group_rows: int = 1,
                 out_dtype=None) -> GpuTensor:
    cols = gt.shape[-1]
    rows = gt.numel // cols if cols else 0
    dev = gt.device_id
    odt = np.dtype(out_dtype) if out_dtype is not None else gt.dtype
    out = _alloc(gt.shape, odt, dev)
    for t, name in ((gamma, "gamma"), (beta, "beta")):
        if t is not None and (t.dtype != np.float32 or t.numel != cols):
            raise ValueError(f"layer norm {name} must be fp32 with {cols} elements")
    if (gamma is None) != (beta is None):
        raise ValueError("layer norm gamma and beta go together")
    mod_ptr, mod_dt, ld_mod = None, DT_F32, 0
    if mod is not None:
        if mod.shape[-1] != 2 * cols:
            raise ValueError(f"modulation rows must hold 2 x {cols} values, got {mod.shape}")
        mod_ptr, mod_dt, ld_mod = C.c_void_p(mod.ptr), E.dtype_code(mod.dtype), 2 * cols
    with E.on_device(dev):
        s = E.get_stream(dev)
        check(lib.sf_layernorm_modulate(rows, cols, C.c_void_p(gt.ptr), E.dtype_code(gt.dtype), cols,
                                        C.c_void_p(gamma.ptr) if gamma is not None else None,
                                        C.c_void_p(beta.ptr) if beta is not None else None,
                                        float(eps), mod_ptr, mod_dt, ld_mod, int(group_rows),
                                        C.c_void_p(out.ptr), E.dtype_code(odt), cols,
                                        C.c_void_p(s) if s else None), "sf_layernorm_modulate")
    return out


def dev_layer_norm(gt: GpuTensor, gt_gamma: GpuTensor | None = None,
                   gt_beta: GpuTensor | None = None, eps: float = 1e-5) -> GpuTensor:
    """LayerNorm over the last dimension (``dev_layer_norm`` behind
    ``nn/layers.py:470-493``; kernel ``_cuda_kernels.cu:1070-1093``), fp32 /
    bf16 / fp16 in and out, fp32 gamma and beta."""
    return _norm_launch(gt, gt_gamma, gt_beta, eps)


def dev_ada_layer_norm(gt: GpuTensor, gt_params: GpuTensor, gt_gamma: GpuTensor | None = None,
                       gt_beta: GpuTensor | None = None, eps: float = 1e-5,
                       out_dtype=None) -> GpuTensor:
    """AdaLayerNorm (``diffusion/models.py:478-487``) of ``x [B, N, C]`` with
    the modulation linear's output ``params [B, 2C]``: LayerNorm, then
    ``h * (1 + params[b, :C]) + params[b, C:]`` for every token of sample b,
    in one kernel.  New (the reference modulates on the host)."""
    if gt.ndim != 3 or gt_params.ndim != 2 or gt_params.shape[0] != gt.shape[0]:
        raise ValueError(f"adaLN shapes: x {gt.shape}, params {gt_params.shape}")
    return _norm_launch(gt, gt_gamma, gt_beta, eps, gt_params, gt.shape[1], out_dtype)


# ───────────────────────────── experts ─────────────────────────────

_F32, _I32, _U32 = np.dtype(np.float32), np.dtype(np.int32), np.dtype(np.uint32)


def _same_device(first: GpuTensor, *others) -> int:
    """Device of the tensors (None skipped); refuses a mix."""
    dev = first.device_id
    for t in others:
        if t is not None and t.device_id != dev:
            raise ValueError(f"operands on different devices ({dev} vs {t.device_id})")
    return dev


def _result(out, shape, dtype, dev, name: str) -> GpuTensor:
    """``out`` when the caller gives the result's buffer, else a new tensor."""
    if out is None:
        return _alloc(shape, dtype, dev)
    if out.shape != shape or out.dtype != dtype:
        raise ValueError(f"{name} must be {shape} {dtype}, got {out.shape} {out.dtype}")
    return out


def _apart(one, *others) -> None:
    """Refuses a result that shares memory with an input, by address (``one``
    is the result, or the input of several results)."""
    if one is None or not one.numel:
        return
    mine = one.buffer
    lo, hi = mine.ptr, mine.ptr + mine.nbytes
    for t in others:
        if t is not None:
            b = t.buffer
            if b is mine or (b.ptr < hi and lo < b.ptr + b.nbytes):
                raise ValueError("out must not share memory with the inputs")


def _int32(t: GpuTensor, name: str) -> GpuTensor:
    if t.dtype != _I32:
        raise TypeError(f"{name} must be int32, got {t.dtype}")
    return t


def _ptr(t):
    """Address of a tensor, None for none (both as ctypes takes a pointer)."""
    return t.buffer.ptr if t is not None else None


class MoeRoute:
    """A batch's choices of experts, as ``dev_moe_route`` gives them:

    * ``experts`` int32 ``[tokens, top_k]``, by falling logit;
    * ``weights`` fp32 ``[tokens, top_k]``;
    * ``offsets`` int32 ``[experts + 1]``: the slots of expert e are
      ``offsets[e] .. offsets[e + 1] - 1``;
    * ``rows`` int32 ``[tokens * top_k]``: the token of each slot;
    * ``slots`` int32 ``[tokens, top_k]``: the slot of each choice."""

    __slots__ = ("experts", "weights", "offsets", "rows", "slots", "scratch")

    def __init__(self, experts, weights, offsets, rows, slots):
        self.experts, self.weights, self.offsets = experts, weights, offsets
        self.rows, self.slots = rows, slots
        self.scratch = None  # per-block counts, kept with the buffers they are used with


def moe_route_scratch(tokens: int, experts: int, top_k: int) -> int:
    """Bytes of counts that routing so many tokens takes (0 for few)."""
    need = C.c_size_t()
    check(lib.sf_moe_route_workspace_size(tokens, experts, top_k, C.byref(need)), "sf_moe_route_workspace_size")
    return need.value


def dev_moe_route(gt_logits: GpuTensor, top_k: int, renormalize: bool = True,
                  out: MoeRoute | None = None) -> MoeRoute:
    """Route ``[tokens, experts]`` logits (fp32 / bf16 / fp16): the ``top_k``
    experts of every token (ties to the lowest expert, NaN as -inf), their
    softmax weights -- over the chosen experts, or over all of them with
    ``renormalize=False`` -- and the choices grouped by expert for
    ``dev_grouped_linear`` (``sf_moe_route``).  ``out``: a MoeRoute whose
    buffers are written instead of new ones (a captured graph, a decoding
    loop), which share no memory with the logits; it must not be read by work in
    flight on another stream.  New (the
    reference has no routed layers)."""
    if gt_logits.ndim != 2:
        raise ValueError(f"router logits must be [tokens, experts], got {gt_logits.shape}")
    T, X = gt_logits.shape
    k = int(top_k)
    dev = gt_logits.device_id
    code = E.dtype_code(gt_logits.dtype)
    need = moe_route_scratch(T, X, k)
    if out is None:
        i32 = np.int32
        out = MoeRoute(_alloc((T, k), i32, dev), _alloc((T, k), np.float32, dev),
                       _alloc((X + 1,), i32, dev), _alloc((T * k,), i32, dev), _alloc((T, k), i32, dev))
    else:
        e, w, o, r, s = out.experts, out.weights, out.offsets, out.rows, out.slots
        _same_device(gt_logits, e, w, o, r, s)
        if not (e.shape == w.shape == s.shape == (T, k) and o.shape == (X + 1,) and r.shape == (T * k,)
                and e.dtype == o.dtype == r.dtype == s.dtype == _I32 and w.dtype == _F32):
            for name, t, shape in (("experts", e, (T, k)), ("weights", w, (T, k)), ("offsets", o, (X + 1,)),
                                   ("rows", r, (T * k,)), ("slots", s, (T, k))):
                _result(t, shape, _F32 if name == "weights" else _I32, dev, name)
        _apart(gt_logits, e, w, o, r, s)
    if need and (out.scratch is None or out.scratch.nbytes < need or out.scratch.device_id != dev):
        out.scratch = _make_buffer(need, dev)
    ws = out.scratch.ptr if need else None
    with E.on_device(dev):
        check(lib.sf_moe_route(T, X, k, _ptr(gt_logits), code, X, 1 if renormalize else 0,
                               _ptr(out.experts), _ptr(out.weights), _ptr(out.offsets),
                               _ptr(out.rows), _ptr(out.slots), ws, need, E.get_stream(dev)),
              "sf_moe_route")
    return out


def dev_grouped_linear(gt_x: GpuTensor, gt_weight: GpuTensor, gt_offsets: GpuTensor,
                       gt_bias: GpuTensor | None = None, activation: str = "none", *,
                       rows: GpuTensor | None = None, out_dtype=None,
                       out: GpuTensor | None = None) -> GpuTensor:
    """One linear per expert over rows grouped by expert, in one launch
    (``sf_gemm_grouped``): output row i, ``offsets[e] <= i < offsets[e + 1]``,
    is ``act(weight[e] @ x[r] + bias[e])`` with ``r = rows[i]`` when ``rows``
    is given (the rows are gathered as they are read), else ``r = i``.

    ``weight`` is ``[experts, N, K]``, each expert as an ``nn.Linear`` weight,
    ``bias`` ``[experts, N]``.  ``activation="silu_gate"`` takes ``[experts,
    2 N, K]``, the first N rows the gate: ``silu(gate) * value``.  The group
    sizes stay on the device.  Rows of the result in no group are not written
    (``dev_moe_route``'s offsets cover every row).  ``out`` shares no memory
    with the inputs."""
    act = E.grouped_act_code(activation)
    if gt_x.ndim != 2 or gt_weight.ndim != 3:
        raise ValueError(f"grouped linear shapes: x {gt_x.shape}, weight {gt_weight.shape}")
    if gt_x.dtype != gt_weight.dtype:
        raise TypeError(f"matmul operands must share a dtype ({gt_x.dtype} vs {gt_weight.dtype})")
    X, wide, K = gt_weight.shape
    if gt_x.shape[1] != K:
        raise ValueError(f"grouped linear shape mismatch: x {gt_x.shape}, weight {gt_weight.shape}")
    if act == ACT_SILU_GATE and wide % 2:
        raise ValueError(f"silu_gate needs gate and value rows, got {wide} rows per expert")
    if _int32(gt_offsets, "offsets").shape != (X + 1,):
        raise ValueError(f"offsets must be ({X + 1},), got {gt_offsets.shape}")
    if rows is not None and _int32(rows, "rows").ndim != 1:
        raise ValueError(f"rows must be 1-d, got {rows.shape}")
    if gt_bias is not None and gt_bias.shape != (X, wide):
        raise ValueError(f"bias must be {(X, wide)}, got {gt_bias.shape}")
    N = wide // 2 if act == ACT_SILU_GATE else wide
    M = rows.shape[0] if rows is not None else gt_x.shape[0]
    dev = _same_device(gt_x, gt_weight, gt_offsets, gt_bias, rows, out)
    _apart(out, gt_x, gt_weight, gt_bias, gt_offsets, rows)
    odt = _out_dtype(gt_x, out_dtype if out is None else out.dtype)
    y = _result(out, (M, N), odt, dev, "out")
    bias_dt = E.dtype_code(gt_bias.dtype) if gt_bias is not None else DT_F32
    stream, code = E.get_stream(dev), E.dtype_code(gt_x.dtype)
    call = (X, M, N, K, _ptr(gt_x), gt_x.shape[0], K, _ptr(rows), _ptr(gt_offsets), _ptr(gt_weight),
            K, wide * K, _ptr(gt_bias), bias_dt, wide, _ptr(y), N, code, E.dtype_code(odt), act)
    with E.on_device(dev):
        if rows is None or M <= 1024:  # short batches need no workspace
            check(lib.sf_gemm_grouped(*call, None, 0, stream), "sf_gemm_grouped")
            return y
        need = C.c_size_t()
        check(lib.sf_gemm_grouped_workspace_size(X, M, N, K, code, stream, C.byref(need)),
              "sf_gemm_grouped_workspace_size")
        with E.workspace_lock:
            buf = E.workspace(dev, stream, need.value)
            ws, ws_bytes = (buf.ptr, buf.nbytes) if buf is not None else (None, 0)
            check(lib.sf_gemm_grouped(*call, ws, ws_bytes, stream), "sf_gemm_grouped")
    return y


def dev_moe_combine(gt_y: GpuTensor, gt_slots: GpuTensor, gt_weights: GpuTensor,
                    residual: GpuTensor | None = None, out: GpuTensor | None = None) -> GpuTensor:
    """Weighted sum of every token's expert rows (``sf_moe_combine``):
    ``residual[t] + sum_j weights[t, j] * y[slots[t, j]]`` in fp32, rounded
    once; ``slots`` and ``weights`` as in a MoeRoute, ``y`` ``[slots, C]``.
    A slot outside ``y`` (-1, say, for a dropped choice) adds nothing.  ``out``
    may be ``residual``, and shares no memory with the other inputs."""
    if gt_y.ndim != 2 or gt_slots.ndim != 2:
        raise ValueError(f"combine shapes: y {gt_y.shape}, slots {gt_slots.shape}")
    T, k = _int32(gt_slots, "slots").shape
    width = gt_y.shape[1]
    if gt_weights.shape != (T, k) or gt_weights.dtype != _F32:
        raise ValueError(f"weights must be {(T, k)} float32, got {gt_weights.shape} {gt_weights.dtype}")
    if residual is not None and (residual.shape != (T, width) or residual.dtype != gt_y.dtype):
        raise ValueError(f"residual must be {(T, width)} {gt_y.dtype}, got {residual.shape} {residual.dtype}")
    dev = _same_device(gt_y, gt_slots, gt_weights, residual, out)
    _apart(out, gt_y, gt_slots, gt_weights,
           None if out is None or residual is None or residual.ptr == out.ptr else residual)
    o = _result(out, (T, width), gt_y.dtype, dev, "out")
    with E.on_device(dev):
        check(lib.sf_moe_combine(T, width, k, _ptr(gt_y), gt_y.shape[0], width,
                                 E.dtype_code(gt_y.dtype), _ptr(gt_slots), _ptr(gt_weights),
                                 _ptr(residual), width, _ptr(o), width, E.get_stream(dev)),
              "sf_moe_combine")
    return o


# ───────────────────────────── 4-bit weights ─────────────────────────────

# Nibble i of a packed word holds column _W4_NIBBLE[i] of its eight.
_W4_NIBBLE = (0, 2, 4, 6, 1, 3, 5, 7)
_W4_MAX_ROWS = 64  # rows of x that sf_linear_w4 takes


def pack_w4(q: np.ndarray) -> np.ndarray:
    """Host ``[N, K]`` values 0..15 to ``[N, 16 * ceil(K / 128)]`` uint32
    words in the order ``sf_linear_w4`` documents; columns past K hold 0."""
    if q.dtype.kind == "V":  # ml_dtypes' small types
        q = q.astype(np.float32)
    if q.ndim != 2 or q.dtype.kind not in "uibf" or (q.size and not (
            q.min() >= 0 and q.max() <= 15 and (q.dtype.kind != "f" or (q == np.rint(q)).all()))):
        raise ValueError("4-bit values are a 2-d array of whole numbers 0..15")
    n, k = q.shape
    blocks = -(-k // 128)
    padded = np.zeros((n, blocks * 128), np.uint32)
    padded[:, :k] = q
    # [n, block, w, t, column of 8] -> words 4 t + w
    cols = padded.reshape(n, blocks, 4, 4, 8).transpose(0, 1, 3, 2, 4)
    words = np.zeros(cols.shape[:-1], np.uint32)
    for i, c in enumerate(_W4_NIBBLE):
        words |= cols[..., c] << np.uint32(4 * i)
    return words.reshape(n, blocks * 16)


class W4Weight:
    """An ``[out_features, in_features]`` weight in 4 bits with group scales:
    ``W[n, k] = scales[k // group, n] * (q[n, k] - zeros[k // group, n])``,
    q in 0..15, zeros 8 where None.

    * ``packed``: uint32 (or int32) ``[N, 16 * ceil(K / 128)]``, nibbles in
      the order ``sf_linear_w4`` documents (``from_arrays`` packs);
    * ``scales`` / ``zeros``: ``[ceil(K / group), N]`` in the type of the
      activations (bf16 / fp16)."""

    def __init__(self, packed: GpuTensor, scales: GpuTensor, zeros: GpuTensor | None = None, *,
                 in_features: int, group: int = 128):
        if group not in (32, 64, 128):
            raise ValueError(f"group of {group} columns (32, 64 or 128)")
        if in_features < 1:
            raise ValueError(f"a 4-bit weight of {in_features} columns")
        if packed.ndim != 2 or packed.dtype not in (_U32, _I32):
            raise ValueError(f"packed must be 2-d uint32, got {packed.shape} {packed.dtype}")
        n = packed.shape[0]
        if packed.shape[1] != -(-in_features // 128) * 16:
            raise ValueError(f"packed rows of {packed.shape[1]} words for {in_features} columns")
        for t, name in ((scales, "scales"), (zeros, "zeros")):
            if t is not None and t.shape != (-(-in_features // group), n):
                raise ValueError(f"{name} must be {(-(-in_features // group), n)}, got {t.shape}")
        if zeros is not None and zeros.dtype != scales.dtype:
            raise TypeError(f"scales and zeros must share a dtype ({scales.dtype} vs {zeros.dtype})")
        _same_device(packed, scales, zeros)
        self.packed, self.scales, self.zeros = packed, scales, zeros
        self.in_features, self.out_features, self.group = int(in_features), n, int(group)

    @property
    def shape(self) -> tuple[int, int]:
        return (self.out_features, self.in_features)

    @property
    def device_id(self) -> int:
        return self.packed.device_id

    @classmethod
    def from_arrays(cls, q: np.ndarray, scales: np.ndarray, zeros: np.ndarray | None = None,
                    group: int = 128, device_id: int = -1) -> "W4Weight":
        """From host arrays as checkpoints hold them: ``q [N, K]`` in 0..15,
        ``scales`` and ``zeros`` ``[N, ceil(K / group)]``; packed on the host."""
        n, k = q.shape
        up = lambda a: gputensor_from_numpy(np.ascontiguousarray(a), device_id)  # noqa: E731
        return cls(up(pack_w4(q)), up(scales.T),
                   up(zeros.T) if zeros is not None else None, in_features=k, group=group)

    def to(self, target_dev: int) -> "W4Weight":
        """Copy on another device."""
        if self.device_id == target_dev:
            return self
        move = lambda t: gputensor_to_device(t, target_dev) if t is not None else None  # noqa: E731
        return W4Weight(move(self.packed), move(self.scales), move(self.zeros),
                        in_features=self.in_features, group=self.group)


def dev_quantize_w4(gt_weight: GpuTensor, group: int = 128, zeros: bool = False,
                    dtype=None) -> W4Weight:
    """Quantise an ``[N, K]`` weight to 4 bits on its device
    (``sf_quantize_w4``): scale max|w| / 7 around 8, or, with ``zeros``, scale
    and zero point of each group's range.  ``dtype``: type of the scales,
    that of the activations the weight will meet (default: the weight's)."""
    if gt_weight.ndim != 2:
        raise ValueError(f"weight must be [N, K], got {gt_weight.shape}")
    if group not in (32, 64, 128):
        raise ValueError(f"group of {group} columns (32, 64 or 128)")
    n, k = gt_weight.shape
    dev = gt_weight.device_id
    sdt = np.dtype(dtype) if dtype is not None else gt_weight.dtype
    words, groups = -(-k // 128) * 16, -(-k // group)
    packed = _alloc((n, words), np.uint32, dev)
    scales = _alloc((groups, n), sdt, dev)
    zs = _alloc((groups, n), sdt, dev) if zeros else None
    with E.on_device(dev):
        check(lib.sf_quantize_w4(n, k, _ptr(gt_weight), E.dtype_code(gt_weight.dtype), k, group,
                                 _ptr(packed), words, _ptr(scales), _ptr(zs), n,
                                 E.dtype_code(sdt), E.get_stream(dev)), "sf_quantize_w4")
    return W4Weight(packed, scales, zs, in_features=k, group=group)


def dev_dequantize_w4(weight: W4Weight, dtype=None) -> GpuTensor:
    """The ``[N, K]`` weight a W4Weight stands for, in ``dtype`` (default: its
    scales' type), each value rounded once."""
    n, k = weight.shape
    w = _alloc((n, k), np.dtype(dtype) if dtype is not None else weight.scales.dtype, weight.device_id)
    _dequantize_into(weight, w)
    return w


def _dequantize_into(weight: W4Weight, w: GpuTensor) -> None:
    n, k = weight.shape
    dev = weight.device_id
    with E.on_device(dev):
        check(lib.sf_dequantize_w4(n, k, _ptr(weight.packed), weight.packed.shape[1],
                                   _ptr(weight.scales), _ptr(weight.zeros), n, weight.group,
                                   E.dtype_code(weight.scales.dtype), _ptr(w), E.dtype_code(w.dtype), k,
                                   E.get_stream(dev)), "sf_dequantize_w4")


def dev_linear_w4(gt_x: GpuTensor, weight: W4Weight, gt_bias: GpuTensor | None = None,
                  activation: str = "none", out_dtype=None, out: GpuTensor | None = None) -> GpuTensor:
    """``dev_linear_forward`` over a 4-bit weight: ``act(x @ W^T + bias)`` for
    bf16 / fp16 x.  Up to 64 rows of x run on ``sf_linear_w4``, which streams
    the packed weight; more rows dequantise it into a 16-bit weight (one more
    rounding per weight, which the streamed product does not make) in the
    stream's workspace and run the GEMM.  During a graph capture more rows run
    64 at a time on ``sf_linear_w4`` instead: a graph must not hold the
    dequantised weight, whose memory the stream's next call uses again.
    ``out`` shares no memory with x, the bias or the weight."""
    act = E.act_code(activation)
    if gt_x.dtype != weight.scales.dtype:
        raise TypeError(f"x and the weight's scales must share a dtype ({gt_x.dtype} vs {weight.scales.dtype})")
    if gt_x.dtype == _F32:
        raise TypeError("4-bit linears take bf16 or fp16 x")
    n, k = weight.shape
    if gt_x.ndim < 1 or gt_x.shape[-1] != k:
        raise ValueError(f"linear shape mismatch: x {gt_x.shape}, W {weight.shape}")
    if gt_bias is not None and gt_bias.numel != n:
        raise ValueError(f"bias has {gt_bias.numel} elements, expected {n}")
    M = int(math.prod(gt_x.shape[:-1]))
    dev = _same_device(gt_x, weight.packed, gt_bias, out)
    _apart(out, gt_x, gt_bias, weight.packed, weight.scales, weight.zeros)
    odt = _out_dtype(gt_x, out_dtype if out is None else out.dtype)
    y = _result(out, gt_x.shape[:-1] + (n,), odt, dev, "out")
    bias_dt = E.dtype_code(gt_bias.dtype) if gt_bias is not None else DT_F32
    in_code, out_code = E.dtype_code(gt_x.dtype), E.dtype_code(odt)
    stream = E.get_stream(dev)
    with E.on_device(dev):
        if M <= _W4_MAX_ROWS or n == 0 or E.stream_capturing(stream):
            x_row, y_row = k * gt_x.dtype.itemsize, n * odt.itemsize
            for m0 in range(0, M, _W4_MAX_ROWS):
                check(lib.sf_linear_w4(min(M - m0, _W4_MAX_ROWS), n, k, gt_x.ptr + m0 * x_row, k,
                                       _ptr(weight.packed), weight.packed.shape[1],
                                       _ptr(weight.scales), _ptr(weight.zeros), n, weight.group,
                                       _ptr(gt_bias), bias_dt, y.ptr + m0 * y_row, n, in_code,
                                       out_code, act, stream), "sf_linear_w4")
        else:
            epi = E.make_epilogue(bias_ptr=gt_bias.ptr if gt_bias is not None else 0,
                                  bias_dt=bias_dt, act=act)
            with E.workspace_lock:
                buf = E.workspace(dev, stream, n * k * gt_x.dtype.itemsize, "weight")
                w = GpuTensor(buf, (n, k), gt_x.dtype, dev)
                _dequantize_into(weight, w)
                E.gemm(M, n, k, gt_x.ptr, k, 0, w.ptr, k, 1, y.ptr, n, in_code, out_code, epi=epi,
                       device=dev)
    return y


def dev_unsqueeze(gt: GpuTensor, dim: int) -> GpuTensor:
    shape = list(gt.shape)
    if dim < 0:
        dim = len(shape) + 1 + dim
    shape.insert(dim, 1)
    return GpuTensor(gt.buffer, tuple(shape), gt.dtype, gt.device_id)


def dev_squeeze(gt: GpuTensor, dim=None) -> GpuTensor:
    shape = list(gt.shape)
    if dim is not None:
        if dim < 0:
            dim = len(shape) + dim
        if 0 <= dim < len(shape) and shape[dim] == 1:
            shape.pop(dim)
    else:
        shape = [s for s in shape if s != 1]
    return GpuTensor(gt.buffer, tuple(shape), gt.dtype, gt.device_id)


def dev_reshape(gt: GpuTensor, new_shape) -> GpuTensor:
    new_shape = tuple(int(s) for s in new_shape)
    if -1 in new_shape:
        known = int(np.prod([s for s in new_shape if s != -1], dtype=np.int64))
        new_shape = tuple(gt.numel // known if s == -1 else s for s in new_shape)
    if int(np.prod(new_shape, dtype=np.int64)) != gt.numel:
        raise ValueError(f"cannot reshape {gt.shape} to {new_shape}")
    return GpuTensor(gt.buffer, new_shape, gt.dtype, gt.device_id)


# ───────────────────────────── host-array variants ─────────────────────────────

def _host_dtype(*arrs):
    dt = np.result_type(*[a.dtype for a in arrs])
    if dt not in (np.float16, np.float32) and not (bfloat16 is not None and dt == bfloat16):
        dt = np.dtype(np.float32)
    return dt


def cuda_matmul(a: np.ndarray, b: np.ndarray) -> np.ndarray:
    """Host C = A @ B through the device (``_cuda_ops.pyx:2120-2147``)."""
    dt = _host_dtype(a, b)
    ga = gputensor_from_numpy(np.ascontiguousarray(a, dtype=dt))
    gb = gputensor_from_numpy(np.ascontiguousarray(b, dtype=dt))
    return gputensor_to_numpy(dev_matmul(ga, gb))


def cuda_matmul_nt(a: np.ndarray, b: np.ndarray) -> np.ndarray:
    """Host C = A @ B^T (``_cuda_ops.pyx:2150-2177``)."""
    dt = _host_dtype(a, b)
    ga = gputensor_from_numpy(np.ascontiguousarray(a, dtype=dt))
    gb = gputensor_from_numpy(np.ascontiguousarray(b, dtype=dt))
    return gputensor_to_numpy(dev_matmul_nt(ga, gb))


def cuda_batched_matmul(a: np.ndarray, b: np.ndarray) -> np.ndarray:
    """Host batched (..., M, K) @ (..., K, N) (``_cuda_ops.pyx:2180-2225``)."""
    dt = _host_dtype(a, b)
    ga = gputensor_from_numpy(np.ascontiguousarray(a, dtype=dt))
    gb = gputensor_from_numpy(np.ascontiguousarray(b, dtype=dt))
    return gputensor_to_numpy(dev_batched_matmul(ga, gb))


def cuda_linear_forward(x: np.ndarray, weight: np.ndarray, bias: np.ndarray | None = None,
                        activation: str = "none") -> np.ndarray:
    """Host y = x @ W^T + bias (``_cuda_ops.pyx:2453-2471``), bias fused on the
    device instead of added in NumPy."""
    dt = _host_dtype(x, weight)
    K = x.shape[-1]
    gx = gputensor_from_numpy(np.ascontiguousarray(x.reshape(-1, K), dtype=dt))
    gw = gputensor_from_numpy(np.ascontiguousarray(weight, dtype=dt))
    gb = gputensor_from_numpy(np.ascontiguousarray(bias, dtype=dt).ravel()) if bias is not None else None
    y = gputensor_to_numpy(dev_linear_forward(gx, gw, gb, activation))
    return y.reshape(x.shape[:-1] + (weight.shape[0],))


def _host_unary(x: np.ndarray, fn) -> np.ndarray:
    """Host array -> device -> ``fn`` -> host, in the array's dtype (fp32 for
    anything the engine does not store), shape kept."""
    dt = _host_dtype(x)
    g = gputensor_from_numpy(np.ascontiguousarray(x, dtype=dt))
    return gputensor_to_numpy(fn(g)).reshape(np.shape(x))


def cuda_muls(a: np.ndarray, scalar: float) -> np.ndarray:
    """Host ``scalar * a`` through the device (``_cuda_ops.pyx:1926-1944``)."""
    return _host_unary(a, lambda g: dev_muls(g, scalar))


def cuda_silu(x: np.ndarray) -> np.ndarray:
    """Host SiLU through the device (``_cuda_ops.pyx:1954-1955``): the path
    ``F.silu`` takes for a ``cuda`` tensor without device data."""
    return _host_unary(x, dev_silu)


def cuda_gelu(x: np.ndarray) -> np.ndarray:
    """Host GELU-tanh through the device (``_cuda_ops.pyx:1957-1958``)."""
    return _host_unary(x, dev_gelu)


def cuda_softmax(x: np.ndarray, dim: int = -1) -> np.ndarray:
    """Host softmax over the last dimension (``_cuda_ops.pyx:2011-2040``)."""
    return _host_unary(x, lambda g: dev_softmax(g, -1))


def cuda_layer_norm(x: np.ndarray, gamma: np.ndarray | None, beta: np.ndarray | None,
                    eps: float = 1e-5) -> np.ndarray:
    """Host LayerNorm of an (N, D) array (``_cuda_ops.pyx:2231-2270``)."""
    g = gputensor_from_numpy(np.ascontiguousarray(x, dtype=np.float32))
    gg = gputensor_from_numpy(np.ascontiguousarray(gamma, dtype=np.float32)) if gamma is not None else None
    gb = gputensor_from_numpy(np.ascontiguousarray(beta, dtype=np.float32)) if beta is not None else None
    return gputensor_to_numpy(dev_layer_norm(g, gg, gb, eps))


def set_tf32_enabled(enable: bool) -> None:
    """``allow_tf32``: True permits single-pass TF32 for fp32 GEMMs; False
    (default) keeps fp32 accuracy via 3xTF32 (``_cuda_ops.pyx:2474-2477``)."""
    check(lib.sf_set_fp32_mode(FP32_TF32 if enable else FP32_ACCURATE), "sf_set_fp32_mode")


# ───────────────────────────── runtime ─────────────────────────────

def get_device_count() -> int:
    return E.device_count()


def set_device(device: int) -> None:
    E.set_device(device)


def get_current_device() -> int:
    return E.current_device()


def device_synchronize() -> None:
    check(lib.sf_device_synchronize(), "sf_device_synchronize")


def get_device_properties(device: int) -> dict:
    p = DeviceProps()
    check(lib.sf_device_properties(int(device), C.byref(p)), "sf_device_properties")
    return {
        "name": p.name.decode(errors="replace"),
        "total_memory": int(p.total_memory),
        "major": p.major,
        "minor": p.minor,
        "multi_processor_count": p.multi_processor_count,
        "shared_mem_per_block": int(p.shared_mem_per_block),
        "max_threads_per_block": p.max_threads_per_block,
        "warp_size": p.warp_size,
        "max_threads_per_mp": p.max_threads_per_mp,
        "l2_cache_size": int(p.l2_cache_size),
    }


def get_device_capability(device: int = 0) -> tuple[int, int]:
    p = get_device_properties(device)
    return (p["major"], p["minor"])


def get_device_name(device: int = 0) -> str:
    return get_device_properties(device)["name"]


def mem_info() -> tuple[int, int]:
    f, t = C.c_size_t(), C.c_size_t()
    check(lib.sf_mem_info(C.byref(f), C.byref(t)), "sf_mem_info")
    return (f.value, t.value)


def empty_cache(device: int = -1) -> None:
    E.release_workspaces()
    check(lib.sf_empty_cache(int(device)), "sf_empty_cache")


def gpu_malloc(nbytes: int) -> CudaBuffer:
    return _make_buffer(nbytes, E.current_device())


def gpu_free(buf: CudaBuffer) -> None:
    buf.free()


def can_access_peer(device: int, peer_device: int) -> bool:
    c = C.c_int32()
    check(lib.sf_can_access_peer(int(device), int(peer_device), C.byref(c)), "sf_can_access_peer")
    return bool(c.value)


def init_p2p() -> None:
    check(lib.sf_enable_peer_access_all(), "sf_enable_peer_access_all")


def init_all_devices() -> None:
    """Touch every device (engine state is created lazily) and enable P2P."""
    prev = E.current_device()
    for d in range(E.device_count()):
        E.set_device(d)
        E.device_error_status(d)
    E.set_device(prev)
    init_p2p()


class CudaStream:
    """Owned CUDA stream (``_cuda_ops.pyx:608-643``)."""

    def __init__(self, device_id: int = 0, non_blocking: bool = True):
        p = C.c_void_p()
        check(lib.sf_stream_create(int(device_id), 1 if non_blocking else 0, C.byref(p)),
              "sf_stream_create")
        self._stream = p.value
        self._device_id = device_id

    def synchronize(self) -> None:
        E.stream_sync(self._stream)

    def wait_event(self, event: "CudaEvent") -> None:
        check(lib.sf_stream_wait_event(C.c_void_p(self._stream), C.c_void_p(event._event)),
              "sf_stream_wait_event")

    @property
    def cuda_stream(self) -> int:
        return self._stream

    @property
    def device_id(self) -> int:
        return self._device_id

    def __del__(self):
        try:
            if self._stream:
                try:
                    E.release_stream(self._stream)
                finally:
                    lib.sf_stream_destroy(C.c_void_p(self._stream))
                    self._stream = None
        except Exception:
            pass


class CudaEvent:
    """CUDA event for timing / sync (``_cuda_ops.pyx:646-673``)."""

    def __init__(self, enable_timing: bool = True):
        p = C.c_void_p()
        check(lib.sf_event_create(1 if enable_timing else 0, C.byref(p)), "sf_event_create")
        self._event = p.value

    def record(self, stream: CudaStream | None = None) -> None:
        s = stream._stream if stream is not None else E.get_stream(E.current_device())
        check(lib.sf_event_record(C.c_void_p(self._event), C.c_void_p(s) if s else None),
              "sf_event_record")

    def synchronize(self) -> None:
        check(lib.sf_event_synchronize(C.c_void_p(self._event)), "sf_event_synchronize")

    def elapsed_time(self, end: "CudaEvent") -> float:
        ms = C.c_float()
        check(lib.sf_event_elapsed_ms(C.c_void_p(self._event), C.c_void_p(end._event),
                                      C.byref(ms)), "sf_event_elapsed_ms")
        return ms.value

    def __del__(self):
        try:
            if self._event:
                lib.sf_event_destroy(C.c_void_p(self._event))
                self._event = None
        except Exception:
            pass


def cublas_set_stream(stream: CudaStream | None = None) -> None:
    """Route subsequent engine launches on the current device to ``stream``
    (the reference set the cuBLAS handle's stream, ``_cuda_ops.pyx:725-729``)."""
    E.set_stream(E.current_device(), stream._stream if stream is not None else None)


# ───────────────────────────── out of scope ─────────────────────────────

_OUT_OF_SCOPE = {
    "dev_exp", "dev_log", "dev_sqrt", "dev_rsqrt", "dev_sigmoid", "dev_tanh", "dev_sin",
    "dev_cos", "dev_neg", "dev_abs", "dev_relu", "dev_add", "dev_sub", "dev_mul", "dev_div",
    "dev_adds", "dev_clamp", "dev_log_softmax", "dev_cross_entropy",
    "dev_rms_norm", "dev_dropout", "dev_embedding", "dev_adamw_step", "dev_sum", "dev_fill",
    "dev_copy", "dev_transpose_2d", "dev_pow_scalar", "dev_expand", "dev_slice", "dev_cat",
    "dev_stack", "dev_chunk", "dev_cumsum", "dev_mean_dim", "dev_sum_dim", "dev_sum_tensor",
    "dev_mean_tensor", "cuda_exp", "cuda_log", "cuda_sqrt", "cuda_rsqrt", "cuda_sigmoid",
    "cuda_tanh", "cuda_sin", "cuda_cos", "cuda_neg", "cuda_abs", "cuda_add", "cuda_sub",
    "cuda_mul", "cuda_div", "cuda_adds", "cuda_relu",
    "cuda_silu_fwd", "cuda_clamp", "cuda_log_softmax", "cuda_cross_entropy",
    "cuda_rms_norm", "cuda_adamw_step", "cuda_dropout", "cuda_embedding",
    "cuda_transpose_2d", "cuda_sum", "cuda_fill",
}


def __getattr__(name: str):
    if name in _OUT_OF_SCOPE:
        def _missing(*_a, **_k):
            raise NotImplementedError(
                f"_cuda_ops.{name} is outside the B200 engine's matmul path "
                "(only the GEMM / linear / attention-product surface is provided)")
        _missing.__name__ = name
        return _missing
    raise AttributeError(name)
