"""Faults of the routed and the 4-bit linears that the host alone decides:
refused shapes, shared memory, the order of launches.  CPU only: the engine's
entry points are stood in for where a call would reach a device."""
import threading

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


class _Engine:
    """Stands in for the entry points behind the engine's launches and memory:
    a log of (call, thread, what), and memory that is only addresses."""

    def __init__(self, monkeypatch):
        from scaffolding_b200._lib import lib
        self.lib, self.log, self.mu = lib, [], threading.Lock()
        self.next, self.freed, self.capture_id = 1 << 20, {}, {}
        self.patch = lambda name, fn: monkeypatch.setattr(lib, name, fn)
        self.patch("sf_malloc", self._malloc)
        self.patch("sf_free", self._free)
        self.patch("sf_get_device", lambda out: self._set(out, 0))
        self.patch("sf_set_device", lambda dev: 0)
        self.patch("sf_device_synchronize", lambda: self.note("device sync", None))
        self.patch("sf_stream_synchronize", lambda s: self.note("sync", s))
        if hasattr(lib, "sf_stream_capture_id"):
            self.patch("sf_stream_capture_id", lambda s, out: self._set(out, self.capture_id.get(s, 0)))

    @staticmethod
    def _set(out, value):
        out._obj.value = value
        return 0

    def note(self, call, what):
        with self.mu:
            self.log.append((call, threading.get_ident(), what))
        return 0

    def _malloc(self, dev, nbytes, out):
        """The pool's rule: a freed block of the same size comes back first."""
        with self.mu:
            size = -(-max(nbytes, 1) // 256) * 256
            if self.freed.get(size):
                return self._set(out, self.freed[size].pop())
            p, self.next = self.next, self.next + size
        return self._set(out, p)

    def _free(self, dev, p, nbytes):
        size = -(-max(nbytes, 1) // 256) * 256
        with self.mu:
            self.freed.setdefault(size, []).append(p.value)
            self.log.append(("free", threading.get_ident(), p.value))
        return 0


@pytest.fixture
def engine(monkeypatch):
    from scaffolding_b200 import engine as E
    monkeypatch.setattr(E, "_workspaces", {})
    if hasattr(E, "_captured"):
        monkeypatch.setattr(E, "_captured", {})
    monkeypatch.setattr(E, "_streams", {})
    return _Engine(monkeypatch)


def _grouped_needs(engine, nbytes):
    engine.patch("sf_gemm_grouped_workspace_size", lambda X, M, N, K, dt, s, out: engine._set(out, nbytes(M)))


def _two_threads(first, second, inside):
    """Runs ``first`` until ``inside`` is set within it, then ``second`` beside it."""
    errors = []

    def guarded(fn):
        try:
            fn()
        except BaseException as e:  # noqa: BLE001 - reported below
            errors.append(e)

    a = threading.Thread(target=guarded, args=(first,))
    b = threading.Thread(target=guarded, args=(second,))
    a.start()
    assert inside.wait(10)
    b.start()
    a.join(20)
    b.join(20)
    assert not a.is_alive() and not b.is_alive() and not errors, errors


@pytest.mark.parametrize("grow", [False, True])
def test_gathered_rows_of_two_threads(ops, engine, grow):
    """A gathered batch makes two launches through the stream's workspace: no
    other thread's launch comes between them, and none frees it for a larger
    one while the first has its address."""
    inside, done = threading.Event(), threading.Event()

    def launch(X, M, N, K, *rest):
        ws = rest[16]
        engine.note("enter", ws)
        if not inside.is_set():
            inside.set()
            done.wait(0.5)  # room for the other thread to come between
        engine.note("leave", ws)
        done.set()
        return 0

    engine.patch("sf_gemm_grouped", launch)
    _grouped_needs(engine, lambda M: M * 32)
    w, off = _fake(ops, (3, 8, 16), F16), _fake(ops, (4,), I32)

    def call(M):
        ops.dev_grouped_linear(_fake(ops, (10, 16), F16), w, off, rows=_fake(ops, (M,), I32),
                               out=ops.GpuTensor(ops.CudaBuffer(64, 16, 0, False), (M, 8), F16, 0))

    _two_threads(lambda: call(3000), lambda: call(9000 if grow else 3000), inside)
    seen = [(c, t) for c, t, _ in engine.log if c in ("enter", "leave", "free")]
    first = seen[0][1]
    end = seen.index(("leave", first))
    assert seen[0][0] == "enter" and all(t == first for _, t in seen[:end]), seen


def test_split_k_of_two_threads(ops, engine):
    """The same rule for a GEMM whose split-K sums lie in the workspace."""
    from scaffolding_b200 import engine as E
    inside, done = threading.Event(), threading.Event()

    def launch(*args):
        engine.note("enter", None)
        if not inside.is_set():
            inside.set()
            done.wait(0.5)
        engine.note("leave", None)
        done.set()
        return 0

    engine.patch("sf_gemm", launch)
    engine.patch("sf_gemm_workspace_size", lambda *a: engine._set(a[-1], a[1] * 64))

    def call(M):
        E.gemm(M, 8, 8, 64, 8, 0, 64, 8, 1, 64, 8, 0, 0, device=0)

    _two_threads(lambda: call(4), lambda: call(400), inside)
    seen = [(c, t) for c, t, _ in engine.log if c in ("enter", "leave", "free")]
    end = seen.index(("leave", seen[0][1]))
    assert all(t == seen[0][1] for _, t in seen[:end]), seen


def test_released_workspaces_are_not_in_use(engine):
    """A workspace goes back to the pool only when no queued launch reads it."""
    from scaffolding_b200 import engine as E
    with E.workspace_lock:
        ptr = E.workspace(0, 77, 4096).ptr
    E.release_workspaces()
    calls = [(c, what) for c, _, what in engine.log]
    assert ("free", ptr) in calls and calls.index(("device sync", None)) < calls.index(("free", ptr))
    assert not E._workspaces


def _w4(ops, N=6, K=256, group=64, dt=F16):
    G = -(-K // group)
    return ops.W4Weight(_fake(ops, (N, K // 8), np.uint32), _fake(ops, (G, N), dt), in_features=K, group=group)


def test_unpacked_weight_stays_out_of_the_pool(ops, engine):
    """More than 64 rows: the 16-bit weight is read by a product that is only
    queued when the call returns, so its memory must not go back to the pool,
    where an upload outside the stream's order could take it."""
    used = {}

    def dequantize(N, K, packed, ldp, scales, zeros, lds, group, sdt, W, wdt, ldw, stream):
        used["written"] = W
        return 0

    def gemm(M, N, K, A, lda, ta, B, *rest):
        used["read"] = B
        return 0

    value = lambda p: p.value if hasattr(p, "value") else p  # noqa: E731
    engine.patch("sf_stream_is_capturing", lambda s, out: engine._set(out, 0))
    engine.patch("sf_dequantize_w4", dequantize)
    engine.patch("sf_gemm", gemm)
    engine.patch("sf_gemm_workspace_size", lambda *a: engine._set(a[-1], 6 * 256 * 2))
    y = ops.dev_linear_w4(_fake(ops, (70, 256), F16), _w4(ops))
    assert y.shape == (70, 6) and value(used["written"]) == value(used["read"])
    assert all(p != value(used["read"]) for c, _, p in engine.log if c == "free")
    assert ops._alloc((6, 256), F16, 0).ptr != value(used["read"])
    # and it is not the product's own workspace, of the same size here
    from scaffolding_b200 import engine as E
    assert sorted(b.ptr for b in E._workspaces.values()).count(value(used["read"])) == 1 and len(E._workspaces) == 2


def test_uploads_keep_the_streams_order(ops, engine):
    """New memory may be what a dropped intermediate of queued work had: what
    is copied into it is ordered behind that work, on the engine's stream (and is
    no part of a graph that is being captured there)."""
    from scaffolding_b200 import engine as E
    engine.patch("sf_memcpy", lambda dst, src, n, kind, s: engine.note("copy", s if s is None else getattr(s, "value", s)))
    engine.patch("sf_memcpy_peer", lambda d, dd, s, sd, n, st: engine.note("copy", getattr(st, "value", st)))
    for stream, capturing, where in ((None, 0, None), (77, 0, 77), (77, 1, None)):
        engine.patch("sf_stream_is_capturing", lambda s, out: engine._set(out, capturing))
        E.set_stream(0, stream)
        engine.log.clear()
        ops.gputensor_from_numpy(np.zeros(8, F32), 0)
        ops._rebuild_cuda_buffer(np.zeros(8, np.uint8), 0)
        ops.gputensor_to_device(_fake(ops, (8,), dev=1), 0)
        assert [what for c, _, what in engine.log if c == "copy"] == [where] * 3
        last = [c for c, _, _ in engine.log if c in ("copy", "sync")]
        assert last[-1] == "sync" and last.count("sync") >= 3  # the source may be reused when a call returns


def test_captures_have_workspaces_of_their_own(engine):
    """A graph uses its workspaces at every replay, beside other calls and
    graphs of the stream it was captured on: none is another's, and none is
    freed for a larger one or by empty_cache."""
    from scaffolding_b200 import engine as E
    ws = lambda n: E.workspace(0, 77, n).ptr  # noqa: E731
    direct = ws(1000)
    engine.capture_id[77] = 5
    first = [ws(1000), ws(1000), ws(9000)]
    engine.capture_id[77] = 6
    second = ws(1000)
    engine.capture_id[77] = 0
    assert ws(1000) == direct and first[0] == first[1]
    assert len({direct, first[0], first[2], second}) == 4
    ws(50000)  # the stream's own grows
    E.release_workspaces()
    freed = [what for c, _, what in engine.log if c == "free"]
    assert direct in freed and not {first[0], first[2], second} & set(freed)
    E.release_workspaces(captured=True)
    freed = [what for c, _, what in engine.log if c == "free"]
    assert {first[0], first[2], second} <= set(freed)


def _moe_engine(engine):
    """Records what the four steps of nn.MoE write: (step, address)."""
    value = lambda p: getattr(p, "value", p)  # noqa: E731
    wrote = []

    def note(step, *ptrs):
        wrote.extend((step, value(p)) for p in ptrs)
        return 0

    engine.patch("sf_stream_is_capturing", lambda s, out: engine._set(out, 1 if engine.capture_id.get(s) else 0))
    engine.patch("sf_gemm_workspace_size", lambda *a: engine._set(a[-1], 0))
    engine.patch("sf_gemm", lambda M, N, K, A, lda, ta, B, ldb, tb, Cp, *r: note("logits", Cp))
    engine.patch("sf_moe_route", lambda T, X, k, z, dt, ld, rn, e, w, o, r, s, ws, n, st: note("route", e, w, o, r, s, ws))
    _grouped_needs(engine, lambda M: 0)
    engine.patch("sf_gemm_grouped", lambda *a: note("product", a[15]))
    engine.patch("sf_moe_combine", lambda *a: note("combine", a[11]))
    return wrote


def test_moe_intermediates_stay_out_of_the_pool(ops, engine):
    """What nn.MoE's steps hand to each other is read by launches that are only
    queued, or captured, when it returns: none of that memory goes back to the
    pool, and a capture's is not that of later direct calls."""
    from scaffolding_b200 import engine as E
    from scaffolding_b200 import nn
    wrote = _moe_engine(engine)
    m = _moe(ops, nn, dtype=F16)
    E.set_stream(0, 77)
    engine.capture_id[77] = 3
    held = m(_fake(ops, (300, 64), F16))
    captured = {p for step, p in wrote if step != "combine"}
    assert len(captured) == 9 and 0 not in captured  # logits, five of the route and its counts, two products
    assert not [p for c, _, p in engine.log if c == "free" and p in captured]
    engine.capture_id[77] = 0
    wrote.clear()
    m(_fake(ops, (300, 64), F16))
    m(_fake(ops, (2000, 64), F16))
    assert not captured & {p for _, p in wrote} and held.shape == (300, 64)
    spans = [(b.ptr, b.ptr + b.nbytes) for bufs in E._captured.values() for b in bufs]
    assert all(any(lo <= p < hi for lo, hi in spans) for p in captured)


def test_modules_write_into_kept_results(ops, engine):
    """out= of nn.MoE and nn.Linear4, and its refusals."""
    from scaffolding_b200 import nn
    wrote = _moe_engine(engine)
    m = _moe(ops, nn, dtype=F16)
    out = ops.GpuTensor(ops.CudaBuffer(512, 2 * 20 * 64, 0, False), (4, 5, 64), F16, 0)
    x = ops.GpuTensor(ops.CudaBuffer(1 << 16, 2 * 20 * 64, 0, False), (4, 5, 64), F16, 0)
    assert m(x, out=out) is out and wrote[-1] == ("combine", 512)
    assert m(x, x, out=x) is x and wrote[-1] == ("combine", 1 << 16)
    for bad in (_fake(ops, (20, 64), F16), _fake(ops, (4, 5, 64))):
        with pytest.raises(ValueError, match="out must be"):
            m(x, out=bad)
    for name in ("router", "up", "down"):  # read before the result is written, but kept by the layer
        kept = getattr(m, name)
        setattr(m, name, ops.GpuTensor(ops.CudaBuffer(500, 64, 0, False), kept.shape, F16, 0))
        with pytest.raises(ValueError, match="share memory"):
            m(x, out=out)
        setattr(m, name, kept)
    engine.patch("sf_linear_w4", lambda *a: engine.note("y", a[13]))
    lin = nn.Linear4(_w4(ops, N=64))
    x = ops.GpuTensor(ops.CudaBuffer(1 << 16, 4096, 0, False), (4, 5, 256), F16, 0)
    assert lin(x, out=out) is out and engine.log[-1][2] == 512


def _at(ops, lo, shape, dtype=F32):
    n = int(np.prod(shape)) * np.dtype(dtype).itemsize
    return ops.GpuTensor(ops.CudaBuffer(lo, n, 0, False), shape, dtype, 0)


def test_results_share_no_memory_with_any_input(ops):
    """By address: views of one allocation are different buffers."""
    from scaffolding_b200.parallel import row_slice
    share = pytest.raises(ValueError, match="share memory")
    # rows 8.. of an allocation as the result, rows 0..11 as the input
    whole = _at(ops, 4096, (24, 16), F16)
    x, out = row_slice(whole, 0, 12), row_slice(whole, 8, 20)
    w, off = _at(ops, 1 << 20, (2, 16, 16), F16), _at(ops, 1 << 21, (3,), I32)
    with share:
        ops.dev_grouped_linear(x, w, off, out=out)
    y = _at(ops, 4096, (12, 16), F16)
    for name, t in (("offsets", _at(ops, 4096 + 32, (3,), I32)), ("bias", _at(ops, 4096, (2, 16), F16)),
                    ("rows", _at(ops, 4096 + 300, (12,), I32)), ("weight", _at(ops, 4096, (2, 16, 16), F16))):
        with share:
            ops.dev_grouped_linear(_at(ops, 1 << 19, (12, 16), F16), t if name == "weight" else w,
                                   t if name == "offsets" else off, t if name == "bias" else None,
                                   rows=t if name == "rows" else None, out=y)
    s, p = _at(ops, 1 << 20, (4, 3), I32), _at(ops, 1 << 21, (4, 3))
    e = _at(ops, 4096, (4, 16))
    for args in ((_at(ops, 4000, (12, 16)), s, p), (_at(ops, 1 << 18, (12, 16)), _at(ops, 4096, (4, 3), I32), p),
                 (_at(ops, 1 << 18, (12, 16)), s, _at(ops, 4100, (4, 3)))):
        with share:
            ops.dev_moe_combine(*args, out=e)
    with share:  # a residual is the result's memory or none of it
        ops.dev_moe_combine(_at(ops, 1 << 18, (12, 16)), s, p, _at(ops, 4096 + 64, (4, 16)), out=e)
    z = _at(ops, 4096, (4, 128), F16)
    packed, scales, zeros = _at(ops, 1 << 20, (128, 16), np.uint32), _at(ops, 1 << 21, (2, 128), F16), None
    for name, t in (("packed", _at(ops, 4090, (128, 16), np.uint32)), ("scales", _at(ops, 4096, (2, 128), F16)),
                    ("zeros", _at(ops, 4608, (2, 128), F16)), ("x", _at(ops, 4096 + 1000, (4, 128), F16))):
        w4 = ops.W4Weight(t if name == "packed" else packed, t if name == "scales" else scales,
                          t if name == "zeros" else zeros, in_features=128, group=64)
        with share:
            ops.dev_linear_w4(t if name == "x" else _at(ops, 1 << 18, (4, 128), F16), w4, out=z)
    r = ops.MoeRoute(_at(ops, 1 << 20, (4, 2), I32), _at(ops, 1 << 21, (4, 2)), _at(ops, 1 << 22, (9,), I32),
                     _at(ops, 4096, (8,), I32), _at(ops, 1 << 23, (4, 2), I32))
    with share:
        ops.dev_moe_route(_at(ops, 4096 + 16, (4, 8)), 2, out=r)


def test_result_next_to_an_input(ops, engine):
    """Neighbours in one allocation are apart."""
    engine.patch("sf_moe_combine", lambda *a: engine.note("combine", a[11]))
    e = _at(ops, 4096, (4, 16))
    args = _at(ops, 4096 + 256, (12, 16)), _at(ops, 4096 - 48, (4, 3), I32), _at(ops, 1 << 21, (4, 3))
    assert ops.dev_moe_combine(*args, out=e) is e
    assert ops.dev_moe_combine(*args, _at(ops, 4096, (4, 16)), out=e) is e


def test_route_leaves_room_for_its_index_arithmetic():
    """A block's chunk of up to 2^22 tokens may end past the last token: that
    end is a 32-bit number too."""
    import ctypes as C

    from scaffolding_b200._lib import SF_ERR_UNSUPPORTED as NO, lib
    sz = C.c_size_t()
    most = (1 << 31) - (1 << 23) - 1
    for k in (1, 2, 32):
        assert lib.sf_moe_route_workspace_size(most // k, 64, k, C.byref(sz)) == 0
        for tokens in (most // k + 1, ((1 << 31) - 1) // k):
            assert lib.sf_moe_route_workspace_size(tokens, 64, k, C.byref(sz)) == NO
    assert lib.sf_moe_route_workspace_size(most, 64, 1, C.byref(sz)) == 0
    blocks = sz.value // (64 * 4)
    chunk = -(-most // 512)
    assert blocks == -(-most // chunk) and blocks * chunk + 16 * 4 < 1 << 31


def test_a_streams_workspaces_go_with_it(ops, engine):
    """A destroyed stream's workspaces return to the pool, waited for: another
    stream may come to have its address."""
    from scaffolding_b200 import engine as E
    engine.patch("sf_stream_create", lambda dev, nb, out: engine._set(out, 4242))
    engine.patch("sf_stream_destroy", lambda s: engine.note("destroy", getattr(s, "value", s)))
    s = ops.CudaStream(0)
    mine, legacy = E.workspace(0, s.cuda_stream, 100).ptr, E.workspace(0, None, 100).ptr
    more = E.workspace(0, s.cuda_stream, 100, "weight").ptr
    engine.capture_id[4242] = 9
    graphs = E.workspace(0, s.cuda_stream, 100).ptr
    engine.capture_id[4242] = 0
    del s
    calls = [(c, getattr(what, "value", what)) for c, _, what in engine.log]
    freed = [p for c, p in calls if c == "free"]
    assert sorted(freed) == sorted([mine, more]) and graphs not in freed and legacy not in freed
    assert calls.index(("sync", 4242)) < calls.index(("free", mine)) and ("destroy", 4242) in calls
    assert list(E._workspaces) == [(0, 0, "sums")]


def test_packing_refuses_what_is_no_whole_number(ops):
    """Values that 4 bits do not hold are not cut to ones that they do."""
    for bad in ([[1.5]], [[np.nan]], [[np.inf]], [[16.0]], [[-1]], [["3"]], [[2 + 0j]]):
        with pytest.raises(ValueError, match="0..15"):
            ops.pack_w4(np.array(bad))
    for dtype in (np.uint8, np.int64, np.float32, np.float16, ops.bfloat16, bool):
        q = np.array([[1, 0] * 70], dtype)
        assert np.array_equal(ops.pack_w4(q), ops.pack_w4(q.astype(np.uint8)))
    assert ops.pack_w4(np.zeros((0, 5), np.uint8)).shape == (0, 16)


def test_outgrown_workspace_waits_on_its_device(engine):
    """The legacy stream that is waited for is that of the workspace's device,
    whichever device is current."""
    from scaffolding_b200 import engine as E
    current = [0]

    def set_device(dev):
        current[0] = dev
        return 0

    engine.patch("sf_get_device", lambda out: engine._set(out, current[0]))
    engine.patch("sf_set_device", set_device)
    engine.patch("sf_stream_synchronize", lambda s: engine.note("sync on", current[0]))
    E.workspace(1, None, 100)
    E.workspace(1, None, 9000)
    assert [what for c, _, what in engine.log if c == "sync on"] == [1] and current == [0]


def test_w4_leaves_room_for_its_index_arithmetic():
    """Row and column numbers rounded up to a tile are 32-bit numbers too (the
    addresses are never read: the refusals, and an empty x, come first)."""
    import ctypes as C

    from scaffolding_b200._lib import SF_ERR_UNSUPPORTED as NO, lib
    p = C.c_void_p(4096)
    most = (1 << 31) - 4097

    def call(N, K):
        return lib.sf_linear_w4(0, N, K, p, K, p, -(-K // 128) * 16, p, None, N, 128, None, 0, p, N, 2, 2, 0, None)

    assert call(most, 128) == 0 and call(8, most) == 0
    for N, K in ((most + 1, 128), ((1 << 31) - 1, 128), (8, most + 1), (8, (1 << 31) - 128)):
        assert call(N, K) == NO


def test_combine_into_a_residual_of_another_stride():
    """In place means row on row: with other strides one token's result would
    be written over another's residual."""
    import ctypes as C

    from scaffolding_b200._lib import SF_ERR_INVALID_ARGUMENT as BAD, lib
    p, r = C.c_void_p(4096), C.c_void_p(1 << 20)

    def call(tokens, ldr, ldo):
        return lib.sf_moe_combine(tokens, 8, 2, p, 8, 8, 2, p, p, r, ldr, r, ldo, None)

    assert call(2, 8, 16) == BAD and call(5, 24, 8) == BAD


def test_workspace_after_running_out_of_memory(engine):
    """A growth that fails leaves no freed buffer behind for smaller calls."""
    from scaffolding_b200 import engine as E
    from scaffolding_b200._lib import EngineError
    E.workspace(0, None, 100)
    malloc = engine._malloc
    engine.patch("sf_malloc", lambda dev, n, out: -4 if n > 1000 else malloc(dev, n, out))
    with pytest.raises(EngineError):
        E.workspace(0, None, 5000)
    buf = E.workspace(0, None, 100)
    assert buf.ptr and buf.nbytes >= 100
