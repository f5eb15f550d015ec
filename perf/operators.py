"""The linears of a sparse (mixture-of-experts) layer: cases, inputs, plain forms and work.

Four operators, each as a case's "op":

  route     the router: top-k experts of every token, their weights, and the
            choices grouped by expert (ops.dev_moe_route)
  grouped   one linear per expert over the rows grouped by expert
            (ops.dev_grouped_linear)
  combine   the weighted sum of a token's expert rows (ops.dev_moe_combine)
  w4        a linear with 4-bit weights and group scales for few rows
            (ops.dev_linear_w4)

Where ``own`` is false, ``run`` computes the plain form with elementary torch
operations in 32 bits; where it is true, it calls the framework's operators.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ───────────────────────────── cases ─────────────────────────────

def listed():
    return [
        # One token in decoding: two of eight experts, first product with SiLU.
        dict(name="grouped one token", op="grouped", tokens=1, top_k=2, experts=8, K=1024, N=4096,
             dtype="bf16", act="silu", bias=False, gather=True, skew=0.0),
        # A decoding batch of 64 over 64 experts with gated first products: a few rows each.
        dict(name="grouped decode gated", op="grouped", tokens=64, top_k=4, experts=64, K=2048,
             N=1408, dtype="bf16", act="silu_gate", bias=False, gather=True, skew=0.5),
        # A ragged prompt batch, second products (rows already grouped), an odd width, fp16.
        dict(name="grouped prompt down", op="grouped", tokens=1003, top_k=2, experts=16, K=7680,
             N=1923, dtype="f16", act="none", bias=True, gather=False, skew=1.0),
        # The widths of the DiT block and the tokens of one of its samples, two experts each.
        dict(name="grouped large", op="grouped", tokens=17776, top_k=2, experts=8, K=1920, N=7680,
             dtype="bf16", act="gelu_tanh", bias=True, gather=True, skew=0.5),
        # Single-token projections.
        dict(name="w4 one row", op="w4", M=1, N=4096, K=4096, group=128, dtype="bf16", zeros=False,
             bias=False, act="none"),
        dict(name="w4 eight rows down", op="w4", M=8, N=4096, K=11008, group=32, dtype="f16",
             zeros=True, bias=True, act="none"),
        # A wide first product for a few sequences, an odd count.
        dict(name="w4 wide", op="w4", M=5, N=28672, K=8192, group=128, dtype="bf16", zeros=False,
             bias=False, act="silu"),
        # The most rows that are still served as a weight stream.
        dict(name="w4 many rows", op="w4", M=64, N=11008, K=4096, group=64, dtype="bf16",
             zeros=True, bias=True, act="gelu_tanh"),
        # Router of a decoding batch (16-bit logits: ties happen) and of a long prompt.
        dict(name="route decode", op="route", tokens=64, top_k=4, experts=64, dtype="bf16",
             renormalize=True),
        dict(name="route prompt", op="route", tokens=17776, top_k=2, experts=64, dtype="f32",
             renormalize=False),
        # The way back, for the same two.
        dict(name="combine decode", op="combine", tokens=64, top_k=4, C=2048, dtype="bf16",
             residual=True),
        dict(name="combine prompt", op="combine", tokens=17776, top_k=2, C=1920, dtype="bf16",
             residual=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["grouped", "grouped", "w4", "w4", "route", "combine"])
    if op == "grouped":
        experts = _log(rng, 4, 64)
        act = rng.choice(["none", "silu", "gelu_tanh", "silu_gate"])
        K, N = 8 * _log(rng, 16, 960), _log(rng, 100, 7680)
        wide = 2 if act == "silu_gate" else 1
        N = max(100, min(N, 360_000_000 // (experts * K * wide)))
        top_k = rng.randint(1, 4)
        tokens = _log(rng, 1, 17776)
        tokens = max(1, min(tokens, int(1.0e12 / (2.0 * top_k * N * K * wide))))
        return dict(op=op, tokens=tokens, top_k=top_k, experts=experts, K=K, N=N,
                    dtype=rng.choice(["bf16", "f16"]), act=act, bias=rng.random() < 0.5,
                    gather=rng.random() < 0.5, skew=round(rng.uniform(0.0, 1.0), 2))
    if op == "w4":
        return dict(op=op, M=_log(rng, 1, 64), N=_log(rng, 100, 11008), K=8 * _log(rng, 16, 1376),
                    group=rng.choice([32, 64, 128]), dtype=rng.choice(["bf16", "f16"]),
                    zeros=rng.random() < 0.5, bias=rng.random() < 0.5,
                    act=rng.choice(["none", "silu", "gelu_tanh"]))
    if op == "route":
        experts = _log(rng, 2, 256)
        return dict(op=op, tokens=_log(rng, 1, 17776), top_k=rng.randint(1, min(8, experts)),
                    experts=experts, dtype=rng.choice(["bf16", "f16", "f32"]),
                    renormalize=rng.random() < 0.5)
    return dict(op=op, tokens=_log(rng, 1, 17776), top_k=rng.randint(1, 2), C=_log(rng, 64, 1920),
                dtype=rng.choice(["bf16", "f16", "f32"]), residual=rng.random() < 0.5)


# ───────────────────────────── inputs ─────────────────────────────

def _choices(logits, top_k):
    """Experts of every token (falling logit, ties to the lowest index) and
    the choices grouped by expert: (experts, offsets, rows, slots, expert of
    each slot)."""
    tokens, experts = logits.shape
    chosen = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :top_k]
    flat = chosen.reshape(-1)
    of_slot, order = torch.sort(flat, stable=True)
    counts = torch.bincount(flat, minlength=experts)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    slots = torch.empty_like(order)
    slots[order] = torch.arange(order.numel(), device=order.device)
    i32 = torch.int32
    return (chosen.to(i32), offsets.to(i32), (order // top_k).to(i32),
            slots.reshape(tokens, top_k).to(i32), of_slot)


def _pack_order(device):
    """Column of nibble i of word 4*t + w in a block of 128 columns:
    32*w + 8*t + (0, 2, 4, 6, 1, 3, 5, 7)[i], as [16, 8]."""
    word = torch.arange(16, device=device)
    t, w = word // 4, word % 4
    nib = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7], device=device)
    return (32 * w + 8 * t)[:, None] + nib[None, :]


def _pack(q):
    """[N, K] values 0..15 -> packed [N, 16 * ceil(K / 128)] int32 words."""
    N, K = q.shape
    blocks = -(-K // 128)
    q = torch.nn.functional.pad(q, (0, blocks * 128 - K))
    q = q.reshape(N, blocks, 128)[:, :, _pack_order(q.device)]
    shift = 4 * torch.arange(8, device=q.device)
    words = (q.to(torch.int64) << shift).sum(-1)
    words = torch.where(words >= 1 << 31, words - (1 << 32), words)
    return words.to(torch.int32).reshape(N, blocks * 16)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed) * 1000003 + 17)

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    def uniform(*shape):
        return torch.rand(*shape, device=dev, generator=g)

    op, dt = case["op"], DTYPES[case["dtype"]]
    s = {"case": case}
    if op == "route":
        s["logits"] = normal(case["tokens"], case["experts"]).to(dt)
        return s
    if op == "w4":
        M, N, K, group = case["M"], case["N"], case["K"], case["group"]
        groups = -(-K // group)
        s["x"] = normal(M, K).to(dt)
        s["packed"] = _pack(torch.randint(0, 16, (N, K), device=dev, generator=g, dtype=torch.uint8))
        # scales such that the weights look like U(-1/sqrt(K), 1/sqrt(K))
        s["scales"] = ((0.5 + uniform(groups, N)) / (8 * math.sqrt(K))).to(dt)
        s["zeros"] = (torch.randint(5, 11, (groups, N), device=dev, generator=g).to(dt)
                      if case["zeros"] else None)
        s["bias"] = ((2 * uniform(N) - 1) / math.sqrt(K)).to(dt) if case["bias"] else None
        return s
    tokens, top_k = case["tokens"], case["top_k"]
    if op == "combine":
        experts = max(8, top_k)
        logits = normal(tokens, experts)
        s["slots"] = _choices(logits, top_k)[3]
        s["weights"] = torch.softmax(torch.topk(logits, top_k, dim=1).values, dim=1)
        s["y"] = normal(tokens * top_k, case["C"]).to(dt)
        s["residual"] = normal(tokens, case["C"]).to(dt) if case["residual"] else None
        return s
    experts, K, N = case["experts"], case["K"], case["N"]
    wide = 2 if case["act"] == "silu_gate" else 1
    logits = normal(tokens, experts) + case["skew"] * normal(experts)
    _, s["offsets"], rows, _, s["of_slot"] = _choices(logits, min(top_k, experts))
    s["most"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())
    s["rows"] = rows if case["gather"] else None
    s["x"] = normal(tokens if case["gather"] else rows.numel(), K).to(dt)
    s["weight"] = torch.empty(experts, wide * N, K, device=dev, dtype=dt)
    s["weight"].uniform_(-1 / math.sqrt(K), 1 / math.sqrt(K), generator=g)
    s["bias"] = (((2 * uniform(experts, wide * N) - 1) / math.sqrt(K)).to(dt) if case["bias"] else None)
    return s


# ───────────────────────────── plain forms ─────────────────────────────

def _act(v, act):
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))
    if act == "silu_gate":
        n = v.shape[-1] // 2
        return v[..., :n] / (1 + torch.exp(-v[..., :n])) * v[..., n:]
    return v


def _plain_route(s, case):
    z = s["logits"].float()
    experts, offsets, rows, slots, _ = _choices(z, case["top_k"])
    picked = torch.gather(z, 1, experts.long())
    top = picked[:, :1]
    total = torch.exp((picked if case["renormalize"] else z) - top).sum(1, keepdim=True)
    return {"experts": experts, "weights": torch.exp(picked - top) / total, "offsets": offsets,
            "rows": rows, "slots": slots}


def _plain_grouped(s, case):
    """Every expert's rows padded to the longest expert's, one batched product."""
    experts, most = case["experts"], s["most"]
    x = s["x"].float()
    if s["rows"] is not None:
        x = x[s["rows"].long()]
    e = s["of_slot"]
    at = e * most + torch.arange(e.numel(), device=e.device) - s["offsets"].long()[e]
    padded = x.new_zeros(experts * most, x.shape[1])
    padded[at] = x
    y = torch.bmm(padded.view(experts, most, -1), s["weight"].float().transpose(1, 2))
    y = y.reshape(experts * most, -1)[at]
    if s["bias"] is not None:
        y = y + s["bias"].float()[e]
    return _act(y, case["act"]).to(s["x"].dtype)


def _plain_combine(s, case):
    y = s["y"].float()[s["slots"].long()]
    o = (y * s["weights"][:, :, None]).sum(1)
    if s["residual"] is not None:
        o = o + s["residual"].float()
    return o.to(s["y"].dtype)


def _unpack(packed, K):
    """Packed words -> [N, K] values 0..15."""
    N = packed.shape[0]
    shift = 4 * torch.arange(8, device=packed.device, dtype=torch.int32)
    nib = (packed.reshape(N, -1, 16, 1) >> shift) & 15
    q = torch.empty(N, nib.shape[1], 128, device=packed.device, dtype=torch.int32)
    q[:, :, _pack_order(packed.device)] = nib
    return q.reshape(N, -1)[:, :K]


def _plain_w4(s, case):
    q = _unpack(s["packed"], case["K"]).float()
    of_col = torch.arange(case["K"], device=q.device) // case["group"]
    z = s["zeros"].float().t()[:, of_col] if s["zeros"] is not None else 8.0
    w = (q - z) * s["scales"].float().t()[:, of_col]
    y = s["x"].float() @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return _act(y, case["act"]).to(s["x"].dtype)


# ───────────────────────────── the framework's operators ─────────────────────────────

def _tensor(t):
    """A GpuTensor over a torch tensor's memory."""
    import numpy as np

    from scaffolding_b200 import _cuda_ops as ops
    if t is None:
        return None
    dt = {torch.bfloat16: ops.bfloat16, torch.float16: np.float16, torch.float32: np.float32,
          torch.int32: np.int32}[t.dtype]
    dev = t.device.index or 0
    return ops.GpuTensor(ops.CudaBuffer(t.data_ptr(), t.numel() * t.element_size(), dev, False),
                         tuple(t.shape), dt, dev)


def _handles(s):
    """The tensors that a program of this framework holds: its inputs, weights
    and the buffers it has its results in."""
    from scaffolding_b200 import _cuda_ops as ops
    case = s["case"]
    op = case["op"]

    def new(*shape, dtype=DTYPES[case["dtype"]]):
        return torch.empty(*shape, device="cuda", dtype=dtype)

    if op == "route":
        T, k, i32 = case["tokens"], case["top_k"], torch.int32
        out = {"experts": new(T, k, dtype=i32), "weights": new(T, k, dtype=torch.float32),
               "offsets": new(case["experts"] + 1, dtype=i32), "rows": new(T * k, dtype=i32),
               "slots": new(T, k, dtype=i32)}
        return _tensor(s["logits"]), ops.MoeRoute(**{n: _tensor(t) for n, t in out.items()}), out
    if op == "combine":
        out = new(case["tokens"], case["C"])
        return (*(_tensor(s[n]) for n in ("y", "slots", "weights", "residual")), _tensor(out), out)
    if op == "grouped":
        out = new(s["of_slot"].numel(), case["N"])
        return (*(_tensor(s[n]) for n in ("x", "weight", "offsets", "bias", "rows")), _tensor(out), out)
    out = new(case["M"], case["N"])
    weight = ops.W4Weight(_tensor(s["packed"]), _tensor(s["scales"]), _tensor(s["zeros"]),
                          in_features=case["K"], group=case["group"])
    return _tensor(s["x"]), weight, _tensor(s["bias"]), _tensor(out), out


def _own(s, case):
    op = case["op"]
    if "handles" not in s:
        from scaffolding_b200 import _cuda_ops
        s["handles"], s["ops"] = _handles(s), _cuda_ops
    h, ops = s["handles"], s["ops"]
    if op == "route":
        logits, route, out = h
        ops.dev_moe_route(logits, case["top_k"], renormalize=case["renormalize"], out=route)
        return out
    if op == "combine":
        y, slots, weights, residual, o, out = h
        ops.dev_moe_combine(y, slots, weights, residual=residual, out=o)
        return out
    if op == "grouped":
        x, weight, offsets, bias, rows, o, out = h
        ops.dev_grouped_linear(x, weight, offsets, bias, case["act"], rows=rows, out=o)
        return out
    x, weight, bias, o, out = h
    ops.dev_linear_w4(x, weight, bias, case["act"], out=o)
    return out


def run(state):
    case = state["case"]
    if own:
        return _own(state, case)
    plain = {"route": _plain_route, "grouped": _plain_grouped, "combine": _plain_combine,
             "w4": _plain_w4}[case["op"]]
    return plain(state, case)


# ───────────────────────────── work ─────────────────────────────

def work(case):
    op = case["op"]
    es = 4 if case["dtype"] == "f32" else 2
    if op == "w4":
        M, N, K = case["M"], case["N"], case["K"]
        groups = -(-K // case["group"])
        per_group = es * (2 if case["zeros"] else 1)
        return {"bytes": N * K / 2 + groups * N * per_group + es * (M * K + M * N + N * case["bias"]),
                "flops": 2.0 * M * N * K}
    T, k = case["tokens"], case["top_k"]
    if op == "route":
        E = case["experts"]
        return {"bytes": es * T * E + 16 * T * k + 4 * (E + 1), "flops": 3.0 * T * E}
    if op == "combine":
        C = case["C"]
        return {"bytes": es * C * T * (k + 1 + case["residual"]) + 8 * T * k, "flops": 2.0 * T * k * C}
    E, K = case["experts"], case["K"]
    k = min(k, E)
    wide = case["N"] * (2 if case["act"] == "silu_gate" else 1)
    touched = E * (1 - (1 - k / E) ** T)  # experts with rows, for an even router
    return {"bytes": es * ((T if case["gather"] else T * k) * K + touched * wide * K +
                           T * k * case["N"] + touched * wide * case["bias"]) + 4 * (E + 1) +
                     4 * T * k * case["gather"],
            "flops": 2.0 * T * k * wide * K}


# ───────────────────────────── exact values ─────────────────────────────

def _exact_act(v, act):
    if act == "none":
        return v
    if act == "gelu_tanh":
        return torch.nn.functional.gelu(v, approximate="tanh")
    if act == "silu":
        return v * torch.sigmoid(v)
    gate, up = v.chunk(2, dim=-1)
    return gate * torch.sigmoid(gate) * up


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "route":
        z = s["logits"].double()
        at = torch.argsort(z, dim=1, descending=True, stable=True)[:, :case["top_k"]]
        w = torch.gather(torch.softmax(z, 1), 1, at)
        if case["renormalize"]:
            w = torch.softmax(torch.gather(z, 1, at), 1)
        return {"experts": None, "weights": w, "offsets": None, "rows": None, "slots": None}
    if op == "combine":
        o = torch.zeros(case["tokens"], case["C"], device="cuda", dtype=torch.float64)
        if s["residual"] is not None:
            o += s["residual"]
        for j in range(case["top_k"]):
            o += s["weights"][:, j:j + 1].double() * s["y"][s["slots"][:, j].long()].double()
        return o
    if op == "grouped":
        parts = []
        bounds = s["offsets"].tolist()
        for e in range(case["experts"]):
            lo, hi = bounds[e], bounds[e + 1]
            x = s["x"][s["rows"][lo:hi].long()] if case["gather"] else s["x"][lo:hi]
            y = x.double() @ s["weight"][e].double().T
            if case["bias"]:
                y += s["bias"][e]
            parts.append(_exact_act(y, case["act"]))
        return torch.cat(parts)
    # 4-bit weights, rebuilt word by word of a block from the layout's definition
    N, K, group = case["N"], case["K"], case["group"]
    words = s["packed"].long() & 0xFFFFFFFF
    w = torch.zeros(N, words.shape[1] * 8, device="cuda", dtype=torch.float64)
    for t in range(4):
        for j in range(4):
            for i, c in enumerate((0, 2, 4, 6, 1, 3, 5, 7)):
                w[:, 32 * j + 8 * t + c::128] = ((words[:, 4 * t + j::16] >> (4 * i)) & 15).double()
    w = w[:, :K]
    for b in range(s["scales"].shape[0]):
        cols = slice(b * group, min(K, (b + 1) * group))
        w[:, cols] -= s["zeros"][b, :, None].double() if case["zeros"] else 8.0
        w[:, cols] *= s["scales"][b, :, None].double()
    y = s["x"].double() @ w.T
    if case["bias"]:
        y += s["bias"]
    return _exact_act(y, case["act"])
