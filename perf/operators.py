"""Cases, plain forms and calls of the 8-bit floating point expert path: rmsnorm_q8, silu_mul_q8, expert_lists,
matmul_q8 and grouped_matmul of inferenz_b200.MoePool (inzg_rmsnorm_q8 ... inzg_grouped_matmul of include/inzg.h).

The path is one mixture-of-experts layer whose weights are e4m3 with a scale per 128 x 128 block (how the model's
checkpoint holds them), or bf16 / f16: norm of the residual with an 8-bit output, the lists by expert from the router's
selections, the gate|up product on gathered rows, SiLU * up with an 8-bit output, the down product into the tokens'
slots; and dense products of the same activations. Widths are those of the framework's layer: hidden 2048 and 2560,
expert FFN 640 (gate|up 1280), 512 experts, top-10, hyper-connection residual 4 * hidden.
"""
import math

import torch

own = False

BLOCK = 128
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}
BYTES = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1}


def listed():
    return [
        # the norm before a layer when one sequence decodes: latency
        {"name": "norm 1 x 2560", "op": "norm", "n": 1, "cols": 2560, "type": "bf16", "res": True, "y": False, "pad": 0},
        # the same in a prefill of 4096 tokens, with the normalised row for the router too
        {"name": "norm 4096 x 2560", "op": "norm", "n": 4096, "cols": 2560, "type": "bf16", "res": True, "y": True,
         "pad": 0},
        # the entries of 32 decoding sequences, top-10: gate|up rows in fp32
        {"name": "silu 320 x 640", "op": "silu", "n": 320, "cols": 640, "type": "f32", "y": False, "pad": 0},
        # the entries of a 4096-token prefill
        {"name": "silu 40960 x 640", "op": "silu", "n": 40960, "cols": 640, "type": "bf16", "y": False, "pad": 0},
        # the router's selections of 32 decoding sequences
        {"name": "lists 32 x 10 of 512", "op": "lists", "tokens": 32, "topk": 10, "experts": 512, "absent": False},
        # the selections of a prefill, on a rank that owns a part of the experts (the others' entries are absent)
        {"name": "lists 4096 x 10 of 512", "op": "lists", "tokens": 4096, "topk": 10, "experts": 512, "absent": True},
        # a dense projection of one decoding token: the weights' bytes are the time
        {"name": "matmul 1 x 10240 x 2560", "op": "matmul", "m": 1, "n": 10240, "k": 2560, "out": "bf16", "pad": 0},
        # the same over a ragged prefill: the tensor pipe is the time
        {"name": "matmul 4000 x 10240 x 2560", "op": "matmul", "m": 4000, "n": 10240, "k": 2560, "out": "bf16",
         "pad": 0},
        # gate|up of one decoding token: ten experts of one row each among 512
        {"name": "experts 1 token e4m3", "op": "grouped", "type": "e4m3", "tokens": 1, "topk": 10, "experts": 512,
         "n": 1280, "k": 2048, "out": "bf16", "gather": True, "scatter": False, "skew": 0.5},
        # gate|up of 32 decoding sequences: a row or two for each of some 240 experts
        {"name": "experts 32 tokens e4m3", "op": "grouped", "type": "e4m3", "tokens": 32, "topk": 10, "experts": 512,
         "n": 1280, "k": 2048, "out": "bf16", "gather": True, "scatter": False, "skew": 0.5},
        # experts kept in bf16, one of eight ranks' share of them, an odd prompt
        {"name": "experts 333 tokens bf16", "op": "grouped", "type": "bf16", "tokens": 333, "topk": 10, "experts": 64,
         "n": 1280, "k": 2560, "out": "bf16", "gather": True, "scatter": False, "skew": 0.5},
        # down of a 4096-token prefill: weighted rows into the tokens' slots, as inzg_combine reads them
        {"name": "experts 4096 tokens e4m3 down", "op": "grouped", "type": "e4m3", "tokens": 4096, "topk": 10,
         "experts": 512, "n": 2048, "k": 640, "out": "f32", "gather": False, "scatter": True, "skew": 0.5},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "silu", "lists", "matmul", "matmul", "grouped", "grouped", "grouped"])
    yes = lambda: rng.random() < 0.5  # noqa: E731
    if op == "norm":
        cols = _log(rng, 64, 16384)
        return {"op": op, "n": _log(rng, 1, max(1, min(8192, (1 << 25) // cols))), "cols": cols,
                "type": rng.choice(["f32", "bf16", "f16"]), "res": yes(), "y": yes(), "pad": rng.choice([0, 0, 8, 3])}
    if op == "silu":
        cols = _log(rng, 16, 4096)
        return {"op": op, "n": _log(rng, 1, max(1, min(40960, (1 << 25) // cols))), "cols": cols,
                "type": rng.choice(["f32", "bf16", "f16"]), "y": yes(), "pad": rng.choice([0, 0, 8, 3])}
    if op == "lists":
        experts = rng.choice([8, 64, 160, 512, rng.randint(2, 1024)])
        return {"op": op, "tokens": _log(rng, 1, 8192), "topk": rng.randint(1, min(16, experts)), "experts": experts,
                "absent": yes()}
    if op == "matmul":
        m, n, k = _log(rng, 1, 4096), _log(rng, 16, 10240), _log(rng, 64, 10240)
        while m * n * k > 4000 * 10240 * 2560:
            m = max(1, m // 2)
        return {"op": op, "m": m, "n": n, "k": k, "out": rng.choice(["f32", "bf16", "f16"]),
                "pad": rng.choice([0, 16, 128])}
    experts = rng.choice([1, 8, 64, 128, 512, rng.randint(2, 300)])
    n, k = _log(rng, 64, 2560), _log(rng, 64, 2560)
    kind = rng.choice(["e4m3", "e4m3", "bf16", "f16"])
    while experts * n * k * BYTES[kind] > 512 * 1280 * 2048:
        n = max(64, n // 2)
    topk = rng.randint(1, min(10, experts))
    tokens = _log(rng, 1, 4096)
    while tokens * topk * n * k > 40960 * 2048 * 640:
        tokens = max(1, tokens // 2)
    return {"op": op, "type": kind, "tokens": tokens, "topk": topk,
            "experts": experts, "n": n, "k": k, "out": rng.choice(["f32", "bf16", "f16"]), "gather": yes(),
            "scatter": yes(), "skew": rng.choice([0.0, 0.5])}


def _up(v, to):
    return -(-v // to) * to


def _wide(shape, ld, g, dtype, scale=1.0):
    """A [rows][cols] view with row pitch `ld` of normal values."""
    rows, cols = shape
    return (torch.randn(rows, ld, generator=g, device="cuda") * scale).to(dtype)[:, :cols]


def _fp8(shape, ld, g):
    """e4m3 values as a block quantizer leaves them: near 448 at a block's largest."""
    rows, cols = shape
    return (torch.randn(rows, ld, generator=g, device="cuda") * 120.0).clamp(-448, 448).to(torch.float8_e4m3fn)[:, :cols]


def _selections(case, g):
    """The router's distinct experts of each token, some chosen more often than others."""
    T, E, K = case["tokens"], case["experts"], case["topk"]
    logits = torch.randn(T, E, generator=g, device="cuda")
    logits += case.get("skew", 0.5) * torch.randn(E, generator=g, device="cuda")
    p, sel = torch.softmax(logits, 1).topk(K, 1)
    return sel.to(torch.int32).contiguous(), (p / p.sum(1, keepdim=True)).contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, st = case["op"], {"case": case, "stream": torch.cuda.current_stream().cuda_stream or 1}  # 1: the legacy stream
    empty = lambda *a, dtype: torch.empty(*a, dtype=dtype, device="cuda")  # noqa: E731
    if op in ("norm", "silu"):
        n, cols, dt = case["n"], case["cols"], TYPES[case["type"]]
        nb, ld = _up(cols, BLOCK) // BLOCK, cols + case["pad"]
        if op == "norm":
            st["x"] = _wide((n, cols), ld, g, dt)
            # a residual has a few large channels
            ch = torch.exp(torch.randn(cols, generator=g, device="cuda"))
            st["res"] = (_wide((n, cols), cols, g, torch.float32) * ch).to(dt) if case["res"] else None
            st["w"] = 1.0 + 0.1 * torch.randn(cols, generator=g, device="cuda")
            st["sum"] = empty(n, cols, dtype=dt) if case["res"] else None
        else:
            st["x"] = _wide((n, 2 * cols), 2 * cols + case["pad"], g, dt)
        st["y"] = empty(n, cols, dtype=dt) if case["y"] else None
        st["q"], st["s"] = empty(n, _up(cols, 16), dtype=torch.float8_e4m3fn)[:, :cols], empty(n, nb, dtype=torch.float32)
    elif op == "lists":
        st["sel"], st["w"] = _selections(case, g)
        T, K, E = case["tokens"], case["topk"], case["experts"]
        if case["absent"]:  # a quarter of the experts live on another rank
            st["sel"] = torch.where(st["sel"] < E // 4, -1, st["sel"] - E // 4).to(torch.int32).contiguous()
        st["groups"] = E - E // 4 if case["absent"] else E
        # entries of absent experts are not listed: what lies behind the last list stays as it was
        st["off"] = empty(st["groups"] + 1, dtype=torch.int32)
        st["rows"], st["slots"] = (torch.full((T * K,), -1, dtype=torch.int32, device="cuda") for _ in range(2))
        st["ws"] = torch.zeros(T * K, device="cuda")
    elif op == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        ld, nb = _up(k, 16) + case["pad"], _up(k, BLOCK) // BLOCK
        st["a"], st["w"] = _fp8((m, k), ld, g), _fp8((n, k), _up(k, 16), g)
        st["as"] = 0.01 * torch.exp(0.5 * torch.randn(m, nb, generator=g, device="cuda"))
        st["ws"] = (0.5 + torch.rand(_up(n, BLOCK) // BLOCK, nb, generator=g, device="cuda")) / (120 * math.sqrt(k))
        st["out"] = empty(m, n, dtype=TYPES[case["out"]])
    else:
        T, K, E, n, k, dt = case["tokens"], case["topk"], case["experts"], case["n"], case["k"], TYPES[case["type"]]
        sel, w = _selections(case, g)
        order = torch.argsort(sel.reshape(-1), stable=True)
        st["off"] = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
        st["off"][1:] = torch.bincount(sel.reshape(-1).long(), minlength=E).cumsum(0)
        st["most"] = int(torch.bincount(sel.reshape(-1).long(), minlength=E).max())  # the plan's largest group
        rows = T if case["gather"] else T * K
        f8, nb = case["type"] == "e4m3", _up(k, BLOCK) // BLOCK
        ld = _up(k, 16)
        if f8:
            st["a"], st["w"] = _fp8((rows, k), ld, g), _fp8((E * n, k), ld, g)
            st["as"] = 0.01 * torch.exp(0.5 * torch.randn(rows, nb, generator=g, device="cuda"))
            st["ws"] = (0.5 + torch.rand(E, _up(n, BLOCK) // BLOCK, nb, generator=g, device="cuda")) / (
                120 * math.sqrt(k))
        else:
            st["a"] = _wide((rows, k), ld, g, dt)
            st["w"] = _wide((E * n, k), ld, g, dt, 1.0 / math.sqrt(k))
            st["as"] = st["ws"] = None
        st["in_rows"] = (order // K).to(torch.int32) if case["gather"] else None
        st["out_rows"] = order.to(torch.int32) if case["scatter"] else None
        st["scale"] = w.reshape(-1)[order].contiguous() if case["scatter"] else None
        st["out"] = empty(T * K, n, dtype=TYPES[case["out"]])
    return st


# ---------------------------------------------------------------------------------------------------------------------
# the plain forms: fp32, rounded once


def _quantize(v):
    n, cols = v.shape
    nb = _up(cols, BLOCK) // BLOCK
    blocks = torch.nn.functional.pad(v, (0, nb * BLOCK - cols)).view(n, nb, BLOCK)
    s = blocks.abs().amax(2).clamp(min=2.0 ** -100) / 448
    return (blocks / s[:, :, None]).to(torch.float8_e4m3fn).view(n, -1)[:, :cols], s


def _dequantize(a, s):
    """a [rows][k] e4m3, s [rows][blocks] -> fp32"""
    return a.float() * s.repeat_interleave(BLOCK, 1)[:, :a.shape[1]]


def _dequantize_weights(w, ws, n):
    """w [E * n][k] e4m3, ws [E][n blocks][k blocks] -> [E][n][k] fp32"""
    E, k = ws.shape[0], w.shape[1]
    s = ws.repeat_interleave(BLOCK, 1)[:, :n].reshape(E * n, -1)
    return _dequantize(w, s).view(E, n, k)


def _plain_norm(st):
    h = st["x"].float()
    h = h + st["res"].float() if st["res"] is not None else h
    v = h * torch.rsqrt((h * h).mean(1, keepdim=True) + 1e-6) * st["w"]
    q, s = _quantize(v)
    return {"sum": h.to(st["x"].dtype) if st["res"] is not None else None,
            "y": v.to(st["x"].dtype) if st["y"] is not None else None, "q": q, "s": s}


def _plain_silu(st):
    cols = st["case"]["cols"]
    gate, up = st["x"][:, :cols].float(), st["x"][:, cols:].float()
    v = gate / (1 + torch.exp(-gate)) * up
    q, s = _quantize(v)
    return {"y": v.to(st["x"].dtype) if st["y"] is not None else None, "q": q, "s": s}


def _plain_lists(st):
    K, E = st["case"]["topk"], st["groups"]
    sel = st["sel"].reshape(-1).long()
    key = torch.where(sel < 0, E, sel)
    order = torch.argsort(key, stable=True)
    off = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    off[1:] = torch.zeros(E + 1, dtype=torch.int64, device="cuda").scatter_add_(0, key, torch.ones_like(key))[:E].cumsum(0)
    listed_ = key[order] < E
    return {"off": off, "rows": torch.where(listed_, order // K, -1).to(torch.int32),
            "slots": torch.where(listed_, order, -1).to(torch.int32),
            "w": torch.where(listed_, st["w"].reshape(-1)[order], 0)}


def _plain_matmul(st):
    w = _dequantize_weights(st["w"], st["ws"][None], st["case"]["n"])[0]
    return (_dequantize(st["a"], st["as"]) @ w.t()).to(st["out"].dtype)


def _plain_grouped(st):
    c = st["case"]
    E, n, k, entries = c["experts"], c["n"], c["k"], c["tokens"] * c["topk"]
    a = _dequantize(st["a"], st["as"]) if st["as"] is not None else st["a"].float()
    a = a[st["in_rows"].long()] if st["in_rows"] is not None else a
    at = torch.arange(entries, device="cuda")
    group = torch.searchsorted(st["off"][1:].long(), at, right=True)
    if entries < E:  # few entries: each with its own expert's weights
        w = st["w"].view(E, n, -1) if st["w"].is_contiguous() else st["w"].unflatten(0, (E, n))
        w = w[group] if st["ws"] is None else w.view(torch.uint8)[group].view(torch.float8_e4m3fn)
        w = w.float() if st["ws"] is None else _dequantize_weights(w.reshape(entries * n, k), st["ws"][group], n)
        out = torch.bmm(w, a[:, :, None])[:, :, 0]
    else:  # every group padded to the largest
        w = st["w"].float().view(E, n, k) if st["ws"] is None else _dequantize_weights(st["w"], st["ws"], n)
        pos = at - st["off"].long()[group]
        padded = torch.zeros(E, st["most"], k, device="cuda")
        padded[group, pos] = a
        out = torch.bmm(padded, w.transpose(1, 2))[group, pos]
    if st["scale"] is not None:
        out = out * st["scale"][:, None]
    if st["out_rows"] is not None:
        out = torch.zeros_like(out).index_copy_(0, st["out_rows"].long(), out)
    return out.to(st["out"].dtype)


# ---------------------------------------------------------------------------------------------------------------------
# the framework's calls

_pool_ = None


def _pool():
    """The context that a program keeps for its layers."""
    global _pool_
    if _pool_ is None:
        from inferenz_b200 import MoePool
        _pool_ = MoePool(max_tokens=16, device=torch.cuda.current_device())
    return _pool_


def _type(t):
    from inferenz_b200 import _lib
    return {torch.float32: _lib.T_F32, torch.bfloat16: _lib.T_BF16, torch.float16: _lib.T_F16,
            torch.float8_e4m3fn: _lib.T_E4M3}[t.dtype]


def _ptr(t):
    return None if t is None else t.data_ptr()


def _own(st):
    op, p = st["case"]["op"], _pool()
    if op == "norm":
        x, q, s = st["x"], st["q"], st["s"]
        p.rmsnorm_q8_device(x.shape[0], x.shape[1], _type(x), x.data_ptr(), st["w"].data_ptr(), 1e-6, ldx=x.stride(0),
                            res_ptr=_ptr(st["res"]), sum_ptr=_ptr(st["sum"]), y_ptr=_ptr(st["y"]), q_ptr=q.data_ptr(),
                            ldq=q.stride(0), s_ptr=s.data_ptr(), stream=st["stream"])
        return {"sum": st["sum"], "y": st["y"], "q": q, "s": s}
    if op == "silu":
        x, q, s = st["x"], st["q"], st["s"]
        p.silu_mul_q8_device(x.shape[0], q.shape[1], _type(x), x.data_ptr(), ldx=x.stride(0), y_ptr=_ptr(st["y"]),
                             q_ptr=q.data_ptr(), ldq=q.stride(0), s_ptr=s.data_ptr(), stream=st["stream"])
        return {"y": st["y"], "q": q, "s": s}
    if op == "lists":
        T, K = st["sel"].shape
        p.expert_lists_device(T, K, st["groups"], st["sel"].data_ptr(), st["off"].data_ptr(), st["rows"].data_ptr(),
                              st["slots"].data_ptr(), w_ptr=st["w"].data_ptr(), w_out_ptr=st["ws"].data_ptr(),
                              stream=st["stream"])
        return {"off": st["off"], "rows": st["rows"], "slots": st["slots"], "w": st["ws"]}
    a, w, out = st["a"], st["w"], st["out"]
    if op == "matmul":
        p.matmul_q8_device(a.shape[0], w.shape[0], a.shape[1], a.data_ptr(), st["as"].data_ptr(), w.data_ptr(),
                           st["ws"].data_ptr(), out.data_ptr(), _type(out), lda=a.stride(0), ldw=w.stride(0),
                           stream=st["stream"])
        return out
    c = st["case"]
    p.grouped_matmul_device(_type(a), c["experts"], c["n"], c["k"], a.shape[0], out.shape[0], a.data_ptr(),
                            w.data_ptr(), st["off"].data_ptr(), out.data_ptr(), _type(out), lda=a.stride(0),
                            ldw=w.stride(0), a_scale_ptr=_ptr(st["as"]), w_scale_ptr=_ptr(st["ws"]),
                            in_rows_ptr=_ptr(st["in_rows"]), out_rows_ptr=_ptr(st["out_rows"]),
                            out_scale_ptr=_ptr(st["scale"]), stream=st["stream"])
    return out


def run(state):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "silu": _plain_silu, "lists": _plain_lists, "matmul": _plain_matmul,
            "grouped": _plain_grouped}[state["case"]["op"]](state)


def work(case):
    op = case["op"]
    if op == "norm":
        n, cols, b = case["n"], case["cols"], BYTES[case["type"]]
        moved = b * (1 + 2 * case["res"] + case["y"])
        return {"bytes": n * cols * (moved + 1) + 4 * n * (_up(cols, BLOCK) // BLOCK) + 4 * cols, "flops": 6 * n * cols}
    if op == "silu":
        n, cols, b = case["n"], case["cols"], BYTES[case["type"]]
        return {"bytes": n * cols * (b * (2 + case["y"]) + 1) + 4 * n * (_up(cols, BLOCK) // BLOCK),
                "flops": 8 * n * cols}
    if op == "lists":
        return {"bytes": 20 * case["tokens"] * case["topk"] + 4 * case["experts"], "flops": 0}
    if op == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        nb = _up(k, BLOCK) // BLOCK
        return {"bytes": (m + n) * k + m * n * BYTES[case["out"]] + 4 * nb * (m + _up(n, BLOCK) // BLOCK),
                "flops": 2 * m * n * k}
    T, K, E, n, k, b = case["tokens"], case["topk"], case["experts"], case["n"], case["k"], BYTES[case["type"]]
    used = E * (1 - (1 - K / E) ** T)  # experts with an entry, were they chosen alike
    return {"bytes": used * n * k * b + (T if case["gather"] else T * K) * k * b + T * K * n * BYTES[case["out"]],
            "flops": 2 * T * K * n * k}


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits


def _e4m3_of(v):
    """The nearest e4m3 value of each (ties to even), |v| < 464: 4 significant bits down to 2^-6, steps of 2^-9 below."""
    e = torch.frexp(v.abs().clamp(min=2.0 ** -6)).exponent - 1
    step = torch.ldexp(torch.ones_like(v), e - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


def _exact_quantized(v):
    n, cols = v.shape
    q, s = torch.empty_like(v), torch.empty(n, _up(cols, BLOCK) // BLOCK, dtype=v.dtype, device=v.device)
    for b in range(s.shape[1]):
        part = v[:, b * BLOCK:(b + 1) * BLOCK]
        s[:, b] = part.abs().max(1).values.clamp(min=2.0 ** -100) / 448
        q[:, b * BLOCK:(b + 1) * BLOCK] = _e4m3_of(part / s[:, b:b + 1])
    return q, s


def _blockwise(a, sa, w, sw):
    """sum over blocks of sa[i][b] sw[j / 128][b] (a_b w_b^T) in 64 bits"""
    out = torch.zeros(a.shape[0], w.shape[0], dtype=torch.float64, device=a.device)
    for b in range(sa.shape[1]):
        at = slice(b * BLOCK, (b + 1) * BLOCK)
        rows = torch.arange(w.shape[0], device=w.device) // BLOCK
        out += (a[:, at].double() @ w[:, at].double().t()) * sa[:, b:b + 1].double() * sw[rows, b].double()[None]
    return out


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        h = st["x"].double() + (st["res"].double() if case["res"] else 0)
        v = h / torch.sqrt(h.square().sum(1, keepdim=True) / case["cols"] + 1e-6) * st["w"].double()
        q, s = _exact_quantized(v)
        return {"sum": h if case["res"] else None, "y": v if case["y"] else None, "q": q, "s": s}
    if op == "silu":
        g, u = st["x"].double()[:, :case["cols"]], st["x"].double()[:, case["cols"]:]
        v = g * torch.sigmoid(g) * u
        q, s = _exact_quantized(v)
        return {"y": v if case["y"] else None, "q": q, "s": s}
    if op == "lists":
        return None
    if op == "matmul":
        return _blockwise(st["a"], st["as"], st["w"], st["ws"])
    off = st["off"].tolist()
    n, out = case["n"], torch.zeros(off[-1], case["n"], dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        if off[e] == off[e + 1]:
            continue
        to = torch.arange(off[e], off[e + 1], device="cuda")
        at = st["in_rows"][to].long() if case["gather"] else to
        w = st["w"][e * n:(e + 1) * n]
        if case["type"] == "e4m3":
            a = st["a"].view(torch.uint8)[at].view(torch.float8_e4m3fn)
            y = _blockwise(a, st["as"][at], w, st["ws"][e])
        else:
            y = st["a"][at].double() @ w.double().t()
        if case["scatter"]:
            y *= st["scale"][to].double()[:, None]
            to = st["out_rows"][to].long()
        out[to] = y
    return out
