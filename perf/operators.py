"""The feed-forward operators of a large language model on 8-bit weights, measured case by case.

Three operators, as a served model uses them one after the other:

- ``rows``: every row (token) of an activation tensor quantized to uint8 with its own scale and zero point. The codes
  are returned as the values they stand for, through the framework's DequantizeLinear.
- ``product``: an int8 product with the dequantization by a scale per row of A and per column of B, a bias, an
  activation and a residual in its epilogue.
- ``moe``: a whole mixture-of-experts layer for a few tokens: router, top-k, the chosen experts' gated feed-forward on
  int8 weights, and the weighted sum.

``run`` computes a case in elementary torch operations (``own`` false) or with the framework's kernels (``own`` true).
"""
import math

import torch

own = False

_ACTIVATIONS = ("none", "relu", "gelu", "gelu_tanh", "silu")
_TYPES = {"f32": torch.float32, "f16": torch.float16}


# ---- cases ----------------------------------------------------------------------------------------------------------

def listed():
    return [
        # One token of a decode step before its projections: latency only.
        {"name": "rows-1-token", "op": "rows", "rows": 1, "columns": 4096, "type": "f16"},
        # A batch of ragged prompts, rows that do not start on 16-byte boundaries.
        {"name": "rows-ragged-f32", "op": "rows", "rows": 777, "columns": 5001, "type": "f32"},
        # A long prompt's activations.
        {"name": "rows-prompt", "op": "rows", "rows": 4096, "columns": 8192, "type": "f16"},
        # The down projection of one decoded token, added to the residual stream.
        {"name": "product-1-token", "op": "product", "m": 1, "n": 8192, "k": 8192, "b": "nk", "a": "u8", "zeros": True,
         "bias": False, "act": "none", "residual": True, "type": "f16"},
        # The up projection of a decode batch (16 x 28672 x 8192).
        {"name": "product-decode", "op": "product", "m": 16, "n": 28672, "k": 8192, "b": "kn", "a": "u8", "zeros": True,
         "bias": True, "act": "silu", "residual": False, "type": "f16"},
        # A small layer of odd sizes, f32 throughout.
        {"name": "product-odd-f32", "op": "product", "m": 333, "n": 2305, "k": 1001, "b": "kn", "a": "u8",
         "zeros": True, "bias": True, "act": "gelu", "residual": True, "type": "f32"},
        # A prompt's output projection into the residual stream.
        {"name": "product-prompt", "op": "product", "m": 4096, "n": 4096, "k": 4096, "b": "nk", "a": "s8",
         "zeros": False, "bias": True, "act": "none", "residual": True, "type": "f16"},
        # A prompt's up projection with its activation, f32 results.
        {"name": "product-prompt-f32", "op": "product", "m": 8192, "n": 8192, "k": 2048, "b": "kn", "a": "u8",
         "zeros": True, "bias": True, "act": "gelu_tanh", "residual": False, "type": "f32"},
        # One decoded token through a layer of many small experts.
        {"name": "moe-1-token", "op": "moe", "tokens": 1, "model": 2048, "expert": 1024, "experts": 64, "top_k": 8,
         "act": "silu", "type": "f16"},
        # A few tokens, odd sizes, f32 activations.
        {"name": "moe-odd-f32", "op": "moe", "tokens": 5, "model": 1001, "expert": 516, "experts": 12, "top_k": 3,
         "act": "gelu_tanh", "type": "f32"},
        # A decode batch through a layer of few large experts.
        {"name": "moe-large-experts", "op": "moe", "tokens": 8, "model": 4096, "expert": 8192, "experts": 8, "top_k": 2,
         "act": "silu", "type": "f16"},
        # A larger decode batch that touches nearly every expert.
        {"name": "moe-batch", "op": "moe", "tokens": 64, "model": 2048, "expert": 1408, "experts": 64, "top_k": 6,
         "act": "silu", "type": "f16"},
    ]


def _between(rng, low, high):
    """A whole number spread evenly over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def _size(rng, low, high):
    """A size: odd ones among multiples of 16, as real layers have more often."""
    v = _between(rng, low, high)
    return v if rng.random() < 0.3 else max(16, v // 16 * 16)


def draw(rng):
    op = rng.choice(["rows", "product", "product", "moe", "moe"])
    kind = rng.choice(["f16", "f16", "f32"])
    if op == "rows":
        columns = _size(rng, 64, 16384)
        return {"op": op, "rows": _between(rng, 1, min(8192, (1 << 25) // columns)), "columns": columns, "type": kind}
    if op == "product":
        n, k = _size(rng, 64, 16384), _size(rng, 64, 16384)
        m = _between(rng, 1, max(1, min(8192, (1 << 37) // (n * k), (1 << 26) // n)))
        return {"op": op, "m": m, "n": n, "k": k, "b": rng.choice(["kn", "nk"]), "a": rng.choice(["u8", "s8"]),
                "zeros": rng.random() < 0.6, "bias": rng.random() < 0.6, "act": rng.choice(_ACTIVATIONS),
                "residual": rng.random() < 0.5, "type": kind}
    model = _size(rng, 64, 4096)
    expert = _size(rng, 64, 4096)
    experts = _between(rng, 2, max(2, min(128, (1 << 27) // (model * expert))))
    return {"op": op, "tokens": _between(rng, 1, 64), "model": model, "expert": expert, "experts": experts,
            "top_k": rng.randint(1, min(8, experts)), "act": rng.choice(["silu", "gelu", "gelu_tanh", "relu"]),
            "type": kind}


def work(case):
    size = 2 if case["type"] == "f16" else 4
    if case["op"] == "rows":
        count = case["rows"] * case["columns"]
        # x read, codes and their values written; two operations an element for the range, two for the code
        return {"bytes": count * (size + 1 + 4) + 5 * case["rows"], "flops": 4 * count}
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        outputs = m * n * size * (2 if case["residual"] else 1)
        vectors = 4 * (m + n) + (4 * n if case["bias"] else 0) + (m + n if case["zeros"] else 0)
        return {"bytes": m * k + k * n + outputs + vectors, "flops": 2 * m * n * k}
    t, d, f, e, k = (case[name] for name in ("tokens", "model", "expert", "experts", "top_k"))
    touched = e * (1 - (1 - k / e) ** t)  # experts that at least one token chose
    return {"bytes": touched * (3 * d * f + 4 * (2 * f + d)) + 4 * e * d + 2 * t * d * size + 8 * t * k,
            "flops": 2 * t * (k * 3 * d * f + e * d)}


# ---- inputs -----------------------------------------------------------------------------------------------------------

def _codes(shape, generator, spread, shift, low, high, kind):
    """8-bit codes of normally distributed values."""
    out = torch.empty(shape, dtype=kind, device="cuda")
    flat = out.view(-1)
    step = 1 << 27  # bounds the float temporaries of the largest weights
    at = 0
    while at < flat.numel():
        part = flat[at:at + step]
        values = torch.randn(part.numel(), generator=generator, device="cuda")
        part.copy_(values.mul_(spread).add_(shift).round_().clamp_(low, high))
        at += step
    return out


def _uniform(shape, generator, low, high):
    return torch.rand(shape, generator=generator, device="cuda") * (high - low) + low


def _activations(rows, columns, generator):
    """Tokens of different magnitudes, with a few channels far above the others."""
    x = torch.randn(rows, columns, generator=generator, device="cuda")
    x *= _uniform((rows, 1), generator, 0.3, 3.0)
    loud = torch.rand(columns, generator=generator, device="cuda") < 0.002
    return torch.where(loud, x * 12.0, x)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind = _TYPES[case["type"]]
    s = {"case": case}
    if case["op"] == "rows":
        s["x"] = _activations(case["rows"], case["columns"], g).to(kind)
    elif case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        unsigned = case["a"] == "u8"
        s["a"] = _codes((m, k), g, 32.0, 128.0 if unsigned else 0.0, 0 if unsigned else -128, 255 if unsigned else 127,
                        torch.uint8 if unsigned else torch.int8)
        s["b"] = _codes((k, n) if case["b"] == "kn" else (n, k), g, 32.0, 0.0, -128, 127, torch.int8)
        s["a_scale"] = _uniform((m,), g, 0.01, 0.05)
        s["b_scale"] = _uniform((n,), g, 0.5, 1.5) / (32.0 * math.sqrt(k))
        if case["zeros"]:
            s["a_zero"] = _codes((m,), g, 10.0, 128.0 if unsigned else 0.0, 0 if unsigned else -128,
                                 255 if unsigned else 127, s["a"].dtype)
            s["b_zero"] = _codes((n,), g, 3.0, 0.0, -128, 127, torch.int8)
        if case["bias"]:
            s["bias"] = torch.randn(n, generator=g, device="cuda") * 0.3
        if case["residual"]:
            s["residual"] = torch.randn(m, n, generator=g, device="cuda").to(kind)
    else:
        t, d, f, e = (case[name] for name in ("tokens", "model", "expert", "experts"))
        s["x"] = torch.randn(t, d, generator=g, device="cuda").to(kind)
        s["router"] = torch.randn(e, d, generator=g, device="cuda") * (1.5 / math.sqrt(d))
        s["w_in"] = _codes((e, 2 * f, d), g, 32.0, 0.0, -127, 127, torch.int8)
        s["in_scale"] = _uniform((e, 2 * f), g, 0.5, 1.5) / (32.0 * math.sqrt(d))
        s["w_out"] = _codes((e, d, f), g, 32.0, 0.0, -127, 127, torch.int8)
        s["out_scale"] = _uniform((e, d), g, 0.5, 1.5) / (32.0 * math.sqrt(f))
    if own:
        _handles(s)
    return s


# ---- the framework's kernels ------------------------------------------------------------------------------------------

_session = {}


def _open():
    """The framework's device on torch's stream, and its kernel objects: a program keeps them for its whole life."""
    if not _session:
        import os
        import sys

        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                        "onegpu-csharp_b200"))
        import onegpu_cuda as og

        device = og.GpuDevice(torch.cuda.current_device())
        device.set_stream(torch.cuda.current_stream().cuda_stream)
        _session.update(og=og, device=device, quantize=og.DynamicQuantizeKernels(device),
                        dequantize=og.DequantizeKernels(device), gemm=og.Int8Gemm(device), moe=og.Int8MoeKernels(device))
    return _session


def _handles(s):
    """The state's tensors as the framework's buffers, its outputs, and the problem descriptions."""
    f = _open()
    og, device, case = f["og"], f["device"], s["case"]
    np_types = {torch.float32: "float32", torch.float16: "float16", torch.uint8: "uint8", torch.int8: "int8",
                torch.int32: "int32"}

    def buffer(tensor):
        return device.wrap(tensor.data_ptr(), np_types[tensor.dtype], tensor.numel())

    def operand(name, vector=True):
        return og.Int8Operand(buffer(s[name]), 0, vector) if name in s else None

    def padded(count, kind):
        """Byte tensors end on a 32-bit word."""
        return torch.empty((count + 3) // 4 * 4, dtype=kind, device="cuda")

    h = {}
    kind = _TYPES[case["type"]]
    if case["op"] == "rows":
        rows, columns = case["rows"], case["columns"]
        h["x"] = buffer(s["x"])
        s["codes"] = padded(rows * columns, torch.uint8)
        s["values"] = torch.empty(rows, columns, dtype=torch.float32, device="cuda")
        s["scale"] = torch.empty(rows, dtype=torch.float32, device="cuda")
        s["zero"] = padded(rows, torch.uint8)
        for name in ("codes", "values", "scale", "zero"):
            h[name] = buffer(s[name])
        s["out"] = {"values": s["values"], "scale": s["scale"], "zero": s["zero"][:rows]}
    elif case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        h["problem"] = og.Int8GemmProblem(m, n, k, transpose_b=case["b"] == "nk")
        s["c"] = torch.empty(m, n, dtype=kind, device="cuda")
        for name in ("a", "b", "c"):
            h[name] = buffer(s[name])
        for name in ("a_scale", "b_scale", "a_zero", "b_zero", "bias"):
            h[name] = operand(name)
        h["residual"] = operand("residual", False)
        h["act"] = getattr(og, "ACTIVATION_" + case["act"].upper())
        s["out"] = {"c": s["c"]}
    else:
        t, d = case["tokens"], case["model"]
        h["problem"] = og.MoeProblem(t, d, case["expert"], case["experts"], case["top_k"],
                                     activation=getattr(og, "ACTIVATION_" + case["act"].upper()))
        s["y"] = torch.empty(t, d, dtype=kind, device="cuda")
        s["ids"] = torch.empty(t, case["top_k"], dtype=torch.int32, device="cuda")
        s["weights"] = torch.empty(t, case["top_k"], dtype=torch.float32, device="cuda")
        for name in ("x", "router", "w_in", "in_scale", "w_out", "out_scale", "y", "ids", "weights"):
            h[name] = buffer(s[name])
        s["out"] = {"y": s["y"], "ids": s["ids"], "weights": s["weights"]}
    s["handles"] = h


def _run_own(s):
    f, h, case = _session, s["handles"], s["case"]
    device = f["device"]
    encoder = device.begin_commands()
    if case["op"] == "rows":
        rows, columns = case["rows"], case["columns"]
        f["quantize"].encode_rows(encoder, h["x"], 0, rows, columns, 0, h["codes"], 0, h["scale"], 0, h["zero"], 0)
        f["dequantize"].encode(encoder, h["codes"], 0, (rows, columns), 0, True, h["scale"], 0, h["zero"], 0,
                               h["values"], 0)
    elif case["op"] == "product":
        f["gemm"].encode_activated(encoder, h["problem"], h["a"], h["b"], h["c"], h["a_scale"], h["b_scale"],
                                   h["a_zero"], h["b_zero"], h["bias"], None, h["act"], h["residual"])
    else:
        f["moe"].encode(encoder, h["problem"], h["x"], h["router"], h["w_in"], h["in_scale"], h["w_out"],
                        h["out_scale"], h["y"], expert_ids=h["ids"], expert_weights=h["weights"])
    device.submit(encoder)
    return s["out"]


# ---- the plain forms --------------------------------------------------------------------------------------------------

def _activate(v, name):
    if name == "relu":
        return torch.clamp(v, min=0.0)
    if name == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    if name == "silu":
        return v / (1.0 + torch.exp(-v))
    return v


def _plain_rows(s):
    x = s["x"].float()
    low = torch.clamp(x.amin(1, keepdim=True), max=0.0)
    high = torch.clamp(x.amax(1, keepdim=True), min=0.0)
    scale = (high - low) / torch.full_like(low, 255.0)
    empty = scale == 0
    zero = torch.where(empty, 0.0, torch.clamp(torch.round(-(low / scale)), 0.0, 255.0))
    scale = torch.where(empty, 1.0, scale)
    codes = torch.clamp(torch.round(x / scale) + zero, 0.0, 255.0)
    return {"values": (codes - zero) * scale, "scale": scale.view(-1), "zero": zero.view(-1).to(torch.uint8)}


def _plain_product(s):
    case = s["case"]
    a, b = s["a"].float(), s["b"].float()
    if case["b"] == "nk":
        b = b.t()
    if case["zeros"]:
        a = a - s["a_zero"].float().unsqueeze(1)
        b = b - s["b_zero"].float()
    v = (a @ b) * (s["a_scale"].unsqueeze(1) * s["b_scale"])
    if case["bias"]:
        v = v + s["bias"]
    v = _activate(v, case["act"])
    if case["residual"]:
        v = v + s["residual"].float()
    return {"c": v.to(_TYPES[case["type"]])}


def _plain_moe(s):
    case = s["case"]
    t, d, f, e, k = (case[name] for name in ("tokens", "model", "expert", "experts", "top_k"))
    x = s["x"].float()
    logits = s["x"].double() @ s["router"].double().t()  # 64 bits: near-equal logits decide which experts run
    ids = torch.sort(logits, dim=1, descending=True, stable=True)[1][:, :k]
    shares = torch.exp(logits - logits.amax(1, keepdim=True)).float()
    chosen = shares.gather(1, ids)
    weights = chosen / chosen.sum(1, keepdim=True)
    if t * k < e:  # the chosen experts' weights, one copy for each (token, expert)
        pick = ids.reshape(-1)
        rows = x.repeat_interleave(k, 0).unsqueeze(2)
        v = (s["w_in"][pick].float() @ rows).squeeze(2) * s["in_scale"][pick]
        h = _activate(v[:, :f], case["act"]) * v[:, f:]
        y = (s["w_out"][pick].float() @ h.unsqueeze(2)).squeeze(2) * s["out_scale"][pick]
        y = (y.view(t, k, d) * weights.unsqueeze(2)).sum(1)
    else:  # every expert on every token, those not chosen with weight zero
        v = (x @ s["w_in"].float().transpose(1, 2)) * s["in_scale"].unsqueeze(1)
        h = _activate(v[..., :f], case["act"]) * v[..., f:]
        y = (h @ s["w_out"].float().transpose(1, 2)) * s["out_scale"].unsqueeze(1)
        mix = torch.zeros(t, e, device="cuda").scatter_(1, ids, weights)
        y = (y * mix.t().unsqueeze(2)).sum(0)
    return {"y": y.to(_TYPES[case["type"]]), "ids": ids.to(torch.int32), "weights": weights}


def run(state):
    if own:
        return _run_own(state)
    return {"rows": _plain_rows, "product": _plain_product, "moe": _plain_moe}[state["case"]["op"]](state)


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------

def _activation64(v, name):
    """The activations from their definitions: Phi(v) is the normal distribution's, sigma(v) the logistic function."""
    if name == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    if name == "gelu":
        return v * torch.special.ndtr(v)
    if name == "gelu_tanh":
        return v * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3))
    if name == "silu":
        return v * torch.sigmoid(v)
    return v


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rows":
        values, scales = [], []
        for part in s["x"].split(512):
            # DynamicQuantizeLinear defines codes by quotients in 32 bits: 64-bit quotients rounded to them are those
            # (53 bits are over twice 24 plus 2, so the second rounding changes nothing).
            x = part.double()
            low, high = x.min(1).values.clamp(max=0.0), x.max(1).values.clamp(min=0.0)
            step = ((high - low).float().double() / 255.0).float().double()
            step = torch.where(step == 0, torch.ones_like(step), step)
            zero = (-low / step).float().round().double()
            code = ((x / step[:, None]).float().round().double() + zero[:, None]).clamp(0.0, 255.0)
            values.append((code - zero[:, None]) * step[:, None])
            scales.append(step)
        return {"values": torch.cat(values), "scale": torch.cat(scales), "zero": None}
    if case["op"] == "product":
        b = s["b"].double() if case["b"] == "kn" else s["b"].double().t().contiguous()
        if case["zeros"]:
            b -= s["b_zero"].double()[None, :]
        out = []
        for i in range(0, case["m"], 1024):
            a = s["a"][i:i + 1024].double()
            if case["zeros"]:
                a -= s["a_zero"][i:i + 1024].double()[:, None]
            v = torch.mm(a, b) * s["a_scale"][i:i + 1024].double()[:, None] * s["b_scale"].double()[None, :]
            if case["bias"]:
                v += s["bias"].double()[None, :]
            v = _activation64(v, case["act"])
            if case["residual"]:
                v += s["residual"][i:i + 1024].double()
            out.append(v)
        return {"c": torch.cat(out)}
    t, f, k = case["tokens"], case["expert"], case["top_k"]
    x = s["x"].double()
    probability = torch.softmax(torch.mm(x, s["router"].double().t()), 1)
    y = torch.zeros_like(x)
    top = torch.argsort(-probability, dim=1, stable=True)[:, :k]
    weights = torch.gather(probability, 1, top)
    weights = weights / weights.sum(1, keepdim=True)
    for e in torch.unique(top).tolist():
        who, place = torch.nonzero(top == e, as_tuple=True)
        up = torch.mm(x[who], (s["w_in"][e].double() * s["in_scale"][e].double()[:, None]).t())
        h = _activation64(up[:, :f], case["act"]) * up[:, f:]
        down = torch.mm(h, (s["w_out"][e].double() * s["out_scale"][e].double()[:, None]).t())
        y.index_add_(0, who, down * weights[who, place][:, None])
    return {"y": y, "ids": None, "weights": weights}
