"""What is timed of the 8-bit matrix products, and how their results are checked: single calls of the operators that serve a
model whose weights and activations are float8 (e4m3: 4 bits of exponent, 3 of mantissa, largest value 448), with scales.

Activations [M, K] carry one scale per row and group of 128 values of K, a power of two held in 8 bits (e8m0: the exponent
alone); weights [N, K] one float32 scale per block of 128 x 128.  A scale is the smallest power of two that brings the largest
magnitude of its group to 448 or less, 2^-126 at least, and 1 for a group of zeros.  A case is one of
  norm      a root-mean-square norm of float32 rows that leaves 8-bit rows: what stands before a projection
  rows      rows of the model's type to 8 bits: what stands before the projection behind the attention
  weight    a weight matrix to 8 bits, once when a model is loaded
  linear    out = A W^T, as bfloat16, as float32, or added to float32 rows (the residual stream)
  gated     act(A Wg^T) * (A Wu^T), gate and up rows of the weight alternating in blocks of 128, as bfloat16 or as the 8-bit
            rows that the product behind it reads"""
import math

import torch

own = False          # True: `run` calls the framework's operators; False: their plain form
DEVICE = "cuda:0"
GROUP = 128
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
_DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ---------------------------------------------------------------------------------------------- the cases

def listed():
    return [
        # eight chats decode one token each: nothing but latency
        {"name": "norm_8x2048", "op": "norm", "m": 8, "k": 2048},
        # a prompt's portion at the width of an 8-billion-parameter model
        {"name": "norm_2048x4096", "op": "norm", "m": 2048, "k": 4096},
        # a few decoded tokens of a model whose width is no multiple of a group
        {"name": "rows_33x2000", "op": "rows", "m": 33, "k": 2000, "dtype": "bfloat16"},
        # long prompts in one step, the width of a feed-forward
        {"name": "rows_8192x14336", "op": "rows", "m": 8192, "k": 14336, "dtype": "bfloat16"},
        # a small model's fused query, key and value matrix while it is loaded
        {"name": "weight_2560x2048", "op": "weight", "n": 2560, "k": 2048, "dtype": "bfloat16"},
        # a large model's feed-forward matrix from a 32-bit checkpoint
        {"name": "weight_14336x4096", "op": "weight", "n": 14336, "k": 4096, "dtype": "float32"},
        # one chat at a time: the weight is read once, for one row
        {"name": "linear_1x2560x2048", "op": "linear", "m": 1, "n": 2560, "k": 2048, "out": "bfloat16"},
        # a full server decodes: the down projection of 64 tokens into the residual stream
        {"name": "linear_64x4096x14336", "op": "linear", "m": 64, "n": 4096, "k": 14336, "out": "add"},
        # odd sizes throughout, in 32 bits
        {"name": "linear_333x1000x1520", "op": "linear", "m": 333, "n": 1000, "k": 1520, "out": "float32"},
        # long prompts in one step
        {"name": "linear_8192x4096x14336", "op": "linear", "m": 8192, "n": 4096, "k": 14336, "out": "bfloat16"},
        # eight chats decode: gate, up and their product for the down projection to read in 8 bits
        {"name": "gated_8x5632x2048", "op": "gated", "m": 8, "i": 5632, "k": 2048, "act": "silu", "out": "e4m3"},
        # a prompt's portion of a large model
        {"name": "gated_2048x14336x4096", "op": "gated", "m": 2048, "i": 14336, "k": 4096, "act": "silu", "out": "e4m3"},
    ]


def _spread(rng, low, high, step=1):
    """A whole number between low and high, even over the logarithm, a multiple of `step`."""
    return max(low, int(math.exp(rng.uniform(math.log(low), math.log(high)))) // step * step)


def draw(rng):
    op = rng.choice(["norm", "rows", "weight", "linear", "linear", "linear", "gated", "gated"])
    step = rng.choice([1, 8, 128])
    k = _spread(rng, 128, 14336, step)
    if op == "norm":
        return {"op": op, "m": _spread(rng, 1, 8192), "k": min(k, 8192)}
    if op == "rows":
        return {"op": op, "m": _spread(rng, 1, 8192), "k": k, "dtype": rng.choice(["bfloat16", "bfloat16", "float32"])}
    if op == "weight":
        return {"op": op, "n": _spread(rng, 128, 14336, step), "k": min(k, 8192), "dtype": rng.choice(["bfloat16", "float32"])}
    most = 8192 * 4096 * 14336
    if op == "linear":
        n = _spread(rng, 128, 14336, step)
        return {"op": op, "m": min(_spread(rng, 1, 8192), max(1, most // (n * k))), "n": n, "k": k,
                "out": rng.choice(["bfloat16", "bfloat16", "float32", "add"])}
    i = _spread(rng, 128, 14336, step)
    return {"op": op, "m": min(_spread(rng, 1, 8192), max(1, most // (2 * i * k))), "i": i, "k": k,
            "act": rng.choice(["silu", "silu", "gelu_tanh"]), "out": rng.choice(["e4m3", "e4m3", "bfloat16"])}


def _groups(k):
    return -(-k // GROUP)


def work(case):
    op, k = case["op"], case["k"]
    if op == "norm":
        return {"bytes": case["m"] * (4 * k + k + _groups(k)) + 4 * k, "flops": 6 * case["m"] * k}
    if op == "rows":
        return {"bytes": case["m"] * (k * _DTYPES[case["dtype"]].itemsize + k + _groups(k)), "flops": 3 * case["m"] * k}
    if op == "weight":
        return {"bytes": case["n"] * k * (_DTYPES[case["dtype"]].itemsize + 1) + 4 * _groups(case["n"]) * _groups(k),
                "flops": 3 * case["n"] * k}
    m = case["m"]
    n = case["n"] if op == "linear" else 2 * case["i"]
    read = m * (k + _groups(k)) + n * k + 4 * _groups(n) * _groups(k)
    if op == "linear":
        return {"bytes": read + m * n * {"bfloat16": 2, "float32": 4, "add": 8}[case["out"]], "flops": 2 * m * n * k}
    i = case["i"]
    return {"bytes": read + m * (2 * i if case["out"] == "bfloat16" else i + _groups(i)), "flops": 2 * m * n * k + 6 * m * i}


# ---------------------------------------------------------------------------------------------- the inputs

def _rows8(m, k):
    """Room for 8-bit rows, whose rows start on 16 bytes, and for their scales."""
    data = torch.empty(m, -(-k // 16) * 16, dtype=torch.uint8, device=DEVICE).view(E4M3)[:, :k]
    scales = torch.empty(m, -(-_groups(k) // 16) * 16, dtype=torch.uint8, device=DEVICE).view(E8M0)[:, : _groups(k)]
    return data, scales


def _weight8(n, k):
    data = torch.empty(n, -(-k // 16) * 16, dtype=torch.uint8, device=DEVICE).view(E4M3)[:, :k]
    return data, torch.empty(_groups(n), _groups(k), dtype=torch.float32, device=DEVICE)


def _activations(g, m, k):
    """Rows of which a few channels are much larger than the rest, as a trained model's are."""
    channel = torch.exp(0.5 * torch.randn(k, generator=g, device=DEVICE))
    channel[torch.rand(k, generator=g, device=DEVICE) < 0.01] *= 20
    return torch.randn(m, k, generator=g, device=DEVICE) * channel


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    op, k = case["op"], case["k"]
    s = {"case": case}
    if op == "norm":
        s |= {"x": _activations(g, case["m"], k), "weight": 1 + 0.2 * torch.randn(k, generator=g, device=DEVICE), "out": _rows8(case["m"], k)}
    elif op == "rows":
        s |= {"x": _activations(g, case["m"], k).to(_DTYPES[case["dtype"]]), "out": _rows8(case["m"], k)}
    elif op == "weight":
        spread = torch.exp(0.3 * torch.randn(case["n"], 1, generator=g, device=DEVICE))
        w = 0.02 * torch.randn(case["n"], k, generator=g, device=DEVICE) * spread
        s |= {"w": w.to(_DTYPES[case["dtype"]]), "out": _weight8(case["n"], k)}
    else:
        m = case["m"]
        s["a"] = _rows8(m, k)
        _put(s["a"], _quantize_rows(_activations(g, m, k)))
        if op == "linear":
            n = case["n"]
            s["w"] = _weight8(n, k)
            _put(s["w"], _quantize_weight(torch.randn(n, k, generator=g, device=DEVICE) / math.sqrt(k)))
            if case["out"] == "add":
                s["resid"] = torch.randn(m, n, generator=g, device=DEVICE)
            s["out"] = torch.empty(m, n, dtype=_DTYPES.get(case["out"], torch.float32), device=DEVICE)
        else:
            i, blocks = case["i"], _groups(case["i"])
            w = torch.zeros(2, blocks * GROUP, k, device=DEVICE)     # rows behind the last of gate and up are zeros
            w[:, :i] = torch.randn(2, i, k, generator=g, device=DEVICE) / math.sqrt(k)
            w = w.view(2, blocks, GROUP, k).transpose(0, 1).reshape(2 * blocks * GROUP, k)
            s["w"] = _weight8(2 * blocks * GROUP, k)
            _put(s["w"], _quantize_weight(w))
            s["out"] = _rows8(m, i) if case["out"] == "e4m3" else torch.empty(m, i, dtype=torch.bfloat16, device=DEVICE)
    return s


def _put(room, values):
    for r, v in zip(room, values):
        r.copy_(v)


# ---------------------------------------------------------------------------------------------- one pass

def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        from tiny_llm_b200 import ops
        if op == "norm":
            ops.rms_norm_fp8(s["x"], s["weight"], 1e-5, *s["out"])
            return s["out"]
        if op == "rows":
            ops.quantize_fp8(s["x"], *s["out"])
            return s["out"]
        if op == "weight":
            ops.quantize_weight_fp8(s["w"], *s["out"])
            return s["out"]
        if op == "linear":
            if case["out"] == "add":
                s["out"].copy_(s["resid"])
            ops.linear_fp8(*s["a"], *s["w"], s["out"], accumulate=case["out"] == "add")
            return s["out"]
        if case["out"] == "e4m3":
            ops.linear_swiglu_fp8(*s["a"], *s["w"], s["out"][0], s["out"][1], act=case["act"])
        else:
            ops.linear_swiglu_fp8(*s["a"], *s["w"], s["out"], act=case["act"])
        return s["out"]
    if op == "norm":
        x = s["x"]
        return _quantize_rows(x / torch.sqrt((x * x).mean(1, keepdim=True) + 1e-5) * s["weight"])
    if op == "rows":
        return _quantize_rows(s["x"].float())
    if op == "weight":
        return _quantize_weight(s["w"].float())
    k = case["k"]
    a = s["a"][0].float() * s["a"][1].float().repeat_interleave(GROUP, 1)[:, :k]
    w, ws = s["w"]
    w = w.float() * ws.repeat_interleave(GROUP, 0)[: w.shape[0]].repeat_interleave(GROUP, 1)[:, :k]
    y = a @ w.T
    if op == "linear":
        return (y + s["resid"] if case["out"] == "add" else y).to(s["out"].dtype)
    i = case["i"]
    y = y.view(case["m"], -1, 2, GROUP)
    gate, up = (y[:, :, side].reshape(case["m"], -1)[:, :i] for side in (0, 1))
    if case["act"] == "silu":
        h = gate / (1 + torch.exp(-gate)) * up
    else:
        h = 0.5 * gate * (1 + torch.tanh(math.sqrt(2 / math.pi) * (gate + 0.044715 * gate ** 3))) * up
    return _quantize_rows(h) if case["out"] == "e4m3" else h.to(torch.bfloat16)


def _exponent_byte(largest):
    """The scale's biased exponent for groups whose largest magnitudes these are: largest / 2^e <= 448 = 1.75 * 2^8."""
    byte = ((largest.contiguous().view(torch.int32) + 0x1FFFFF) >> 23) - 8
    return torch.where(largest == 0, 127, byte.clamp(min=1))


def _power(byte):
    return (byte << 23).view(torch.float32)


def _quantize_rows(x):
    m, k = x.shape
    grouped = torch.nn.functional.pad(x, (0, _groups(k) * GROUP - k)).view(m, -1, GROUP)
    byte = _exponent_byte(grouped.abs().amax(2))
    data = (grouped * _power(254 - byte)[:, :, None]).to(E4M3)
    return data.view(m, -1)[:, :k], byte.to(torch.uint8).view(E8M0)


def _quantize_weight(w):
    n, k = w.shape
    gn, gk = _groups(n), _groups(k)
    blocks = torch.nn.functional.pad(w, (0, gk * GROUP - k, 0, gn * GROUP - n)).view(gn, GROUP, gk, GROUP)
    byte = _exponent_byte(blocks.abs().amax((1, 3)))
    data = (blocks * _power(254 - byte)[:, None, :, None]).to(E4M3)
    return data.view(gn * GROUP, gk * GROUP)[:n, :k], _power(byte)


# ---------------------------------------------------------------------------------------------- in 64 bits

def _two_to(exponent):
    """2^e in 64 bits, to the bit (a power function may be a unit off, which would move a value across a border)."""
    return ((exponent.long() + 1023) << 52).view(torch.float64)


def _exact_e4m3(x, largest):
    """The values that x / scale rounds to (to the nearest multiple of the step at its size, the even one of two), and the
    scale, for magnitudes that are at most `largest`."""
    exponent = torch.ceil(torch.log2(largest / 448)).clamp(min=-200)
    exponent = torch.where(largest > 448 * _two_to(exponent), exponent + 1, exponent)
    exponent = torch.where(largest <= 448 * _two_to(exponent - 1), exponent - 1, exponent).clamp(min=-126)
    scale = torch.where(largest == 0, 1.0, _two_to(exponent))
    y = x / scale
    step = _two_to((torch.frexp(y)[1] - 1).clamp(min=-6) - 3)
    return torch.round(y / step) * step, scale


def _exact_rows(x):
    pieces = [_exact_e4m3(x[:, g: g + GROUP], x[:, g: g + GROUP].abs().amax(1, keepdim=True)) for g in range(0, x.shape[1], GROUP)]
    return torch.cat([p[0] for p in pieces], 1), torch.cat([p[1] for p in pieces], 1)


def exact(case, seed):
    s = prepare(case, seed)
    op, k = case["op"], case["k"]
    if op == "norm":
        x = s["x"].double()
        return _exact_rows(s["weight"].double() * x * ((x ** 2).sum(1, keepdim=True) / k + 1e-5) ** -0.5)
    if op == "rows":
        return _exact_rows(s["x"].double())
    if op == "weight":
        data, scales = torch.empty(s["w"].shape, dtype=torch.float64, device=DEVICE), torch.empty(s["out"][1].shape, dtype=torch.float64, device=DEVICE)
        for b in range(scales.shape[0]):
            rows = s["w"][b * GROUP: (b + 1) * GROUP].double()
            for c in range(scales.shape[1]):
                block = rows[:, c * GROUP: (c + 1) * GROUP]
                data[b * GROUP: (b + 1) * GROUP, c * GROUP: (c + 1) * GROUP], scales[b, c] = _exact_e4m3(block, block.abs().max())
        return data, scales
    # the blocks of K one after the other: a product of the 8-bit values, then the scales of its rows and columns
    (a, sa), (w, sw) = s["a"], s["w"]
    column = torch.arange(w.shape[0], device=DEVICE) // GROUP
    y = torch.zeros(a.shape[0], w.shape[0], dtype=torch.float64, device=DEVICE)
    for g in range(_groups(k)):
        part = a[:, g * GROUP: (g + 1) * GROUP].double() @ w[:, g * GROUP: (g + 1) * GROUP].double().T
        y += part * sa[:, g: g + 1].double() * sw[column, g].double()
    if op == "linear":
        return y + s["resid"].double() if case["out"] == "add" else y
    blocks = [y[:, 2 * GROUP * b: 2 * GROUP * (b + 1)] for b in range(_groups(case["i"]))]
    gate, up = torch.cat([b[:, :GROUP] for b in blocks], 1)[:, : case["i"]], torch.cat([b[:, GROUP:] for b in blocks], 1)[:, : case["i"]]
    if case["act"] == "silu":
        h = gate * torch.sigmoid(gate) * up
    else:   # z / 2 (1 + tanh(y)) = z sigmoid(2 y)
        h = gate * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (gate + 0.044715 * gate ** 3)) * up
    return _exact_rows(h) if case["out"] == "e4m3" else h
