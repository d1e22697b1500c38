"""Cases of the 8-bit path: rows quantized to int8 with a scale each, the RMS norm and the gated activation that
write such rows, the matrix product of int8 rows, and a feed-forward block of all of them.

Definitions (T: the 16-bit type of the activations; a row with its scale stands for scale * values):
  quantize   scale = max|x| / 127, values = round(x / scale), half to even
  norm       h = T(x + residual) where there is one; y = h / sqrt(mean(h^2) + eps) * weight, then quantized by row
  silu_mul   y = gate / (1 + exp(-gate)) * up, then quantized by row
  linear     T(x_scale[m] * w_scale[n] * sum_k x[m, k] w[n, k] + bias[n])
"""
import math

import torch

own = False

EPS = 1e-5
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one token before a projection, and the weights of a projection quantized once, channel by channel
        {"name": "quantize token", "op": "quantize", "rows": 1, "cols": 4096, "type": "fp16"},
        {"name": "quantize weights", "op": "quantize", "rows": 11008, "cols": 4096, "type": "fp16"},
        # the norm in front of the projections of a decode step of 16 sequences, and of a prefill of an odd length
        # whose width is no multiple of a vector
        {"name": "norm decode", "op": "norm", "rows": 16, "cols": 8192, "type": "bf16", "residual": True},
        {"name": "norm prefill", "op": "norm", "rows": 4095, "cols": 8192, "type": "fp16", "residual": True},
        # between the two products of a feed-forward block: a decode step, and a prefill of a wide one; gate and up are
        # the halves of one product's output
        {"name": "silu_mul decode", "op": "silu_mul", "rows": 4, "cols": 11008, "type": "fp16"},
        {"name": "silu_mul prefill", "op": "silu_mul", "rows": 2048, "cols": 28672, "type": "bf16"},
        # the product: one token, a batch of 16, a ragged one with a bias, and two prefills
        {"name": "linear token", "op": "linear", "rows": 1, "cols": 4096, "outs": 11008, "type": "fp16", "bias": False},
        {"name": "linear batch", "op": "linear", "rows": 16, "cols": 8192, "outs": 28672, "type": "bf16", "bias": False},
        {"name": "linear ragged", "op": "linear", "rows": 333, "cols": 5001, "outs": 1237, "type": "fp16", "bias": True},
        {"name": "linear prefill", "op": "linear", "rows": 4096, "cols": 8192, "outs": 28672, "type": "bf16", "bias": False},
        # a whole feed-forward block with its norm: one token, and a prompt
        {"name": "block token", "op": "block", "rows": 1, "cols": 4096, "ffn": 11008, "type": "fp16"},
        {"name": "block prompt", "op": "block", "rows": 2048, "cols": 4096, "ffn": 11008, "type": "bf16"},
    ]


def draw(rng):
    def size(low, high):
        return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))

    op = rng.choice(["quantize", "norm", "silu_mul", "linear", "linear", "block"])
    case = {"op": op, "type": rng.choice(["fp16", "bf16"])}
    if op in ("quantize", "norm", "silu_mul"):
        cols = size(64, 28672)
        case |= {"rows": size(1, min(16384, 45000000 // cols)), "cols": cols}
        if op == "norm":
            case["residual"] = rng.random() < 0.7
    elif op == "linear":
        cols, outs = size(64, 28672), size(16, 28672)
        if rng.random() < 0.5:  # the widths that models have
            cols, outs = -(-cols // 64) * 64, -(-outs // 64) * 64
        case |= {"rows": size(1, 8192), "cols": cols, "outs": outs, "bias": rng.random() < 0.3}
        while case["rows"] * cols * outs > 4096 * 8192 * 28672:
            case["rows"] = max(1, case["rows"] // 2)
    else:
        cols, ffn = 64 * size(4, 80), 64 * size(8, 200)
        case |= {"rows": size(1, 2048), "cols": cols, "ffn": ffn}
    return case


def _rows(n, k, gen):
    """Rows of int8 as the quantization of a normal distribution gives them, and the scales that leave the products near 1."""
    x = torch.randn(n, k, generator=gen, device="cuda")
    top = x.abs().amax(1, keepdim=True)
    pitch = -(-k // 16) * 16  # rows begin on 16 bytes
    values = torch.zeros(n, pitch, dtype=torch.int8, device="cuda")[:, :k]
    values.copy_((x * (127 / top)).round())
    return values, (top / 127).reshape(-1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    m, k, t = case["rows"], case["cols"], TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def spread():  # channels of different sizes, as activations have them
        return torch.exp(0.5 * normal(k))

    s = {"op": case["op"], "type": t}
    if case["op"] == "quantize":
        s["x"] = (normal(m, k) * spread()).to(t)
    elif case["op"] == "norm":
        s |= {"x": normal(m, k).to(t), "weight": (1 + 0.2 * normal(k)).to(t)}
        s["residual"] = (2 * normal(m, k) * spread()).to(t) if case["residual"] else None
    elif case["op"] == "silu_mul":
        both = (1.5 * normal(m, 2 * k)).to(t)
        s |= {"gate": both[:, :k], "up": both[:, k:]}
    elif case["op"] == "linear":
        s["x"], s["x_scales"] = _rows(m, k, gen)
        s["w"], s["w_scales"] = _rows(case["outs"], k, gen)
        s["w_scales"] = s["w_scales"] / math.sqrt(k)
        s["bias"] = normal(case["outs"]).to(t) if case["bias"] else None
    else:
        f = case["ffn"]
        s |= {"x": normal(m, k).to(t), "residual": (2 * normal(m, k) * spread()).to(t), "weight": (1 + 0.2 * normal(k)).to(t)}
        s["gate_up"], scales = _rows(2 * f, k, gen)
        s["gate_up_scales"] = scales / math.sqrt(k)
        s["down"], scales = _rows(k, f, gen)
        s["down_scales"] = scales / math.sqrt(f)
    return s


def _quantized(y):
    """Values and scales of the rows of `y`, in 32 bits."""
    top = y.abs().amax(1)
    inverse = torch.where(top > 0, 127 / top, 0.0)
    return (y * inverse[:, None]).round(), top / 127


def _normed(x, residual, weight):
    if residual is not None:
        x = (x.float() + residual.float()).to(x.dtype)
    h = x.float()
    return h * torch.rsqrt(h.square().mean(1, keepdim=True) + EPS) * weight.float(), x


def _gated(gate, up):
    gate = gate.float()
    return gate / (1 + torch.exp(-gate)) * up.float()


def _product(x, x_scales, w, w_scales, bias, t):
    y = (x.float() @ w.float().T) * x_scales[:, None] * w_scales[None, :]
    return (y if bias is None else y + bias.float()).to(t)


def run(state):
    s, t = state, state["type"]
    if own:
        return _run_own(s, t)
    if s["op"] == "linear":
        return _product(s["x"], s["x_scales"], s["w"], s["w_scales"], s["bias"], t)
    if s["op"] == "block":
        y, residual = _normed(s["x"], s["residual"], s["weight"])
        both = _product(*_quantized(y), s["gate_up"], s["gate_up_scales"], None, t)
        f = both.shape[1] // 2
        return {"out": _product(*_quantized(_gated(both[:, :f], both[:, f:])), s["down"], s["down_scales"], None, t),
                "residual": residual}
    more = {}
    if s["op"] == "quantize":
        y = s["x"].float()
    elif s["op"] == "norm":
        y, residual = _normed(s["x"], s["residual"], s["weight"])
        if s["residual"] is not None:
            more["residual"] = residual
    else:
        y = _gated(s["gate"], s["up"])
    values, scales = _quantized(y)
    return {"values": (values * scales[:, None]).to(t), "scales": scales, **more}


def _run_own(s, t):
    from gemmlib_b200.int8_linear import Int8Rows, int8_linear, quantize_int8, rms_norm_int8, silu_mul_int8

    if s["op"] == "linear":
        return int8_linear(Int8Rows(s["x"], s["x_scales"]), Int8Rows(s["w"], s["w_scales"]), s["bias"], dtype=t)
    if s["op"] == "block":
        rows, residual = rms_norm_int8(s["x"], s["weight"], EPS, residual=s["residual"])
        both = int8_linear(rows, Int8Rows(s["gate_up"], s["gate_up_scales"]), dtype=t)
        f = both.shape[1] // 2
        rows = silu_mul_int8(both[:, :f], both[:, f:])
        return {"out": int8_linear(rows, Int8Rows(s["down"], s["down_scales"]), dtype=t), "residual": residual}
    more = {}
    if s["op"] == "quantize":
        rows = quantize_int8(s["x"])
    elif s["op"] == "norm":
        rows = rms_norm_int8(s["x"], s["weight"], EPS, residual=s["residual"])
        if s["residual"] is not None:
            rows, more["residual"] = rows
    else:
        rows = silu_mul_int8(s["gate"], s["up"])
    return {"values": rows.dequantize(t), "scales": rows.scales, **more}


def work(case):
    m, k = case["rows"], case["cols"]
    if case["op"] == "linear":
        n = case["outs"]
        return {"bytes": m * k + n * k + 2 * m * n + 4 * (m + n) + 2 * n * case["bias"], "flops": 2 * m * n * k}
    if case["op"] == "block":
        f = case["ffn"]
        # the norm's inputs and outputs, the weights and their scales, the product's outputs and the rows between them
        return {"bytes": 2 * k * 3 * m + 2 * m * k + 3 * f * k + 4 * (2 * f + k) + 2 * m * (2 * f) * 2 + 2 * m * f + 2 * m * k + 2 * k,
                "flops": 2 * m * 3 * f * k}
    # the 16-bit rows read, the int8 ones written; what they stand for is returned: read as int8 and written in 16 bits
    read = {"quantize": 2, "norm": 6 if case.get("residual") else 2, "silu_mul": 4}[case["op"]]
    return {"bytes": m * k * (read + 1 + 1 + 2) + 4 * m + (2 * k if case["op"] == "norm" else 0),
            "flops": m * k * {"quantize": 3, "norm": 7, "silu_mul": 8}[case["op"]]}


def exact(case, seed):
    s = prepare(case, seed)

    def rounded(v):  # to the 16-bit type, where the definition says so
        return v.to(s["type"]).double()

    def by_row(y):
        scale = y.abs().max(dim=1).values / 127
        whole = torch.round(y / torch.where(scale > 0, scale, 1.0).unsqueeze(1))
        return whole, scale

    def product(a, a_scale, w, w_scale):
        out = torch.matmul(a, w.double().t())
        out *= a_scale.double().unsqueeze(1)
        out *= w_scale.double()
        return out

    def norm():
        h = s["x"].double()
        if s["residual"] is not None:
            h = rounded(h + s["residual"].double())
        return s["weight"].double() * h / torch.sqrt((h * h).sum(1, keepdim=True) / h.shape[1] + EPS), h

    if case["op"] == "linear":
        out = product(s["x"].double(), s["x_scales"], s["w"], s["w_scales"])
        if s["bias"] is not None:
            out += s["bias"].double()
        return out
    if case["op"] == "block":
        y, h = norm()
        both = rounded(product(*by_row(y), s["gate_up"], s["gate_up_scales"]))
        gate, up = both.chunk(2, dim=1)
        return {"out": product(*by_row(gate * torch.sigmoid(gate) * up), s["down"], s["down_scales"]), "residual": h}
    more = {}
    if case["op"] == "quantize":
        y = s["x"].double()
    elif case["op"] == "norm":
        y, h = norm()
        if s["residual"] is not None:
            more["residual"] = h
    else:
        y = s["gate"].double() * torch.sigmoid(s["gate"].double()) * s["up"].double()
    whole, scale = by_row(y)
    return {"values": whole * scale.unsqueeze(1), "scales": scale, **more}
