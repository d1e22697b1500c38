"""Cases of the 8-bit floating-point path: rows and weights in e4m3 with a scale for each block of 128, their product, and
the same for a layer of experts: tokens sorted by expert and back, and the product of every expert with its rows.

Definitions (T: the 16-bit type of the activations; blocks at an edge hold what is left):
  rows       a row's block of 128 elements:   scale = max|x| / 448, values = e4m3(x * 448 / max|x|), half to even
  weights    a block of 128 x 128 elements:   the same
  gate       y = gate / (1 + exp(-gate)) * up, then as rows
  linear     T(sum over the blocks b of k of x_scale[m, b] * w_scale[n / 128, b] * sum_(k in b) x[m, k] w[n, k]  + bias[n])
  route      the choices (token t, number j) of experts[t, j], stably sorted by expert, those of no expert behind all others: source
             names the choice at each place, places the place of each choice (-1: no expert), offsets where each expert's rows begin;
             rows[p] = x[token of source[p]] (0 where there is no expert); out[t] = T(sum_j weights[t, j] * y[places[t, j]])
  experts    of the rows of each expert: linear with its weight; a block of them: route, rows, gate and up, gate, down, route back
"""
import math

import torch

own = False

E4M3 = torch.float8_e4m3fn
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one token ahead of a projection, and the weights of a projection, once, when a model is loaded
        {"name": "rows token", "op": "rows", "rows": 1, "cols": 4096, "type": "fp16"},
        {"name": "weights", "op": "weights", "rows": 11008, "cols": 4096, "type": "bf16"},
        # between the two products of a wide feed-forward block in a prefill; gate and up are halves of one product's output
        {"name": "gate prompt", "op": "gate", "rows": 2048, "cols": 28672, "type": "bf16"},
        # the product: one token, a batch of 16, a ragged one with a bias, a prefill
        {"name": "linear token", "op": "linear", "rows": 1, "cols": 4096, "outs": 11008, "type": "fp16", "bias": False},
        {"name": "linear batch", "op": "linear", "rows": 16, "cols": 8192, "outs": 28672, "type": "bf16", "bias": False},
        {"name": "linear ragged", "op": "linear", "rows": 333, "cols": 5001, "outs": 1237, "type": "fp16", "bias": True},
        {"name": "linear prompt", "op": "linear", "rows": 4096, "cols": 8192, "outs": 28672, "type": "bf16", "bias": False},
        # tokens to their experts and back: a decode step of 16 sequences, and a training step with its gradients
        {"name": "route decode", "op": "route", "tokens": 16, "cols": 4096, "experts": 64, "choices": 8, "dropped": 0.0, "train": False, "type": "bf16"},
        {"name": "route train", "op": "route", "tokens": 8192, "cols": 4096, "experts": 32, "choices": 4, "dropped": 0.0, "train": True, "type": "bf16"},
        # one product of experts where half of the choices belong to another GPU's experts and sizes are odd
        {"name": "experts ragged", "op": "experts", "tokens": 501, "cols": 1237, "outs": 1000, "experts": 7, "choices": 2, "dropped": 0.5, "type": "fp16"},
        # a whole layer of experts: a decode step of 16 sequences, and a prompt
        {"name": "layer decode", "op": "layer", "tokens": 16, "cols": 2048, "ffn": 1408, "experts": 64, "choices": 8, "dropped": 0.0, "type": "bf16"},
        {"name": "layer prompt", "op": "layer", "tokens": 4096, "cols": 4096, "ffn": 1408, "experts": 32, "choices": 4, "dropped": 0.0, "type": "bf16"},
    ]


def draw(rng):
    def size(low, high):
        return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))

    op = rng.choice(["rows", "weights", "gate", "linear", "linear", "route", "route", "experts", "layer"])
    case = {"op": op, "type": rng.choice(["fp16", "bf16"])}
    if op in ("rows", "weights", "gate"):
        cols = size(64, 28672)
        return case | {"rows": size(1, min(16384, 45000000 // cols)), "cols": cols}
    whole = rng.random() < 0.5  # the widths that models have
    if op == "linear":
        cols, outs = size(64, 28672), size(16, 28672)
        if whole:
            cols, outs = -(-cols // 64) * 64, -(-outs // 64) * 64
        case |= {"rows": size(1, 8192), "cols": cols, "outs": outs, "bias": rng.random() < 0.3}
        while case["rows"] * cols * outs > 4096 * 8192 * 28672:
            case["rows"] = max(1, case["rows"] // 2)
        return case
    experts = size(2, 128)
    case |= {"tokens": size(1, 4096), "cols": size(64, 4096), "experts": experts, "choices": rng.randint(1, min(8, experts)),
             "dropped": rng.choice([0.0, 0.0, 0.1, 0.7])}
    if op == "route":
        return case | {"train": rng.random() < 0.5}
    wide = "outs" if op == "experts" else "ffn"
    case[wide] = size(64, 2048)
    if whole:
        case["cols"], case[wide] = -(-case["cols"] // 64) * 64, -(-case[wide] // 64) * 64
    while case["experts"] * case["cols"] * case[wide] > 32 * 4096 * 1408:
        case[wide] = max(64, case[wide] // 2)
    while case["tokens"] * case["choices"] > 16384:
        case["tokens"] //= 2
    return case


def _blocks(n):
    return -(-n // 128)


def _spread(s, rows, cols):
    """A scale for each element, from one for each block."""
    return s.repeat_interleave(128, -1)[..., :cols] if rows is None else s.repeat_interleave(128, -2)[..., :rows, :].repeat_interleave(128, -1)[..., :cols]


def _pitched(values):
    """Rows that begin on 16 bytes, as a loaded or quantized weight has them."""
    k = values.size(-1)
    held = torch.zeros(*values.shape[:-1], -(-k // 16) * 16, dtype=values.dtype, device=values.device)[..., :k]
    held.copy_(values)
    return held


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    k, t, op = case["cols"], TYPES[case["type"]], case["op"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def spread():  # channels of different sizes, as activations have them
        return torch.exp(0.5 * normal(k))

    def weight(*shape):
        """Values with the scales that leave products near 1, as the quantization of a normal distribution gives them."""
        scales = (0.8 + 0.4 * torch.rand(*shape[:-2], _blocks(shape[-2]), _blocks(shape[-1]), generator=gen, device="cuda")) * (4.5 / 448)
        values = torch.empty(shape, dtype=E4M3, device="cuda")
        for part, out in zip([normal(*shape)] if len(shape) == 2 else (normal(*shape[1:]) for _ in range(shape[0])),
                             [values] if len(shape) == 2 else values):
            out.copy_((part * (448 / 4.5)).clamp(-448, 448))
        return _pitched(values), scales / math.sqrt(shape[-1])

    s = {"op": op, "type": t}
    if op in ("rows", "weights", "gate", "linear"):
        m = case["rows"]
    if op == "rows":
        return s | {"x": (normal(m, k) * spread()).to(t)}
    if op == "weights":
        return s | {"x": (0.02 * normal(m, k)).to(t)}
    if op == "gate":
        both = (1.5 * normal(m, 2 * k)).to(t)
        return s | {"gate": both[:, :k], "up": both[:, k:]}
    if op == "linear":
        values, scales = _rows(normal(m, k) * spread())
        s["w"], s["w_scales"] = weight(case["outs"], k)
        return s | {"x": _pitched(values), "x_scales": scales, "bias": normal(case["outs"]).to(t) if case["bias"] else None}
    n, e, c = case["tokens"], case["experts"], case["choices"]
    # a token's experts are different ones, some of them wanted more often than others; -1 for those that are not this GPU's
    liked = normal(n, e) + normal(e)
    s["experts"] = liked.argsort(1, descending=True)[:, :c].contiguous()
    s["experts"] = torch.where(torch.rand(n, c, generator=gen, device="cuda") < case["dropped"], -1, s["experts"])
    s["n_experts"] = e
    if op == "experts":
        order = _sorted(s["experts"], e)
        values, scales = _rows(normal(n * c, k) * spread())
        s["w"], s["w_scales"] = weight(e, case["outs"], k)
        # the number of rows that the plain form leaves each expert room for
        return s | {"x": _pitched(values), "x_scales": scales, "offsets": order[2], "most": max(1, int(order[2].diff().max()))}
    s["x"] = (normal(n, k) * spread()).to(t)
    s["weights"] = torch.softmax(normal(n, c), 1)
    if op == "route":
        s["y"] = normal(n * c, k).to(t)
        s["train"] = case["train"]
        if case["train"]:
            s |= {"d_rows": normal(n * c, k).to(t), "d_out": normal(n, k).to(t)}
        return s
    f = case["ffn"]
    s["most"] = max(1, int(_sorted(s["experts"], e)[2].diff().max()))
    s["gate_up"], s["gate_up_scales"] = weight(e, 2 * f, k)
    s["down"], s["down_scales"] = weight(e, k, f)
    return s


def _quantized(y, top):
    """Values of `y` where the largest magnitude of each element's block is `top`; in 64 bits, so that halves fall as defined."""
    return (y.double() * torch.where(top > 0, 448 / top.double(), 0.0)).to(torch.float32).to(E4M3)


def _rows(y):
    n, k = y.shape
    pad = torch.nn.functional.pad(y, (0, -k % 128)).view(n, -1, 128)
    top = pad.float().abs().amax(-1)
    y, top64 = y.double(), _spread(top, None, k).double()
    values = torch.where(top64 > 0, y * 448 / top64, 0.0).to(torch.float32).to(E4M3)
    return values, (top.double() / 448).float()


def _weights(w):
    n, k = w.shape
    pad = torch.nn.functional.pad(w, (0, -k % 128, 0, -n % 128)).view(_blocks(n), 128, _blocks(k), 128)
    top = pad.float().abs().amax((1, 3))
    top64 = _spread(top, n, k).double()
    values = torch.where(top64 > 0, w.double() * 448 / top64, 0.0).to(torch.float32).to(E4M3)
    return values, (top.double() / 448).float()


def _gated(gate, up):
    gate = gate.float()
    return gate / (1 + torch.exp(-gate)) * up.float()


def _real(values, scales, rows=None):
    return values.float() * _spread(scales, rows, values.size(-1))


def _sorted(experts, n_experts):
    flat = experts.reshape(-1)
    flat = torch.where((flat >= 0) & (flat < n_experts), flat, n_experts)
    mine = flat[:, None] == torch.arange(n_experts + 1, device=flat.device)
    counts = mine.sum(0)
    begins = counts.cumsum(0) - counts
    place = begins[flat] + (mine.cumsum(0) - 1).gather(1, flat[:, None])[:, 0]
    source = torch.zeros_like(flat).index_put_((place,), torch.arange(flat.numel(), device=flat.device))
    places = torch.where(flat < n_experts, place, -1).view(experts.shape)
    return source.int(), places.int(), begins.int()


def _expert_product(x, w, w_scales, offsets, most, t):
    """x: real rows in 32 bits.  Every expert's rows in a block of its own with room for `most`."""
    e, n, k = w.shape
    place = torch.arange(x.size(0), device=x.device)
    expert = (place[:, None] >= offsets[None, 1:]).sum(1)
    kept = expert < e
    expert = torch.where(kept, expert, 0)
    at = torch.where(kept, expert * most + place - offsets[expert], e * most)
    room = torch.zeros(e * most + 1, k, device=x.device).index_put_((at,), torch.where(kept[:, None], x, 0.0))[:-1].view(e, most, k)
    y = (room @ _real(w, w_scales, n).transpose(1, 2)).view(e * most, n)
    return torch.where(kept[:, None], y[torch.where(kept, at, 0)], 0.0).to(t)


def _gather(x, order):
    source, places, offsets = order
    kept = torch.arange(source.numel(), device=x.device) < offsets[-1]
    return torch.where(kept[:, None], x[source // places.size(1)], 0)


def _combine(y, places, weights, t):
    if y.size(0) == 0:
        return y.new_zeros(places.size(0), y.size(1))
    taken = torch.where(places[:, :, None] >= 0, y[places.clamp(min=0)].float(), 0.0)
    return (taken * weights[:, :, None]).sum(1).to(t)


def run(state):
    s, t, op = state, state["type"], state["op"]
    if own:
        return _run_own(s, t, op)
    if op in ("rows", "gate", "weights"):
        values, scales = _weights(s["x"]) if op == "weights" else _rows(s["x"] if op == "rows" else _gated(s["gate"], s["up"]))
        return {"values": _real(values, scales, values.size(0) if op == "weights" else None).to(t), "scales": scales}
    if op == "linear":
        y = _real(s["x"], s["x_scales"]) @ _real(s["w"], s["w_scales"], s["w"].size(0)).T
        return (y if s["bias"] is None else y + s["bias"].float()).to(t)
    if op == "experts":
        return _expert_product(_real(s["x"], s["x_scales"]), s["w"], s["w_scales"], s["offsets"], s["most"], t)
    order = _sorted(s["experts"], s["n_experts"])
    source, places, offsets = order
    if op == "layer":
        both = _expert_product(_real(*_rows(_gather(s["x"], order))), s["gate_up"], s["gate_up_scales"], offsets, s["most"], t)
        f = both.size(1) // 2
        y = _expert_product(_real(*_rows(_gated(both[:, :f], both[:, f:]))), s["down"], s["down_scales"], offsets, s["most"], t)
        return _combine(y, places, s["weights"], t)
    result = {"source": source, "places": places, "offsets": offsets, "rows": _gather(s["x"], order),
              "out": _combine(s["y"], places, s["weights"], t)}
    if s["train"]:
        token, c = source // places.size(1), places.size(1)
        kept = (torch.arange(source.numel(), device=token.device) < offsets[-1])[:, None]
        d_out = s["d_out"].float()
        result["d_x"] = _combine(s["d_rows"], places, torch.ones_like(s["weights"]), t)
        result["d_y"] = torch.where(kept, s["weights"].reshape(-1)[source][:, None] * d_out[token], 0.0).to(t)
        dots = torch.where(kept, s["y"].float() * d_out[token], 0.0).sum(1)
        result["d_weights"] = torch.zeros_like(dots).index_put_((source,), dots).view(-1, c)
    return result


def _run_own(s, t, op):
    from gemmlib_b200.experts import combine_rows, fp8_expert_linear, gather_rows, sort_by_expert
    from gemmlib_b200.fp8_linear import Fp8Rows, Fp8Weight, fp8_linear, quantize_fp8, quantize_fp8_weight, silu_mul_fp8

    if op in ("rows", "gate", "weights"):
        rows = quantize_fp8_weight(s["x"]) if op == "weights" else quantize_fp8(s["x"]) if op == "rows" else silu_mul_fp8(s["gate"], s["up"])
        return {"values": rows.dequantize(t), "scales": rows.scales}
    if op == "linear":
        return fp8_linear(Fp8Rows(s["x"], s["x_scales"]), Fp8Weight(s["w"], s["w_scales"]), s["bias"], dtype=t)
    if op == "experts":
        return fp8_expert_linear(Fp8Rows(s["x"], s["x_scales"]), Fp8Weight(s["w"], s["w_scales"]), s["offsets"], dtype=t)
    order = sort_by_expert(s["experts"], s["n_experts"])
    if op == "layer":
        both = fp8_expert_linear(quantize_fp8(s["x"], order), Fp8Weight(s["gate_up"], s["gate_up_scales"]), order.offsets, dtype=t)
        f = both.size(1) // 2
        y = fp8_expert_linear(silu_mul_fp8(both[:, :f], both[:, f:]), Fp8Weight(s["down"], s["down_scales"]), order.offsets, dtype=t)
        return combine_rows(y, order, s["weights"])
    result = {"source": order.source, "places": order.places, "offsets": order.offsets}
    if not s["train"]:
        return result | {"rows": gather_rows(s["x"], order), "out": combine_rows(s["y"], order, s["weights"])}
    leaves = [s[name].detach().requires_grad_() for name in ("x", "y", "weights")]
    rows, out = gather_rows(leaves[0], order), combine_rows(leaves[1], order, leaves[2])
    grads = torch.autograd.grad((rows, out), leaves, (s["d_rows"], s["d_out"]))
    return result | {"rows": rows.detach(), "out": out.detach(), "d_x": grads[0], "d_y": grads[1], "d_weights": grads[2]}


def work(case):
    k, op = case["cols"], case["op"]
    if op in ("rows", "gate", "weights"):
        # the 16-bit rows read, the 8-bit ones written; what they stand for is returned: read in 8 bits and written in 16
        m = case["rows"]
        return {"bytes": m * k * ((4 if op == "gate" else 2) + 1 + 1 + 2) + 4 * _blocks(k) * (_blocks(m) if op == "weights" else m),
                "flops": m * k * (8 if op == "gate" else 3)}
    if op == "linear":
        m, n = case["rows"], case["outs"]
        return {"bytes": m * k + n * k + 2 * m * n + 4 * _blocks(k) * (m + _blocks(n)) + 2 * n * case["bias"], "flops": 2 * m * n * k}
    n, c, e = case["tokens"], case["choices"], case["experts"]
    rows = round(n * c * (1 - case["dropped"]))
    used = e * (1 - (1 - 1 / e) ** rows)  # experts that have rows, where each is as likely as another
    if op == "experts":
        m = case["outs"]
        return {"bytes": round(used * (m * k + 4 * _blocks(m) * _blocks(k)) + rows * (k + 4 * _blocks(k)) + 2 * n * c * m), "flops": 2 * rows * m * k}
    sort = 8 * n * c + 4 * (2 * n * c + e + 1)
    if op == "layer":
        f = case["ffn"]
        # the weights, the tokens in and out; between the operators: the rows in 8 bits, gate and up, the gated rows, the outputs
        return {"bytes": round(used * 3 * f * k + sort + 4 * n * c + 4 * n * k + rows * (2 * k + 8 * f + 2 * f + 4 * k)),
                "flops": 2 * rows * 3 * f * k}
    passes = 2 * n * k + 2 * n * c * k + 2 * rows * k + 4 * n * c + 2 * n * k  # x and the rows of it; y, the weights and out
    if case["train"]:  # the gradients of rows and out read, y and the weights again, the gradients of x, y and the weights written
        passes += 2 * rows * k + 2 * n * k + 2 * rows * k + 4 * n * c + 2 * n * k + 2 * n * c * k + 4 * n * c
    return {"bytes": sort + passes, "flops": rows * k * (2 + 5 * case["train"])}


def exact(case, seed):
    s = prepare(case, seed)
    t, op = s["type"], case["op"]

    def rounded(v):  # to the 16-bit type, where the definition says so
        return v.to(t).double()

    def to_e4m3(v):
        """The nearest of the numbers that e4m3 has, half to even: a step is 2^-3 of the power of two below, at least 2^-9."""
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
        return torch.round(v / step) * step

    def each(scale, length, dim):
        index = torch.arange(length, device=scale.device) // 128
        return scale.double().index_select(dim, index)

    def by_block(y, high):
        n, k = y.shape
        scale = torch.empty(-(-n // high), _blocks(k), dtype=torch.float64, device=y.device)
        for b in range(_blocks(k)):
            top = y[:, b * 128:(b + 1) * 128].abs().max(dim=1).values
            scale[:, b] = top if high == 1 else torch.nn.functional.pad(top, (0, -n % high)).view(-1, high).max(dim=1).values
        full = each(scale, k, 1)
        full = full if high == 1 else each(full, n, 0)
        return to_e4m3(y * 448 / torch.where(full > 0, full, 1.0)) * full / 448, scale / 448

    def product(a, w, w_scales):
        return a @ (w.double() * each(each(w_scales, w.size(0), 0), w.size(1), 1)).t()

    def silu(v):
        return v * torch.sigmoid(v)

    def of_experts(a, w, w_scales, offsets):
        out = torch.zeros(a.size(0), w.size(1), dtype=torch.float64, device=a.device)
        for e, (lo, hi) in enumerate(zip(offsets[:-1], offsets[1:])):
            if hi > lo:
                out[lo:hi] = product(a[lo:hi], w[e], w_scales[e])
        return out

    if op in ("rows", "weights", "gate"):
        y = silu(s["gate"].double()) * s["up"].double() if op == "gate" else s["x"].double()
        values, scales = by_block(y, 128 if op == "weights" else 1)
        return {"values": values, "scales": scales}
    if op == "linear":
        out = product(s["x"].double() * each(s["x_scales"], s["x"].size(1), 1), s["w"], s["w_scales"])
        return out if s["bias"] is None else out + s["bias"].double()
    if op == "experts":
        return of_experts(s["x"].double() * each(s["x_scales"], s["x"].size(1), 1), s["w"], s["w_scales"], s["offsets"].tolist())

    e, c = s["n_experts"], s["experts"].size(1)
    flat = s["experts"].flatten()
    key = flat.masked_fill((flat < 0) | (flat >= e), e)
    by_expert, source = torch.sort(key, stable=True)
    offsets = torch.searchsorted(by_expert, torch.arange(e + 1, device=flat.device))
    kept = int(offsets[-1])
    places = torch.full_like(flat, -1)
    places[source[:kept]] = torch.arange(kept, device=flat.device)
    tokens, used = source[:kept] // c, s["weights"].double().flatten()[source[:kept]].unsqueeze(1)

    def back(y, factor):
        return torch.zeros(s["x"].shape, dtype=torch.float64, device=y.device).index_add_(0, tokens, y[:kept].double() * factor)

    if op == "layer":
        rows = by_block(s["x"].double(), 1)[0][tokens]
        at = offsets.tolist()
        both = rounded(of_experts(rows, s["gate_up"], s["gate_up_scales"], at))
        gate, up = both.chunk(2, dim=1)
        return back(rounded(of_experts(by_block(silu(gate) * up, 1)[0], s["down"], s["down_scales"], at)), used)

    def padded(v):
        return torch.nn.functional.pad(v, (0, 0, 0, flat.numel() - kept))

    result = {"source": source.int(), "places": places.view(-1, c).int(), "offsets": offsets.int(),
              "rows": padded(s["x"].double()[tokens]), "out": back(s["y"], used)}
    if s["train"]:
        d_out = s["d_out"].double()[tokens]
        d_weights = torch.zeros(flat.numel(), dtype=torch.float64, device=flat.device)
        d_weights[source[:kept]] = (s["y"][:kept].double() * d_out).sum(1)
        result |= {"d_x": back(s["d_rows"], 1.0), "d_y": padded(d_out * used), "d_weights": d_weights.view(-1, c)}
    return result
