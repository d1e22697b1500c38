"""Layers of experts on the GPU: the sort against a stable one, the moves and their gradients against 64 bits, the experts' product.

Bounds: the weighted sum has `choices` fused additions of 2^-24 of the magnitudes so far and one rounding to its type; a weight's gradient is a sum
of n products, of which a lane adds n / 32 and then five more are added: (n / 32 + 6) * 2^-24 of the magnitudes.  Tolerances of the product as in
test_fp8_linear_gpu.py.
"""
import pytest

from tests.test_fp8_linear_gpu import check_close, rows_of, weight_of

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16]


def choices_of(tokens, choices, n_experts, seed, dropped=0.2, dtype=torch.int64):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ids = torch.randint(0, n_experts, (tokens, choices), generator=g, device="cuda")  # the same expert twice, too
    gone = torch.rand(tokens, choices, generator=g, device="cuda")
    return torch.where(gone < dropped / 2, -1, torch.where(gone < dropped, n_experts + 3, ids)).to(dtype)


def check_order(order, ids, n_experts):
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < n_experts), flat, n_experts)
    sorted_key, source = torch.sort(key, stable=True)
    offsets = torch.searchsorted(sorted_key, torch.arange(n_experts + 1, device=key.device))
    places = torch.empty_like(source)
    places[source] = torch.arange(len(source), device=key.device)
    places = torch.where(key < n_experts, places, -1)
    for got, want in ((order.source, source), (order.places, places.view(ids.shape)), (order.offsets, offsets)):
        assert got.dtype == torch.int32 and got.shape == want.shape and torch.equal(got.long(), want)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64], ids=str)
@pytest.mark.parametrize("tokens,choices,n_experts", [
    (1, 1, 1), (1, 8, 8), (3, 2, 1024), (16, 8, 64), (31, 1, 5), (33, 3, 7), (1000, 8, 128), (1024, 8, 256), (1025, 8, 3), (4097, 4, 32), (20000, 6, 1000),
    (8192, 1, 1), (100000, 3, 1024), (600001, 2, 17)])
def test_sort(tokens, choices, n_experts, dtype):
    from gemmlib_b200.experts import ExpertOrder, sort_by_expert

    for dropped in (0.0, 0.3, 1.0):
        ids = choices_of(tokens, choices, n_experts, tokens, dropped, dtype)
        order = sort_by_expert(ids, n_experts)
        assert type(order) is ExpertOrder
        check_order(order, ids, n_experts)


def test_sort_of_other_layouts_and_values():
    from gemmlib_b200.experts import sort_by_expert

    ids = choices_of(60, 4, 9, 1)
    check_order(sort_by_expert(ids.view(3, 20, 4), 9), ids.view(3, 20, 4), 9)
    check_order(sort_by_expert(ids.t().contiguous().t(), 9), ids, 9)
    check_order(sort_by_expert(ids[:, 1:3], 9), ids[:, 1:3].contiguous(), 9)
    check_order(sort_by_expert(ids[0], 9), ids[0], 9)
    far = torch.tensor([[2 ** 40, -2 ** 60, 3, 2 ** 32 + 1]], device="cuda")
    check_order(sort_by_expert(far, 9), far, 9)
    same = torch.full((5000, 2), 6, device="cuda")
    check_order(sort_by_expert(same, 9), same, 9)
    empty = sort_by_expert(ids[:0], 9)
    assert empty.source.shape == (0,) and empty.places.shape == (0, 4) and torch.equal(empty.offsets, torch.zeros(10, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="1 to 1024 experts"):
        sort_by_expert(ids, 1025)
    with pytest.raises(RuntimeError, match="int32 or int64"):
        sort_by_expert(ids.float(), 9)


def problem(tokens, choices, n_experts, k, dtype, seed, dropped=0.2):
    from gemmlib_b200.experts import sort_by_expert

    g = torch.Generator(device="cuda").manual_seed(seed)
    ids = choices_of(tokens, choices, n_experts, seed, dropped)
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return dict(order=sort_by_expert(ids, n_experts), x=normal(tokens, k).to(dtype), y=normal(tokens * choices, k).to(dtype),
                weights=torch.softmax(normal(tokens, choices), 1), d_rows=normal(tokens * choices, k).to(dtype), d_out=normal(tokens, k).to(dtype))


def rounded_close(got, want, magnitude, additions):
    half = torch.finfo(got.dtype).eps / 2
    smallest = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}[got.dtype]
    bound = want.abs() * half * (1 + 1e-3) + smallest + additions * 2.0 ** -24 * magnitude
    off = (got.double() - want).abs()
    assert (off <= bound).all(), float((off - bound).max())


MOVES = [(1, 1, 1, 1), (1, 8, 8, 4096), (16, 8, 64, 4096), (7, 3, 5, 1237), (300, 2, 7, 24), (501, 4, 128, 640), (3000, 6, 33, 130), (64, 13, 20, 512), (5000, 2, 4, 1032)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("tokens,choices,n_experts,k", MOVES)
def test_moves_and_their_gradients(tokens, choices, n_experts, k, dtype):
    from gemmlib_b200.experts import combine_rows, gather_rows

    p = problem(tokens, choices, n_experts, k, dtype, tokens + k)
    order = p["order"]
    kept = int(order.offsets[-1])
    token = order.source.long() // choices
    p["y"][kept:] = float("nan")  # rows of no expert are not read
    p["d_rows"][kept:] = float("nan")
    x, y, weights = (p[n].clone().requires_grad_() for n in ("x", "y", "weights"))
    rows, out = gather_rows(x, order), combine_rows(y, order, weights)
    assert torch.equal(rows[:kept], p["x"][token[:kept]]) and (rows[kept:] == 0).all() and rows.shape == (tokens * choices, k)
    with torch.no_grad():
        assert torch.equal(gather_rows(x, order), rows) and torch.equal(combine_rows(y, order, weights), out)

    def back(values, factor):
        total = torch.zeros(tokens, k, dtype=torch.float64, device="cuda")
        return total.index_add_(0, token[:kept], values[:kept].double() * factor)

    used = p["weights"].double().reshape(-1)[order.source.long()][:kept, None]
    rounded_close(out.detach(), back(p["y"], used), back(p["y"].abs(), used), choices)
    d_x, d_y, d_weights = torch.autograd.grad((rows, out), (x, y, weights), (p["d_rows"], p["d_out"]))
    rounded_close(d_x, back(p["d_rows"], 1.0), back(p["d_rows"].abs(), 1.0), choices)
    d_out = p["d_out"].double()[token]
    want = torch.zeros(tokens * choices, k, dtype=torch.float64, device="cuda")
    want[:kept] = used * d_out[:kept]
    rounded_close(d_y, want, want.abs(), 1)
    dots, size = torch.zeros(2, tokens * choices, dtype=torch.float64, device="cuda")
    dots[order.source.long()[:kept]] = (p["y"].double() * d_out)[:kept].sum(1)
    size[order.source.long()[:kept]] = (p["y"].double() * d_out).abs()[:kept].sum(1)
    assert d_weights.dtype == torch.float32
    rounded_close(d_weights, dots.view(tokens, choices), size.view(tokens, choices), k / 32 + 6)
    dropped = order.places < 0
    assert (d_weights[dropped] == 0).all()


def test_gradients_against_differences():
    """The weighted sum is linear in each of its arguments: a difference over any step is the derivative times the step, up to the roundings."""
    from gemmlib_b200.experts import combine_rows, gather_rows

    p = problem(40, 3, 6, 64, torch.float16, 8)
    order = p["order"]
    kept = int(order.offsets[-1])
    x, y, weights = (p[n].clone().requires_grad_() for n in ("x", "y", "weights"))
    x.grad = y.grad = None
    g = torch.Generator(device="cuda").manual_seed(9)
    loss = lambda a, b, w: (combine_rows(b, order, w).double() * p["d_out"].double()).sum() + (  # noqa: E731
        gather_rows(a, order)[:kept].double() * p["d_rows"][:kept].double()).sum()
    loss(x, y, weights).backward()
    with torch.no_grad():
        base = loss(x, y, weights)
        for leaf, i in ((x, 0), (y, 1), (weights, 2)):
            step = torch.randint(-1, 2, leaf.shape, generator=g, device="cuda").to(leaf.dtype) * (0.5 if i < 2 else 0.25)
            moved = [x, y, weights]
            moved[i] = leaf + step  # (16-bit sums are rounded: the difference is taken of what came out)
            got = loss(*moved) - base
            want = (leaf.grad.double() * (moved[i].double() - leaf.double())).sum()
            # outputs are rounded to fp16 (2^-11 of up to 8), the gradients of x and y too; 40 x 64 and 120 x 64 of them with random signs
            bound = 2.0 ** -11 * ((2 * combine_rows(y, order, weights).double().abs() + 4) * p["d_out"].double().abs()).sum() + 2.0 ** -11 * (
                leaf.grad.double().abs() * (moved[i].double() - leaf.double()).abs()).sum()
            assert (got - want).abs() <= bound, (i, float(got), float(want), float(bound))


@pytest.mark.parametrize("weights_type", [torch.float32, torch.float16, torch.bfloat16], ids=str)
def test_types_and_layouts_of_weights_and_gradients(weights_type):
    from gemmlib_b200.experts import combine_rows, gather_rows

    p = problem(50, 4, 6, 200, torch.bfloat16, 3)
    order, w = p["order"], p["weights"].to(weights_type)
    want = combine_rows(p["y"], order, w.float())
    assert torch.equal(combine_rows(p["y"], order, w), want)
    assert torch.equal(combine_rows(p["y"], order, w.t().contiguous().t()), want)
    wide = torch.zeros(200, 207, dtype=torch.bfloat16, device="cuda")[:, 3:203]
    wide.copy_(p["y"])
    assert torch.equal(combine_rows(wide, order, w), want)
    leaf = w.clone().requires_grad_()
    out = combine_rows(p["y"], order, leaf)  # y needs no gradient
    out.sum().backward()  # a gradient of ones that is expanded
    assert leaf.grad.dtype == weights_type
    expect = torch.zeros(200, dtype=torch.float64, device="cuda")
    kept = int(order.offsets[-1])
    expect[order.source.long()[:kept]] = p["y"].double().sum(1)[:kept]
    size = p["y"].double().abs().sum(1).max()
    half = torch.finfo(weights_type).eps / 2
    assert ((leaf.grad.double().reshape(-1) - expect).abs() <= expect.abs() * half * 1.001 + size * 14 * 2.0 ** -24).all()
    x = p["x"].clone().requires_grad_()
    gather_rows(x, order).sum().backward()
    assert torch.equal(x.grad, (order.places >= 0).sum(1, keepdim=True).expand(50, 200).to(x.dtype))
    shaped = problem(50, 4, 6, 200, torch.bfloat16, 3)["order"]._replace(places=order.places.view(5, 10, 4))
    assert combine_rows(p["y"], shaped, w.view(5, 10, 4)).shape == (5, 10, 200)
    assert torch.equal(gather_rows(p["x"].view(5, 10, 200), shaped), gather_rows(p["x"], order))


def test_infinite_weights_of_dropped_choices_do_not_count():
    from gemmlib_b200.experts import combine_rows

    p = problem(30, 3, 4, 64, torch.float16, 5, dropped=0.5)
    order = p["order"]
    want = combine_rows(p["y"], order, p["weights"])
    w = torch.where(order.places < 0, float("nan"), p["weights"])
    assert torch.equal(combine_rows(p["y"], order, w), want)
    none = problem(30, 3, 4, 64, torch.float16, 5, dropped=1.0)
    assert (combine_rows(none["y"], none["order"], none["weights"]) == 0).all()


def test_refusals():
    from gemmlib_b200.experts import ExpertOrder, combine_rows, fp8_expert_linear, gather_rows
    from gemmlib_b200.fp8_linear import Fp8Weight, quantize_fp8

    p = problem(10, 2, 4, 64, torch.float16, 5)
    order = p["order"]
    w, x = stack_of(3, 40, 64, 1), rows_of(20, 64, 2)
    offsets = torch.tensor([0, 5, 9, 20], dtype=torch.int32, device="cuda")
    for call, text in [
        (lambda: gather_rows(p["x"][:9], order), "order's tokens"),
        (lambda: quantize_fp8(p["x"][:9], order), "order's tokens"),
        (lambda: combine_rows(p["y"][:19], order, p["weights"]), "one row a choice"),
        (lambda: combine_rows(p["y"], order, p["weights"][:, :1]), "shape of the order's places"),
        (lambda: combine_rows(p["y"], order, p["weights"].double()), "float32, float16 or bfloat16"),
        (lambda: combine_rows(p["y"], order, p["weights"].cpu()), "device"),
        (lambda: gather_rows(p["x"], ExpertOrder(*(t.long() for t in order))), "int32"),
        (lambda: gather_rows(p["x"], order._replace(source=order.source[:-1])), "source"),
        (lambda: fp8_expert_linear(x, w, offsets.long()), "int32"),
        (lambda: fp8_expert_linear(x, w, offsets[:-1]), "experts \\+ 1"),
        (lambda: fp8_expert_linear(x, Fp8Weight(w.values[0], w.scales[0]), offsets), "experts, out_features"),
        (lambda: fp8_expert_linear(x, Fp8Weight(w.values, w.scales[:2]), offsets), "of shape"),
        (lambda: fp8_expert_linear(x, stack_of(3, 40, 80, 1), offsets), "in_features"),
        (lambda: fp8_expert_linear(x, w, offsets, out=torch.empty(20, 41, dtype=torch.float16, device="cuda")), "out must have"),
        (lambda: fp8_expert_linear(x, Fp8Weight(w.values.expand(3, 40, 64)[:1].expand(3, 40, 64), w.scales), offsets), "one pitch|behind one another"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            call()
    # an order of the caller's own that names no token or place: no access out of bounds
    wrong = order._replace(source=torch.full_like(order.source, 1 << 30))
    assert (gather_rows(p["x"], wrong) == 0).all()
    for far in (1 << 30, -(1 << 30), 20):
        wrong = order._replace(places=torch.full_like(order.places, far))
        assert (combine_rows(p["y"], wrong, p["weights"]) == 0).all()
        assert quantize_fp8(p["x"], wrong).values.shape == (20, 64)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_quantized_in_the_experts_order(dtype):
    from gemmlib_b200.experts import gather_rows
    from gemmlib_b200.fp8_linear import quantize_fp8

    for tokens, choices, n_experts, k in MOVES:
        p = problem(tokens, choices, n_experts, k, dtype, 2)
        q, want = quantize_fp8(p["x"], p["order"]), quantize_fp8(gather_rows(p["x"], p["order"]))
        assert torch.equal(q.values.float(), want.values.float()) and torch.equal(q.scales, want.scales)


def stack_of(experts, n, k, seed):
    from gemmlib_b200.fp8_linear import Fp8Weight

    each = [weight_of(n, k, seed + 100 * e) for e in range(experts)]
    pitch = -(-k // 16) * 16
    values = torch.full((experts, n, pitch), 0x7f, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[..., :k]
    for v, e in zip(values, each):
        v.copy_(e.values)
    return Fp8Weight(values, torch.stack([e.scales for e in each]))


def check_experts(out, x, w, offsets):
    from gemmlib_b200.fp8_linear import Fp8Rows, Fp8Weight

    at = offsets.tolist()
    for e, (lo, hi) in enumerate(zip(at[:-1], at[1:])):
        if hi > lo:
            check_close(out[lo:hi], Fp8Rows(x.values[lo:hi], x.scales[lo:hi]), Fp8Weight(w.values[e], w.scales[e]))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("counts,behind,k,n", [
    ([1], 0, 128, 128), ([0, 0, 5, 0], 3, 200, 130), ([1] * 64, 0, 2048, 256), ([3, 0, 40, 17, 128, 1, 200], 100, 1237, 1000), ([300, 0, 1000, 129], 0, 640, 1408),
    ([700, 650, 900], 50, 1408, 520), ([0] * 1023 + [9], 0, 64, 48), ([2000], 7, 256, 24), ([33] * 30, 5, 300, 777), ([0, 0], 40, 64, 64)])
def test_expert_product(counts, behind, k, n, dtype):
    from gemmlib_b200.experts import fp8_expert_linear

    offsets = torch.tensor([0] + counts, device="cuda").cumsum(0).int()
    rows = sum(counts) + behind
    x, w = rows_of(rows, k, 1), stack_of(len(counts), n, k, 2)
    out = fp8_expert_linear(x, w, offsets, dtype)
    assert out.shape == (rows, n) and out.dtype == dtype
    check_experts(out, x, w, offsets)
    assert (out[sum(counts):] == 0).all()
    held = torch.full((rows, n + 8), 5.0, dtype=dtype, device="cuda")
    fp8_expert_linear(x, w, offsets, dtype, out=held[:, :n])
    assert torch.equal(held[:sum(counts), :n], out[:sum(counts)]) and (held[sum(counts):] == 5).all() and (held[:, n:] == 5).all()
    if behind > 1:  # rows ahead of the first expert's, too
        moved = offsets.clone()
        moved += 1
        shifted = fp8_expert_linear(x, w, moved, dtype)
        check_experts(shifted, x, w, moved)
        assert (shifted[0] == 0).all() and (shifted[1 + sum(counts):] == 0).all()


@pytest.mark.parametrize("rows", [40, 900])
def test_offsets_that_are_none_stay_within_bounds(rows):
    """A value is taken for the nearest that fits behind those before."""
    from gemmlib_b200.experts import fp8_expert_linear

    x, w = rows_of(rows, 200, 1), stack_of(5, 136, 200, 2)
    for raw, taken in (([-7, 10, 5, 1 << 30, 3, 12], [0, 10, 10, rows, rows, rows]), ([rows + 1] * 6, [rows] * 6), ([0, 0, 0, 0, 0, -1], [0] * 6),
                       ([-(1 << 31), 20, 20, 30, 30, (1 << 31) - 1], [0, 20, 20, 30, 30, rows])):
        out = fp8_expert_linear(x, w, torch.tensor(raw, dtype=torch.int32, device="cuda"))
        offsets = torch.tensor(taken)
        check_experts(out, x, w, offsets)
        assert (out[:taken[0]] == 0).all() and (out[taken[-1]:] == 0).all()


def layer(experts, k, f, dtype, seed):
    from gemmlib_b200.experts import Fp8Experts

    g = torch.Generator(device="cuda").manual_seed(seed)
    return Fp8Experts((torch.randn(experts, 2 * f, k, generator=g, device="cuda") / k ** 0.5).to(dtype),
                      (torch.randn(experts, k, f, generator=g, device="cuda") / f ** 0.5).to(dtype))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("tokens,choices,n_experts,k,f", [(1, 2, 4, 256, 128), (16, 8, 64, 512, 1408), (7, 3, 5, 200, 77), (600, 2, 6, 640, 200), (2000, 4, 8, 256, 384)])
def test_a_layer_of_experts(tokens, choices, n_experts, k, f, dtype):
    """As a layer for each expert on its own rows."""
    import copy

    from gemmlib_b200.experts import Fp8Experts, combine_rows, gather_rows, sort_by_expert
    from gemmlib_b200.fp8_linear import Fp8Rows, Fp8Weight, fp8_linear, quantize_fp8, silu_mul_fp8

    m = layer(n_experts, k, f, dtype, 1)
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(tokens, k, generator=g, device="cuda").to(dtype)
    ids = choices_of(tokens, choices, n_experts, 3, dropped=0.1)
    weights = torch.softmax(torch.randn(tokens, choices, generator=g, device="cuda"), 1)
    got = m(x, ids, weights)
    order = sort_by_expert(ids, n_experts)
    rows, at = quantize_fp8(gather_rows(x, order)), order.offsets.tolist()
    y = torch.zeros(tokens * choices, k, dtype=dtype, device="cuda")
    for e, (lo, hi) in enumerate(zip(at[:-1], at[1:])):
        if hi == lo:
            continue
        both = fp8_linear(Fp8Rows(rows.values[lo:hi], rows.scales[lo:hi]), Fp8Weight(m.gate_up[e, :, :k], m.gate_up_scales[e]), dtype=dtype)
        y[lo:hi] = fp8_linear(silu_mul_fp8(both[:, :f], both[:, f:]), Fp8Weight(m.down[e, :, :f], m.down_scales[e]), dtype=dtype)
    want = combine_rows(y, order, weights)
    # the two ways may split K otherwise, and a sum that is rounded otherwise can move an e4m3 value by a step: 2^-3 of it, of one in many
    assert (got.double() - want.double()).norm() <= 2.0 ** -7 * want.double().norm()
    assert torch.equal(m(x.view(1, tokens, k), ids.view(1, tokens, choices), weights.view(1, tokens, choices))[0], got)
    other = Fp8Experts.from_weights(Fp8Weight(m.gate_up[..., :k], m.gate_up_scales), Fp8Weight(m.down[..., :f], m.down_scales))
    assert torch.equal(other(x, ids, weights), got)
    assert torch.equal(copy.deepcopy(m)(x, ids, weights), got) and m.weight_bytes() > 3 * n_experts * k * f
    fresh = layer(n_experts, k, f, dtype, 9)
    fresh.load_state_dict(m.state_dict())
    assert torch.equal(fresh(x, ids, weights), got)
    leaf = weights.clone().requires_grad_()
    m(x, ids, leaf).double().sum().backward()
    expect = torch.zeros(tokens * choices, dtype=torch.float64, device="cuda")
    expect[order.source.long()[:at[-1]]] = y.double()[:at[-1]].sum(1)
    size = y.double().abs().sum(1).max()
    assert (leaf.grad.double().reshape(-1) - expect).abs().max() <= 2.0 ** -5 * size
    with pytest.raises(RuntimeError, match="no backward pass"):
        m(x.clone().requires_grad_(), ids, weights)


def test_captured_layers_on_streams_beside_each_other():
    """Two graphs of a layer, replayed with new tokens, choices and weights, on two streams at a time."""
    m = layer(16, 512, 384, torch.bfloat16, 1)
    graphs = []
    for seed in range(2):
        x = torch.zeros(64, 512, dtype=torch.bfloat16, device="cuda")
        ids, weights = torch.zeros(64, 4, dtype=torch.long, device="cuda"), torch.zeros(64, 4, device="cuda")
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            m(x, ids, weights)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            out = m(x, ids, weights)
        graphs.append((g, stream, x, ids, weights, out))
    for seed in range(4):
        want = []
        for i, (g, stream, x, ids, weights, out) in enumerate(graphs):
            gen = torch.Generator(device="cuda").manual_seed(10 * seed + i)
            x.copy_(torch.randn(64, 512, generator=gen, device="cuda"))
            ids.copy_(choices_of(64, 4, 16, 10 * seed + i, dropped=0.3 * i))
            weights.copy_(torch.rand(64, 4, generator=gen, device="cuda"))
            want.append(m(x, ids, weights))
        torch.cuda.synchronize()
        for _ in range(3):
            for g, stream, *_ in graphs:
                with torch.cuda.stream(stream):
                    g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(t[5], w) for t, w in zip(graphs, want))
    from gemmlib_b200 import capi

    assert capi.last_kernel_status() == 0


def test_a_captured_backward_pass():
    """Forward and backward of the moves in one graph, replayed with other inputs."""
    from gemmlib_b200.experts import combine_rows, gather_rows, sort_by_expert

    def step(ids, x, weights, d):
        order = sort_by_expert(ids, 6)
        out = combine_rows(gather_rows(x, order) * 2, order, weights)
        return (out, *torch.autograd.grad(out, (x, weights), d))

    def fresh(seed):
        p = problem(40, 3, 6, 200, torch.float16, seed)
        return choices_of(40, 3, 6, seed), p["x"], p["weights"], p["d_out"]

    held = [t.clone() for t in fresh(1)]
    held[1].requires_grad_(), held[2].requires_grad_()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(*held)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        got = step(*held)
    for seed in (2, 3):
        new = fresh(seed)
        with torch.no_grad():
            for h, n in zip(held, new):
                h.copy_(n)
        g.replay()
        torch.cuda.synchronize()
        want = step(new[0], new[1].requires_grad_(), new[2].requires_grad_(), new[3])
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_no_tokens():
    from gemmlib_b200.experts import combine_rows, gather_rows, sort_by_expert
    from gemmlib_b200.fp8_linear import quantize_fp8

    m = layer(3, 64, 32, torch.float16, 1)
    x, ids, weights = (torch.empty(0, n, device="cuda") for n in (64, 2, 2))
    x, ids = x.half().requires_grad_(), ids.long()
    order = sort_by_expert(ids, 3)
    rows, out = gather_rows(x, order), combine_rows(torch.empty(0, 64, dtype=torch.float16, device="cuda"), order, weights.requires_grad_())
    assert rows.shape == (0, 64) and out.shape == (0, 64) and quantize_fp8(x.detach(), order).values.shape == (0, 64)
    grads = torch.autograd.grad((rows, out), (x, weights), (torch.empty_like(rows), torch.empty_like(out)))
    assert grads[0].shape == (0, 64) and grads[1].shape == (0, 2)
    assert m(x.detach(), ids, weights.detach()).shape == (0, 64)


def test_products_of_many_experts_after_products_of_split_tiles():
    """What a kernel may have of shared memory is the most that any call asks for, whichever came first."""
    from gemmlib_b200.experts import fp8_expert_linear
    from gemmlib_b200.fp8_linear import fp8_linear

    for m in (16, 30, 60, 100):  # split tiles of every height
        x, w = rows_of(m, 4096, 1), weight_of(512, 4096, 2)
        check_close(fp8_linear(x, w), x, w)
    w = stack_of(1024, 40, 64, 2)
    for each in (1, 20, 40, 80):
        offsets = torch.arange(0, 1025 * each, each, device="cuda").int()
        x = rows_of(1024 * each, 64, 1)
        out = fp8_expert_linear(x, w, offsets)
        for e in (0, 511, 1023):
            lo, hi = e * each, (e + 1) * each
            check_close(out[lo:hi], type(x)(x.values[lo:hi], x.scales[lo:hi]), type(w)(w.values[e], w.scales[e]))


def test_first_calls_from_several_threads():
    import threading

    from gemmlib_b200.experts import fp8_expert_linear
    from gemmlib_b200.fp8_linear import fp8_linear

    problems = [(rows_of(m, k, i), weight_of(n, k, 10 + i)) for i, (m, k, n) in enumerate([(5, 999, 333), (70, 2048, 500), (200, 1111, 800), (900, 640, 640)])]
    offsets = torch.tensor([0, 100, 900], dtype=torch.int32, device="cuda")
    stack = stack_of(2, 640, 640, 5)
    want = [fp8_linear(x, w) for x, w in problems] + [fp8_expert_linear(problems[3][0], stack, offsets)]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got = fp8_linear(*problems[i]) if i < 4 else fp8_expert_linear(problems[3][0], stack, offsets)
                    torch.cuda.current_stream().synchronize()
                    assert torch.equal(got, want[i])
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(5)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not failed, failed


def test_a_backward_pass_captured_while_an_eager_graph_of_the_same_leaves_lives():
    """On another stream that is refused (autograd's node for a leaf's gradient has the eager stream, and its wait would end the capture), for
    either leaf, and the process goes on; on the same stream, and once the eager graph is gone, it is captured."""
    from gemmlib_b200.experts import combine_rows, gather_rows

    p = problem(40, 3, 6, 200, torch.float16, 1)
    order = p["order"]
    x, weights = p["x"].clone().requires_grad_(), p["weights"].clone().requires_grad_()
    stream = torch.cuda.Stream()

    def step():
        out = combine_rows(gather_rows(x, order), order, weights)
        return out, lambda: torch.autograd.grad(out, (x, weights), p["d_out"])

    eager, backward = step()
    stream.wait_stream(torch.cuda.current_stream())
    for call in (lambda: gather_rows(x, order), lambda: combine_rows(p["y"], order, weights)):
        with pytest.raises(RuntimeError, match="lives on another stream"):
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=stream):
                call()
    want = [t.clone() for t in backward()]
    del eager, backward
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        eager, backward = step()
        backward()
        eager, backward = step()  # lives, on the stream that is captured
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        got = step()[1]()
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and eager is not None


def test_more_than_2_to_the_31_elements():
    """Rows, outputs and weights whose last elements lie beyond: compared at both ends and in the middle."""
    from gemmlib_b200.experts import combine_rows, fp8_expert_linear, gather_rows, sort_by_expert
    from gemmlib_b200.fp8_linear import Fp8Rows, Fp8Weight, fp8_linear, quantize_fp8, quantize_fp8_weight, silu_mul_fp8

    g = torch.Generator(device="cuda").manual_seed(1)
    n, k = 70000, 32768
    few = torch.tensor([0, 1, 40000, 65535, 65536, 69999], device="cuda")
    x = torch.empty(n, k, dtype=torch.bfloat16, device="cuda")
    x[:1000].normal_(generator=g)
    for at in range(1000, n, 1000):
        x[at:at + 1000] = x[:1000] * (1 + at / n)
    own = x[few]
    q, want = quantize_fp8(x), quantize_fp8(own)
    assert torch.equal(q.values[few].float(), want.values.float()) and torch.equal(q.scales[few], want.scales)
    assert torch.equal(q.dequantize(torch.bfloat16)[few], want.dequantize(torch.bfloat16))
    assert torch.equal(silu_mul_fp8(x, x).values[few].float(), silu_mul_fp8(own, own).values.float())
    w = quantize_fp8_weight(x)
    last = quantize_fp8_weight(x[-(n % 128):])
    assert torch.equal(w.values[-(n % 128):].float(), last.values.float()) and torch.equal(w.scales[-1:], last.scales)
    # weights beyond 2^31 bytes, then outputs beyond 2^31 elements
    a = rows_of(5, k, 1)
    out = fp8_linear(a, w, dtype=torch.bfloat16)
    tail = Fp8Weight(w.values[-(n % 128):], w.scales[-1:])
    check_close(out[:, -(n % 128):], a, tail)
    del out
    b, c = rows_of(n, 128, 2), weight_of(k, 128, 3)
    out = fp8_linear(b, c, dtype=torch.bfloat16)
    check_close(out[few], Fp8Rows(b.values[few], b.scales[few]), c)
    offsets = torch.tensor([0, 66000, n], dtype=torch.int32, device="cuda")
    two = Fp8Weight(torch.stack([c.values.view(torch.uint8), c.values.view(torch.uint8).flip(0)]).view(torch.float8_e4m3fn), torch.stack([c.scales, c.scales]))
    fp8_expert_linear(b, two, offsets, torch.bfloat16, out=out)
    check_close(out[few[:5]], Fp8Rows(b.values[few[:5]], b.scales[few[:5]]), c)
    check_close(out[few[5:]], Fp8Rows(b.values[few[5:]], b.scales[few[5:]]), Fp8Weight(two.values[1], two.scales[1]))
    del out, two, q, want
    # tokens to experts: 35000 of two choices
    ids = torch.randint(-1, 5, (n // 2, 2), generator=g, device="cuda")
    order = sort_by_expert(ids, 5)
    rows = gather_rows(x[:n // 2], order)
    kept = int(order.offsets[-1])
    at = torch.tensor([0, kept // 2, kept - 1], device="cuda")
    assert torch.equal(rows[at], x[order.source[at].long() // 2]) and (rows[kept:kept + 3] == 0).all() and (rows[-1] == 0).all()
    weights = torch.rand(n // 2, 2, generator=g, device="cuda")
    out = combine_rows(rows, order, weights)
    t = torch.tensor([0, 20000, n // 2 - 1], device="cuda")
    used = torch.where(order.places[t] >= 0, weights[t], 0.0).double().sum(1, keepdim=True)
    rounded_close(out[t], x[t].double() * used, x[t].double().abs() * used, 3)
    q = quantize_fp8(x[:n // 2], order)
    assert torch.equal(q.values[at].float(), quantize_fp8(rows[at]).values.float()) and (q.scales[kept:] == 0).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("tokens,choices,n_experts,k", [(1, 8, 8, 4096), (7, 3, 5, 1237), (300, 2, 7, 24)])
def test_a_gradient_by_itself(tokens, choices, n_experts, k, dtype):
    """Of the rows or of the weights alone: bit for bit as together."""
    from gemmlib_b200.experts import combine_rows

    p = problem(tokens, choices, n_experts, k, dtype, 4)
    y, weights = p["y"].clone().requires_grad_(), p["weights"].clone().requires_grad_()
    want = torch.autograd.grad(combine_rows(y, p["order"], weights), (y, weights), p["d_out"])
    assert torch.equal(torch.autograd.grad(combine_rows(y, p["order"], p["weights"]), y, p["d_out"])[0], want[0])
    out = combine_rows(p["y"], p["order"], weights)
    assert torch.equal(torch.autograd.grad(out, weights, p["d_out"])[0], want[1])
    out = combine_rows(y, p["order"], weights)  # both have one, one is asked for
    assert torch.equal(torch.autograd.grad(out, weights, p["d_out"], retain_graph=True)[0], want[1])
    assert torch.equal(torch.autograd.grad(out, y, p["d_out"])[0], want[0])


def test_the_abi_computes_either_gradient():
    from gemmlib_b200 import capi

    p = problem(9, 3, 5, 40, torch.float16, 6)
    source, count = p["order"].source, p["order"].offsets.data_ptr() + 4 * 5
    new = lambda: (torch.full((27, 40), 7.0, dtype=torch.float16, device="cuda"), torch.full((9, 3), 7.0, device="cuda"))  # noqa: E731
    run = lambda d_y, d_weights: capi.experts_combine_backward(  # noqa: E731
        0, 9, 3, 40, (p["d_out"], 40), (p["y"], 40), p["weights"], 2, source, count, d_y, d_weights, stream=torch.cuda.current_stream().cuda_stream)
    both, alone = new(), new()
    run((both[0], 40), both[1])
    run((alone[0], 40), None)
    run(None, alone[1])
    assert all(torch.equal(a, b) for a, b in zip(both, alone)) and not (both[0] == 7).all()
    with pytest.raises(capi.BlkQ4Error, match="Null tensor pointer: d_weights"):
        run(None, None)


def test_a_second_differentiation_is_refused():
    """A first one with a graph is not."""
    from gemmlib_b200.experts import combine_rows, gather_rows

    p = problem(9, 3, 5, 40, torch.float16, 6)
    for leaf, call in ((p["x"], lambda t: gather_rows(t, p["order"])), (p["weights"], lambda t: combine_rows(p["y"], p["order"], t))):
        leaf = leaf.clone().requires_grad_()
        out = call(leaf)
        plain, = torch.autograd.grad(out, leaf, torch.ones_like(out), retain_graph=True)
        grad, = torch.autograd.grad(out, leaf, torch.ones_like(out), create_graph=True)
        assert torch.equal(grad, plain) and grad.requires_grad
        with pytest.raises(RuntimeError, match="cannot be differentiated twice"):
            grad.float().sum().backward()


def test_what_was_saved_for_a_gradient_must_not_change():
    from gemmlib_b200.experts import combine_rows

    p = problem(9, 3, 5, 40, torch.float16, 6)
    y, weights = p["y"].clone(), p["weights"].clone().requires_grad_()
    out = combine_rows(y, p["order"], weights)
    y.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.float().sum().backward()
    out = combine_rows(y, p["order"], weights).float().sum()
    out.backward()
    with pytest.raises(RuntimeError, match="backward through the graph a second time"):
        out.backward()


def test_tangents_are_refused():
    import torch.autograd.forward_ad as fwAD

    from gemmlib_b200.experts import combine_rows, gather_rows

    p = problem(9, 3, 5, 40, torch.float16, 6)
    for wanted in (False, True):
        with fwAD.dual_level():
            x = fwAD.make_dual(p["x"].clone().requires_grad_(wanted), torch.ones_like(p["x"]))
            weights = fwAD.make_dual(p["weights"].clone().requires_grad_(wanted), torch.ones_like(p["weights"]))
            with pytest.raises(RuntimeError, match="no forward derivatives"):
                gather_rows(x, p["order"])
            with pytest.raises(RuntimeError, match="no forward derivatives"):
                combine_rows(p["y"], p["order"], weights)
    assert torch.equal(gather_rows(p["x"], p["order"]), gather_rows(p["x"].clone().requires_grad_(), p["order"]))


def test_hooks_shared_leaves_and_sums_of_gradients():
    """The same rows and weights in two sums, and a leaf's gradient that is added to."""
    from gemmlib_b200.experts import combine_rows, gather_rows

    p = problem(31, 2, 4, 72, torch.float16, 9)
    order = p["order"]
    x, weights = p["x"].clone().requires_grad_(), p["weights"].clone().requires_grad_()
    seen = []
    x.register_hook(lambda g: seen.append(g.clone()))
    rows = gather_rows(x, order)
    out = combine_rows(rows, order, weights) + combine_rows(rows * 2, order, weights)
    for i in (1, 2):
        out.backward(p["d_out"], retain_graph=True)
        assert len(seen) == i
    one = torch.autograd.grad(combine_rows(gather_rows(x, order), order, weights), weights, p["d_out"])[0]
    # each gradient of the weights is a sum of 72 products in fp32, three times as large as one together; twice added up
    size = 6 * (p["x"].double().abs() * p["d_out"].double().abs()).sum(1, keepdim=True)
    assert ((weights.grad.double() - 6 * one.double()).abs() <= (72 / 32 + 10) * 2.0 ** -23 * size + 1e-30).all()
    kept = (order.places >= 0).double() * p["weights"].double()
    want = 2 * 3 * kept.sum(1, keepdim=True) * p["d_out"].double()
    # rounded to fp16: each d_y (two of them, the one of the doubled rows again), their sum, the sum over a token's rows, the two backward passes' sum
    bound = 2.0 ** -11 * 8 * 2 * 3 * kept.sum(1, keepdim=True) * p["d_out"].double().abs() + 2.0 ** -23
    assert ((x.grad.double() - want).abs() <= bound).all()
