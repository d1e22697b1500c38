"""Weights of experts that do not lie behind one another, scales that are parts of others; transforms of functions; a layer as its steps."""
import pytest

from tests.test_experts_gpu import TYPES, choices_of, layer, problem, stack_of
from tests.test_fp8_linear_gpu import rows_of

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


def room(values, before, behind):
    """The matrices [experts, rows, columns] of `values` inside ones of NaN that are larger by so much in every dimension."""
    shape = [b + s + e for b, s, e in zip(before, values.shape, behind)]
    held = torch.full(shape, 0x7f, dtype=torch.uint8, device="cuda").view(E4M3)
    inside = held[tuple(slice(b, b + s) for b, s in zip(before, values.shape))]
    return inside.copy_(values)


@pytest.mark.parametrize("each,n,k", [(3, 200, 272), (20, 130, 300), (400, 520, 640), (70, 1, 48)])
def test_stacks_with_gaps(each, n, k):
    """`each` rows an expert (tiles of few rows and of many): every second expert, rows and columns of larger matrices, scales of every layout."""
    from gemmlib_b200.experts import fp8_expert_linear
    from gemmlib_b200.fp8_linear import Fp8Rows, Fp8Weight

    experts = 4
    x, w = rows_of(experts * each, k, 1), stack_of(experts, n, k, 2)
    offsets = torch.arange(0, experts * each + 1, each, device="cuda").int()
    want = fp8_expert_linear(x, w, offsets)
    assert want.isfinite().all()
    pitch = -k % 16  # what makes a row whole pieces of 16 bytes
    doubled = torch.full((2 * experts, n, k + pitch), 0x7f, dtype=torch.uint8, device="cuda").view(E4M3)[..., :k]
    doubled[::2] = w.values
    two = torch.full((2 * experts, *w.scales.shape[1:]), float("nan"), device="cuda")
    two[::2] = w.scales
    for values, scales in (
            (doubled[::2], two[::2]),
            (doubled[::2], w.scales),
            (w.values, two[::2]),
            (room(w.values, (1, 7, 16), (2, 5, 32 + pitch)), w.scales),
            (room(w.values, (0, 0, 0), (0, 3, 16 + pitch)), w.scales.transpose(1, 2).contiguous().transpose(1, 2)),
            (w.values, w.scales.permute(2, 0, 1).contiguous().permute(1, 2, 0)),
            (w.values, torch.nn.functional.pad(w.scales, (2, 1, 1, 3), value=float("nan"))[:, 1:1 + w.scales.size(1), 2:2 + w.scales.size(2)])):
        assert torch.equal(fp8_expert_linear(x, Fp8Weight(values, scales), offsets), want)
    kb = x.scales.size(1)
    for scales in (x.scales.t().contiguous().t(), torch.nn.functional.pad(x.scales, (3, 2), value=float("nan"))[:, 3:3 + kb],
                   x.scales.repeat_interleave(2, 0)[::2]):
        assert torch.equal(fp8_expert_linear(Fp8Rows(x.values, scales), w, offsets), want)
    odd = torch.empty(experts * each, k + 1, dtype=torch.uint8, device="cuda").view(E4M3)[:, 1:].copy_(x.values)
    assert torch.equal(fp8_expert_linear(Fp8Rows(odd, x.scales), w, offsets), want)


def test_stacks_that_are_refused():
    from gemmlib_b200.experts import fp8_expert_linear
    from gemmlib_b200.fp8_linear import Fp8Weight

    x, w = rows_of(30, 256, 1), stack_of(3, 64, 256, 2)
    offsets = torch.tensor([0, 10, 20, 30], dtype=torch.int32, device="cuda")
    wide = torch.zeros(3, 64, 256 + 16, dtype=torch.uint8, device="cuda").view(E4M3)
    odd_pitch = torch.zeros(3, 64, 257, dtype=torch.uint8, device="cuda").view(E4M3)[..., :256]
    for values, text in ((w.values[:1].expand(3, 64, 256), "behind one another"),  # one expert in all places
                         (w.values[:, :1].expand(3, 64, 256), "contiguous rows"),
                         (w.values.transpose(1, 2).contiguous().transpose(1, 2), "contiguous rows"),
                         (w.values.transpose(0, 1).contiguous().transpose(0, 1), "behind one another"),  # experts between one another's rows
                         (wide[..., 8:264], "16 bytes"), (odd_pitch, "16 bytes")):
        with pytest.raises(RuntimeError, match=text):
            fp8_expert_linear(x, Fp8Weight(values, w.scales), offsets)
    with pytest.raises(RuntimeError, match="of shape"):
        fp8_expert_linear(x, Fp8Weight(w.values, w.scales[:2]), offsets)
    with pytest.raises(RuntimeError, match="must be on the device"):
        fp8_expert_linear(x, Fp8Weight(w.values, w.scales.cpu()), offsets)


def test_transforms_are_refused():
    """A tensor that stands for a batch of others, or is wrapped for a derivative, has no memory of its own: an error, and what follows is as before."""
    from gemmlib_b200.experts import combine_rows, fp8_expert_linear, gather_rows, sort_by_expert
    from gemmlib_b200.fp8_linear import fp8_linear, quantize_fp8, silu_mul_fp8

    p = problem(9, 3, 5, 48, torch.float16, 6)
    order = p["order"]
    want = combine_rows(gather_rows(p["x"], order), order, p["weights"])
    x2, w2, y2 = (torch.stack([p[n], p[n]]) for n in ("x", "weights", "y"))
    ids = choices_of(9, 3, 5, 1)
    rows, w, stack = rows_of(9, 48, 1), stack_of(1, 16, 48, 2), stack_of(2, 16, 48, 2)
    one = type(w)(w.values[0], w.scales[0])
    offsets = torch.tensor([0, 4, 9], dtype=torch.int32, device="cuda")
    batched = [
        (lambda x: gather_rows(x, order), x2),
        (lambda t: combine_rows(p["y"], order, t), w2),
        (lambda y: combine_rows(y, order, p["weights"]), y2),
        (lambda i: sort_by_expert(i, 5).places, torch.stack([ids, ids])),
        (lambda x: quantize_fp8(x).scales, x2),
        (lambda x: silu_mul_fp8(x, p["x"]).scales, x2),
        (lambda s: fp8_linear(type(rows)(rows.values, s), one), torch.stack([rows.scales, rows.scales])),
        (lambda s: fp8_expert_linear(type(rows)(rows.values, s), stack, offsets), torch.stack([rows.scales, rows.scales])),
    ]
    for call, t in batched:
        with pytest.raises(RuntimeError):
            torch.func.vmap(call)(t)
    for call, t in ((lambda x: gather_rows(x, order).float().sum(), p["x"]), (lambda t: combine_rows(p["y"], order, t).float().sum(), p["weights"]),
                    (lambda y: combine_rows(y, order, p["weights"]).float().sum(), p["y"])):
        with pytest.raises(RuntimeError):
            torch.func.grad(call)(t)
        with pytest.raises(RuntimeError):
            torch.func.jvp(call, (t,), (torch.ones_like(t),))
    assert torch.equal(combine_rows(gather_rows(p["x"], order), order, p["weights"]), want)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("tokens,choices,n_experts,k,f,dropped", [(1, 2, 4, 256, 128, 0.0), (16, 8, 64, 512, 1408, 0.1), (7, 3, 5, 200, 77, 0.3), (700, 4, 8, 640, 384, 0.875),
                                                                  (5, 2, 3, 64, 64, 1.0)])
def test_a_layer_is_its_steps(tokens, choices, n_experts, k, f, dropped, dtype):
    """Bit for bit the public calls one by one; the weights' gradient is the sum of k products of a row of y with the output's gradient, of which a lane
    adds k / 32 and five more are added: (k / 32 + 6) * 2^-24 of their magnitudes."""
    from gemmlib_b200.experts import combine_rows, fp8_expert_linear, sort_by_expert
    from gemmlib_b200.fp8_linear import Fp8Weight, quantize_fp8, silu_mul_fp8

    m = layer(n_experts, k, f, dtype, 1)
    g = torch.Generator(device="cuda").manual_seed(2)
    x, d = (torch.randn(tokens, k, generator=g, device="cuda").to(dtype) for _ in range(2))
    ids = choices_of(tokens, choices, n_experts, 3, dropped)
    weights = torch.softmax(torch.randn(tokens, choices, generator=g, device="cuda"), 1).requires_grad_()
    out = m(x, ids, weights)
    order = sort_by_expert(ids, n_experts)
    both = fp8_expert_linear(quantize_fp8(x, order), Fp8Weight(m.gate_up[..., :k], m.gate_up_scales), order.offsets, dtype)
    y = fp8_expert_linear(silu_mul_fp8(both[:, :f], both[:, f:]), Fp8Weight(m.down[..., :f], m.down_scales), order.offsets, dtype)
    assert torch.equal(out, combine_rows(y, order, weights.detach()))
    out.backward(d)
    kept = order.places >= 0
    products = y.double()[order.places.long().clamp(min=0)] * d.double()[:, None]
    want, size = products.sum(-1) * kept, products.abs().sum(-1) * kept
    assert ((weights.grad.double() - want).abs() <= (k / 32 + 6) * 2.0 ** -24 * size).all()
