"""The gate where exp(-gate) is no float any more: blocks that have nothing larger, against 64 bits.

t = gate / (1 + exp(-gate)) * up is a normal float down to a gate of -181 where up is large.  Below -87.3 it comes from four factors exp(gate / 4)
(1 ulp: 2^-22 with the rounding, relative, each) and five products of 2^-24: less than 2^-19; the gates above it are off by up to 2^-17 (exp's
argument of up to 88 rounded to 2^-24).  A t, and a scale, below the normal floats are rounded to multiples of 2^-149.
"""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16]
FAR, LEAST = 2.0 ** -17, 2.0 ** -150


def e4m3(v):
    """The nearest e4m3 number of every float64, half to even, in float64."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def check(gate, up):
    from gemmlib_b200.fp8_linear import silu_mul_fp8

    n, k = gate.shape
    q = silu_mul_fp8(gate, up)
    g = gate.double()
    y = g * torch.sigmoid(g) * up.double()
    top = torch.nn.functional.pad(y.abs(), (0, -k % 128)).view(n, -1, 128).amax(-1)
    assert (top < 2.0 ** 127).all()
    assert ((q.scales.double() - top / 448).abs() <= (top + LEAST) / 448 * (FAR + 2.0 ** -24) + 2 * LEAST).all()
    # a block whose largest t is no more than some steps of the subnormals has values that depend on their rounding
    told = (top > 2.0 ** -130).repeat_interleave(128, 1)[:, :k]
    each = top.clamp(min=2.0 ** -130).repeat_interleave(128, 1)[:, :k]
    t, off = y * 448 / each, (y.abs() * 2 * FAR + 2 * LEAST) * 448 / each  # the value's own distance and the scale's
    got = q.values.double()
    assert ((got >= e4m3(t - off)) & (got <= e4m3(t + off)))[told].all()
    return q, top


def normal(n, k, seed):
    return torch.randn(n, k, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda", dtype=torch.float64)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("k", [1, 77, 128, 1000, 4096])
def test_gates_whose_reciprocal_is_no_normal_float(k, dtype):
    """From -88.7 to -87.3: 1 / (1 + exp(-gate)) lies between 2^-128 and 2^-126."""
    g = torch.Generator(device="cuda").manual_seed(k)
    gate = (-88.7 + 1.4 * torch.rand(40, k, generator=g, device="cuda")).to(dtype)
    high = 15 if dtype == torch.float16 else 120
    up = (normal(40, k, 1).clamp(-2, 2) * torch.exp2(torch.linspace(0, high - 1, 40, device="cuda", dtype=torch.float64))[:, None]).to(dtype)
    q, top = check(gate, up)
    assert ((q.scales > 0) == (top > 0)).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_every_gate_below(dtype):
    """A row for each gate of the type from -80 to -200, alone in its blocks, and one beside gates of 0 and the largest ones of the type."""
    gate = torch.arange(-200, -80, 1 / 16, device="cuda").to(dtype).unique()
    big = 2.0 ** 15 if dtype == torch.float16 else 2.0 ** 126
    up = (big * (0.5 + torch.rand(len(gate), 256, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda"))).to(dtype)
    up[:, ::3] *= -1
    rows = gate[:, None].expand(-1, 256).contiguous()
    q, top = check(rows, up)
    assert (top[gate > -181].min() > 2.0 ** -126 or dtype == torch.float16) and (q.scales[gate > -90] > 0).all()
    rows[:, 1:128:2] = 0
    check(rows, up)
    rows[:, 1:128:2] = torch.finfo(dtype).min  # exp of it is 0, whatever up is
    check(rows, up)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_beside_ordinary_gates(dtype):
    """Their values are those of the block without them, and rows that begin anywhere have the same bits."""
    from gemmlib_b200.fp8_linear import silu_mul_fp8

    gate, up = (2 * normal(33, 500, 3)).to(dtype), normal(33, 500, 4).to(dtype)
    want = silu_mul_fp8(gate, up)
    far = gate.clone()
    far[:, 7::16] = -95.0
    got, _ = check(far, up)
    same = torch.ones(500, dtype=torch.bool, device="cuda")
    same[7::16] = False
    alone = gate.clone()
    alone[:, 7::16] = 0
    want = silu_mul_fp8(alone, up)
    assert torch.equal(got.scales, want.scales) and torch.equal(got.values.float()[:, same], want.values.float()[:, same])
    assert (got.values.float()[:, ~same] == 0).all()
    far[:, :128] = -88.0
    held = silu_mul_fp8(far, up)
    for before in (1, 3, 5):
        wide = torch.full((2, 33, 500 + before), float("nan"), dtype=dtype, device="cuda")
        g, u = wide[:, :, before:]
        g.copy_(far), u.copy_(up)
        odd = silu_mul_fp8(g, u)
        assert torch.equal(odd.values.view(torch.uint8), held.values.view(torch.uint8)) and torch.equal(odd.scales, held.scales)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_infinite_gates_and_factors_spoil_their_block(dtype):
    from gemmlib_b200.fp8_linear import silu_mul_fp8

    gate, up = torch.full((4, 256), -88.0, dtype=dtype, device="cuda"), torch.ones(4, 256, dtype=dtype, device="cuda")
    gate[1, 5], gate[2, 130] = float("-inf"), float("nan")
    up[3, 9] = float("inf")
    spoiled = torch.zeros(4, 2, dtype=torch.bool, device="cuda")
    spoiled[1, 0] = spoiled[2, 1] = spoiled[3, 0] = True
    assert torch.equal(silu_mul_fp8(gate, up).scales.isnan(), spoiled)
