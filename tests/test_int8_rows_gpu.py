"""int8 rows on the GPU, against their definition in 64 bits.

Bounds.  u = 127 t / max|t| is what the values round.  The kernel multiplies t with fp32(127 / max|t|), off by 2^-24 of itself, and
rounds the product to fp32, off by half a step of 2^-17 up to 128, and then to an integer: for t known exactly
|u - value| <= 1/2 + 127 * 2^-24 + 2^-18.
"""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

EPS24 = 2.0 ** -24
TYPES = [torch.float16, torch.bfloat16]
# one to many threads and chunks a row, rows that end inside a vector, in several CTAs (over 32768), and read twice (over 65536)
WIDTHS = [1, 2, 7, 8, 9, 16, 100, 128, 255, 512, 513, 1000, 2048, 2056, 4096, 5001, 8192, 8200, 11008, 28672, 32768, 32769, 40000, 65529, 65537, 70000]


def ids(v):
    return str(v).replace("torch.", "")


def normal(*shape, dtype, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def check_rows(rows, t, factor=None, t_error=0.0, factor_error=0.0):
    """`t`: the rows in 64 bits, known up to the relative error t_error (a number or a tensor like t); `factor`: by row, times the
    scale."""
    values, scales = rows
    assert values.dtype == torch.int8 and values.shape == t.shape and scales.dtype == torch.float32
    assert scales.shape == t.shape[:-1]
    top = t.abs().amax(-1, keepdim=True)
    error = torch.as_tensor(t_error, device=t.device, dtype=torch.float64).expand_as(t)
    top_error = error.amax()
    u = torch.where(top > 0, 127 * t / torch.where(top > 0, top, 1.0), 0.0)
    off = (u - values.double()).abs()
    assert (off <= 0.5 + 127 * EPS24 + 2.0 ** -18 + u.abs() * (error + top_error) * 1.01).all(), float((off - 0.5).max())
    want = top[..., 0] / 127 * (1.0 if factor is None else factor)
    # below 2^-126 floats are 2^-149 apart, so that a rounding is off by up to 2^-150 whatever the value
    assert ((scales.double() - want).abs() <= want * (EPS24 * 1.01 + top_error * 1.01 + factor_error) + 2.0 ** -150).all()


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("cols", WIDTHS)
def test_quantize(dtype, cols):
    from gemmlib_b200.int8_linear import quantize_int8

    x = normal(5, cols, dtype=dtype, seed=cols)
    x[2] = 0
    x[3] *= 1e-3
    rows = quantize_int8(x)
    check_rows(rows, x.double())
    assert rows.scales[2] == 0 and not rows.values[2].any()
    assert int(rows.values[0].abs().max()) == 127
    if cols > 1:
        assert rows.values.stride(0) % 32 == 0  # rows that the product takes as they are


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows", [1, 3, 4, 5, 127, 1000])
@pytest.mark.parametrize("cols", [64, 4096])
def test_quantize_many_rows(dtype, rows, cols):
    from gemmlib_b200.int8_linear import quantize_int8

    x = normal(rows, cols, dtype=dtype, seed=rows)
    check_rows(quantize_int8(x), x.double())


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("cols,pitch,offset", [
    (1025, 1025, 0), (1025, 1025, 3), (1032, 1040, 8), (1100, 1100, 1), (2047, 2049, 5), (4096, 4096, 0), (4096, 4099, 7), (4097, 4097, 2),
    (5003, 5003, 0), (8192, 8192, 0), (8191, 8193, 6), (8200, 8200, 0), (11008, 11008, 4), (11007, 11007, 1), (20001, 20001, 0),
    (28672, 28672, 0), (31743, 31744, 0), (31745, 31745, 0), (33000, 33001, 1)])
def test_many_rows(dtype, cols, pitch, offset):
    """More rows than the GPU takes at a time, which begin anywhere: against the definition, against a few of the same rows alone bit
    for bit, and nothing is read but the rows (their surroundings are NaN)."""
    from gemmlib_b200.int8_linear import quantize_int8, rms_norm_int8, silu_mul_int8

    rows = 1301
    flat = torch.full((2, rows * pitch + 64), float("nan"), dtype=dtype, device="cuda")
    x, y = (f[offset: offset + (rows - 1) * pitch + cols].as_strided((rows, cols), (pitch, 1)) for f in flat)
    x.copy_(normal(rows, cols, dtype=dtype, seed=cols))
    y.copy_(normal(rows, cols, dtype=dtype, seed=cols + 1))
    w = normal(cols, dtype=dtype, seed=3)
    check_rows(quantize_int8(x), x.double())
    t, factor = norm_reference(x, w, 1e-5)
    check_rows(rms_norm_int8(x, w), t, factor, factor_error=NORM_ERROR)
    made, h = rms_norm_int8(x, w, residual=y)
    assert torch.equal(h, x + y)
    t, factor = norm_reference(h, w, 1e-5)
    check_rows(made, t, factor, factor_error=NORM_ERROR)
    g = x.double()
    check_rows(silu_mul_int8(x, y), g * torch.sigmoid(g) * y.double(), t_error=silu_error(x))
    for call in (quantize_int8, lambda v: rms_norm_int8(v, w), lambda v: silu_mul_int8(v, y[: len(v)])):
        few, all_ = call(x[:5]), call(x)
        assert torch.equal(few.values, all_.values[:5]) and torch.equal(few.scales, all_.scales[:5])
    out = y.clone(memory_format=torch.preserve_format) if pitch == cols else y
    made2, h2 = rms_norm_int8(x, w, residual=out, residual_out=out)
    assert torch.equal(h2, h) and torch.equal(made2.values, made.values) and torch.equal(made2.scales, made.scales)
    if pitch != cols:
        assert torch.isnan(flat[1, offset: offset + rows * pitch].view(rows, pitch)[:-1, cols:]).all()


def test_rounding_is_half_to_even_and_symmetric():
    from gemmlib_b200.int8_linear import quantize_int8

    # max 127: the values are the inputs themselves, rounded
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 0.499, 126.5, -126.5, -127.0, 3.0]], dtype=torch.float16, device="cuda")
    assert quantize_int8(x).values.tolist() == [[127, 0, 2, 2, 0, -2, -2, 0, 126, -126, -127, 3]]


def test_extreme_magnitudes():
    from gemmlib_b200.int8_linear import quantize_int8

    for dtype, top in ((torch.float16, [65504.0, 2.0 ** -24, 2.0 ** -14]), (torch.bfloat16, [3.3e38, 1e-30, 2.0 ** -126])):
        x = torch.tensor([[t, -t / 2, 0.0, t / 4] for t in top], dtype=torch.float64, device="cuda").to(dtype)
        check_rows(quantize_int8(x), x.double())
    # a scale below the smallest normal float keeps what bits it has: within half a step of 2^-149
    x = torch.tensor([[2.0 ** -133, -(2.0 ** -133), 0.0]], dtype=torch.bfloat16, device="cuda")
    r = quantize_int8(x)
    assert r.values.tolist() == [[127, -127, 0]]
    assert abs(float(r.scales[0].double()) - 2.0 ** -133 / 127) <= 2.0 ** -150


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("cols,at", [(1, 0), (40, 39), (4096, 4095), (5001, 5000), (40000, 8191), (40000, 39999), (70000, 69999)])
def test_a_row_with_an_infinity_or_nan_is_nan_alone(dtype, bad, cols, at):
    from gemmlib_b200.int8_linear import quantize_int8, rms_norm_int8, silu_mul_int8

    x = normal(3, cols, dtype=dtype)
    x[1, at] = bad
    w = torch.ones(cols, dtype=dtype, device="cuda")
    w[at] = 0  # 0 * inf is NaN
    good = normal(3, cols, dtype=dtype, seed=1)
    made = [quantize_int8(x), rms_norm_int8(x, w), rms_norm_int8(good, w, residual=x)[0], silu_mul_int8(good, x)]
    for r in made:
        assert torch.isnan(r.scales).tolist() == [False, True, False]
        assert not r.values[1].any() and torch.isnan(r.dequantize(dtype)[1]).all()
        assert torch.isfinite(r.dequantize(dtype)[[0, 2]]).all()


def norm_reference(h, w, eps):
    h, w = h.double(), w.double()
    return h * w, 1 / torch.sqrt(h.square().mean(-1) + eps)


# fp32 sums of up to 72 squares a thread and a tree of ten: (72 + 10 + 2) * 2^-24, halved by the root, and five more roundings
NORM_ERROR = 47 * EPS24


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("cols", WIDTHS)
def test_rms_norm(dtype, residual, cols):
    from gemmlib_b200.int8_linear import rms_norm_int8

    x, w = normal(5, cols, dtype=dtype, seed=cols), normal(cols, dtype=dtype, seed=7)
    x[3] *= 100
    eps = 1e-5
    if residual:
        r = normal(5, cols, dtype=dtype, seed=cols + 1, scale=3.0)
        rows, h = rms_norm_int8(x, w, eps, residual=r)
        assert torch.equal(h, x + r)
    else:
        x[2] = 0
        rows, h = rms_norm_int8(x, w, eps), x
        assert rows.scales[2] == 0
    t, factor = norm_reference(h, w, eps)
    check_rows(rows, t, factor, factor_error=NORM_ERROR)


@pytest.mark.parametrize("place", ["x", "residual", "other", "slice of x's matrix"])
@pytest.mark.parametrize("cols", [256, 4097, 40000, 70001])
def test_rms_norm_residual_out_in_place(place, cols):
    from gemmlib_b200.int8_linear import rms_norm_int8

    both = normal(6, 2 * cols, dtype=torch.float16)
    x, r, w = both[:, :cols], normal(6, cols, dtype=torch.float16, seed=1), normal(cols, dtype=torch.float16, seed=2)
    want, sum_ = rms_norm_int8(x, w, residual=r)
    keep = both[:, cols:].clone()
    out = {"x": x, "residual": r, "other": torch.empty_like(r), "slice of x's matrix": both[:, cols:]}[place]
    rows, h = rms_norm_int8(x, w, residual=r, residual_out=out)
    assert h.data_ptr() == out.data_ptr() and torch.equal(out, sum_)
    assert torch.equal(rows.values, want.values) and torch.equal(rows.scales, want.scales)
    if place == "x":
        assert torch.equal(both[:, cols:], keep)


def test_rms_norm_of_values_whose_squares_overflow():
    from gemmlib_b200.int8_linear import rms_norm_int8

    x = normal(4, 300, dtype=torch.bfloat16)
    x[1] *= 1e20
    x[2] *= 1e16
    rows = rms_norm_int8(x, torch.ones(300, dtype=torch.bfloat16, device="cuda"))
    assert torch.isnan(rows.scales).tolist() == [False, True, False, False]
    top = float(x[2].double().abs().max() / x[2].double().square().mean().sqrt()) / 127
    assert abs(float(rows.scales[2]) - top) <= top * (NORM_ERROR + EPS24)


@pytest.mark.parametrize("cols", [512, 9000, 70000])
def test_rms_norm_of_a_tensor_added_to_itself_in_place(cols):
    from gemmlib_b200.int8_linear import rms_norm_int8

    x, w = normal(700, cols, dtype=torch.float16), normal(cols, dtype=torch.float16, seed=1)
    want, h = rms_norm_int8(x, w, residual=x)
    got, same = rms_norm_int8(x, w, residual=x, residual_out=x)
    assert same.data_ptr() == x.data_ptr() and torch.equal(x, h)
    assert torch.equal(got.values, want.values) and torch.equal(got.scales, want.scales)


def test_rms_norm_refusals():
    from gemmlib_b200.int8_linear import rms_norm_int8

    both = normal(4, 64, dtype=torch.float16)
    x, w = both[:, :32], normal(32, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="not overlap them otherwise"):
        rms_norm_int8(x, w, residual=x.clone(), residual_out=both[:, 16:48])
    with pytest.raises(RuntimeError, match="not overlap them otherwise"):
        rms_norm_int8(both.view(8, 32)[:4], w, residual=x.clone(), residual_out=both.view(8, 32)[1:5])
    with pytest.raises(RuntimeError, match="overlaps the weight"):
        rms_norm_int8(x[:1].clone(), both[3, :32], residual=x[:1].clone(), residual_out=both[3:, :32])
    with pytest.raises(RuntimeError, match="contiguous rows of one pitch"):
        rms_norm_int8(x, w, residual=x.clone(), residual_out=normal(32, 4, dtype=torch.float16).t())
    with pytest.raises(RuntimeError, match="one row of the input's length and type"):
        rms_norm_int8(x, w[:31])
    with pytest.raises(RuntimeError, match="one row of the input's length and type"):
        rms_norm_int8(x, w.bfloat16())
    with pytest.raises(RuntimeError, match="the residual must have the input's shape"):
        rms_norm_int8(x, w, residual=x[:3])
    with pytest.raises(RuntimeError, match="must be on the device"):
        rms_norm_int8(x, w.cpu())


def silu_error(gate):
    """Relative: exp of -g 2 + 1.173 |g| ulp, the quotient 2 ulp, the sum and two products half an ulp each; an ulp is 2^-23."""
    return (1.173 * gate.double().abs() + 2 + 2 + 1.5) * 2.0 ** -23


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("cols", WIDTHS)
def test_silu_mul(dtype, cols):
    from gemmlib_b200.int8_linear import silu_mul_int8

    both = normal(5, 2 * cols, dtype=dtype, seed=cols, scale=3.0)
    both[2, :cols] = 0
    gate, up = both[:, :cols], both[:, cols:]
    g = gate.double()
    check_rows(silu_mul_int8(gate, up), g / (1 + torch.exp(-g)) * up.double(), t_error=silu_error(gate))


def test_silu_mul_far_from_zero():
    from gemmlib_b200.int8_linear import silu_mul_int8

    gate = torch.tensor([[-60000.0, -100.0, -89.0, -60.0, 60.0, 100.0, 60000.0, 1.0]], dtype=torch.float16, device="cuda")
    up = torch.ones_like(gate)
    r = silu_mul_int8(gate, up)
    assert r.values.tolist() == [[0, 0, 0, 0, 0, 0, 127, 0]] and abs(float(r.scales[0]) * 127 - 60000) < 0.01
    r = silu_mul_int8(gate[:, :4].contiguous(), up[:, :4])  # -60 exp(-60) is the largest
    g = gate[:, :4].double()
    check_rows(r, g * torch.sigmoid(g), t_error=silu_error(torch.full_like(g, 61.0)))


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("cols", [1, 15, 16, 17, 100, 4096, 5001, 28672])
def test_dequantize(dtype, cols):
    from gemmlib_b200.int8_linear import quantize_int8

    r = quantize_int8(normal(7, cols, dtype=torch.bfloat16, seed=cols))
    out = r.dequantize(dtype)
    assert out.dtype == dtype and out.is_contiguous()
    assert torch.equal(out, (r.values.float() * r.scales[:, None]).to(dtype))


@pytest.mark.parametrize("q_pitch,q_offset,pitch,offset", [(512, 0, 507, 0), (512, 0, 507, 5), (504, 8, 512, 3), (509, 3, 512, 0), (509, 1, 511, 7)])
def test_dequantize_rows_that_begin_anywhere(q_pitch, q_offset, pitch, offset):
    from gemmlib_b200 import capi

    rows, cols = 37, 501
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randint(-128, 128, (rows * q_pitch + 16,), generator=g, device="cuda", dtype=torch.int8)[q_offset:]
    scales = torch.rand(rows, generator=g, device="cuda")
    out = torch.full((rows * pitch + 16,), 7.0, dtype=torch.bfloat16, device="cuda")
    capi.int8_rows_dequant(capi.INT8_BF16, rows, cols, (q, q_pitch), scales, (out[offset:], pitch))
    torch.cuda.synchronize()
    want = (q.as_strided((rows, cols), (q_pitch, 1)).float() * scales[:, None]).bfloat16()
    inside = out[offset:].as_strided((rows, cols), (pitch, 1))
    assert torch.equal(inside, want)
    inside.fill_(7.0)
    assert (out == 7).all()


LAYOUTS = {
    "slice": lambda x: torch.cat([x, x], -1)[..., : x.shape[-1]],
    "odd offset": lambda x: torch.cat([x[..., :1], x], -1)[..., 1:],
    "transposed": lambda x: x.transpose(-1, -2).contiguous().transpose(-1, -2),
    "every second row": lambda x: x.repeat_interleave(2, -2)[..., ::2, :],
    "expanded": lambda x: x[..., :1, :].expand_as(x),
    "three dimensions": lambda x: x.reshape(2, 3, -1),
    "permuted": lambda x: x.reshape(2, 3, -1).transpose(0, 1),
    "one row": lambda x: x[0],
    "no rows": lambda x: x[:0],
}


@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("cols", [40, 4096])
def test_layouts_give_the_same_rows(layout, cols):
    """A view gives what a contiguous copy of it gives, bit for bit, and no input is written."""
    from gemmlib_b200.int8_linear import quantize_int8, rms_norm_int8, silu_mul_int8

    x, y = (LAYOUTS[layout](normal(6, cols, dtype=torch.float16, seed=s)) for s in (0, 1))
    w = normal(cols, dtype=torch.float16, seed=2)
    before = x.clone()
    calls = [quantize_int8, lambda v: rms_norm_int8(v, w), lambda v: silu_mul_int8(v, y), lambda v: silu_mul_int8(y, v),
             lambda v: rms_norm_int8(v, w, residual=y)[0], lambda v: rms_norm_int8(y, w, residual=v)[0]]
    for call in calls:
        got, want = call(x), call(x.contiguous())
        assert torch.equal(got.values, want.values) and torch.equal(got.scales, want.scales)
        assert got.values.shape == x.shape and got.scales.shape == x.shape[:-1]
        assert torch.equal(got.dequantize(), want.dequantize())
    assert torch.equal(x, before)


@pytest.mark.parametrize("cols", [96, 2000, 9000])
def test_offsets_beyond_32_bits(cols):
    from gemmlib_b200.int8_linear import quantize_int8, rms_norm_int8, silu_mul_int8

    rows, pitch, end = 70000, 32768, slice(70000 - 300, 70000)
    wide = torch.empty(rows, pitch, dtype=torch.bfloat16, device="cuda").normal_()
    a, b = wide[:, :cols], wide[:, pitch - cols:]
    assert rows * pitch > 2 ** 31
    w = normal(cols, dtype=torch.bfloat16, seed=1)
    tail_a, tail_b = a[end].clone(), b[end].clone()

    def check(got, want):
        assert torch.equal(got.values[end], want.values) and torch.equal(got.scales[end], want.scales)

    got = quantize_int8(a)
    check(got, quantize_int8(tail_a))
    assert torch.equal(got.dequantize(torch.bfloat16)[end], quantize_int8(tail_a).dequantize(torch.bfloat16))
    check(silu_mul_int8(a, b), silu_mul_int8(tail_a, tail_b))
    check(rms_norm_int8(b, w), rms_norm_int8(tail_b, w))
    want, h = rms_norm_int8(tail_a, w, residual=tail_b)
    got, total = rms_norm_int8(a, w, residual=b, residual_out=b)
    check(got, want)
    assert torch.equal(b[end], h) and total.data_ptr() == b.data_ptr()


def test_nothing_is_written_outside_the_rows():
    """Through the C entry points, into buffers with guards between the rows and behind them."""
    from gemmlib_b200 import capi

    for cols, pitch in ((40, 48), (41, 43), (4096, 4112), (5001, 5003)):
        x, w = normal(4, cols, dtype=torch.float16), normal(cols, dtype=torch.float16, seed=1)
        values = torch.full((4 * pitch + 64,), 99, dtype=torch.int8, device="cuda")
        sums = torch.full((4 * pitch + 64,), 7.0, dtype=torch.float16, device="cuda")
        scales = torch.full((8,), 5.0, device="cuda")
        capi.int8_rows_rms_norm(capi.INT8_FP16, 4, cols, (x, cols), (x, cols), w, 1e-5, (sums, pitch), (values, pitch), scales)
        torch.cuda.synchronize()
        inside = torch.zeros(4 * pitch + 64, dtype=torch.bool, device="cuda")
        inside[: 4 * pitch].view(4, pitch)[:, :cols] = True
        assert (values[~inside] == 99).all() and (sums[~inside] == 7).all() and (scales[4:] == 5).all()
        assert torch.equal(sums[: 4 * pitch].view(4, pitch)[:, :cols], x + x)
        out = torch.full((4 * pitch + 64,), 7.0, dtype=torch.float16, device="cuda")
        capi.int8_rows_dequant(capi.INT8_FP16, 4, cols, (values, pitch), scales, (out, pitch))
        torch.cuda.synchronize()
        assert (out[~inside] == 7).all()


def test_repeats_are_equal_and_streams_and_graphs_work():
    from gemmlib_b200.int8_linear import quantize_int8, rms_norm_int8

    x, w = normal(64, 4096, dtype=torch.bfloat16), normal(4096, dtype=torch.bfloat16, seed=1)
    want, h = rms_norm_int8(x, w, residual=x)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(3):
            got, _ = rms_norm_int8(x, w, residual=x)
    stream.synchronize()
    assert torch.equal(got.values, want.values) and torch.equal(got.scales, want.scales)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, _ = rms_norm_int8(x, w, residual=x)
        again = quantize_int8(got.dequantize(torch.bfloat16))
    x.copy_(normal(64, 4096, dtype=torch.bfloat16, seed=3))
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    want, _ = rms_norm_int8(x, w, residual=x)
    assert torch.equal(got.values, want.values) and torch.equal(got.scales, want.scales)
    assert torch.equal(again.values, quantize_int8(want.dequantize(torch.bfloat16)).values)
