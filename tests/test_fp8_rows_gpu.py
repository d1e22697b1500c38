"""Rows and weights of e4m3 on the GPU, against their definition in 64 bits.

Of 16-bit inputs every value is decided: the quotient 448 x / max|x| of numbers of 11 bits is exact in 64 bits where it is half-way between two e4m3
numbers, and further from that than any rounding otherwise; the scale is max / 448 rounded to fp32.  So both have to be equal.  The gate's
values come from fp32 arithmetic (ex2 and rcp of 2^-22, three roundings of 2^-24, exp's argument of up to 90 rounded to 2^-24: 2^-17 in all,
relative), so a value may be that of a t as far away.
"""
import copy
import io

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16]
E4M3 = torch.float8_e4m3fn


def e4m3(v):
    """The nearest e4m3 number of every float64, half to even, in float64."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def top_of(y, high):
    """The largest magnitude of each element's block, and of each block."""
    n, k = y.shape
    pad = torch.nn.functional.pad(y.abs(), (0, -k % 128, 0, -n % high)).view(-(-n // high), high, -(-k // 128), 128)
    top = pad.amax((1, 3))
    return top.repeat_interleave(high, 0)[:n].repeat_interleave(128, 1)[:, :k], top


def check(q, x, high=1):
    """`q` against `x` [n, k] of finite 16-bit numbers."""
    y = x.double()
    each, top = top_of(y, high)
    assert torch.equal(q.scales.reshape(top.shape), (top / 448).float())
    want = e4m3(torch.where(each > 0, y * 448 / torch.where(each > 0, each, 1.0), 0.0))
    got = q.values.reshape(x.shape).double()
    assert torch.equal(got, want), (got != want).nonzero()[:5]


def inputs(n, k, dtype, seed, spread=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(n, k, generator=g, device="cuda") * torch.exp(spread * torch.randn(k, generator=g, device="cuda"))).to(dtype)


SIZES = [(1, 1), (1, 127), (1, 128), (1, 129), (2, 200), (3, 4096), (5, 5001), (17, 384), (100, 640), (333, 1237), (1000, 2048), (4100, 520), (70000, 24), (64, 28672)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,k", SIZES)
def test_rows(n, k, dtype):
    from gemmlib_b200.fp8_linear import quantize_fp8

    x = inputs(n, k, dtype, n + k)
    q = quantize_fp8(x)
    assert q.values.dtype == E4M3 and q.values.shape == (n, k) and q.scales.shape == (n, -(-k // 128)) and q.values.stride(0) % 32 == 0
    check(q, x)
    each = q.values.double() * q.scales.double().repeat_interleave(128, 1)[:, :k]
    assert torch.equal(q.dequantize(dtype), each.float().to(dtype))  # (the product of 4 and 24 bits is rounded twice, as here)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, 1), (127, 129), (128, 128), (300, 200), (11, 4096), (1237, 5001), (3, 130, 257), (2, 2, 64, 384), (7, 1, 1)], ids=str)
def test_weights(shape, dtype):
    from gemmlib_b200.fp8_linear import quantize_fp8_weight

    *lead, n, k = shape
    x = inputs(x_rows := torch.Size(lead).numel() * n, k, dtype, 3).view(shape)
    q = quantize_fp8_weight(x)
    assert q.values.shape == x.shape and q.scales.shape == (*lead, -(-n // 128), -(-k // 128))
    for e, (v, s) in enumerate(zip(q.values.reshape(-1, n, k), q.scales.reshape(-1, *q.scales.shape[-2:]))):
        check(type(q)(v, s), x.reshape(-1, n, k)[e], 128)
    real = q.values.double() * q.scales.double().repeat_interleave(128, -2)[..., :n, :].repeat_interleave(128, -1)[..., :k]
    assert torch.equal(q.dequantize(dtype), real.float().to(dtype)) and x_rows > 0


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_halves_between_two_values(dtype):
    """Largest magnitudes that are multiples of 7 put 16-bit numbers exactly half-way; three in 64 of any largest magnitude do too."""
    from gemmlib_b200.fp8_linear import quantize_fp8, quantize_fp8_weight

    rows = []
    for top in [7, 3.5, 0.4375, 448, 49, 231, 245, 1785 if dtype == torch.float16 else 1792, 12, 1, 0.3, 100, 5 / 64]:
        top = torch.tensor(top, dtype=torch.float64)
        mids = torch.tensor([m * 2.0 ** e for e in range(-10, 5) for m in range(16, 33)], dtype=torch.float64)  # all values and midpoints but few
        row = (mids * top / 448).clamp(max=float(top))[:255]
        rows.append(torch.cat([row, top.view(1)]).view(2, 128))
        rows.append(torch.cat([top.view(1), -row]).view(2, 128))
    for r in rows:
        r[:, 0] = r.abs().max()
    x = torch.cat(rows).to(dtype).cuda()
    check(quantize_fp8(x), x)
    check(quantize_fp8_weight(x), x, 128)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_ranges(dtype):
    """Blocks of every magnitude that the type has, and of zeros."""
    from gemmlib_b200.fp8_linear import quantize_fp8

    info = torch.finfo(dtype)
    g = torch.Generator(device="cuda").manual_seed(1)
    low = -24 if dtype == torch.float16 else -133
    x = torch.rand(400, 128, generator=g, device="cuda", dtype=torch.float64) * 2 - 1
    x = x * torch.exp2(torch.linspace(low, 15 if dtype == torch.float16 else 127, 400, device="cuda", dtype=torch.float64))[:, None]
    x = x.clamp(-info.max, info.max).to(dtype)
    x[5] = 0
    x[6, ::2] = -0.0
    x[6, 1::2] = 0
    x[7, 3] = info.max
    q = quantize_fp8(x)
    y = x.double()
    top = y.abs().amax(1, keepdim=True)
    want = e4m3(torch.where(top > 0, y * 448 / torch.where(top > 0, top, 1.0), 0.0))
    assert torch.equal(q.values.double(), want)
    # a scale below fp32's normal numbers is rounded to a multiple of 2^-149
    assert ((q.scales.double() - top / 448).abs() <= top / 448 * 2.0 ** -24 + 2.0 ** -150).all()
    assert (q.scales[5] == 0).all() and (q.scales[6] == 0).all()


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_infinities_and_nan_spoil_their_block_alone(dtype, bad):
    from gemmlib_b200.fp8_linear import quantize_fp8, quantize_fp8_weight, silu_mul_fp8

    x = inputs(300, 400, dtype, 2)
    clean = quantize_fp8(x)
    y = x.clone()
    y[7, 130] = bad
    y[299, 399] = bad
    q = quantize_fp8(y)
    spoiled = torch.zeros_like(clean.scales, dtype=torch.bool)
    spoiled[7, 1] = spoiled[299, 3] = True
    assert torch.equal(q.scales.isnan(), spoiled) and torch.equal(q.scales[~spoiled], clean.scales[~spoiled])
    wide = spoiled.repeat_interleave(128, 1)[:, :400]
    assert (q.values.float()[wide] == 0).all() and torch.equal(q.values.float()[~wide], clean.values.float()[~wide])
    w = quantize_fp8_weight(y)
    want = torch.zeros(3, 4, dtype=torch.bool, device="cuda")
    want[0, 1] = want[2, 3] = True
    assert torch.equal(w.scales.isnan(), want)
    assert torch.equal(silu_mul_fp8(x, y).scales.isnan(), spoiled)
    assert torch.equal(q.dequantize(dtype).isnan(), wide)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,k", [(1, 1), (4, 11008), (17, 130), (333, 1237), (2048, 704), (3000, 64)])
def test_gate(n, k, dtype):
    from gemmlib_b200.fp8_linear import silu_mul_fp8

    both = inputs(n, 2 * k, dtype, 5, 0.3) * 3
    gate, up = both[:, :k], both[:, k:]
    q = silu_mul_fp8(gate, up)
    y = gate.double() * torch.sigmoid(gate.double()) * up.double()
    each, top = top_of(y, 1)
    far = 2.0 ** -17
    assert ((q.scales.double() - top / 448).abs() <= top / 448 * (far + 2.0 ** -24)).all()
    t = torch.where(each > 0, y * 448 / torch.where(each > 0, each, 1.0), 0.0)
    lo, hi = e4m3(t - t.abs() * 2 * far), e4m3(t + t.abs() * 2 * far)  # the value's own distance and the scale's
    got = q.values.double()
    assert ((got >= lo) & (got <= hi)).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_extreme_gates(dtype):
    """exp of either end: silu(-large) is 0, silu(large) the gate itself; products that overflow are infinite and spoil the block."""
    from gemmlib_b200.fp8_linear import silu_mul_fp8

    big = torch.finfo(dtype).max
    gate = torch.tensor([[-big, -1000.0, -0.0, 0.0, 1000.0, 20.0, -20.0, 1.0]], device="cuda").to(dtype)
    q = silu_mul_fp8(gate, torch.ones_like(gate))
    assert q.dequantize(torch.bfloat16).isfinite().all() and (q.values.float()[0, :4] == 0).all()
    if dtype == torch.bfloat16:
        assert silu_mul_fp8(torch.full_like(gate, big), torch.full_like(gate, big)).scales.isnan().all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("k", [64, 129, 1000])
def test_layouts(k, dtype):
    """Rows that begin anywhere, leading dimensions, transposed inputs: as the same rows on their own."""
    from gemmlib_b200.fp8_linear import Fp8Rows, quantize_fp8, quantize_fp8_weight

    wide = inputs(24, k + 11, dtype, 9)
    for at in (0, 1, 2, 3, 8, 11):
        x = wide[:, at:at + k]
        own = quantize_fp8(x.clone())
        for q in (quantize_fp8(x), quantize_fp8(x.reshape(2, 3, 4, k)), quantize_fp8(x.t().contiguous().t())):
            assert torch.equal(q.values.reshape(24, k).float(), own.values.float()) and torch.equal(q.scales.reshape(24, -1), own.scales)
        every = quantize_fp8(x[::2])
        assert torch.equal(every.values.float(), own.values[::2].float())
        w = quantize_fp8_weight(x)
        assert torch.equal(w.values.float(), quantize_fp8_weight(x.clone()).values.float())
        # values and scales out of the middle of wider ones
        values = torch.zeros(24, k + 7, dtype=torch.uint8, device="cuda").view(E4M3)[:, 5:5 + k]
        values.copy_(own.values)
        scales = torch.zeros(24, own.scales.size(1) + 3, device="cuda")[:, 1:1 + own.scales.size(1)]
        scales.copy_(own.scales)
        assert torch.equal(Fp8Rows(values, scales).dequantize(dtype), own.dequantize(dtype))


def test_empty_and_saved_rows(tmp_path):
    from gemmlib_b200.fp8_linear import Fp8Rows, Fp8Weight, quantize_fp8, quantize_fp8_weight, silu_mul_fp8

    x = torch.empty(0, 300, dtype=torch.float16, device="cuda")
    for q in (quantize_fp8(x), silu_mul_fp8(x, x)):
        assert q.values.shape == (0, 300) and q.scales.shape == (0, 3) and q.dequantize().shape == (0, 300)
    q = quantize_fp8(inputs(5, 300, torch.float16, 1))
    held = io.BytesIO()
    torch.save(q, held)
    held.seek(0)
    for other in (torch.load(held), copy.deepcopy(q)):
        assert type(other) is Fp8Rows and torch.equal(other.values.float(), q.values.float()) and torch.equal(other.scales, q.scales)
    w = quantize_fp8_weight(inputs(130, 300, torch.float16, 1))
    torch.save(w, tmp_path / "w")
    other = torch.load(tmp_path / "w")
    assert type(other) is Fp8Weight and torch.equal(other.values.float(), w.values.float()) and torch.equal(other.scales, w.scales)


def test_refusals_on_the_gpu():
    from gemmlib_b200.fp8_linear import Fp8Rows, Fp8Weight, quantize_fp8, quantize_fp8_weight, silu_mul_fp8

    x = inputs(4, 256, torch.float16, 1)
    q, w = quantize_fp8(x), quantize_fp8_weight(x)
    with pytest.raises(RuntimeError, match="of shape"):
        Fp8Rows(q.values, q.scales[:, :1]).dequantize()
    with pytest.raises(RuntimeError, match="of shape"):
        Fp8Weight(w.values, q.scales).dequantize()
    with pytest.raises(RuntimeError, match="float32"):
        Fp8Rows(q.values, q.scales.half()).dequantize()
    with pytest.raises(RuntimeError, match="device"):
        Fp8Rows(q.values, q.scales.cpu()).dequantize()
    with pytest.raises(RuntimeError, match="CUDA tensor|device"):
        silu_mul_fp8(x, x.cpu())
    with pytest.raises(RuntimeError, match="out_features, in_features"):
        quantize_fp8_weight(x[0])
    with pytest.raises(RuntimeError, match="at least one element"):
        quantize_fp8(x[:, :0])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_rows_that_begin_anywhere(dtype):
    """Bit for bit as rows that begin on 16 bytes, for every width around a piece and a block, and every beginning within 16 bytes; what stands
    beside the rows is NaN."""
    from gemmlib_b200.fp8_linear import quantize_fp8, quantize_fp8_weight, silu_mul_fp8

    def same(a, b, case):
        assert torch.equal(a.values.view(torch.uint8), b.values.view(torch.uint8)) and torch.equal(a.scales, b.scales), case

    g = torch.Generator(device="cuda").manual_seed(1)
    for k in [*range(1, 35), 127, 128, 129, 255, 257, 500, 1237]:
        for before in range(9):
            for behind in (0, 1, 4):
                wide = torch.full((2, 19, before + k + behind), float("nan"), dtype=dtype, device="cuda")
                gate, up = wide[:, :, before:before + k].copy_(torch.randn(2, 19, k, generator=g, device="cuda").to(dtype))
                held = torch.zeros(2, 19, -(-k // 8) * 8, dtype=dtype, device="cuda")[:, :, :k].copy_(wide[:, :, before:before + k])
                same(quantize_fp8(gate), quantize_fp8(held[0]), (k, before, behind))
                same(quantize_fp8_weight(gate), quantize_fp8_weight(held[0]), (k, before, behind))
                same(silu_mul_fp8(gate, up), silu_mul_fp8(*held), (k, before, behind))
