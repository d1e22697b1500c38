"""The product of int8 rows on the GPU, against exact integer sums.

Bound: the sum (an integer) is rounded to fp32, multiplied with the activation's scale and then, with the bias added, with the
weight's: three roundings of 2^-24; then the result is rounded to its type, by half a step of it.
"""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

EPS24 = 2.0 ** -24
TYPES = [torch.float16, torch.bfloat16]


def rows_of(n, k, seed):
    """Random int8 rows, on pitches of any multiple of 16 bytes, with the whole range of int8 (-128 too), and scales."""
    from gemmlib_b200.int8_linear import Int8Rows

    g = torch.Generator(device="cuda").manual_seed(seed)
    v = torch.full((n, -(-k // 16) * 16), 77, dtype=torch.int8, device="cuda")[:, :k]  # the padding is no part of the rows
    v.copy_(torch.randint(-128, 128, (n, k), generator=g, device="cuda"))
    s = (0.5 + torch.rand(n, generator=g, device="cuda")) / (74 * k ** 0.25)
    return Int8Rows(v, s)


def check_close(got, x, w, bias=None):
    k = x.values.shape[-1]
    sums = x.values.double().reshape(-1, k) @ w.values.double().t()  # exact: below 2^53
    product = sums * x.scales.double().reshape(-1, 1) * w.scales.double()
    want = product if bias is None else product + bias.double()
    eps = torch.finfo(got.dtype).eps / 2
    smallest = 2.0 ** -25 if got.dtype == torch.float16 else 2.0 ** -134  # half a step of a subnormal result
    bound = want.abs() * eps * (1 + 1e-3) + smallest + 3.01 * EPS24 * (product.abs() + want.abs())
    off = (got.double().reshape(want.shape) - want).abs()
    assert (off <= bound).all(), (float(off.max()), int((off > bound).sum()))


SHAPES = [  # rows, in_features, out_features: tiles and steps that end inside, one to many rows, K split or not
    (1, 1, 1), (1, 16, 8), (1, 500, 3001), (2, 512, 777), (1, 1000, 2050), (2, 1024, 99), (2, 530, 1500), (3, 5001, 70), (1, 20000, 300), (4, 9000, 2000), (1, 128, 128), (1, 100, 130), (1, 4096, 4096), (2, 4096, 1000), (7, 5001, 129), (8, 8192, 256),
    (15, 129, 127), (16, 256, 64), (17, 1000, 1237), (31, 2048, 384), (33, 640, 2048), (64, 4096, 512), (65, 127, 100),
    (100, 11008, 96), (127, 384, 641), (128, 1024, 1024), (129, 1024, 136), (200, 2000, 520), (255, 130, 300), (256, 512, 256),
    (257, 512, 513), (300, 4096, 768), (333, 5001, 1237), (512, 256, 1024), (513, 1040, 264), (1000, 136, 2000), (1024, 1024, 1024),
    (2048, 2048, 1536), (1500, 704, 3000), (4097, 64, 520), (20000, 48, 24),
]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_product(shape, dtype):
    from gemmlib_b200.int8_linear import int8_linear

    m, k, n = shape
    x, w = rows_of(m, k, 1), rows_of(n, k, 2)
    out = int8_linear(x, w, dtype=dtype)
    assert out.shape == (m, n) and out.dtype == dtype
    check_close(out, x, w)
    bias = torch.linspace(-3, 3, n, device="cuda").to(dtype)
    check_close(int8_linear(x, w, bias, dtype=dtype), x, w, bias)


@pytest.mark.parametrize("m", [1, 16, 300])
def test_sums_are_exact_to_the_end_of_int32(m):
    """The longest K with the largest magnitudes: 128 * 128 * 131071 < 2^31."""
    from gemmlib_b200.int8_linear import Int8Rows, int8_linear

    k = 131071
    v = torch.full((m, k + 1), -128, dtype=torch.int8, device="cuda")[:, :k]
    x = Int8Rows(v, torch.full((m,), 2.0 ** -20, device="cuda"))
    w = torch.full((24, k + 1), -128, dtype=torch.int8, device="cuda")[:, :k]
    w[1] = 127
    w[2, ::2] = 127
    check_close(int8_linear(x, Int8Rows(w, torch.ones(24, device="cuda")), dtype=torch.bfloat16), x, Int8Rows(w, torch.ones(24, device="cuda")))


@pytest.mark.parametrize("m,k,n", [(3, 300, 200), (40, 4096, 201), (700, 512, 520)])
def test_strided_operands_and_output(m, k, n):
    from gemmlib_b200.int8_linear import Int8Rows, int8_linear

    x, w = rows_of(m, k, 3), rows_of(n, k, 4)
    want = int8_linear(x, w)
    wide = torch.zeros(n, 1024 * 5, dtype=torch.int8, device="cuda")
    wide[:, 16:16 + k] = w.values
    assert torch.equal(int8_linear(x, Int8Rows(wide[:, 16:16 + k], w.scales)), want)
    # activations that begin anywhere, and scales that are not contiguous
    far = torch.zeros(m, k + 7, dtype=torch.int8, device="cuda")
    far[:, 3:3 + k] = x.values
    scales = torch.stack([x.scales, x.scales], 1)[:, 0]
    assert torch.equal(int8_linear(Int8Rows(far[:, 3:3 + k], scales), w), want)
    # leading dimensions
    if m % 2 == 0:
        three = Int8Rows(x.values.unflatten(0, (2, m // 2)), x.scales.view(2, m // 2))
        assert torch.equal(int8_linear(three, w), want.view(2, m // 2, n))
    one = int8_linear(Int8Rows(x.values[0], x.scales[0]), w)
    assert one.shape == (n,) and torch.equal(one, want[0])
    for pad in (1, 6, 8):  # outputs into a wider matrix, and nothing beside them
        out = torch.full((m, n + pad), 9.0, dtype=torch.float16, device="cuda")
        view = out[:, pad - 1: pad - 1 + n]
        got = int8_linear(x, w, out=view)
        assert got.data_ptr() == view.data_ptr() and torch.equal(view, want)
        assert (out[:, :pad - 1] == 9).all() and (out[:, pad - 1 + n:] == 9).all()


@pytest.mark.parametrize("m,k,n", [(2, 256, 4), (40, 512, 201), (600, 256, 4927), (600, 256, 4924), (600, 256, 4920), (4000, 64, 1001)])
@pytest.mark.parametrize("wider", [1, 4, 7, 8, 16])
def test_nothing_is_written_beside_an_output_in_a_wider_matrix(m, k, n, wider):
    """Whatever its rows end on: 16, 8 or 2 bytes of the wider matrix's aligned rows."""
    from gemmlib_b200.int8_linear import int8_linear

    x, w = rows_of(m, k, 6), rows_of(n, k, 7)
    want = int8_linear(x, w)
    for pitch in {n + wider, -(-(n + wider) // 8) * 8}:
        out = torch.full((m + 1, pitch), 9.0, dtype=torch.float16, device="cuda")
        assert torch.equal(int8_linear(x, w, out=out[:m, :n]), want)
        assert (out[:, n:] == 9).all() and (out[m] == 9).all()


@pytest.mark.parametrize("n", [32776, 32767])  # outputs by TMA, and one by one
def test_offsets_beyond_32_bits(n):
    from gemmlib_b200.int8_linear import Int8Rows, int8_linear

    m, k = 70000, 48
    wide = torch.randint(-128, 128, (m, 32768), dtype=torch.int8, device="cuda")
    x = Int8Rows(wide[:, 32000:32000 + k], torch.rand(m, device="cuda") / 100)
    w = rows_of(n, k, 2)
    out = int8_linear(x, w)
    assert m * 32768 > 2 ** 31 and out.numel() > 2 ** 31
    for at in (0, m // 2, m - 300):
        part = Int8Rows(x.values[at:at + 300], x.scales[at:at + 300])
        check_close(out[at:at + 300], part, w)


@pytest.mark.parametrize("m", [1, 4, 40])  # the weights beyond 2^31 bytes, by loads and by copies
def test_weights_beyond_32_bits(m):
    from gemmlib_b200.int8_linear import Int8Rows, int8_linear

    n, k = 70000, 500
    wide = torch.randint(-128, 128, (n, 32768), dtype=torch.int8, device="cuda")
    x, w = rows_of(m, k, 1), Int8Rows(wide[:, 32000:32000 + k], torch.rand(n, device="cuda") / 100)
    check_close(int8_linear(x, w, dtype=torch.bfloat16), x, w)


def test_no_rows_and_nan_rows():
    from gemmlib_b200.int8_linear import Int8Rows, int8_linear, quantize_int8

    w = rows_of(50, 64, 5)
    empty = Int8Rows(torch.empty(0, 64, dtype=torch.int8, device="cuda"), torch.empty(0, device="cuda"))
    assert int8_linear(empty, w).shape == (0, 50)
    x = torch.randn(4, 64, device="cuda").half()
    x[2, 5] = float("inf")
    x[3] = 0
    out = int8_linear(quantize_int8(x), w)
    assert torch.isnan(out[2]).all() and torch.isfinite(out[[0, 1]]).all() and not out[3].any()


def test_refusals():
    from gemmlib_b200.int8_linear import Int8Rows, int8_linear

    x, w = rows_of(4, 64, 1), rows_of(8, 64, 2)
    for bad, text in [
        (lambda: int8_linear(x, rows_of(8, 48, 2)), "cannot be multiplied"),
        (lambda: int8_linear(x, Int8Rows(w.values[:, :63].contiguous(), w.scales)), "cannot be multiplied"),
        (lambda: int8_linear(Int8Rows(x.values[:, :63], x.scales), Int8Rows(w.values[:, :63].contiguous(), w.scales)), "must begin on 16 bytes"),
        (lambda: int8_linear(x, Int8Rows(w.values[0], w.scales)), "must be .out_features, in_features."),
        (lambda: int8_linear(x, Int8Rows(w.values[:0], w.scales[:0])), "the weight is empty"),
        (lambda: int8_linear(x, Int8Rows(w.values, w.scales[:7])), "one float32 scale a row"),
        (lambda: int8_linear(Int8Rows(x.values, x.scales.half()), w), "one float32 scale a row"),
        (lambda: int8_linear(x, w, torch.zeros(8, device="cuda")), "the bias must be"),
        (lambda: int8_linear(x, w, torch.zeros(7, dtype=torch.float16, device="cuda")), "the bias must be"),
        (lambda: int8_linear(x, w, out=torch.empty(4, 7, dtype=torch.float16, device="cuda")), "shape and type of the result"),
        (lambda: int8_linear(x, w, out=torch.empty(4, 8, dtype=torch.bfloat16, device="cuda")), "shape and type of the result"),
        (lambda: int8_linear(x, w, out=torch.empty(8, 4, dtype=torch.float16, device="cuda").t()), "contiguous rows of one pitch"),
        (lambda: int8_linear(x, Int8Rows(w.values.cpu(), w.scales)), "must be a CUDA tensor"),
        (lambda: int8_linear(rows_of(2, 131088, 1), rows_of(2, 131088, 2)), "int32 sums hold up to"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            bad()


@pytest.mark.parametrize("m", [1, 5, 64, 400])
def test_repeats_streams_and_graphs(m):
    """The same bits every time: on side streams, two at once, captured, and with the weights fetched early."""
    from gemmlib_b200 import capi
    from gemmlib_b200.int8_linear import int8_linear

    x, w = rows_of(m, 2048, 1), rows_of(1100, 2048, 2)
    want = int8_linear(x, w)
    check_close(want, x, w)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(int8_linear(x, w, flags=i % 2 * capi.EARLY_WEIGHT_FETCH))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs.append(int8_linear(x, w))
        outs.append(int8_linear(x, w, flags=capi.EARLY_WEIGHT_FETCH))
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, want)
    assert capi.last_kernel_status() == 0
