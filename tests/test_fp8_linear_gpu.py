"""The product of e4m3 rows and weights on the GPU, against 64 bits.

Bound: products of two e4m3 numbers are exact in fp32.  A sum over k has at most k additions; the tensor cores' may drop what lies below
the last bit instead of rounding it, so each is off by up to 2^-23 of what has been added in magnitude: for a block's 128, the blocks behind
one another and the parts of a split K, (128 + blocks + 8) * 2^-23 of the sum of magnitudes, with the scales' product (2^-24) among them.  Then
the result is rounded to its type, by half a step.
"""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16]
E4M3 = torch.float8_e4m3fn


def values(n, k, g, pitch=16):
    """e4m3 values over the whole range, on rows of any multiple of 16 bytes; the padding is NaN, which is no part of the rows."""
    v = torch.full((n, -(-k // pitch) * pitch), 0x7f, dtype=torch.uint8, device="cuda").view(E4M3)[:, :k]
    r = torch.randn(n, k, generator=g, device="cuda") * torch.exp(torch.randn(n, k, generator=g, device="cuda"))
    v.copy_((60 * r).clamp(-448, 448))
    return v


def rows_of(m, k, seed):
    from gemmlib_b200.fp8_linear import Fp8Rows

    g = torch.Generator(device="cuda").manual_seed(seed)
    return Fp8Rows(values(m, k, g), torch.exp(torch.randn(m, -(-k // 128), generator=g, device="cuda")) / (60 * k ** 0.25))


def weight_of(n, k, seed):
    from gemmlib_b200.fp8_linear import Fp8Weight

    g = torch.Generator(device="cuda").manual_seed(seed)
    return Fp8Weight(values(n, k, g), torch.exp(0.5 * torch.randn(-(-n // 128), -(-k // 128), generator=g, device="cuda")) / (60 * k ** 0.25))


def real(q, high=1):
    n, k = q.values.shape[-2:]
    s = q.scales.double().repeat_interleave(128, -1)[..., :k]
    return q.values.double() * (s if high == 1 else s.repeat_interleave(high, -2)[..., :n, :])


def check_close(got, x, w, bias=None):
    a, b = real(x), real(w, 128)
    want, magnitude = a @ b.t(), a.abs() @ b.abs().t()
    if bias is not None:
        want, magnitude = want + bias.double(), magnitude + bias.double().abs()
    k = a.size(1)
    half = torch.finfo(got.dtype).eps / 2
    smallest = 2.0 ** -25 if got.dtype == torch.float16 else 2.0 ** -134
    bound = want.abs() * half * (1 + 1e-3) + smallest + (128 + -(-k // 128) + 8) * 2.0 ** -23 * magnitude
    off = (got.double() - want).abs()
    assert (off <= bound).all(), (float((off / bound).max()), int((off > bound).sum()))


SHAPES = [  # rows, in_features, out_features: tiles and steps that end inside, one to many rows, K split or not
    (1, 1, 1), (1, 16, 8), (1, 500, 3001), (2, 512, 777), (1, 4096, 4096), (2, 4096, 1000), (3, 5001, 70), (1, 20000, 300), (7, 5001, 129), (8, 8192, 256),
    (15, 129, 127), (16, 256, 64), (17, 1000, 1237), (31, 2048, 384), (33, 640, 2048), (64, 4096, 512), (65, 127, 100), (100, 11008, 96), (127, 384, 641),
    (128, 1024, 1024), (129, 1024, 136), (200, 2000, 520), (255, 130, 300), (256, 512, 256), (257, 512, 513), (300, 4096, 768), (333, 5001, 1237),
    (512, 256, 1024), (513, 1040, 264), (1000, 136, 2000), (1024, 1024, 1024), (2048, 2048, 1536), (1500, 704, 3000), (4097, 64, 520), (20000, 48, 24),
    (48, 8192, 28672), (1000, 1, 1000),
]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_product(shape, dtype):
    from gemmlib_b200.fp8_linear import fp8_linear

    m, k, n = shape
    x, w = rows_of(m, k, 1), weight_of(n, k, 2)
    out = fp8_linear(x, w, dtype=dtype)
    assert out.shape == (m, n) and out.dtype == dtype
    check_close(out, x, w)
    bias = torch.linspace(-3, 3, n, device="cuda").to(dtype)
    check_close(fp8_linear(x, w, bias, dtype=dtype), x, w, bias)
    assert torch.equal(fp8_linear(x, w, dtype=dtype), out)  # the same every time


@pytest.mark.parametrize("m,k,n", [(3, 300, 200), (40, 4096, 201), (200, 1000, 513), (700, 512, 520), (1300, 640, 3000)])
def test_strided_operands_and_output(m, k, n):
    from gemmlib_b200.fp8_linear import Fp8Rows, Fp8Weight, fp8_linear

    x, w = rows_of(m, k, 3), weight_of(n, k, 4)
    want = fp8_linear(x, w)
    kb, pitch = x.scales.size(1), -(-k // 16) * 16
    wide = torch.full((m, pitch + 48), 0x7f, dtype=torch.uint8, device="cuda").view(E4M3)[:, 16:16 + k]
    wide.copy_(x.values)
    scales = torch.full((m, kb + 5), float("nan"), device="cuda")[:, 2:2 + kb]
    scales.copy_(x.scales)
    w_scales = torch.full((w.scales.size(0), kb + 3), float("nan"), device="cuda")[:, 3:]
    w_scales.copy_(w.scales)
    assert torch.equal(fp8_linear(Fp8Rows(wide, scales), Fp8Weight(w.values, w_scales)), want)
    # rows that begin anywhere are laid out first, transposed scales copied
    odd = torch.empty(m, k + 1, dtype=torch.uint8, device="cuda").view(E4M3)[:, 1:]
    odd.copy_(x.values)
    assert torch.equal(fp8_linear(Fp8Rows(odd, x.scales.t().contiguous().t()), w), want)
    # every second row
    two = torch.empty(2 * m, pitch, dtype=torch.uint8, device="cuda").view(E4M3)[::2, :k]
    two.copy_(x.values)
    assert torch.equal(fp8_linear(Fp8Rows(two, x.scales), w), want)
    for at, room in ((0, 0), (3, 8), (8, 24)):
        held = torch.full((m, n + room), 7.0, dtype=torch.float16, device="cuda")
        out = held[:, at:at + n]
        assert fp8_linear(x, w, out=out).data_ptr() == out.data_ptr()
        assert torch.equal(out, want) and (held[:, :at] == 7).all() and (held[:, at + n:] == 7).all()
    shaped = fp8_linear(Fp8Rows(x.values.unsqueeze(0), x.scales.unsqueeze(0)), w)
    assert shaped.shape == (1, m, n) and torch.equal(shaped[0], want)


@pytest.mark.parametrize("m", [1, 20, 300, 1500])
def test_nan_scales_and_values_stay_where_they_belong(m):
    from gemmlib_b200.fp8_linear import Fp8Rows, Fp8Weight, fp8_linear

    k, n = 1000, 700
    x, w = rows_of(m, k, 5), weight_of(n, k, 6)
    want = fp8_linear(x, w)
    scales = x.scales.clone()
    scales[m - 1, 3] = float("nan")
    got = fp8_linear(Fp8Rows(x.values, scales), w)
    assert got[m - 1].isnan().all() and torch.equal(got[:m - 1], want[:m - 1])
    w_scales = w.scales.clone()
    w_scales[2, 7] = float("nan")
    got = fp8_linear(x, Fp8Weight(w.values, w_scales))
    spoiled = torch.zeros(n, dtype=torch.bool, device="cuda")
    spoiled[256:384] = True
    assert torch.equal(got.isnan().all(0), spoiled) and torch.equal(got[:, ~spoiled], want[:, ~spoiled])
    spoiled_weight = weight_of(n, k, 6)
    spoiled_weight.values.view(torch.uint8)[5, 77] = 0x7f  # e4m3's own NaN
    got = fp8_linear(x, spoiled_weight)
    assert got[:, 5].isnan().all() and torch.equal(got[:, :5], want[:, :5]) and torch.equal(got[:, 6:], want[:, 6:])


@pytest.mark.parametrize("m", [1, 30, 400])
def test_overflowing_results_are_infinite(m):
    from gemmlib_b200.fp8_linear import Fp8Rows, Fp8Weight, fp8_linear

    x = Fp8Rows(torch.full((m, 256), 448.0, device="cuda").to(E4M3), torch.ones(m, 2, device="cuda"))
    w = Fp8Weight(torch.full((130, 256), 448.0, device="cuda").to(E4M3), torch.ones(2, 2, device="cuda"))
    assert (fp8_linear(x, w) == float("inf")).all()
    assert torch.equal(fp8_linear(x, w, dtype=torch.bfloat16), torch.full((m, 130), 448.0 ** 2 * 256, device="cuda").bfloat16())
    assert (fp8_linear(Fp8Rows(x.values, torch.zeros_like(x.scales)), w) == 0).all()


def test_refusals():
    from gemmlib_b200.fp8_linear import Fp8Rows, Fp8Weight, fp8_linear

    x, w = rows_of(4, 256, 1), weight_of(200, 256, 2)
    cases = [
        (lambda: fp8_linear(x, weight_of(200, 240, 2)), "in_features"),
        (lambda: fp8_linear(Fp8Rows(x.values, x.scales[:, :1]), w), "of shape"),
        (lambda: fp8_linear(x, Fp8Weight(w.values, w.scales[:1])), "of shape"),
        (lambda: fp8_linear(x, Fp8Weight(w.values[:, 1:], w.scales)), "in_features|16 bytes"),
        (lambda: fp8_linear(rows_of(4, 255, 1), Fp8Weight(w.values[:, 1:], w.scales)), "16 bytes"),
        (lambda: fp8_linear(x, w, torch.zeros(199, dtype=torch.float16, device="cuda")), "bias"),
        (lambda: fp8_linear(x, w, torch.zeros(200, dtype=torch.bfloat16, device="cuda")), "bias"),
        (lambda: fp8_linear(x, w, out=torch.zeros(4, 199, dtype=torch.float16, device="cuda")), "out must have"),
        (lambda: fp8_linear(x, w, out=torch.zeros(4, 200, dtype=torch.bfloat16, device="cuda")), "out must have"),
        (lambda: fp8_linear(x, w, out=torch.zeros(200, 4, dtype=torch.float16, device="cuda").t()), "contiguous rows"),
        (lambda: fp8_linear(x, w, out=x.scales.view(torch.float16)[:, :1].expand(4, 200)), "contiguous rows"),
        (lambda: fp8_linear(x, Fp8Weight(w.values.cpu(), w.scales)), "device|CUDA"),
    ]
    for call, text in cases:
        with pytest.raises(RuntimeError, match=text):
            call()
    buffer = torch.zeros(200 * 256, dtype=torch.uint8, device="cuda")
    inside = Fp8Weight(buffer.view(E4M3).view(200, 256), w.scales)
    with pytest.raises(RuntimeError, match="overlaps"):
        fp8_linear(x, inside, out=buffer.view(torch.float16)[:800].view(4, 200))
    assert fp8_linear(Fp8Rows(x.values[:0], x.scales[:0]), w).shape == (0, 200)


@pytest.mark.parametrize("m", [1, 24, 64, 700])
def test_streams_and_graphs(m):
    """Calls beside each other, captured first calls, the early fetch of weights: the same bits."""
    from gemmlib_b200 import ms_blkq4linear_ext as ext
    from gemmlib_b200.fp8_linear import fp8_linear

    problems = [(rows_of(m, k, i), weight_of(n, k, 10 + i)) for i, (k, n) in enumerate([(4096, 1408), (1408, 4096), (2048, 2048), (5001, 333)])]
    want = [fp8_linear(x, w) for x, w in problems]
    streams = [torch.cuda.Stream() for _ in problems]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, (x, w) in zip(streams, problems):
            with torch.cuda.stream(s):
                got.append([fp8_linear(x, w, flags=ext.EARLY_WEIGHT_FETCH) for _ in range(4)])
        torch.cuda.synchronize()
        assert all(torch.equal(o, t) for o4, t in zip(got, want) for o in o4)
    graphs = []
    for x, w in problems:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = [fp8_linear(x, w) for _ in range(3)]
        graphs.append((g, out))
    for _ in range(3):
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, t) for (_, out), t in zip(graphs, want) for o in out)
    from gemmlib_b200 import capi

    assert capi.last_kernel_status() == 0


def test_early_fetch_sees_weights_that_are_written_ahead_of_the_kernel_before():
    """w -> quantization -> a product of other tensors -> the product of w with the early fetch."""
    from gemmlib_b200 import ms_blkq4linear_ext as ext
    from gemmlib_b200.fp8_linear import fp8_linear, quantize_fp8, quantize_fp8_weight

    g = torch.Generator(device="cuda").manual_seed(1)
    x = quantize_fp8(torch.randn(4, 2048, generator=g, device="cuda").half())
    other = weight_of(512, 2048, 3)
    for seed in range(5):
        w16 = torch.randn(1024, 2048, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").half()
        w = quantize_fp8_weight(w16)
        fp8_linear(x, other)
        got = fp8_linear(x, w, flags=ext.EARLY_WEIGHT_FETCH)
        torch.cuda.synchronize()
        assert torch.equal(got, fp8_linear(x, w))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("bias", [False, True])
def test_module(dtype, bias):
    import copy

    from gemmlib_b200.fp8_linear import Fp8Linear, Fp8Weight, fp8_linear, quantize_fp8, quantize_fp8_weight

    g = torch.Generator(device="cuda").manual_seed(4)
    n, k = 333, 1000
    w = (torch.randn(n, k, generator=g, device="cuda") / 30).to(dtype)
    b = torch.randn(n, generator=g, device="cuda").to(dtype) if bias else None
    layer = Fp8Linear(w, b)
    x = torch.randn(2, 5, k, generator=g, device="cuda").to(dtype)
    rows, weight = quantize_fp8(x), quantize_fp8_weight(w)
    want = fp8_linear(rows, weight, b, dtype=dtype)
    for _ in range(3):  # the first one is a plain launch
        assert torch.equal(layer(x), want) and torch.equal(layer(rows), want)
    out = torch.empty(2, 5, n, dtype=dtype, device="cuda")
    assert layer(rows, out=out) is not None and torch.equal(out, want)
    for other in (Fp8Linear.from_weight(weight, b, dtype), copy.deepcopy(layer)):
        assert torch.equal(other(x), want)
    given = Fp8Weight(weight.values.t().contiguous().t(), weight.scales.t().contiguous().t())
    kept = Fp8Linear.from_weight(given, b, dtype)
    given.values.view(torch.uint8).zero_()
    assert torch.equal(kept(x), want)
    state = layer.state_dict()
    fresh = Fp8Linear(torch.zeros_like(w), b)
    fresh.load_state_dict(state)
    assert torch.equal(fresh(x), want)
    moved = copy.deepcopy(layer).cpu().cuda()
    assert torch.equal(moved(x), want) and moved.half().q_scales.dtype == torch.float32 and moved.q_weights.dtype == E4M3


def test_layers_in_a_stack():
    """Beside int8 and 4-bit layers, sharing a buffer's rows, with rows from a gate."""
    from gemmlib_b200.fp8_linear import Fp8Linear, silu_mul_fp8
    from gemmlib_b200.int8_linear import Int8Linear
    from gemmlib_b200.ms_blkq4linear import BlkQ4Linear
    from gemmlib_b200.stack import LinearStack

    g = torch.Generator(device="cuda").manual_seed(5)
    h, f = 512, 768
    make = lambda n, k: (torch.randn(n, k, generator=g, device="cuda") / k ** 0.5).half()  # noqa: E731
    q, gate, up, down = Fp8Linear(make(h, h)), Fp8Linear(make(f, h)), Fp8Linear(make(f, h)), Fp8Linear(make(h, f))
    four, eight = BlkQ4Linear(64, True, True, make(h, h), None), Int8Linear(make(h, h))
    steps = [(four, "x", "a"), (q, "a", "b"), (eight, "a", "i"), (gate, "b", "gate"), (up, "b", "up"), (down, "gate", "down")]
    stack = LinearStack(steps, fp8_inputs={5: lambda bufs: silu_mul_fp8(bufs["gate"], bufs["up"])})
    with pytest.raises(ValueError, match="no Fp8Linear"):
        LinearStack(steps, fp8_inputs={2: lambda bufs: None})
    for m in (1, 20, 300):
        x = torch.randn(m, h, generator=g, device="cuda").half()
        got = stack.forward(x, "down").clone()
        a = four(x)
        b = q(a)
        want = down(silu_mul_fp8(gate(b), up(b)))
        assert torch.equal(stack.buffers(m)["i"], eight(a)) and torch.equal(got, want)
    assert stack.weight_bytes() > 0
