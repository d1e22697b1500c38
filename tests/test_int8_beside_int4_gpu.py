"""The int8 product and the 4-bit kernels at work at the same time, on streams of their own: clusters of both wait for shared memory,
tensor memory and each other's CTAs, and both end with the results that they have alone."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def test_products_on_three_streams():
    from gemmlib_b200 import capi
    from gemmlib_b200.int8_linear import Int8Rows, int8_linear
    from gemmlib_b200.ms_blkq4linear import BlkQ4Linear

    g = torch.Generator(device="cuda").manual_seed(0)

    def rows(n, k):
        pitch = -(-k // 32) * 32
        v = torch.randint(-127, 128, (n, pitch), generator=g, device="cuda", dtype=torch.int8)[:, :k]
        return Int8Rows(v, torch.rand(n, generator=g, device="cuda") / 1000)

    # tiles of 48 to 112 rows in one to four parts, some of which leave an SM room for a second CTA; pairs of CTAs
    eight = [(rows(m, k), rows(n, k)) for m, k, n in ((51, 4096, 14697), (64, 4096, 4096), (100, 2048, 8192), (275, 512, 11849),
                                                     (16, 8192, 512), (600, 1024, 4096))]
    # up to 16 rows in parts (all of an SM's tensor memory), and prompts
    four = []
    for m, k, n in ((16, 4096, 4096), (8, 8192, 1024), (40, 4096, 4096), (300, 2048, 4096)):
        for block in (64, 128):
            w = (torch.randn(n, k, generator=g, device="cuda") * 0.02).half()
            four.append((BlkQ4Linear(block, True, False, w), torch.randn(m, k, generator=g, device="cuda").half()))
    want8 = [int8_linear(x, w) for x, w in eight]
    want4 = [layer(x) for layer, x in four]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got8, got4 = [], []
    for turn in range(12):
        for i in range(max(len(eight), len(four))):
            with torch.cuda.stream(streams[0]):
                got8.append((i % len(eight), int8_linear(*eight[i % len(eight)])))
            with torch.cuda.stream(streams[1]):
                layer, x = four[(i + turn) % len(four)]
                got4.append(((i + turn) % len(four), layer(x)))
            with torch.cuda.stream(streams[2]):
                j = (i + turn) % len(eight)
                got8.append((j, int8_linear(*eight[j])))
    torch.cuda.synchronize()
    for i, y in got8:
        assert torch.equal(y, want8[i]), i
    for i, y in got4:
        assert torch.equal(y, want4[i]), i
    assert capi.last_kernel_status() == 0
