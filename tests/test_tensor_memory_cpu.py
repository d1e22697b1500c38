"""Which kernels can stand on one SM: those whose tensor memory does not fit together must not fit together in shared memory, or
two clusters of different streams can wait for each other's columns for good."""
import random

SM, RESERVED = 228 * 1024, 1024  # shared memory of an SM, what of it is the system's for each CTA
# of the 4-bit tensor-core kernels the one that asks for the least: up to 16 rows, all 512 columns.  Six stages of activations, twelve
# of packed weights with scales and zero points, barriers, alignment.
SKINNY = 6 * 4096 + 12 * (8192 + 512 + 256) + 512 + 1024


def columns(tile_m):
    c = 32
    while c < tile_m:
        c *= 2
    return c


def test_int8_products_share_an_sm_only_where_their_tensor_memory_does(lib_built):
    from gemmlib_b200 import capi

    rng = random.Random(1)
    size = lambda top: round(2 ** rng.uniform(0, top))
    shapes = [(51, 14697, 16802), (275, 11849, 25)] + [(size(10), size(15), size(15)) for _ in range(5000)]
    seen = set()
    for m, n, k in shapes:
        p = capi.int8_gemm_plan(m, n, k)
        seen.add(p["kernel"])
        if p["kernel"] == "stream":
            continue
        taken = 512 if p["kernel"] == "pair" else columns(p["tile_m"])
        for others in (1, 2):  # further CTAs of the same kind
            fits = (others + 1) * (p["smem"] + RESERVED) <= SM
            assert not fits or (others + 1) * taken <= 512, (m, n, k, p)
        assert p["smem"] + SKINNY + 2 * RESERVED > SM, (m, n, k, p)
    assert seen == {"stream", "one-cta", "pair"}
