"""The 8-bit path without a GPU: the C entry points' checks of their arguments, and the extension's."""
import ctypes
import os
import re

import pytest

from tests._util import ROOT

torch = pytest.importorskip("torch")


def test_symbols_match_the_header(lib_built):
    from gemmlib_b200 import capi

    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "ms_blkq4gemm.h")).read(), flags=re.S)
    declared = sorted(set(re.findall(r"\b(int8_\w+)\s*\(", text)))
    assert sorted(capi.INT8_SYMBOLS) == declared
    lib = ctypes.CDLL(lib_built)
    for s in declared:
        assert hasattr(lib, s)


# never dereferenced: every call below is refused before a launch
P = 1 << 20


def quant_args(**other):
    a = dict(dtype=0, rows=4, cols=40, x=(P, 4 * 40 * 2), ldx=40, values=(P, 3 * 48 + 40), ldv=48, scales=(P, 16))
    return {**a, **other}


@pytest.mark.parametrize("change,text", [
    ({"dtype": 2}, "Unsupported type: 2"),
    ({"rows": 0}, "Empty problem size: 0x40"),
    ({"cols": -1}, "Empty problem size"),
    ({"cols": (1 << 28) + 1}, "Too many columns"),
    ({"x": (0, 320)}, "Null tensor pointer: x"),
    ({"x": (P + 1, 320)}, "Misaligned tensor: x"),
    ({"x": (P, 319)}, "Unexpected size of x: 319 expected: 320"),
    ({"ldx": 39}, "Leading dimension of x is smaller"),
    ({"ldx": -40}, "Leading dimension of x is smaller"),
    ({"ldx": 1 << 62}, "Leading dimension of x is out of range"),
    ({"ldx": 41}, "Unexpected size of x"),
    ({"values": (P, 3 * 48 + 39)}, "Unexpected size of values"),
    ({"values": (0, 0)}, "Null tensor pointer: values"),
    ({"scales": (P, 15)}, "Unexpected size of scales: 15 expected: 16"),
    ({"scales": (P + 2, 16)}, "Misaligned tensor: scales"),
])
def test_quant_refusals(lib_built, change, text):
    from gemmlib_b200 import capi

    a = quant_args(**change)
    with pytest.raises(capi.BlkQ4Error, match=re.escape(text)):
        capi.int8_rows_quant(a["dtype"], a["rows"], a["cols"], (a["x"], a["ldx"]), (a["values"], a["ldv"]), a["scales"])


@pytest.mark.parametrize("change,text", [
    ({"weight": (P, 79)}, "Unexpected size of weight"),
    ({"weight": None}, "Null tensor pointer: weight"),
    ({"eps": -1e-5}, "eps must not be negative"),
    ({"eps": float("nan")}, "eps must not be negative"),
    ({"residual": ((P, 320), 40)}, "Null tensor pointer: residual_out"),
    ({"residual": ((P, 318), 40), "residual_out": ((P, 320), 40)}, "Unexpected size of residual"),
    ({"residual": ((2 * P, 1000), 40), "residual_out": ((2 * P, 1000), 48)}, "must have its leading dimension"),
    ({"residual": ((2 * P, 1000), 40), "residual_out": ((P, 1000), 48)}, "must have its leading dimension"),
])
def test_norm_refusals(lib_built, change, text):
    from gemmlib_b200 import capi

    a = {"weight": (P, 80), "eps": 1e-5, "residual": None, "residual_out": None, **change}
    with pytest.raises(capi.BlkQ4Error, match=re.escape(text)):
        capi.int8_rows_rms_norm(0, 4, 40, ((P, 320), 40), a["residual"], a["weight"], a["eps"], a["residual_out"],
                                ((P, 192), 48), (P, 16))


def test_silu_mul_and_dequant_refusals(lib_built):
    from gemmlib_b200 import capi

    with pytest.raises(capi.BlkQ4Error, match="Unexpected size of up"):
        capi.int8_rows_silu_mul(1, 4, 40, ((P, 320), 40), ((P, 300), 40), ((P, 192), 48), (P, 16))
    with pytest.raises(capi.BlkQ4Error, match="Unexpected size of out"):
        capi.int8_rows_dequant(1, 4, 40, ((P, 192), 48), (P, 16), ((P, 318), 40))


def gemm_args(**other):
    return {**dict(dtype=0, m=3, n=5, k=40, x=(P, 3 * 48), ldx=48, xs=(P, 12), w=(P, 5 * 48), ldw=48, ws=(P, 20), bias=None,
                   out=(P, 30), ldo=5), **other}


@pytest.mark.parametrize("change,text", [
    ({"dtype": -1}, "Unsupported type: -1"),
    ({"k": 0}, "Empty problem size: 3x5x0"),
    ({"k": 131072}, "int32 sums hold up to 131071 k"),
    ({"m": (1 << 28) + 1}, "Too many rows"),
    ({"x": (P + 8, 200)}, "must begin on 16 bytes"),
    ({"w": (P + 8, 300)}, "must begin on 16 bytes"),
    ({"ldx": 40, "x": (P, 200)}, "must begin on 16 bytes"),
    ({"ldw": 40}, "must begin on 16 bytes"),
    ({"x": (P, 2 * 48 + 39)}, "Unexpected size of x"),
    ({"w": (P, 4 * 48 + 39)}, "Unexpected size of w"),
    ({"xs": (P, 8)}, "Unexpected size of x_scales"),
    ({"ws": (P, 19)}, "Unexpected size of w_scales"),
    ({"bias": (P, 9)}, "Unexpected size of bias"),
    ({"out": (P, 29)}, "Unexpected size of out"),
    ({"ldo": 4}, "Leading dimension of out is smaller"),
])
def test_gemm_refusals(lib_built, change, text):
    from gemmlib_b200 import capi

    a = gemm_args(**change)
    with pytest.raises(capi.BlkQ4Error, match=re.escape(text)):
        capi.int8_gemm(a["dtype"], a["m"], a["n"], a["k"], (a["x"], a["ldx"]), a["xs"], (a["w"], a["ldw"]), a["ws"], a["bias"],
                       (a["out"], a["ldo"]))


def test_a_refusal_without_a_place_for_its_text(lib_built):
    from gemmlib_b200 import capi

    assert capi.lib.int8_rows_quant_sm100(0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, None) == -1


def test_extension_refuses_cpu_tensors_and_wrong_types():
    from gemmlib_b200.int8_linear import Int8Rows, int8_linear, quantize_int8, rms_norm_int8, silu_mul_int8

    x = torch.zeros(2, 32, dtype=torch.float16)
    q = Int8Rows(torch.zeros(2, 32, dtype=torch.int8), torch.ones(2))
    for call in (lambda: quantize_int8(x), lambda: rms_norm_int8(x, x[0]), lambda: silu_mul_int8(x, x), q.dequantize,
                 lambda: int8_linear(q, q)):
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            call()
    for call in (lambda: quantize_int8(x.float()), lambda: rms_norm_int8(x.double(), x[0]), lambda: silu_mul_int8(q.values, x),
                 lambda: q.dequantize(torch.float32), lambda: int8_linear(q, q, dtype=torch.float32)):
        with pytest.raises(RuntimeError, match="must be float16 or bfloat16"):
            call()
    with pytest.raises(RuntimeError, match="must be int8"):
        int8_linear(Int8Rows(x, torch.ones(2)), q)
    with pytest.raises(RuntimeError, match="no backward pass"):
        quantize_int8(x.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="one shape and type"):
        silu_mul_int8(x, x[:1])
    with pytest.raises(RuntimeError, match="residual_out without a residual"):
        rms_norm_int8(x, x[0], residual_out=x)
    with pytest.raises(TypeError, match="a tensor is wanted"):
        quantize_int8(None)


def test_plans_cover_k_and_fit_on_an_sm(lib_built):
    """Sizes from one to the largest: every part of K has steps, the stages a round of them, and the shared memory its place
    (227 KB a CTA, and two of 110 KB with their barriers on an SM)."""
    import random

    from gemmlib_b200 import capi

    rng = random.Random(0)
    size = lambda top: round(2 ** rng.uniform(0, top))
    seen = set()
    for _ in range(5000):
        m, n, k = size(14), size(16), min(131071, size(17))
        p = capi.int8_gemm_plan(m, n, k)
        seen.add(p["kernel"])
        steps = -(-k // 128)
        if p["kernel"] == "stream":
            assert m <= 4
            continue
        assert p["smem"] <= 227 * 1024 and p["stages"] >= 3
        assert p["tiles"] == -(-m // p["tile_m"]) * -(-n // p["tile_n"])
        assert (p["split"] - 1) * p["steps"] < steps <= p["split"] * p["steps"]
        if p["kernel"] == "one-cta":
            assert p["tile_m"] % 16 == 0 and 16 <= p["tile_m"] <= 256 and p["tile_n"] == 128
            rows = min(m, p["tile_m"])
            collected = (p["split"] - 1) * (-(-(-(-rows // p["split"])) // 8) * 8) * 512 if p["split"] > 1 else 0
            assert p["smem"] >= p["stages"] * (128 + p["tile_m"]) * 128 + collected + 1536
            assert p["split"] == 1 or p["tiles"] * p["split"] <= 2 * 148
        else:
            assert p["tile_m"] == 256 and p["tile_n"] % 32 == 0 and 128 <= p["tile_n"] <= 256
    assert seen == {"stream", "one-cta", "pair"}


@pytest.mark.parametrize("m,n,k", [(0, 1, 1), (1, 0, 1), (1, 1, 0), (1, 1, 131072), (1 << 29, 1, 1)])
def test_plans_that_there_are_none_of(lib_built, m, n, k):
    from gemmlib_b200 import capi

    with pytest.raises(capi.BlkQ4Error):
        capi.int8_gemm_plan(m, n, k)
