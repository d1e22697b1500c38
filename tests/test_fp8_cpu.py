"""The 8-bit floating-point path and layers of experts without a GPU: the C entry points' checks of their arguments, the extension's, and the
plans."""
import ctypes
import os
import random
import re

import pytest

from tests._util import ROOT

torch = pytest.importorskip("torch")


def test_symbols_match_the_header(lib_built):
    from gemmlib_b200 import capi

    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "ms_blkq4gemm.h")).read(), flags=re.S)
    for prefix, symbols in (("fp8", capi.FP8_SYMBOLS), ("experts", capi.EXPERTS_SYMBOLS)):
        declared = sorted(set(re.findall(r"\b(%s_\w+)\s*\(" % prefix, text)))
        assert sorted(symbols) == declared
        for s in declared:
            assert hasattr(ctypes.CDLL(lib_built), s)


# never dereferenced: every call below is refused before a launch
P = 1 << 20


def refused(call, text):
    from gemmlib_b200 import capi

    with pytest.raises(capi.BlkQ4Error, match=re.escape(text)):
        call(capi)


@pytest.mark.parametrize("change,text", [
    ({"dtype": 2}, "Unsupported type: 2"),
    ({"rows": 0}, "Empty problem size: 0x200"),
    ({"rows": (1 << 28) + 1}, "Too many rows"),
    ({"cols": (1 << 28) + 1}, "Too many columns"),
    ({"x": ((0, 1600), 200)}, "Null tensor pointer: x"),
    ({"x": ((P + 1, 1600), 200)}, "Misaligned tensor: x"),
    ({"x": ((P, 1599), 200)}, "Unexpected size of x: 1599 expected: 1600"),
    ({"x": ((P, 1600), 199)}, "Leading dimension of x is smaller"),
    ({"values": ((P, 3 * 224 + 199), 224)}, "Unexpected size of values"),
    ({"scales": ((P, 31), 2)}, "Unexpected size of scales: 31 expected: 32"),
    ({"scales": ((P, 32), 1)}, "Leading dimension of scales is smaller"),
    ({"scales": ((P + 2, 32), 2)}, "Misaligned tensor: scales"),
])
def test_rows_refusals(lib_built, change, text):
    a = {**dict(dtype=0, rows=4, cols=200, x=((P, 1600), 200), values=((P, 3 * 224 + 200), 224), scales=((P, 32), 2)), **change}
    refused(lambda c: c.fp8_rows_quant(*a.values()), text)
    if "x" not in change:
        refused(lambda c: c.fp8_rows_silu_mul(a["dtype"], a["rows"], a["cols"], a["x"], a["x"], a["values"], a["scales"]), text)


@pytest.mark.parametrize("change,text", [
    ({"experts": 0}, "Empty problem size: 0 experts"),
    ({"n": 1 << 28}, "Too many weight rows"),
    ({"w": ((P, 2 * 130 * 200 * 2 - 1), 200)}, "Unexpected size of w"),
    ({"values": ((P, 259 * 224 + 199), 224)}, "Unexpected size of values"),
    ({"scales": ((P, 31), 2)}, "Unexpected size of scales"),
])
def test_weight_refusals(lib_built, change, text):
    a = {**dict(dtype=1, experts=2, n=130, k=200, w=((P, 2 * 130 * 200 * 2), 200), values=((P, 259 * 224 + 200), 224), scales=((P, 32), 2)), **change}
    refused(lambda c: c.fp8_weight_quant(*a.values()), text)
    if "w" not in change:
        refused(lambda c: c.fp8_weight_dequant(a["dtype"], a["experts"], a["n"], a["k"], a["values"], a["scales"], a["w"]), text)


GEMM = dict(dtype=0, m=3, n=130, k=200, x=((P, 2 * 208 + 200), 208), xs=((P, 24), 2), w=((P, 129 * 208 + 200), 208), ws=((P, 16), 2), bias=None,
            out=((P, 780), 130))


@pytest.mark.parametrize("change,text", [
    ({"dtype": -1}, "Unsupported type: -1"),
    ({"k": 0}, "Empty problem size"),
    ({"m": (1 << 28) + 1}, "Too many rows"),
    ({"x": ((P + 8, 1000), 208)}, "must begin on 16 bytes"),
    ({"w": ((P, 1 << 20), 200)}, "must begin on 16 bytes"),
    ({"x": ((P, 615), 208)}, "Unexpected size of x"),
    ({"xs": ((P, 23), 2)}, "Unexpected size of x_scales"),
    ({"ws": ((P, 15), 2)}, "Unexpected size of w_scales"),
    ({"bias": (P, 259)}, "Unexpected size of bias"),
    ({"out": ((P, 779), 130)}, "Unexpected size of out"),
])
def test_gemm_refusals(lib_built, change, text):
    refused(lambda c: c.fp8_gemm(*{**GEMM, **change}.values()), text)


EXPERTS = dict(dtype=0, experts=3, rows=5, n=130, k=200, x=((P, 4 * 208 + 200), 208), xs=((P, 40), 2), w=((P, 3 * 130 * 208), 208),
               w_stride=130 * 208, ws=((P, 48), 2), ws_stride=4, offsets=(P, 16), out=((P, 1300), 130))


@pytest.mark.parametrize("change,text", [
    ({"experts": 0}, "Empty problem size: 0 experts"),
    ({"experts": 1025, "offsets": (P, 1026 * 4)}, "Up to 1024 experts"),
    ({"offsets": (P, 15)}, "Unexpected size of offsets"),
    ({"offsets": None}, "Null tensor pointer: offsets"),
    ({"w_stride": 130 * 208 + 8, "w": ((P, 1 << 20), 208)}, "must begin on 16 bytes"),
    ({"w_stride": 0}, "Stride of w is smaller"),
    ({"w_stride": 1 << 61}, "Stride of w is smaller than an expert, or out of range"),
    ({"w": ((P, 2 * 130 * 208 + 129 * 208 + 199), 208)}, "Unexpected size of w"),
    ({"ws": ((P, 47), 2)}, "Unexpected size of w_scales"),
    ({"ws_stride": 3}, "Stride of w_scales is smaller"),
])
def test_experts_gemm_refusals(lib_built, change, text):
    refused(lambda c: c.fp8_experts_gemm(*{**EXPERTS, **change}.values()), text)


@pytest.mark.parametrize("change,text", [
    ({"n": 0}, "Empty problem size: 0 choices"),
    ({"n": (1 << 28) + 1}, "Too many choices"),
    ({"n_experts": 1025, "offsets": (P, 1 << 20)}, "Up to 1024 experts"),
    ({"id_bytes": 2}, "Unsupported type of ids: 2 bytes"),
    ({"ids": (P, 79)}, "Unexpected size of ids"),
    ({"ids": (P + 4, 80)}, "Misaligned tensor: ids"),
    ({"source": (P, 39)}, "Unexpected size of source"),
    ({"places": None}, "Null tensor pointer: places"),
    ({"offsets": (P, 15)}, "Unexpected size of offsets"),
])
def test_sort_refusals(lib_built, change, text):
    a = {**dict(n=10, n_experts=3, id_bytes=8, ids=(P, 80), source=(P, 40), places=(P, 40), offsets=(P, 16)), **change}
    refused(lambda c: c.experts_sort(*a.values()), text)


def test_a_large_sort_wants_its_workspace(lib_built):
    from gemmlib_b200 import capi

    n = 1 << 20
    need = capi.lib.experts_sort_workspace_size(n, 64)
    assert need > 0 and capi.lib.experts_sort_workspace_size(8, 64) == 0
    assert capi.lib.experts_sort_workspace_size(n, 0) == 0 and capi.lib.experts_sort_workspace_size(n, 1025) == 0
    big = (P, 4 * n)
    refused(lambda c: c.experts_sort(n, 64, 4, big, big, big, (P, 260), (P, need - 1)), "Unexpected size of workspace")


@pytest.mark.parametrize("change,text", [
    ({"choices": 0}, "Empty problem size: 0 choices"),
    ({"tokens": 1 << 20, "choices": 1 << 10}, "Too many choices"),
    ({"source": (P, 23)}, "Unexpected size of source"),
    ({"count": 0}, "Null tensor pointer: count"),
    ({"count": P + 1}, "Misaligned tensor: count"),
    ({"out": ((P, 479), 40)}, "Unexpected size of out"),
])
def test_gather_refusals(lib_built, change, text):
    a = {**dict(dtype=0, tokens=3, choices=2, cols=40, x=((P, 240), 40), source=(P, 24), count=P, out=((P, 480), 40)), **change}
    refused(lambda c: c.experts_gather(*a.values()), text)


@pytest.mark.parametrize("change,text", [
    ({"y": ((P, 479), 40)}, "Unexpected size of y"),
    ({"places": (P, 20)}, "Unexpected size of places"),
    ({"weights": (P, 23)}, "Unexpected size of weights"),
    ({"weights_type": 3}, "Unsupported type of weights: 3"),
    ({"out": ((P, 239), 40)}, "Unexpected size of out"),
])
def test_combine_refusals(lib_built, change, text):
    a = {**dict(dtype=0, tokens=3, choices=2, cols=40, y=((P, 480), 40), places=(P, 24), weights=(P, 24), weights_type=2, out=((P, 240), 40)), **change}
    refused(lambda c: c.experts_combine(*a.values()), text)
    if "places" not in change and "out" not in change:
        refused(lambda c: c.experts_combine_backward(0, 3, 2, 40, ((P, 240), 40), a["y"], a["weights"], a["weights_type"], (P, 24), P, ((P, 480), 40),
                                                     (P, 24)), text)


def test_a_refusal_without_a_place_for_its_text(lib_built):
    from gemmlib_b200 import capi

    assert capi.lib.fp8_rows_quant_sm100(0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, None) == -1
    assert capi.lib.fp8_gemm_plan_sm100(0, 0, 1, 1, (ctypes.c_int * 8)()) == -1
    assert capi.lib.fp8_gemm_plan_sm100(0, 1, 1, 1, None) == -1


def rows(*shape):
    from gemmlib_b200.fp8_linear import Fp8Rows

    return Fp8Rows(torch.zeros(*shape, dtype=torch.float8_e4m3fn), torch.ones(*shape[:-1], -(-shape[-1] // 128)))


def weight(*shape):
    from gemmlib_b200.fp8_linear import Fp8Weight

    return Fp8Weight(torch.zeros(*shape, dtype=torch.float8_e4m3fn), torch.ones(*shape[:-2], -(-shape[-2] // 128), -(-shape[-1] // 128)))


def order_of(tokens, choices, experts):
    from gemmlib_b200.experts import ExpertOrder

    i = torch.int32
    return ExpertOrder(torch.zeros(tokens * choices, dtype=i), torch.zeros(tokens, choices, dtype=i), torch.zeros(experts + 1, dtype=i))


def test_extension_refuses_cpu_tensors_and_wrong_types():
    from gemmlib_b200 import experts as E, fp8_linear as F

    x = torch.zeros(2, 32, dtype=torch.float16)
    offsets = torch.zeros(4, dtype=torch.int32)
    for call in (lambda: F.quantize_fp8(x), lambda: F.quantize_fp8_weight(x), lambda: F.silu_mul_fp8(x, x), rows(2, 32).dequantize, weight(2, 32).dequantize,
                 lambda: F.fp8_linear(rows(2, 32), weight(3, 32)), lambda: E.fp8_expert_linear(rows(2, 32), weight(3, 8, 32), offsets),
                 lambda: E.sort_by_expert(torch.zeros(2, 2, dtype=torch.long), 3), lambda: E.gather_rows(x, order_of(2, 2, 3)),
                 lambda: E.combine_rows(x, order_of(1, 2, 3), torch.ones(1, 2))):
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            call()
    for call in (lambda: F.quantize_fp8(x.float()), lambda: F.quantize_fp8_weight(x.double()), lambda: F.silu_mul_fp8(x.float(), x),
                 lambda: rows(2, 32).dequantize(torch.float32), lambda: F.fp8_linear(rows(2, 32), weight(3, 32), dtype=torch.float32),
                 lambda: E.gather_rows(x.float(), order_of(2, 2, 3))):
        with pytest.raises(RuntimeError, match="must be float16 or bfloat16"):
            call()
    for call in (lambda: F.fp8_linear(F.Fp8Rows(x, torch.ones(2, 1)), weight(3, 32)), lambda: F.Fp8Rows(x, torch.ones(2, 1)).dequantize()):
        with pytest.raises(RuntimeError, match="must be float8_e4m3fn"):
            call()
    with pytest.raises(RuntimeError, match="one shape and type"):
        F.silu_mul_fp8(x, x[:1])
    with pytest.raises(TypeError, match="a tensor is wanted"):
        F.quantize_fp8(None)


def calls():
    """Each call with one tensor that the argument makes."""
    from gemmlib_b200 import experts as E, fp8_linear as F

    x, scales, out = torch.zeros(2, 32, dtype=torch.float16), torch.ones(2, 1), torch.zeros(2, 2, dtype=torch.float16)
    offsets = torch.zeros(4, dtype=torch.int32)
    w, experts = weight(2, 32), weight(3, 2, 32)
    return {
        "quantize": (x, F.quantize_fp8),
        "weight": (x, F.quantize_fp8_weight),
        "gate": (x, lambda t: F.silu_mul_fp8(t, x)),
        "up": (x, lambda t: F.silu_mul_fp8(x, t)),
        "dequantized scales": (scales, lambda t: F.Fp8Rows(rows(2, 32).values, t).dequantize()),
        "scales": (scales, lambda t: F.fp8_linear(F.Fp8Rows(rows(2, 32).values, t), w)),
        "weight's scales": (torch.ones(1, 1), lambda t: F.fp8_linear(rows(2, 32), F.Fp8Weight(w.values, t))),
        "bias": (out[0], lambda t: F.fp8_linear(rows(2, 32), w, t)),
        "out": (out, lambda t: F.fp8_linear(rows(2, 32), w, out=t)),
        "experts' scales": (scales, lambda t: E.fp8_expert_linear(F.Fp8Rows(rows(2, 32).values, t), experts, offsets)),
        "experts' out": (out, lambda t: E.fp8_expert_linear(rows(2, 32), experts, offsets, out=t)),
    }


NAMES = ["quantize", "weight", "gate", "up", "dequantized scales", "scales", "weight's scales", "bias", "out", "experts' scales", "experts' out"]


def test_every_call_is_named():
    assert sorted(calls()) == sorted(NAMES)


@pytest.mark.parametrize("name", NAMES)
def test_tensors_that_require_a_gradient_or_have_a_tangent_are_refused(name):
    t, call = calls()[name]
    with pytest.raises(RuntimeError, match="no backward pass"):
        call(t.clone().requires_grad_())
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="no forward derivatives"):
            call(torch.autograd.forward_ad.make_dual(t.clone(), torch.ones_like(t)))


def test_moves_refuse_tangents():
    from gemmlib_b200 import experts as E

    x = torch.zeros(2, 32, dtype=torch.float16)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x.clone(), torch.ones_like(x))
        with pytest.raises(RuntimeError, match="no forward derivatives"):
            E.gather_rows(dual, order_of(2, 2, 3))
        with pytest.raises(RuntimeError, match="no forward derivatives"):
            E.combine_rows(dual, order_of(1, 2, 3), torch.ones(1, 2))


def test_modules_refuse_weights_that_are_not_theirs():
    from gemmlib_b200.experts import Fp8Experts
    from gemmlib_b200.fp8_linear import Fp8Linear, Fp8Weight

    with pytest.raises(ValueError, match="out_features, in_features"):
        Fp8Linear.from_weight(weight(2, 2, 32))
    with pytest.raises(ValueError, match="float8_e4m3fn"):
        Fp8Linear.from_weight(Fp8Weight(torch.zeros(2, 32), torch.ones(1, 1)))
    with pytest.raises(ValueError, match="one scale for each 128 x 128"):
        Fp8Linear.from_weight(Fp8Weight(weight(2, 32).values, torch.ones(1, 2)))
    with pytest.raises(ValueError, match="not those of one layer"):
        Fp8Experts.from_weights(weight(2, 64, 48), weight(2, 48, 31))
    with pytest.raises(ValueError, match="one scale for each 128 x 128"):
        Fp8Experts.from_weights(Fp8Weight(weight(2, 64, 48).values, torch.ones(2, 1, 2)), weight(2, 48, 32))
    layer = Fp8Linear.from_weight(weight(300, 200))
    assert layer.q_weights.shape == (300, 224) and layer.q_scales.shape == (3, 2) and layer.weight_bytes() == 300 * 200 + 24
    half = layer.half()
    assert half.q_weights.dtype == torch.float8_e4m3fn and half.q_scales.dtype == torch.float32


# shared memory of an SM, what of it is the system's for each CTA
SM, RESERVED = 228 * 1024, 1024
# of the 4-bit tensor-core kernels the one that asks for the least: up to 16 rows, all 512 columns
SKINNY = 6 * 4096 + 12 * (8192 + 512 + 256) + 512 + 1024


def test_plans_fit_on_an_sm_and_share_it_only_where_their_tensor_memory_does(lib_built):
    """Every part of K has steps; CTAs whose tensor memory does not fit together do not fit together in shared memory."""
    from gemmlib_b200 import capi

    rng = random.Random(1)
    size = lambda top: round(2 ** rng.uniform(0, top))  # noqa: E731
    shapes = [(size(13), size(15), size(15), 0) for _ in range(3000)] + [(size(15), size(12), size(13), size(10)) for _ in range(3000)]
    shapes += [(1, 1, 1, 0), (1 << 28, 1, 1 << 28, 1024), (4096, 4096, 4096, 1024)]
    seen = set()
    for m, n, k, experts in shapes:
        p = capi.fp8_gemm_plan(m, n, k, experts)
        seen.add((p["kernel"], p["tile_m"], p["split"] > 1))
        if p["kernel"] == "stream":
            assert experts == 0
            continue
        steps = -(-k // 128)
        assert p["stages"] >= 3 and p["smem"] <= 227 * 1024 and p["columns"] <= 512
        assert p["steps"] * p["split"] >= steps and p["steps"] * (p["split"] - 1) < steps
        assert experts == 0 or p["split"] == 1
        for others in (1, 2):  # further CTAs of the same kind
            fits = (others + 1) * (p["smem"] + RESERVED) <= SM
            assert not fits or (others + 1) * p["columns"] <= 512, (m, n, k, p)
        assert p["smem"] + SKINNY + 2 * RESERVED > SM, (m, n, k, p)
        if p["columns"] > 128:  # beside any CTA that has up to 512
            assert p["smem"] + 97 * 1024 + 2 * RESERVED > SM
    assert {"few", "many", "stream"} == {k for k, _, _ in seen} and {16, 32, 64, 128} <= {t for _, t, _ in seen} and any(s for _, _, s in seen)


def test_loads_from_tensor_memory_are_waited_for_with_their_registers_named():
    """tcgen05.ld is asynchronous: a statement that waits for it has to name the registers that it fills, or arithmetic on them may be moved
    ahead of the wait."""
    for name, loads in (("fp8_gemm.cu", 0), ("fp8_gemm_wide.cuh", 1)):
        text = open(os.path.join(ROOT, "gemmlib_b200", "csrc", name)).read()
        helper = re.search(r"__device__ __forceinline__ void tmem_ld_wait_for\(.*?\n}\n", text, flags=re.S)
        if helper:
            assert '"+r"(r[' in helper.group()
            text = text.replace(helper.group(), "")
        assert "tmem_ld_wait()" not in text
        for s in re.findall(r"asm volatile\((.*?)\);\n", text, flags=re.S):
            assert ("tcgen05.ld." in s) == ("wait::ld" in s), s
        assert len(re.findall(r"tmem_ld_32x32b_x\d+\(", text)) == loads
