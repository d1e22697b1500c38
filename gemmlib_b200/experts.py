"""Layers of experts: tokens sorted by expert and back, the product of every expert's rows with its weight, and a whole layer of e4m3 weights.

A router gives every token some choices: ``experts`` [..., choices] (int32 or int64) names them, ``weights`` of that shape says how much each counts.  An
expert that is none of 0 .. n_experts - 1 (-1 for padding, or another GPU's experts) drops its choice: it has no row, adds nothing and gets no gradient.

    order = sort_by_expert(experts, n_experts)
    rows = gather_rows(x, order)                # [choices of all tokens, features], expert by expert; zeros behind the last expert's rows
    y = ...                                     # the experts, on rows[order.offsets[e]:order.offsets[e + 1]]
    out = combine_rows(y, order, weights)       # [..., features]

``gather_rows`` and ``combine_rows`` have a backward pass (of one order).  All sums are float32, taken in the order of a token's choices, and
rounded once; nothing depends on the order of atomics.  Offsets stay on the device: no call waits for the GPU, and all of them can be captured, with
their backward pass (not while an eager graph of the same leaves lives on another stream: autograd would make the capture wait for it; such a
call is refused, or its backward pass where the leaf stands behind other operators).
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch import nn

from . import ms_blkq4linear_ext
from .fp8_linear import BLOCK, Fp8Rows, Fp8Weight, KeepsScales, own_weight, quantize_fp8, quantize_fp8_weight, silu_mul_fp8

_sort = ms_blkq4linear_ext.experts_sort
_gather = ms_blkq4linear_ext.experts_gather
_combine = ms_blkq4linear_ext.experts_combine
_expert_linear = ms_blkq4linear_ext.fp8_expert_linear


class ExpertOrder(NamedTuple):
    """The choices, stably sorted by expert (all int32, on the device).

    ``source`` [n]: the choice (token * choices + number) at each place, those of no expert behind all others;
    ``places`` [..., choices]: the place of each choice, -1 for those of no expert;
    ``offsets`` [n_experts + 1]: where each expert's rows begin, and behind them the number of rows that belong to one."""

    source: torch.Tensor
    places: torch.Tensor
    offsets: torch.Tensor


ms_blkq4linear_ext.fp8_types(2, ExpertOrder)
torch.serialization.add_safe_globals([ExpertOrder])


def sort_by_expert(experts: torch.Tensor, n_experts: int) -> ExpertOrder:
    """The order of the choices ``experts`` [..., choices], for up to 1024 experts."""
    return _sort(experts, n_experts)


def gather_rows(x: torch.Tensor, order: ExpertOrder) -> torch.Tensor:
    """The row of ``x`` [..., features] (float16 or bfloat16) of every choice, in the order's places: [n, features]; zeros behind
    ``order.offsets[-1]``.  A token's gradient is the sum of its rows'."""
    return _gather(x, *order)


def combine_rows(y: torch.Tensor, order: ExpertOrder, weights: torch.Tensor) -> torch.Tensor:
    """The sum of each token's rows of ``y`` [n, features], with ``weights`` (float32, float16 or bfloat16) of the shape of ``order.places``:
    [..., features], in the type of ``y``.  What stands behind ``order.offsets[-1]`` is not read."""
    return _combine(y, *order, weights)


def fp8_expert_linear(x: Fp8Rows, weight: Fp8Weight, offsets: torch.Tensor, dtype: torch.dtype = torch.float16,
                      out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``fp8_linear`` of rows ``offsets[e]`` to ``offsets[e + 1]`` of ``x`` [rows, in_features] with ``weight`` e of [experts, out_features,
    in_features].  Rows of no expert are zero, or left as they are in an ``out`` that is given."""
    return _expert_linear(x[0], x[1], weight[0], weight[1], offsets, dtype, 0, out)


class Fp8Experts(KeepsScales):
    """A layer of gated feed-forward experts with e4m3 weights: ``gate_up`` [experts, 2 * ffn, features] (gate first) and ``down`` [experts,
    features, ffn], 16-bit tensors that are quantized in the constructor, each in one call (with a second copy of the e4m3 values for as long as it
    lasts where rows are no whole 32 bytes).

    ``forward(x, experts, weights)``: the weighted sum of the experts' ``down(silu(gate) * up)`` for ``x`` [..., features], choices ``experts`` [...,
    choices] and their ``weights``.  The weights' gradient is computed (a router can be trained); there is none for ``x``."""

    _scale_names = ("gate_up_scales", "down_scales")

    def __init__(self, gate_up: torch.Tensor, down: torch.Tensor):
        super().__init__()
        with torch.no_grad():
            self._set(quantize_fp8_weight(gate_up), quantize_fp8_weight(down), copy=False)

    def _set(self, gate_up: Fp8Weight, down: Fp8Weight, copy):
        for name, w in (("gate_up", gate_up), ("down", down)):
            if w.values.dim() != 3 or w.values.dtype != torch.float8_e4m3fn:
                raise ValueError(f"{name} must be float8_e4m3fn [experts, out_features, in_features], instead got {w.values.dtype} {tuple(w.values.shape)}")
            n, k = w.values.shape[1:]
            if tuple(w.scales.shape) != (w.values.size(0), -(-n // BLOCK), -(-k // BLOCK)):
                raise ValueError(f"{name}: one scale for each 128 x 128 is wanted, instead got {tuple(w.scales.shape)}")
        self.n_experts, double, self.features = gate_up.values.shape
        self.ffn = double // 2
        if double % 2 or tuple(down.values.shape) != (self.n_experts, self.features, self.ffn):
            raise ValueError(f"gate_up {tuple(gate_up.values.shape)} and down {tuple(down.values.shape)} are not those of one layer")
        values, scales = own_weight(gate_up, copy)
        self.register_buffer("gate_up", values)
        self.register_buffer("gate_up_scales", scales)
        values, scales = own_weight(down, copy)
        self.register_buffer("down", values)
        self.register_buffer("down_scales", scales)

    @classmethod
    def from_weights(cls, gate_up: Fp8Weight, down: Fp8Weight):
        """A layer of weights that are e4m3 with their scales already, as a checkpoint has them: it keeps a copy."""
        self = cls.__new__(cls)
        nn.Module.__init__(self)
        self._set(Fp8Weight(*gate_up), Fp8Weight(*down), copy=True)
        return self

    def forward(self, x: torch.Tensor, experts: torch.Tensor, weights: torch.Tensor) -> torch.Tensor:
        order = sort_by_expert(experts, self.n_experts)
        offsets, f = order.offsets, self.ffn
        both = fp8_expert_linear(quantize_fp8(x, order), Fp8Weight(self.gate_up[..., :self.features], self.gate_up_scales), offsets, x.dtype)
        rows = silu_mul_fp8(both[:, :f], both[:, f:])
        y = fp8_expert_linear(rows, Fp8Weight(self.down[..., :f], self.down_scales), offsets, x.dtype)
        return combine_rows(y, order, weights)

    def weight_bytes(self) -> int:
        return self.n_experts * self.features * 3 * self.ffn + 4 * (self.gate_up_scales.numel() + self.down_scales.numel())

    def extra_repr(self):
        return f"experts={self.n_experts}, features={self.features}, ffn={self.ffn}"
