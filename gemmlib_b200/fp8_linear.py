"""8-bit floating point with a scale for each block of 128: e4m3 activations (a scale for each 128 elements of a row) and e4m3 weights (one
for each 128 x 128), as 8-bit checkpoints have them.

``Fp8Linear`` is a linear layer like ``Int8Linear``; blocks keep an outlier from costing its whole row the precision.  Its input is a float16 or
bfloat16 tensor, which it quantizes by row, or the ``Fp8Rows`` that an operator ahead of it wrote: ``silu_mul_fp8`` or ``quantize_fp8``,
shared by the layers that read the same activations.

Rows: any leading dimensions, the last one is a row.  Rows of one pitch (slices of a wider tensor among them) are read in place, other layouts
are copied first.  Work is enqueued on the current stream of the tensors' device.  A block with an infinity or NaN gets the scale NaN: the row is NaN in
every output that reads it (of a weight: its 128 outputs are, for every row).  There is no backward pass: a tensor of a call that requires one is refused while
gradients are enabled, and so is one with a forward-mode tangent.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Union

import torch
from torch import nn

from . import ms_blkq4linear_ext
from .layers import KeepsBias, SettlesAnew

BLOCK = 128

_EARLY = ms_blkq4linear_ext.EARLY_WEIGHT_FETCH
_quantize = ms_blkq4linear_ext.fp8_quantize
_quantize_weight = ms_blkq4linear_ext.fp8_quantize_weight
_silu_mul = ms_blkq4linear_ext.silu_mul_fp8
_dequantize = ms_blkq4linear_ext.fp8_dequantize
_linear = ms_blkq4linear_ext.fp8_linear


class Fp8Rows(NamedTuple):
    """Rows of float8_e4m3fn [..., k] and their float32 scales [..., ceil(k / 128)]: a block of 128 stands for scale * values.  (The
    operators' rows and scales share an allocation; what is pickled, saved or copied as ``Fp8Rows`` has one of its own for each.)"""

    values: torch.Tensor
    scales: torch.Tensor

    def __reduce__(self):  # tensors of two types in one storage cannot be saved
        return Fp8Rows, (self.values, self.scales.clone())

    def dequantize(self, dtype: torch.dtype = torch.float16) -> torch.Tensor:
        return _dequantize(self.values, self.scales, dtype, False)


class Fp8Weight(NamedTuple):
    """Weights of float8_e4m3fn [..., out_features, in_features] and their float32 scales [..., ceil(out_features / 128), ceil(in_features /
    128)]: a block of 128 x 128 stands for scale * values."""

    values: torch.Tensor
    scales: torch.Tensor

    def dequantize(self, dtype: torch.dtype = torch.float16) -> torch.Tensor:
        return _dequantize(self.values, self.scales, dtype, True)


ms_blkq4linear_ext.fp8_types(0, Fp8Rows)  # what the extension's functions return
ms_blkq4linear_ext.fp8_types(1, Fp8Weight)
torch.serialization.add_safe_globals([Fp8Rows, Fp8Weight])  # two tensors: torch.load takes them with weights_only, its default


def quantize_fp8(x: torch.Tensor, order=None) -> Fp8Rows:
    """Every block of 128 of a row by its largest magnitude: scale = max|x| / 448, values = e4m3(x * 448 / max|x|), half to even.  With an
    ``order`` (``experts.sort_by_expert``): the rows of ``experts.gather_rows(x, order)``, which are not written in 16 bits first."""
    if order is None:
        return _quantize(x, None, None, None)
    source, places, offsets = order
    return _quantize(x, source, places, offsets)


def quantize_fp8_weight(w: torch.Tensor) -> Fp8Weight:
    """``w`` [..., out_features, in_features], every block of 128 x 128 by its largest magnitude."""
    return _quantize_weight(w)


def silu_mul_fp8(gate: torch.Tensor, up: torch.Tensor) -> Fp8Rows:
    """``gate / (1 + exp(-gate)) * up``, quantized by blocks of a row; gate and up may be halves of one tensor."""
    return _silu_mul(gate, up)


def fp8_linear(x: Fp8Rows, weight: Fp8Weight, bias: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.float16,
               out: Optional[torch.Tensor] = None, flags: int = 0) -> torch.Tensor:
    """``x`` [..., in_features] times ``weight`` [out_features, in_features], transposed, plus ``bias`` (of the output's type), as float16 or
    bfloat16.  Sums, scales and bias are held in float32 and the result is rounded once."""
    return _linear(x[0], x[1], weight[0], weight[1], bias, dtype, flags, out)


def own_weight(weight: Fp8Weight, copy: bool) -> Fp8Weight:
    """The weight as the layers keep it: rows of whole 32 bytes, contiguous scales; a copy where it is the caller's."""
    values, scales = weight
    pad = -values.size(-1) % 32
    if pad:  # (of bytes: padding is not defined for e4m3)
        values = nn.functional.pad(values.view(torch.uint8), (0, pad)).view(torch.float8_e4m3fn)
    elif copy or not values.is_contiguous():
        values = values.clone(memory_format=torch.contiguous_format)
    return Fp8Weight(values.detach(), scales.detach().to(torch.float32, copy=copy).contiguous())


class KeepsScales(nn.Module):
    """Layers whose float32 scales and e4m3 weights stay what they are when the model is converted."""

    _scale_names = ()

    def _apply(self, fn, recurse=True):
        held = {name: getattr(self, name) for name in self._scale_names}
        values = {name: b for name, b in self._buffers.items() if b is not None and b.dtype == torch.float8_e4m3fn}
        super()._apply(fn, recurse)
        for name, scales in held.items():
            if getattr(self, name).dtype != torch.float32:  # .half() and the like are for the model's 16-bit tensors
                setattr(self, name, scales.to(getattr(self, name).device))
        for name, v in values.items():
            if self._buffers[name].dtype != torch.float8_e4m3fn:
                self._buffers[name] = v.to(self._buffers[name].device)
        return self


class Fp8Linear(KeepsBias, SettlesAnew, KeepsScales):
    """Linear layer with e4m3 weights: ``weights`` [out_features, in_features] (float16 or bfloat16, on the GPU) are quantized in the constructor.
    ``forward`` takes a float16 or bfloat16 tensor, and answers in its type, or ``Fp8Rows``, and answers in ``out``'s type or the weights'.
    From the second call on the weights' first tiles are fetched while the kernel ahead still runs (``early_weight_fetch = False`` on a layer
    whose weights are rewritten by work queued on the stream of ``forward``)."""

    _scale_names = ("q_scales",)

    def __init__(self, weights: torch.Tensor, bias_tensor: Optional[torch.Tensor] = None):
        super().__init__()
        with torch.no_grad():
            weight = quantize_fp8_weight(weights)
        self._set(weight, bias_tensor, weights.dtype, copy=False)

    def _set(self, weight: Fp8Weight, bias_tensor, dtype, copy):
        if weight.values.dim() != 2:
            raise ValueError("weights must be [out_features, in_features]")
        if weight.values.dtype != torch.float8_e4m3fn:
            raise ValueError(f"weights must be float8_e4m3fn, instead got {weight.values.dtype}")
        self.out_features, self.in_features = weight.values.shape
        if tuple(weight.scales.shape) != (-(-self.out_features // BLOCK), -(-self.in_features // BLOCK)):
            raise ValueError(f"one scale for each 128 x 128 of {tuple(weight.values.shape)} is wanted, instead got {tuple(weight.scales.shape)}")
        self.dtype = dtype
        values, scales = own_weight(weight, copy)
        self.register_buffer("q_weights", values)
        self.register_buffer("q_scales", scales)
        self._keep_bias(bias_tensor, copy)
        self.early_weight_fetch = True
        self._settled = False  # the first forward is a plain launch

    @classmethod
    def from_weight(cls, weight: Fp8Weight, bias_tensor: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16):
        """A layer of weights that are e4m3 with their scales already, as a checkpoint has them, of any layout: it keeps a copy of them and the bias."""
        self = cls.__new__(cls)
        nn.Module.__init__(self)
        self._set(Fp8Weight(*weight), bias_tensor, dtype, copy=True)
        return self

    def weight_bytes(self) -> int:
        return self.out_features * self.in_features + 4 * self.q_scales.numel()

    def forward(self, input: Union[torch.Tensor, Fp8Rows], out: Optional[torch.Tensor] = None) -> torch.Tensor:
        if isinstance(input, torch.Tensor):
            values, scales = _quantize(input, None, None, None)
            dtype = input.dtype
        else:
            values, scales = input
            dtype = self.dtype if out is None else out.dtype
        w, bias = self.q_weights, self.bias
        if w.size(1) != self.in_features:
            w = w[:, :self.in_features]
        if bias is not None and bias.dtype != dtype:
            bias = bias.to(dtype)
        settled = self._settled
        output = _linear(values, scales, w, self.q_scales, bias, dtype, _EARLY if settled and self.early_weight_fetch else 0, out)
        if not settled:
            self._settled = True
        return output

    def extra_repr(self):
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"
