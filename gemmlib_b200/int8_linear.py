"""The 8-bit path beside the 4-bit weights: int8 weights by output channel, int8 activations by token (W8A8).

Where a product is bound by the tensor cores - prompts, large batches - 8-bit operands run at twice the 16-bit rate.
``Int8Linear`` is a linear layer like ``BlkQ4Linear``; its input is a float16 or bfloat16 tensor, which it quantizes by row, or the
``Int8Rows`` that an operator ahead of it wrote: the RMS norm (``RMSNormInt8``, ``rms_norm_int8``), the gated activation
(``silu_mul_int8``) or ``quantize_int8``, shared by the layers that read the same activations.

Rows: any leading dimensions, the last one is a row.  Rows of one pitch (slices of a wider tensor among them) are read
in place, other layouts are copied first.  Work is enqueued on the current stream of the tensors' device.  A row with an infinity
or NaN gets the scale NaN, and is NaN in every output.  There is no backward pass: a tensor of a call (inputs,
scales, weights, bias, what is written) that requires one is refused while gradients are enabled, and so is one with a
forward-mode tangent.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Union

import torch
from torch import nn

from . import ms_blkq4linear_ext

_EARLY = ms_blkq4linear_ext.EARLY_WEIGHT_FETCH
_quantize = ms_blkq4linear_ext.int8_quantize
_rms_norm = ms_blkq4linear_ext.rms_norm_int8
_silu_mul = ms_blkq4linear_ext.silu_mul_int8
_dequantize = ms_blkq4linear_ext.int8_dequantize
_linear = ms_blkq4linear_ext.int8_linear


class Int8Rows(NamedTuple):
    """Rows of int8 and a float32 scale for each: row r stands for ``scales[r] * values[r]``.  (The operators' rows and scales share
    an allocation; what is pickled, saved or copied as ``Int8Rows`` has one of its own for each.)"""

    values: torch.Tensor
    scales: torch.Tensor

    def __reduce__(self):  # tensors of two types in one storage cannot be saved
        return Int8Rows, (self.values, self.scales.clone())

    def dequantize(self, dtype: torch.dtype = torch.float16) -> torch.Tensor:
        return _dequantize(self.values, self.scales, dtype)


ms_blkq4linear_ext.int8_rows_type(Int8Rows)  # what the extension's functions return
torch.serialization.add_safe_globals([Int8Rows])  # two tensors: torch.load takes them with weights_only, its default


def quantize_int8(x: torch.Tensor) -> Int8Rows:
    """Every row of ``x`` by its largest magnitude: scale = max|x| / 127, values = round(x * (127 / max|x|))."""
    return _quantize(x)


def rms_norm_int8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5, residual: Optional[torch.Tensor] = None,
                  residual_out: Optional[torch.Tensor] = None):
    """``h / sqrt(mean(h^2) + eps) * weight`` of every row, quantized.  Without a residual h = x and the result is an
    ``Int8Rows``.  With one h = x + residual, rounded to their type, and the result is (``Int8Rows``, h); h goes to
    ``residual_out`` where that is given, which may be ``x`` or ``residual``."""
    return _rms_norm(x, weight, eps, residual, residual_out)


def silu_mul_int8(gate: torch.Tensor, up: torch.Tensor) -> Int8Rows:
    """``gate / (1 + exp(-gate)) * up``, quantized by row; gate and up may be halves of one tensor."""
    return _silu_mul(gate, up)


def int8_linear(x: Int8Rows, weight: Int8Rows, bias: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.float16,
                out: Optional[torch.Tensor] = None, flags: int = 0) -> torch.Tensor:
    """``x`` [..., in_features] times ``weight`` [out_features, in_features], transposed, plus ``bias`` (of the output's type),
    as float16 or bfloat16.  Sums are exact; scales and bias are applied in float32 and the result is rounded once."""
    return _linear(x[0], x[1], weight[0], weight[1], bias, dtype, flags, out)


class RMSNormInt8(nn.Module):
    """RMS norm in front of ``Int8Linear`` layers: ``rms_norm_int8`` with a weight of its own."""

    def __init__(self, weight: torch.Tensor, eps: float = 1e-5):
        super().__init__()
        self.weight = nn.Parameter(weight.detach(), requires_grad=False)
        self.eps = float(eps)

    def forward(self, x, residual=None, residual_out=None):
        return rms_norm_int8(x, self.weight, self.eps, residual, residual_out)

    def extra_repr(self):
        return f"{self.weight.numel()}, eps={self.eps}"


class Int8Linear(nn.Module):
    """Linear layer with int8 weights, one scale an output channel: ``weights`` [out_features, in_features] (float16 or
    bfloat16, on the GPU) are quantized in the constructor.  ``forward`` takes a float16 or bfloat16 tensor, and answers in its
    type, or ``Int8Rows``, and answers in ``out``'s type or the weights'.  From the second call on the weights' first tiles are
    fetched while the kernel ahead still runs (``early_weight_fetch = False`` on a layer whose packed weights are rewritten
    by work queued on the stream of ``forward``)."""

    def __init__(self, weights: torch.Tensor, bias_tensor: Optional[torch.Tensor] = None):
        super().__init__()
        with torch.no_grad():
            rows = quantize_int8(weights)
        self._set(rows, bias_tensor, weights.dtype)

    def _set(self, rows: Int8Rows, bias_tensor, dtype, copy=False):
        if rows.values.dim() != 2:
            raise ValueError("weights must be [out_features, in_features]")
        self.out_features, self.in_features = rows.values.shape
        self.dtype = dtype
        pad, values = -self.in_features % 32, rows.values
        if pad:  # kept with whole rows of 32 bytes, so that copies of the buffer have them too
            values = nn.functional.pad(values, (0, pad))
        elif copy:
            values = values.clone(memory_format=torch.contiguous_format)
        self.register_buffer("q_weights", values)
        self.register_buffer("q_scales", rows.scales.detach().clone())  # (the operators' rows and scales share their memory)
        self.bias = bias_tensor
        self.early_weight_fetch = True
        self._settled = False  # the first forward is a plain launch

    @classmethod
    def from_rows(cls, weight: Int8Rows, bias_tensor: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.float16):
        """A layer of weights that are int8 rows already, [out_features, in_features], of any layout: it keeps a copy."""
        self = cls.__new__(cls)
        nn.Module.__init__(self)
        self._set(Int8Rows(*weight), bias_tensor, dtype, copy=True)
        return self

    def _apply(self, fn, recurse=True):
        scales = self.q_scales
        super()._apply(fn, recurse)
        if self.q_scales.dtype != torch.float32:  # .half() and the like are for the model's 16-bit tensors
            self.q_scales = scales.to(self.q_scales.device)
        self._settled = False
        return self

    def __setstate__(self, state):
        super().__setstate__(state)
        self._settled = False  # a copy's buffers are written on some stream too

    def _load_from_state_dict(self, *args, **kwargs):
        self._settled = False  # the buffers are about to be overwritten by a copy on some stream
        return super()._load_from_state_dict(*args, **kwargs)

    def weight_bytes(self) -> int:
        return self.out_features * self.in_features + 4 * self.out_features

    def forward(self, input: Union[torch.Tensor, Int8Rows], out: Optional[torch.Tensor] = None) -> torch.Tensor:
        if isinstance(input, torch.Tensor):
            values, scales = _quantize(input)
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
