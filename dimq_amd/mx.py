"""Microscaled formats: 4-bit linear layers and 8-bit activation checkpoints.

Along a tensor's last dimension, blocks of 32 elements (a last one may be short) share one power of two, kept as a byte
(exponent + 127); a block's codes are 4-bit floats {0, .5, 1, 1.5, 2, 3, 4, 6} with sign (two a byte, the earlier element in
the low half, 16 bytes a block) or 8-bit integers -127..127 in units of 1/64 of the scale.  A block that holds a NaN or an
infinity stands for NaN throughout.  ``Q4(x)`` and ``Q8(x)`` are the values that x's codes stand for.

* Serving: ``quantize_mxfp4`` packs a weight once; ``mxfp4_linear`` runs the layer, quantizing its input on the way in
  (``modules.DIMQMXFP4Linear`` holds both), and as a frozen layer passes gradients on.
* Training: ``linear`` (``MXFP4TrainLinear``) runs that layer on the master weights with straight-through gradients and
  keeps its input in 8 bits for the weight gradient; ``gelu`` keeps its input in 8 bits too.

All but ``linear`` and ``gelu`` are torch ops too (``torch.ops.dimq.quantize_mxfp4`` and so on), which traces, dispatch
modes and vmap see; those two, and gradients through a frozen layer, refuse to be traced.  All of it is for CUDA
(HIP) tensors in fp32, fp16 and bf16; the gradients are those of the formulas in each function's
description and have no gradients of their own.
"""

from __future__ import annotations

import torch
import torch.nn as nn
from torch import Tensor

from .ops import ACTIVATIONS, require_extension


class _Unbuilt:
    """Stands for the compiled half while it cannot be loaded: an operator's call looks for it again, or raises."""

    def __getattr__(self, name: str):
        global _native
        require_extension()
        from ._C import _native
        return getattr(_native, name)


try:  # now, so that torch.ops.dimq is there after the package's import
    from ._C import _native
except Exception:
    _native = _Unbuilt()


def quantize_mxfp4(x: Tensor) -> tuple[Tensor, Tensor]:
    """(codes, scales) of x's last dimension in 4 bits: uint8 ``[..., 16 * blocks]`` and ``[..., blocks]``."""
    return _native.quantize_mxfp4(x)


def compress_activation(x: Tensor) -> tuple[Tensor, Tensor]:
    """(codes, scales) of x's last dimension in 8 bits: int8 ``[..., 32 * blocks]`` and uint8 ``[..., blocks]``."""
    return _native.compress_activation(x)


def quantize_and_compress(x: Tensor) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """``quantize_mxfp4(x) + compress_activation(x)`` from one read of x."""
    return _native.quantize_and_compress(x)


def dequantize_mxfp4(codes: Tensor, scales: Tensor, size: int, dtype: torch.dtype = torch.float32) -> Tensor:
    """The values of 4-bit codes, ``[..., size]``, rounded to ``dtype`` (exact in fp32 and bf16)."""
    return _native.dequantize_mxfp4(codes, scales, size, dtype)


def decompress_activation(codes: Tensor, scales: Tensor, size: int, dtype: torch.dtype = torch.float32) -> Tensor:
    """The values of 8-bit codes, ``[..., size]``, rounded to ``dtype`` (exact in fp32 and bf16)."""
    return _native.decompress_activation(codes, scales, size, dtype)


def mxfp4_linear(x: Tensor, codes: Tensor, scales: Tensor, bias: Tensor | None = None, *, residual: Tensor | None = None,
                 activation: str | None = None, out_dtype: torch.dtype | None = None) -> Tensor:
    """``act(Q4(x) W^T + bias + residual)`` for the weight W that ``quantize_mxfp4`` packed (codes ``[out_features, ...]``);
    activation None, "relu" or "gelu" (exact); the output in ``out_dtype`` (x's by default).  W is frozen: gradients go
    straight through the quantization to x (``g W``), to the bias (``sum g``) and to the residual (``g``); a backward pass
    through a fused activation raises."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}")
    return _native.mxfp4_linear(x, codes, scales, bias, residual, ACTIVATIONS[activation], out_dtype)


def mxfp4_linear_grad_input(grad: Tensor, codes: Tensor, scales: Tensor, in_features: int,
                            out_dtype: torch.dtype | None = None) -> Tensor:
    """``grad W``: the gradient to that layer's input, straight through its quantization."""
    return _native.mxfp4_linear_grad_input(grad, codes, scales, in_features, out_dtype)


def linear_grad_weight(grad: Tensor, codes: Tensor, scales: Tensor, in_features: int, bias: bool = True,
                       out_dtype: torch.dtype = torch.float32) -> tuple[Tensor, Tensor | None]:
    """``(grad^T Q8(x), grad summed over the rows)`` for the 8-bit codes of a layer's input x; the second is None without
    ``bias``."""
    gw, gb = _native.linear_grad_weight(grad, codes, scales, in_features, bias, out_dtype, None)
    return gw, gb if bias else None


def linear(x: Tensor, weight: Tensor, bias: Tensor | None = None) -> Tensor:
    """``Q4(x) Q4(weight)^T + bias`` in x's dtype, with gradients straight through the quantizations:
    ``g Q4(weight)`` to x, ``g^T Q8(x)`` to the weight, ``sum g`` to the bias.  Of x the graph keeps the 8-bit form, about
    half of its 16-bit size."""
    return _native.mx_linear(x, weight, bias)


def gelu(h: Tensor) -> Tensor:
    """``h Phi(h)`` in h's dtype; backward ``g gelu'(Q8(h))``: the graph keeps h's 8-bit form."""
    return _native.mx_gelu(h)


class MXFP4TrainLinear(nn.Linear):
    """nn.Linear whose forward and backward are ``linear``: the same parameters, which an optimiser updates."""

    def forward(self, x: Tensor) -> Tensor:
        return linear(x, self.weight, self.bias)

    @classmethod
    def from_linear(cls, linear_: nn.Linear) -> "MXFP4TrainLinear":
        m = cls(linear_.in_features, linear_.out_features, linear_.bias is not None, device="meta")
        m.weight, m.bias = linear_.weight, linear_.bias
        return m
