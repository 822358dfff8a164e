"""Python entry points for the DIMQ operators (MI355X HIP backend).

Mirrors ``dimq_backend/ops.py`` (reference ``dimq_cuda_backend/dimq_backend/ops.py:12-125``):
same function names, arguments and errors, with ``is_available()`` testing that
the HIP library (``dimq_amd._C``) loads.  The generalised operators for
b-bit / per-channel / weight-only layers are added alongside.
"""

from __future__ import annotations

import importlib
from functools import lru_cache
from typing import Sequence

import torch


@lru_cache(maxsize=1)
def _extension_available() -> bool:
    try:
        importlib.import_module("dimq_amd._C")
    except Exception:
        return False
    return True


def is_available() -> bool:
    """Return whether the compiled HIP library is loadable (ops.py:21-24)."""

    return _extension_available()


def require_extension() -> None:
    if not is_available():
        raise RuntimeError(
            "dimq_amd HIP library is not available. "
            "Build it with `make -C dimq_amd/csrc` (or `python -c 'import __graft_entry__ as g; g.build()'`)."
        )


@lru_cache(maxsize=1)
def _native():
    """The compiled half of the operators that are called past the dispatcher."""
    require_extension()
    from ._C import _native as compiled

    return compiled


def pack_u4(indices: torch.Tensor) -> torch.Tensor:
    require_extension()
    return torch.ops.dimq.pack_u4(indices)


def unpack_u4(packed: torch.Tensor, numel: int) -> torch.Tensor:
    require_extension()
    return torch.ops.dimq.unpack_u4(packed, int(numel))


def quantize_activation_u4(x: torch.Tensor, act_scale: float, act_zero_point: int) -> torch.Tensor:
    require_extension()
    return torch.ops.dimq.quantize_activation_u4(x, float(act_scale), int(act_zero_point))


def build_product_table(codebook: torch.Tensor, act_scale: float, act_zero_point: int) -> torch.Tensor:
    require_extension()
    return torch.ops.dimq.build_product_table(codebook, float(act_scale), int(act_zero_point))


def dimq_linear_lut(
    x: torch.Tensor,
    packed_weight: torch.Tensor,
    codebook: torch.Tensor,
    act_scale: float,
    act_zero_point: int,
    bias: torch.Tensor | None,
    out_features: int,
    in_features: int,
) -> torch.Tensor:
    require_extension()
    return torch.ops.dimq.linear_lut(
        x, packed_weight, codebook, float(act_scale), int(act_zero_point), bias, int(out_features), int(in_features)
    )


def dimq_conv2d_lut(
    x: torch.Tensor,
    packed_weight: torch.Tensor,
    codebook: torch.Tensor,
    act_scale: float,
    act_zero_point: int,
    bias: torch.Tensor | None,
    weight_shape: Sequence[int],
    stride: Sequence[int],
    padding: Sequence[int],
    dilation: Sequence[int],
    groups: int,
) -> torch.Tensor:
    require_extension()
    out_channels, cin_per_group, kernel_h, kernel_w = [int(v) for v in weight_shape]
    stride_h, stride_w = _pair(stride)
    pad_h, pad_w = _pair(padding)
    dil_h, dil_w = _pair(dilation)
    return torch.ops.dimq.conv2d_lut(
        x, packed_weight, codebook, float(act_scale), int(act_zero_point), bias, out_channels, cin_per_group,
        kernel_h, kernel_w, stride_h, stride_w, pad_h, pad_w, dil_h, dil_w, int(groups),
    )


# ---------------------------------------------------------------------------
# generalised operators (no reference counterpart: the reference is W4A4 only)
# ---------------------------------------------------------------------------

VARIANTS = {"auto": 0, "small_m": 1, "mfma": 2}
ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "gelu": 2}


def pack_bits(indices: torch.Tensor, bits: int) -> torch.Tensor:
    require_extension()
    return torch.ops.dimq.pack_bits(indices, int(bits))


def unpack_bits(packed: torch.Tensor, numel: int, bits: int) -> torch.Tensor:
    require_extension()
    return torch.ops.dimq.unpack_bits(packed, int(numel), int(bits))


def hard_quantize(w: torch.Tensor, centers: torch.Tensor, per_channel: bool = False):
    """Nearest-centre (indices, values), quant/dimq.py:197-221 semantics."""
    require_extension()
    return torch.ops.dimq.hard_quantize(w, centers, bool(per_channel))


def build_product_table_grouped(codebook: torch.Tensor, act_scale: float, act_zero_point: int) -> torch.Tensor:
    require_extension()
    return torch.ops.dimq.build_product_table_grouped(codebook, float(act_scale), int(act_zero_point))


def dimq_linear_codebook(
    x: torch.Tensor,
    packed_weight: torch.Tensor,
    codebook: torch.Tensor,
    bits: int,
    bias: torch.Tensor | None,
    out_features: int,
    in_features: int,
    *,
    out_dtype: torch.dtype | None = None,
    variant: str = "auto",
    residual: torch.Tensor | None = None,
    activation: str | None = None,
    decoded: torch.Tensor | None = None,
) -> torch.Tensor:
    """y = act(x @ W_hat^T + bias + residual) with W_hat[n, k] = codebook[n or 0, idx[n, k]].

    ``residual`` (output shape) and ``activation`` ("relu" or "gelu", exact erf
    form) are fused into the kernel's store; without them this is the plain
    weight-only Linear.  ``decoded``: this layer's buffer from
    ``predecode_codebook_weights`` (same packed weights and codebook), used by
    the large-M path in place of its own per-call weight decode."""
    require_extension()
    return torch.ops.dimq.linear_codebook(
        x, packed_weight, codebook, int(bits), bias, int(out_features), int(in_features), out_dtype,
        VARIANTS[variant], residual, ACTIVATIONS[activation], decoded,
    )


def predecode_codebook_weights(layers):
    """Decodes the weights of several codebook Linears in one batch of launches.

    ``layers``: (packed_weight, codebook, bits, out_features, in_features)
    tuples on one GPU.  Returns (buffer, views): views[i] is layer i's decode
    (None when bits is 8 or in_features % 32 != 0), to pass as
    ``dimq_linear_codebook(..., decoded=views[i])`` while the packed weights
    and codebook stay unchanged.  No counterpart in the reference, whose LUT
    kernels decode inside every call."""
    require_extension()
    from . import _C
    return _C.predecode_codebook_weights_impl(layers)


def dimq_conv2d_codebook(
    x: torch.Tensor,
    packed_weight: torch.Tensor,
    codebook: torch.Tensor,
    bits: int,
    bias: torch.Tensor | None,
    weight_shape: Sequence[int],
    stride: Sequence[int],
    padding: Sequence[int],
    dilation: Sequence[int],
    groups: int,
    *,
    out_dtype: torch.dtype | None = None,
    variant: str = "auto",
    prepared_weight: torch.Tensor | None = None,
    residual: torch.Tensor | None = None,
    activation: str | None = None,
) -> torch.Tensor:
    """Weight-only codebook conv2d; NCHW or channels_last input, output in the same memory format.

    ``prepared_weight`` (from :func:`prepare_conv_weight`) enables the LDS-halo
    and large-tile implicit-GEMM kernels for the shapes they support.
    ``residual`` (output shape) and ``activation`` ("relu" / "gelu") are fused
    into the kernel's store: y = act(conv + bias + residual)."""
    require_extension()
    out_channels, cin_per_group, kernel_h, kernel_w = [int(v) for v in weight_shape]
    stride_h, stride_w = _pair(stride)
    pad_h, pad_w = _pair(padding)
    dil_h, dil_w = _pair(dilation)
    return torch.ops.dimq.conv2d_codebook(
        x, packed_weight, codebook, int(bits), bias, out_channels, cin_per_group, kernel_h, kernel_w, stride_h,
        stride_w, pad_h, pad_w, dil_h, dil_w, int(groups), out_dtype, VARIANTS[variant], prepared_weight, residual,
        ACTIVATIONS[activation],
    )


def prepare_conv_weight(packed_weight: torch.Tensor, bits: int, weight_shape: Sequence[int]) -> torch.Tensor | None:
    """Kernel-layout copy of a conv_kcrs packed weight, or None when the shape has no kernel layout."""
    require_extension()
    from . import _C

    out_channels, cin, kernel_h, kernel_w = [int(v) for v in weight_shape]
    if _C.prepared_conv_words(out_channels, cin, kernel_h, kernel_w, int(bits)) <= 0:
        return None
    return torch.ops.dimq.prepare_conv_weight(packed_weight, int(bits), out_channels, cin, kernel_h, kernel_w)


def dimq_linear_codebook_act(x: torch.Tensor, packed_weight: torch.Tensor, codebook: torch.Tensor, bits: int,
                             act_centers: torch.Tensor, bias: torch.Tensor | None, out_features: int,
                             in_features: int, out_dtype: torch.dtype | None = None,
                             variant: str = "auto") -> torch.Tensor:
    """Weight x activation codebook Linear: x quantized to its nearest activation centre (the QAT wrapper's
    activation_centers, quant/dimq_wrapper.py:80-85), then the weight-codebook GEMM."""
    require_extension()
    return torch.ops.dimq.linear_codebook_act(x, packed_weight, codebook, int(bits), act_centers, bias,
                                              int(out_features), int(in_features), out_dtype, VARIANTS[variant])


def build_codebook_product_table(codebook: torch.Tensor, act_values: torch.Tensor) -> torch.Tensor:
    """[rows, Kw, Ka] fp32 table codebook[g][w] * act_values[a] (one rounding): the weight x activation codebook
    products a LUT GEMM gathers from.  act_values: the activation centres as the activations take them (in the
    activations' dtype)."""
    require_extension()
    from . import _C

    return _C.build_codebook_product_table_impl(codebook, act_values)


def dimq_linear_lut_act(act_idx: torch.Tensor, packed_weight: torch.Tensor, codebook: torch.Tensor, bits: int,
                        act_centers: torch.Tensor, x_dtype: torch.dtype, bias: torch.Tensor | None, out_features: int,
                        in_features: int, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Index x index LUT GEMM (M <= 16): y[m, n] = sum_k (C_w[n][w[n, k]] * C_a[a[m, k]]) + bias[n], act_idx the
    uint8 activation-centre indices, C_a rounded to x_dtype (the reference's centers[idx].to(x.dtype))."""
    require_extension()
    from . import _C

    return _C.linear_lut_act_impl(act_idx, packed_weight, codebook, int(bits), act_centers, x_dtype, bias,
                                  int(out_features), int(in_features), out_dtype)


def dimq_conv2d_codebook_act(x: torch.Tensor, packed_weight: torch.Tensor, codebook: torch.Tensor, bits: int,
                             act_centers: torch.Tensor, bias: torch.Tensor | None, weight_shape: Sequence[int],
                             stride=1, padding=0, dilation=1, groups: int = 1, *,
                             out_dtype: torch.dtype | None = None, prepared_weight: torch.Tensor | None = None,
                             variant: str = "auto") -> torch.Tensor:
    """Weight x activation codebook Conv2d: x quantized to its nearest activation centre (the QAT wrapper's
    activation_centers, quant/dimq_wrapper.py:80-85), then the weight-codebook conv."""
    require_extension()
    from . import _C

    oc, cin_g, kh, kw = [int(v) for v in weight_shape]
    sh, sw = _pair(stride)
    ph, pw = _pair(padding)
    dh, dw = _pair(dilation)
    return _C.conv2d_codebook_act_impl(x, packed_weight, codebook, int(bits), act_centers, bias, oc, cin_g, kh, kw,
                                       sh, sw, ph, pw, dh, dw, int(groups), out_dtype, prepared_weight,
                                       VARIANTS[variant])


# ---------------------------------------------------------------------------
# Chained W4A4 layers.  Between layers the activations travel as the fp16
# integers a - zp (a = clamp(rint(x / s) + zp, 0, 15), the reference's u4 code,
# dimq_backend/reference.py:11-21), so a layer's epilogue can quantize its
# output for the next layer instead of the next layer re-reading a float tensor.
def quantize_activation_f16(x: torch.Tensor, act_scale: float, act_zp: int) -> torch.Tensor:
    """fp16 tensor of x's shape holding a - zp: the input form of linear_lut_q / conv2d_lut_q."""
    require_extension()
    from . import _C

    return _C.quantize_activation_f16_impl(x, act_scale, act_zp)


def dimq_linear_lut_q(xq: torch.Tensor, packed_weight: torch.Tensor, codebook: torch.Tensor, act_scale: float,
                      bias: torch.Tensor | None, out_features: int, in_features: int, *,
                      activation: str | None = None, out_act: tuple[float, int] | None = None,
                      out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """linear_lut on pre-quantized activations: y = act(s * sum_k C[w] (a - zp) + bias), xq = a - zp (fp16),
    s = act_scale.  With out_act = (s', zp') the result is returned as the next layer's codes (fp16 q' - zp');
    otherwise as out_dtype (default fp32).  codebook: the 16-entry fp16 codebook of the packed export."""
    require_extension()
    from . import _C

    return _C.linear_lut_q_impl(xq, packed_weight, codebook, act_scale, bias, int(out_features), int(in_features),
                                ACTIVATIONS[activation], out_act, out_dtype)


def dimq_conv2d_lut_q(xq: torch.Tensor, packed_weight: torch.Tensor, codebook: torch.Tensor, act_scale: float,
                      bias: torch.Tensor | None, weight_shape: Sequence[int], stride=1, padding=0, dilation=1,
                      groups: int = 1, *, prepared_weight: torch.Tensor | None = None,
                      activation: str | None = None, out_act: tuple[float, int] | None = None,
                      out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """conv2d_lut on pre-quantized NCHW activations (xq = a - zp, fp16); output NCHW.  prepared_weight: the 4-bit
    kernel layout of prepare_conv_weight (optional).  activation / out_act / out_dtype as dimq_linear_lut_q."""
    require_extension()
    from . import _C

    oc, cin_g, kh, kw = [int(v) for v in weight_shape]
    sh, sw = _pair(stride)
    ph, pw = _pair(padding)
    dh, dw = _pair(dilation)
    return _C.conv2d_lut_q_impl(xq, packed_weight, codebook, act_scale, bias, oc, cin_g, kh, kw, sh, sw, ph, pw, dh,
                                dw, int(groups), prepared_weight, ACTIVATIONS[activation], out_act, out_dtype)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None,
               eps: float = 1e-5, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """LayerNorm over the last dimension on the HIP kernel (fp16/bf16 x; the ViT workload's LayerNorms); the
    output in out_dtype (fp16 / bf16, default x's dtype)."""
    require_extension()
    return torch.ops.dimq.layer_norm(x, int(x.shape[-1]), weight, bias, float(eps), out_dtype)


def quantize_grouped(w: torch.Tensor, group_size: int = 128, *, symmetric: bool = False,
                     scale_dtype: torch.dtype = torch.float16):
    """``(codes, scales, zeros)`` of a weight ``[out_features, in_features]`` in 4 bits with a scale per group of
    ``group_size`` (a multiple of 32) elements of a row, for :func:`dimq_linear_grouped`.  The grid runs from a group's
    smallest value (0 if that is positive) to its largest (0 if negative) in 15 steps, with a zero point that stands for 0
    exactly; ``symmetric``: around 0 (codes 1..15, zero point 8, zeros None).  codes: uint8 ``[out_features, 16 * blocks]``,
    rows padded to blocks of 32, two a byte, the earlier element in the low half.  Done once, at load, in torch operations;
    a weight that is not finite raises."""
    if w.dim() != 2 or w.numel() == 0:
        raise RuntimeError("quantize_grouped expects a weight [out_features, in_features]")
    if group_size <= 0 or group_size % 32:
        raise RuntimeError("quantize_grouped: the group size must be a positive multiple of 32")
    if scale_dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise RuntimeError("quantize_grouped: scales must be fp32, fp16 or bf16")
    w = w.detach().float()
    if not bool(torch.isfinite(w).all()):
        raise RuntimeError("quantize_grouped: the weight must be finite")
    n, k = w.shape
    groups, blocks = -(-k // group_size), -(-k // 32)
    v = torch.nn.functional.pad(w, (0, groups * group_size - k)).view(n, groups, group_size)
    low, high = v.amin(2).clamp(max=0), v.amax(2).clamp(min=0)
    steps = torch.maximum(-low, high) / 7 if symmetric else (high - low) / 15
    # a scale that its type rounds to 0 could not be divided by
    scales = steps.clamp(min=torch.finfo(scale_dtype).tiny, max=torch.finfo(scale_dtype).max).to(scale_dtype)
    s = scales.float()
    zeros = None if symmetric else torch.round(-low / s).clamp(0, 15)
    q = torch.round(v / s[..., None] + (8 if symmetric else zeros[..., None])).clamp(0, 15).to(torch.uint8)
    q = torch.nn.functional.pad(q.view(n, -1)[:, :k], (0, blocks * 32 - k)).view(n, blocks * 16, 2)
    return q[..., 0] + q[..., 1] * 16, scales, None if symmetric else zeros.to(torch.uint8)


def dimq_linear_grouped(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None,
                        group_size: int, bias: torch.Tensor | None = None, *, x_scales: torch.Tensor | None = None,
                        residual: torch.Tensor | None = None, activation: str | None = None,
                        out_dtype: torch.dtype | None = None, variant: str = "auto") -> torch.Tensor:
    """``act(x W^T + bias + residual)`` with ``W[n, k] = scales[n, k // group_size] * (q[n, k] - zeros[n, k // group_size])``,
    q the 4-bit codes as :func:`quantize_grouped` packs them, zeros (uint8, at most 15) 8 where None.  x in fp32, fp16 or
    bf16, or in torch.float8_e4m3fn with ``x_scales`` (fp32, one for each row, as :func:`rms_norm_e4m3` gives), which
    multiplies the row.  Neither x nor W is rounded, sums are fp32; a row of x that holds a NaN or an infinity gives outputs that
    are not finite; the output in ``out_dtype`` (x's by default, bf16 for
    float8).  ``variant``: "small_m" one launch, "mfma" tiles (a workspace and up to three launches), "auto" by size.  For
    serving: a backward pass through it raises."""
    return _native().linear_grouped(x, codes, scales, zeros, int(group_size), bias, x_scales, residual,
                                    ACTIVATIONS[activation], out_dtype, VARIANTS[variant])


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, eps: float = 1e-6, *,
             residual: torch.Tensor | None = None, out_dtype: torch.dtype | None = None):
    """``y = h / sqrt(mean(h^2) + eps) * weight`` over the last dimension, h = x; with a residual (x's shape and dtype)
    ``(y, h)``, h = x + residual rounded to their dtype.  x in fp32, fp16 or bf16, y in ``out_dtype`` (x's by default).
    Gradients reach x, the residual and the weight; they have none of their own."""
    y, h = _native().rms_norm(x, weight, float(eps), residual, out_dtype)
    return y if residual is None else (y, h)


def rms_norm_e4m3(x: torch.Tensor, weight: torch.Tensor | None = None, eps: float = 1e-6, *,
                  residual: torch.Tensor | None = None):
    """``rms_norm`` with its rows in 8 bits, the input that ``dimq_linear_grouped`` takes: ``(codes, scales)``, with a
    residual ``(codes, scales, h)``.  codes: torch.float8_e4m3fn of y / scale, to nearest even; scales: fp32, max|y| / 448
    of each row (at least 2^-126; 0 for a row of zeros).  A row with a y that is not finite has the scale NaN.  For serving:
    it has no gradients."""
    codes, scales, h = _native().rms_norm_e4m3(x, weight, float(eps), residual)
    return (codes, scales) if residual is None else (codes, scales, h)


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0):
    """``(logprobs, entropy, top_logprobs, top_ids)`` of rows of logits ``[..., vocab]`` in fp32, fp16 or bf16, p their
    softmax: log p of each row's token (tokens ``[...]``, int64 or int32; 0 for a negative token, NaN for one beyond the
    vocabulary), the entropy -sum p log p, and the ``top`` (at most 128) largest log p with their tokens, in order, the lower
    token first among equals.  The values are fp32.  A row that holds a NaN or +infinity, or nothing above -infinity, has
    no distribution: its values are NaN, its alternatives' tokens -1.  Gradients reach the logits from the log
    probabilities and the entropy (zero where both of a row's are); they have none of their own."""
    return _native().token_logprobs(logits, tokens, int(top))


def max_pool2d_nhwc(x: torch.Tensor, kernel_size, stride=None, padding=0) -> torch.Tensor:
    """2-D max pooling of a channels-last fp16/bf16 tensor on the HIP kernel (the ResNet workload's stem pool)."""
    require_extension()
    kh, kw = _pair(kernel_size)
    sh, sw = _pair(stride if stride is not None else kernel_size)
    ph, pw = _pair(padding)
    return torch.ops.dimq.max_pool2d_nhwc(x, kh, kw, sh, sw, ph, pw)


def _pair(value: Sequence[int] | int) -> tuple[int, int]:
    if isinstance(value, int):
        return int(value), int(value)
    if len(value) != 2:
        raise ValueError(f"expected pair, got {value!r}")
    return int(value[0]), int(value[1])
