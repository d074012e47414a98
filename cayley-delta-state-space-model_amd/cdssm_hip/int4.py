"""Decode products with 4-bit weights in groups, on the HIP kernel.

``quantize_int4`` turns a weight into codes of -8 .. 7 with a bf16 scale for every ``group_size`` of them along a row, laid out
for ``int4_linear``, the counterpart of ``lm.skinny_linear`` at a quarter of the weight's bytes; ``pack_int4`` takes codes and
scales that come from elsewhere.  ``CDSSMLMHeadModel.quantize_int4_`` has a model's decode steps use them.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib
from .distill import _native

Tensor = torch.Tensor

GROUP_SIZES = (32, 64, 128)
MAX_ROWS = 64


@dataclass(frozen=True, eq=False)
class Int4Weight:
    """A weight (out_features, in_features) as ``int4_linear`` reads it.  ``words`` and ``scales`` are in the kernel's order."""

    words: Tensor
    scales: Tensor
    out_features: int
    in_features: int
    group_size: int

    def unpack(self) -> tuple:
        """(codes (N, K) int8, scales (N, ceil(K / group_size)) bf16)."""
        return _native().int4_unpack(self.words, self.scales, self.out_features, self.in_features, self.group_size)

    def dequantize(self, dtype: torch.dtype = torch.float32) -> Tensor:
        """The weight (N, K) that the codes and scales stand for, in fp32 or rounded once to ``dtype``."""
        codes, scales = self.unpack()
        wide = scales.float().repeat_interleave(self.group_size, 1)[:, :self.in_features]
        return (codes.float() * wide).to(dtype)


def _check_group(op: str, group_size: int) -> None:
    if group_size not in GROUP_SIZES:
        raise ValueError(f"{op}: group_size must be one of {GROUP_SIZES}, got {group_size}")


def pack_int4(codes: Tensor, scales: Tensor, group_size: int) -> Int4Weight:
    """codes (N, K) int8 of -8 .. 7 and scales (N, ceil(K / group_size)) bf16, W[n, k] = scales[n, k // group_size] codes[n, k],
    as ``int4_linear`` reads them.  Codes outside -8 .. 7 are refused (which waits for the GPU)."""
    op = "pack_int4"
    _check_group(op, group_size)
    if not codes.is_cuda:
        raise RuntimeError(f"{op} runs on the GPU only")
    if scales.device != codes.device:
        raise RuntimeError(f"{op}: codes are on {codes.device}, scales on {scales.device}")
    if codes.dtype != torch.int8 or scales.dtype != torch.bfloat16:
        raise TypeError(f"{op}: codes must be int8 and scales bfloat16, got {codes.dtype} and {scales.dtype}")
    if codes.dim() != 2 or 0 in codes.shape or tuple(scales.shape) != (codes.shape[0], -(-codes.shape[1] // group_size)):
        raise ValueError(f"{op}: codes must be (N, K) with N, K >= 1 and scales (N, ceil(K / {group_size})), got "
                         f"{tuple(codes.shape)} and {tuple(scales.shape)}")
    lo, hi = torch.aminmax(codes)
    if int(lo) < -8 or int(hi) > 7:
        raise ValueError(f"{op}: codes must be within -8 .. 7, got {int(lo)} .. {int(hi)}")
    words, laid = _native().int4_pack(codes, scales.detach(), group_size)
    return Int4Weight(words, laid, codes.shape[0], codes.shape[1], group_size)


def quantize_int4(weight: Tensor, group_size: int = 64) -> Int4Weight:
    """weight (N, K) fp32 or bf16 in 4 bits: of every ``group_size`` weights of a row (32, 64 or 128; the last ones of a row may
    be fewer) the scale is the largest magnitude over 7, rounded to bf16, and a code the nearest whole number to weight / scale
    (even ones at a half).  Groups below 2^-120 throughout become 0; a group that holds an infinity or NaN is NaN."""
    op = "quantize_int4"
    _check_group(op, group_size)
    if not weight.is_cuda:
        raise RuntimeError(f"{op} runs on the GPU only")
    if weight.dtype not in _lib.DTYPE_CODE:
        raise TypeError(f"{op}: weight must be float32 or bfloat16, got {weight.dtype}")
    if weight.dim() != 2 or 0 in weight.shape:
        raise ValueError(f"{op}: weight must be (N, K) with N, K >= 1, got {tuple(weight.shape)}")
    codes, scales = _native().int4_quantize(weight.detach(), group_size)
    words, laid = _native().int4_pack(codes, scales, group_size)
    return Int4Weight(words, laid, weight.shape[0], weight.shape[1], group_size)


def fingerprints(weights: list) -> list:
    """A number of what each of these weights (N, K) fp32 or bf16 on one GPU holds (their bits and places, not their addresses or
    strides): another for any change, but for chance of 2^-64.  Waits for the GPU."""
    return _native().int4_fingerprints([w.detach() for w in weights]).tolist()


def int4_linear(x: Tensor, weight: Int4Weight, bias: Optional[Tensor] = None, residual: Optional[Tensor] = None,
                norm_weight: Optional[Tensor] = None, eps: float = 0.0) -> Tensor:
    """x' @ W^T (+ bias) (+ residual) for a 4-bit weight W (N, K): x (..., K) bf16 of at most 64 rows -> (..., N) bf16, with
    x' = x, or with a norm weight x rsqrt(mean(x^2) + eps) norm_weight.  bias (N), residual (..., N) and norm_weight (K) are
    taken in bf16.  Sums in fp32, rounded once; the weight is not rounded, and x' to 2^-17 (without a norm x' is x itself, and an
    element costs the columns whose weight is 0 there nothing, however large).  Where x holds an infinity or NaN its row is not
    finite in any column (with a norm it is NaN), and where 8 |x'| summed over a group passes fp32 it may not be.  With a norm
    x^2 summed over a row is held in fp32: a row where it passes that (|x| from 2^64 / sqrt(K) on) is NaN.  Without a gradient:
    refused where one would be followed."""
    return _native().int4_linear(x, weight.words, weight.scales, weight.out_features, weight.in_features, weight.group_size,
                                 bias, residual, norm_weight, eps)


def int4_linear_conv_step(x: Tensor, weight: Int4Weight, bias: Optional[Tensor], norm_weight: Tensor, eps: float, conv_col: int,
                          window: Tensor, conv_weight: Tensor, conv_bias: Tensor) -> tuple:
    """``int4_linear`` with a norm weight, and ``lm.conv1d_silu_step`` on its columns conv_col .. conv_col + C, in one launch up to
    K = 1024, as ``lm.skinny_linear_conv_step`` does it: x (M, K) -> (product (M, N), conv output (M, C)), window (M, taps - 1, C) bf16
    updated in place.  The same bits as the two calls."""
    return _native().int4_linear_conv_step(x, weight.words, weight.scales, weight.out_features, weight.in_features,
                                           weight.group_size, bias, norm_weight, eps, conv_col, window, conv_weight, conv_bias)
