"""Operators on fp8 operands with block scales.

The reference's block-wise path (comfy/int8_kernels.py) in 8-bit floating
point, with the same blocks: 128 columns of a row for activations, 128 x 128
tiles for weights.

* ``act_quant_fp8`` / ``act_dequant_fp8``        activations and back
* ``weight_quant_fp8`` / ``weight_dequant_fp8``  weights and back
* ``fp8_gemm``                                   product of quantized operands
* ``fp8_linear``                                 linear layer: quantizes its input

Codes are ``float8_e4m3fn``, scales ``float8_e8m0fnu``: powers of two, the
smallest for which a block's largest value is at most 448 times its scale (and at
least 2^-100).  Dividing by one is exact, so a code is a single rounding away from
its value.  The last block of a row or column may be smaller; rows of codes lie
whole 16 bytes apart in memory, so codes of rows of another length are a view
(contiguous ones are taken too, at the cost of a copy per product).  A block with
an infinity or a NaN reads back as NaN as a whole.  Sums are fp32.  Inference
only: inputs that require a gradient are refused while gradients are enabled, and
such that carry a forward-mode tangent always (``weight_quant_fp8`` reads a
parameter as it is).
"""

from typing import Optional, Tuple

import torch

from .. import ops


def _block(block_size: int) -> None:
    if block_size != 128:
        raise NotImplementedError(f"fp8 scales cover blocks of 128, got block_size={block_size}")


def act_quant_fp8(x: torch.Tensor, block_size: int = 128) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(q [..., n], scale [..., ceil(n / 128)])`` of ``x`` (bf16, fp16 or fp32)."""
    _block(block_size)
    return ops.quant_rows_f8(x)


def act_dequant_fp8(q: torch.Tensor, scale: torch.Tensor, block_size: int = 128,
                    output_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The activations that ``q`` and ``scale`` stand for."""
    _block(block_size)
    return ops.dequant_f8(q, scale, 1, output_dtype or torch.get_default_dtype())


def weight_quant_fp8(w: torch.Tensor, block_size: int = 128) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(q [N, K], scale [ceil(N / 128), ceil(K / 128)])`` of ``w`` (bf16, fp16 or fp32)."""
    _block(block_size)
    return ops.quant_weight_f8(w)


def weight_dequant_fp8(q: torch.Tensor, scale: torch.Tensor, block_size: int = 128,
                       output_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The weight [N, K] that ``q`` and ``scale`` stand for."""
    _block(block_size)
    return ops.dequant_f8(q, scale, 128, output_dtype or torch.get_default_dtype())


def fp8_gemm(a: torch.Tensor, a_s: torch.Tensor, b: torch.Tensor, b_s: torch.Tensor,
             bias: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``A B^T + bias``: ``a`` [..., K] and ``a_s`` as from ``act_quant_fp8`` (or a producer in
    ``fused_quant_kernels``), ``b`` [N, K] and ``b_s`` as from ``weight_quant_fp8``."""
    return ops.gemm_f8(a, a_s, b, b_s, bias, out_dtype)


def fp8_linear(x: torch.Tensor, w: torch.Tensor, w_s: torch.Tensor,
               bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``fp8_gemm(*act_quant_fp8(x), w, w_s, bias)`` in x's dtype, from one token on."""
    return ops.linear_f8(x, w, w_s, bias)
