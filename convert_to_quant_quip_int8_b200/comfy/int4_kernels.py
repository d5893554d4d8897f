"""Operators on weights of 4 bits with group scales.

The reference stops at int8; these are the same steps one precision lower, for
models whose weights have to be read once per token:

* ``weight_quant_int4`` / ``weight_dequant_int4``  a weight to codes and scales and back
* ``int4_linear``                                  linear layer, any number of tokens
* ``moe_int4``                                     mixture-of-experts layer for a few tokens

A weight [..., N, K] is held as ``q`` uint8 [..., N, Kp/2] and ``scale`` bf16
[..., N, Kp/group_size], Kp being K rounded up to whole 128s (the order of the
codes: include/qi8.h).  Scales have at most five significant bits, so that
code * scale is exact in bf16.  Activations are bf16 or fp16 and stay so (no
activation quantization); sums are fp32.  Inference only: inputs, scales among
them, that require a gradient are refused while gradients are enabled, and such
that carry a forward-mode tangent always (the quantizer reads a parameter as it
is).
"""

from typing import Optional, Tuple

import torch

from .. import _lib as L
from .. import ops

_ACTS = {"silu": L.QI8_ACT_SILU, "gelu": L.QI8_ACT_GELU}


def weight_quant_int4(w: torch.Tensor, group_size: int = 128) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(q, scale)`` of ``w`` [..., N, K] (bf16, fp16 or fp32): per group of ``group_size`` (32, 64 or 128) input
    features ``scale = amax / 7`` to five significant bits, ``code = rint(w / scale)``.  A group that holds an
    infinity or a NaN reads back as NaN."""
    return ops.quant_weight_i4(w, group_size)


def weight_dequant_int4(q: torch.Tensor, scale: torch.Tensor, in_features: int, group_size: int = 128,
                        output_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The weight [..., N, in_features] that ``q`` and ``scale`` stand for."""
    if output_dtype is None:
        output_dtype = torch.get_default_dtype()
    return ops.dequant_i4(q, scale, in_features, group_size, output_dtype)


def int4_linear(x: torch.Tensor, q: torch.Tensor, scale: torch.Tensor, group_size: int = 128,
                bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x [..., K] W^T + bias`` in x's dtype (bf16 or fp16), ``W`` [N, K] in 4 bits."""
    return ops.gemm_w4(x, q, scale, group_size, bias)


def moe_int4(x: torch.Tensor, router: torch.Tensor, w13: torch.Tensor, w13_scale: torch.Tensor, w2: torch.Tensor,
             w2_scale: torch.Tensor, top_k: int, group_size: int = 128, renormalize: bool = True,
             activation: str = "silu") -> torch.Tensor:
    """Mixture-of-experts layer: ``y = sum_e p_e W2_e (act(G_e x) * (U_e x))`` over the ``top_k`` experts with the
    largest router logits ``x router^T`` (equal ones: lowest expert first), ``p = softmax(logits)`` on them, divided
    by their sum with ``renormalize``.

    ``router`` [E, H] in x's dtype or fp32; ``w13``/``w13_scale`` 4-bit [E, 2 I, H], gate rows above up rows;
    ``w2``/``w2_scale`` 4-bit [E, H, I]; ``activation`` "silu" or "gelu" (erf).  E <= 1024, top_k <= min(E, 64).
    Meant for a few tokens: they run 64 at a time.
    """
    if activation not in _ACTS:
        raise ValueError(f"activation must be 'silu' or 'gelu', got {activation!r}")
    return ops.moe_w4(x, router, w13, w13_scale, w2, w2_scale, top_k, group_size, renormalize, _ACTS[activation])
