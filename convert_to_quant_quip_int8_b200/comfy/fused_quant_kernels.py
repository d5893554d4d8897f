"""Producers of quantized activations: what stands before a quantized linear
layer, in one pass with the quantization.

* ``rms_norm_quant``   root-mean-square norm, with the residual's addition
* ``gated_act_quant``  ``act(gate) * up`` of a gated feed-forward

``output`` says which product reads the result:

* ``"fp8"``         codes and scales of ``fp8_kernels.act_quant_fp8``, for ``fp8_gemm``
* ``"int8"``        one scale per row, for the tensor- and axis-wise layers (``ops.gemm_i8``)
* ``"int8_block"``  one scale per row and 128 columns, for ``int8_kernels.int8_gemm``

int8 codes are rounded to nearest, in ``"int8_block"`` too, where
``int8_kernels.act_quant`` truncates like the reference does.  Between the inputs
and the codes nothing is rounded to 16 bits but the residual's sum, which is
returned.  Inference only, like the other operators of this package.
"""

from typing import Optional, Tuple, Union

import torch

from .. import _lib as L
from .. import ops

_MODES = {"fp8": L.QI8_Q_FP8, "int8": L.QI8_Q_TOKEN, "int8_block": L.QI8_Q_BLOCK}
_ACTS = {"silu": L.QI8_ACT_SILU, "gelu": L.QI8_ACT_GELU, "gelu_tanh": L.QI8_ACT_GELU_TANH}


def _choice(table: dict, what: str, name: str) -> int:
    if name not in table:
        raise ValueError(f"{what} must be one of {sorted(table)}, got {name!r}")
    return table[name]


def rms_norm_quant(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                   residual: Optional[torch.Tensor] = None, output: str = "fp8"
                   ) -> Union[Tuple[torch.Tensor, torch.Tensor], Tuple[torch.Tensor, torch.Tensor, torch.Tensor]]:
    """``(q, scale)`` of ``h / sqrt(mean(h^2) + eps) * weight`` over the last dimension; with ``residual``
    ``h = x + residual``, rounded to x's dtype, and the result is ``(q, scale, h)``.  ``eps`` 0 (a row of zeros
    is NaN then) or at least 1e-37."""
    return ops.rms_norm_quant(x, weight, eps, residual, _choice(_MODES, "output", output))


def gated_act_quant(gate: torch.Tensor, up: torch.Tensor, activation: str = "silu",
                    output: str = "fp8") -> Tuple[torch.Tensor, torch.Tensor]:
    """``(q, scale)`` of ``act(gate) * up``; ``activation`` "silu", "gelu" (erf) or "gelu_tanh".  ``gate`` and ``up``
    may be the halves of one tensor."""
    return ops.gated_quant(gate, up, _choice(_ACTS, "activation", activation), _choice(_MODES, "output", output))
