"""CPU tests of the fp8 operators' host side at its edges: tangents, metadata, layouts and the schedule of a kernel."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from convert_to_quant_quip_int8_b200 import ops
from convert_to_quant_quip_int8_b200.comfy import fp8_kernels as F8
from convert_to_quant_quip_int8_b200.comfy import fused_quant_kernels as FQ

BF = torch.bfloat16


@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(monkeypatch, grad):
    monkeypatch.setattr(ops, "_one_device", lambda *t: torch.device("cpu"))  # past the check of the device
    x = torch.ones(4, 256, dtype=BF)
    with torch.set_grad_enabled(grad), fwd.dual_level():
        d = fwd.make_dual(x, torch.ones_like(x))
        for f in (F8.weight_quant_fp8, F8.act_quant_fp8, FQ.rms_norm_quant, lambda t: FQ.gated_act_quant(x, t)):
            with pytest.raises(RuntimeError, match="forward mode"):
                f(d)
