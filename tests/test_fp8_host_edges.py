"""CPU tests of the fp8 operators' host side at its edges: tangents, metadata, layouts and the schedule of a kernel."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from convert_to_quant_quip_int8_b200 import ops
from convert_to_quant_quip_int8_b200.comfy import fp8_kernels as F8
from convert_to_quant_quip_int8_b200.comfy import fused_quant_kernels as FQ
from convert_to_quant_quip_int8_b200.comfy.quant_ops import QUANT_ALGOS, QuantizedTensor
from convert_to_quant_quip_int8_b200.utils import comfy_quant as CQ

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


def test_codes_get_rows_of_whole_16_bytes():
    q = torch.arange(7 * 40, dtype=torch.uint8).view(7, 40)
    for v in (q, q[:, 3:], q[:, :33], q[1:2, 5:], q.t(), q[:0], q[:, :0], q[:, 7:8]):
        c = v.contiguous().view(torch.float8_e4m3fn)
        for t in (c, v.view(torch.float8_e4m3fn)):
            a = ops.aligned_codes(t)
            assert a.shape == t.shape and torch.equal(a.view(torch.uint8), t.view(torch.uint8))
            if a.numel():
                assert a.storage_offset() % 16 == 0 and (a.shape[0] == 1 or a.stride(0) % 16 == 0)
            assert ops.aligned_codes(a) is a
    for v in (q[0], q.view(7, 2, 20), q.view(7, 1, 40)[:, :, :7], q[0, 3:]):  # no weights, but no error here either
        t = v.view(torch.float8_e4m3fn)
        assert torch.equal(ops.aligned_codes(t).view(torch.uint8), v)
    whole = torch.zeros(3, 48, dtype=torch.uint8).view(torch.float8_e4m3fn)
    assert ops.aligned_codes(whole) is whole
    assert ops.aligned_codes(whole[:, :33]).data_ptr() == whole.data_ptr()


@pytest.mark.parametrize("layout,code", [("BlockWiseFP8Layout", torch.float8_e4m3fn), ("TensorWiseINT8Layout", torch.int8)])
def test_a_transfer_keeps_the_type_that_is_dequantized_to(layout, code):
    t = QuantizedTensor(torch.zeros(4, 256).to(code), layout, {"scale": torch.zeros(1), "orig_dtype": BF,
                                                               "block_size": 128, "is_weight": True})
    assert t.to("meta")._layout_params["orig_dtype"] == BF
    assert t.to("meta", torch.float16)._layout_params["orig_dtype"] == torch.float16


def test_metadata_keeps_the_block_size():
    for name, algo in QUANT_ALGOS.items():
        size = algo.get("group_size", 128)
        meta = CQ.tensor_to_dict(CQ.create_comfy_quant_tensor(name, block_size=size))
        assert meta == ({"format": name, "group_size": size} if "group_size" in algo else {"format": name})


def test_rows_of_no_columns_have_the_least_scale(monkeypatch):
    monkeypatch.setattr(ops, "_one_device", lambda *t: torch.device("cpu"))  # nothing is launched
    torch.full((3 * 5,), 7.0)  # memory that a fresh tensor may get
    x = torch.empty(3, 5, 0, dtype=BF)
    for got in (FQ.rms_norm_quant(x, output="int8"), FQ.gated_act_quant(x, x, output="int8")):
        assert got[0].shape == x.shape and got[1].shape == (3, 5, 1) and (got[1] == torch.tensor(1e-30)).all()
    for output in ("fp8", "int8_block"):
        assert FQ.gated_act_quant(x, x, output=output)[1].shape == (3, 5, 0)
