"""GPU tests of the fp8 operators where their kernels, layouts and launches change over."""

import pytest
import torch
import torch.nn.functional as F

from convert_to_quant_quip_int8_b200 import _lib as L
from convert_to_quant_quip_int8_b200 import ops
from convert_to_quant_quip_int8_b200.comfy import fp8_kernels as F8
from convert_to_quant_quip_int8_b200.comfy.quant_ops import QuantizedTensor
from test_gpu_fp8 import randn

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _status():
    yield
    ops.device_status(reset=True)


@pytest.mark.parametrize("k", [200, 256, 333])
def test_copies_of_a_weight_keep_rows_that_products_take(k):
    x, w = randn(5, k, dtype=BF), randn(130, k, seed=1, scale=0.02, dtype=BF)
    wq = QuantizedTensor.from_float(w, "BlockWiseFP8Layout", is_weight=True)
    codes = wq._qdata.cpu().contiguous().cuda()  # as they come from a file
    reload = QuantizedTensor(codes, "BlockWiseFP8Layout", dict(wq._layout_params))
    expected = F.linear(x, wq)
    copied = wq.clone()
    copied.copy_(reload)
    for t in (wq, wq.clone(), wq.cpu().cuda(), reload, wq.detach(), torch.empty_like(wq).copy_(wq), copied):
        q = t._qdata
        assert q.is_cuda and L.load().qi8_gemm_f8_workspace_bytes(q.data_ptr(), 130, k, q.stride(0), q.data_ptr(), 130,
                                                                   q.stride(0)) == 0
        assert torch.equal(F.linear(x, t), expected) and torch.equal(t.dequantize(), wq.dequantize())
    assert wq.detach()._qdata.data_ptr() == wq._qdata.data_ptr()
    assert wq.cpu()._qdata.is_contiguous()
