"""CPU tests of the fp8 path and of the fused producers: the oracle's format, and the refusals that need no device."""

import numpy as np
import pytest
import torch

import oracle as O
from convert_to_quant_quip_int8_b200 import _lib as L
from convert_to_quant_quip_int8_b200 import ops
from convert_to_quant_quip_int8_b200.comfy import fp8_kernels as F8
from convert_to_quant_quip_int8_b200.comfy import fused_quant_kernels as FQ
from convert_to_quant_quip_int8_b200.comfy import quant_ops as Q

E4, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def test_oracle_rounds_like_the_type():
    # every code, every midpoint and its neighbours
    codes = torch.arange(0, 127, dtype=torch.uint8).view(E4).double()
    mid = (codes[1:] + codes[:-1]) / 2
    v = torch.cat([codes, mid, mid * (1 + 2.0 ** -20), mid * (1 - 2.0 ** -20)])
    v = torch.cat([v, -v])
    assert np.array_equal(O.f8_round(v.numpy()), v.float().to(E4).double().numpy())


def test_scale_is_the_smallest_that_holds_the_block():
    amax = np.array([448.0, 448.0 * (1 + 2 ** -23), 1.0, 1.75, 1.7500001, 1e-38, 0.0, 3e38, np.inf, np.nan])
    s = O.f8_scale(amax)
    assert np.isnan(s[-2:]).all()
    s, amax = s[:-2], amax[:-2]
    assert (amax <= 448 * s).all() and ((amax > 448 * s / 2) | (s == 2.0 ** -100)).all()
    assert s[0] == 1 and s[1] == 2 and s[5] == s[6] == 2.0 ** -100


def test_quantize_ragged_blocks():
    rng = np.random.default_rng(0)
    v = rng.standard_normal((130, 200))
    for tile, shape in ((1, (130, 2)), (128, (2, 2))):
        q, s = O.f8_quantize(v, tile)
        assert s.shape == shape and np.abs(q).max() <= 448
        # half a step of a normal number, or of a subnormal one
        tol = np.maximum(2.0 ** -4 * np.abs(v), 2.0 ** -10 * O.f8_values(np.ones_like(q), s, tile))
        assert (np.abs(O.f8_values(q, s, tile) - v) <= tol).all()


def _operands(m=3, n=130, k=200):
    return (torch.zeros(m, k).to(E4), torch.zeros(m, 2, dtype=torch.uint8).view(E8),
            torch.zeros(n, k).to(E4), torch.zeros(2, 2, dtype=torch.uint8).view(E8))


def test_wrappers_reject_cpu_tensors():
    a, a_s, b, b_s = _operands()
    x = torch.zeros(3, 200, dtype=torch.bfloat16)
    w = Q.QuantizedTensor(b, "BlockWiseFP8Layout", {"scale": b_s, "block_size": 128, "is_weight": True,
                                                    "orig_dtype": torch.bfloat16})
    for call in (lambda: F8.act_quant_fp8(x), lambda: F8.weight_quant_fp8(x), lambda: F8.act_dequant_fp8(a, a_s),
                 lambda: F8.weight_dequant_fp8(b, b_s), lambda: F8.fp8_gemm(a, a_s, b, b_s),
                 lambda: F8.fp8_linear(x, b, b_s), lambda: FQ.rms_norm_quant(x), lambda: FQ.gated_act_quant(x, x),
                 lambda: torch.nn.functional.linear(x, w)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_format_checks():
    a, a_s, b, b_s = _operands()
    ops._check_f8(a, a_s, 1)
    ops._check_f8(b, b_s, 128)
    for q, s, tile in ((a, b_s, 1), (b, a_s, 128), (a, a_s[:, :1], 1), (b[None], b_s[None], 128), (b[:128], b_s, 128)):
        with pytest.raises(AssertionError):
            ops._check_f8(q, s, tile)
    with pytest.raises(AssertionError, match="contiguous"):
        ops._check_f8(torch.zeros(2, 200).to(E4), a_s[:2].t(), 1)
    for q, s in ((a.float(), a_s), (a, a_s.float()), (a.to(torch.float8_e5m2), a_s), (a, a_s.view(torch.uint8))):
        with pytest.raises(TypeError):
            ops._check_f8(q, s, 1)


def test_choices_by_name():
    with pytest.raises(ValueError, match="int8_block"):
        FQ.rms_norm_quant(None, output="int4")
    with pytest.raises(ValueError, match="gelu_tanh"):
        FQ.gated_act_quant(None, None, activation="relu")
    for f in (F8.act_quant_fp8, F8.weight_quant_fp8):
        with pytest.raises(NotImplementedError):
            f(None, block_size=64)


def test_code_rows_start_on_16_bytes():
    for shape in ((3, 200), (2, 5, 16), (4, 1), (0, 7), (3, 0)):
        q = ops._new_codes(shape, E4, "cpu")
        assert tuple(q.shape) == shape
        if q.numel():
            q2, ld = ops._code_rows(q)
            assert ld == -(-shape[-1] // 16) * 16 and q2.data_ptr() == q.data_ptr()
            assert q2.shape[0] == q.numel() // shape[-1]


def test_row_strides():
    x = torch.zeros(6, 40)
    assert ops._strided_rows(x[:, :30])[1] == 40
    assert ops._strided_rows(x[::2])[1] == 80
    y, ld = ops._strided_rows(x.t())
    assert ld == 6 and y.is_contiguous()
    y, ld = ops._strided_rows(x[:1].expand(6, 40))  # rows that overlap
    assert ld == 40 and y.is_contiguous()
    assert ops._strided_rows(x.view(2, 3, 40)[:, :2])[1] == 40
    assert ops._strided_rows(x[0, :30])[1] >= 30
    assert ops._strided_rows(torch.zeros(5, 2)[:, :1])[1] >= 1


def test_layout_is_registered():
    assert Q.LAYOUTS[Q.QUANT_ALGOS["float8_blockwise"]["comfy_tensor_layout"]] is Q.BlockWiseFP8Layout


def test_layout_refuses_lost_writes():
    _, _, b, b_s = _operands()
    w = Q.QuantizedTensor(b, "BlockWiseFP8Layout", {"scale": b_s, "block_size": 128, "is_weight": True,
                                                    "orig_dtype": torch.bfloat16})
    with pytest.raises(RuntimeError, match="packed"):
        w.add_(1.0)
    with pytest.raises(TypeError):
        w.copy_(torch.zeros(130, 200))


def test_c_entries_fail_without_a_device():
    lib = L.load()
    assert lib.qi8_quant_rows_f8(None, 0, 1, 128, 128, None, 128, None, None) == L.QI8_EUNSUPPORTED
    assert lib.qi8_quant_weight_f8(None, 0, 1, 128, 128, None, 128, None, None) == L.QI8_EUNSUPPORTED
    assert lib.qi8_dequant_f8(None, 1, 128, 128, None, 1, None, 0, 128, None) == L.QI8_EUNSUPPORTED
    assert lib.qi8_gemm_f8(None, None, 1, 128, 128, None, None, 1, 128, None, 0, None, 0, 1, None, 0,
                           None) == L.QI8_EUNSUPPORTED
    assert lib.qi8_linear_f8(None, 0, 1, 128, 128, None, None, 1, 128, None, 0, None, 0, 1, None, 0,
                             None) == L.QI8_EUNSUPPORTED
    assert lib.qi8_rms_norm_quant(None, 0, 1, 128, 128, None, 0, None, 0, 1e-6, 2, None, 128, None, None, 0,
                                  None) == L.QI8_EUNSUPPORTED
    assert lib.qi8_gated_quant(None, 128, None, 128, 0, 1, 128, 2, 2, None, 128, None, None) == L.QI8_EUNSUPPORTED
    assert "sm_100" in L.last_error()
