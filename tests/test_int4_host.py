"""CPU tests of the 4-bit weight path: the oracle's format and the refusals that need no device."""

import numpy as np
import pytest
import torch

import oracle as O
from convert_to_quant_quip_int8_b200 import _lib as L
from convert_to_quant_quip_int8_b200 import ops
from convert_to_quant_quip_int8_b200.comfy import int4_kernels as I4
from convert_to_quant_quip_int8_b200.comfy import quant_ops as Q


@pytest.mark.parametrize("k,group", [(1, 32), (77, 64), (128, 128), (300, 32)])
def test_pack_unpack_and_exact_products(k, group):
    rng = np.random.default_rng(k)
    w = rng.standard_normal((5, k)) * 0.02
    codes, scale = O.i4_quantize(w, group)
    q = O.i4_pack(codes)
    assert q.shape == (5, O.i4_padded(k) // 2)
    assert np.array_equal(O.i4_unpack(q), codes)
    assert np.abs(codes).max() <= 7 and not codes[:, k:].any()
    v = O.i4_values(q, scale, k, group)
    # five significant bits times three: exact in bf16
    assert np.array_equal(O.round_bf16(v.astype(np.float32)).astype(np.float64), v)
    # at most half a step off; 7 / (1 - 1/33) = 7.22: the largest by a quarter step
    assert (np.abs(v - w) <= 0.5 * np.repeat(scale, group, 1)[:, :k] + 1e-300).all()


def test_positions_are_a_permutation():
    byte, shift = O.i4_positions(256)
    assert len(set(zip(byte.tolist(), shift.tolist()))) == 256 and byte.max() == 127
    # feature 0 is the lowest nibble of byte 0; feature 1 the fifth nibble of its word; 32 starts word 1
    assert (byte[0], shift[0]) == (0, 0) and (byte[1], shift[1]) == (2, 0) and (byte[32], shift[32]) == (4, 0)
    assert (byte[8], shift[8]) == (16, 0)


def test_non_finite_groups_and_zeros():
    w = np.zeros((1, 128))
    w[0, 3], w[0, 40] = np.inf, np.nan
    codes, scale = O.i4_quantize(w, 32)
    assert np.isnan(scale[0, :2]).all() and (scale[0, 2:] == 2.0 ** -100).all() and not codes.any()


def _weight(n=16, k=256, group=128):
    return (torch.zeros(n, k // 2, dtype=torch.uint8), torch.zeros(n, k // group, dtype=torch.bfloat16))


def test_wrappers_reject_cpu_tensors():
    q, s = _weight()
    x = torch.zeros(2, 256, dtype=torch.bfloat16)
    for call in (lambda: I4.weight_quant_int4(torch.zeros(4, 128)), lambda: I4.weight_dequant_int4(q, s, 256),
                 lambda: I4.int4_linear(x, q, s), lambda: torch.nn.functional.linear(x, Q.QuantizedTensor(
                     q, "GroupWiseINT4Layout", {"scale": s, "group_size": 128, "in_features": 256,
                                                "orig_dtype": torch.bfloat16})),
                 lambda: I4.moe_int4(x, torch.zeros(4, 256), torch.stack([q] * 4), torch.stack([s] * 4), q, s, 2)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_format_checks():
    q, s = _weight()
    ops._check_i4(q, s, 256, 128, 2)
    ops._check_i4(q, s, 129, 128, 2)
    for k, group, dims in ((257, 128, 2), (128, 128, 2), (256, 64, 2), (256, 48, 2), (256, 128, 3)):
        with pytest.raises(AssertionError):
            ops._check_i4(q, s, k, group, dims)
    with pytest.raises(AssertionError):
        ops._check_i4(q[:, ::2], s, 128, 128, 2)
    with pytest.raises(AssertionError):
        ops._check_i4(q[1:], s, 256, 128, 2)
    with pytest.raises(TypeError):
        ops._check_i4(q.to(torch.int8), s, 256, 128, 2)
    with pytest.raises(TypeError):
        ops._check_i4(q, s.float(), 256, 128, 2)


def test_gradients_are_refused():
    x = torch.zeros(2, 2, requires_grad=True)
    with pytest.raises(RuntimeError, match="backward"):
        ops._no_grad(None, x)
    with torch.no_grad():
        ops._no_grad(x)
    ops._no_grad(x.detach())


def test_activation_name():
    with pytest.raises(ValueError, match="silu"):
        I4.moe_int4(None, None, None, None, None, None, 1, activation="relu")


def test_layout_is_registered():
    assert Q.LAYOUTS[Q.QUANT_ALGOS["int4_groupwise"]["comfy_tensor_layout"]] is Q.GroupWiseINT4Layout


def test_workspace_refuses_bad_sizes():
    f = L.load().qi8_moe_w4_workspace_bytes
    assert f(5, 256, 8, 64, 2) > 0
    for t, h, e, i, k in ((5, 0, 8, 64, 2), (5, 256, 0, 64, 1), (5, 256, 8, 64, 9), (5, 256, 8, 64, 0),
                          (5, 256, 1025, 64, 2), (5, 256, 128, 64, 65), (-1, 256, 8, 64, 2)):
        assert f(t, h, e, i, k) == 0
        assert L.last_error()


def test_route_breaks_ties_by_index():
    p = O.moe_route(np.array([[1.0, 3.0, 3.0, 3.0, 0.0]]), 2, True)
    assert np.array_equal(p, [[0, 0.5, 0.5, 0, 0]])
