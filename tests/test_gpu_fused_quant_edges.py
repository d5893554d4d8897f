"""GPU tests of the quantized gate at far values and of the int8 read-back of short rows."""

import math

import pytest
import torch

from convert_to_quant_quip_int8_b200 import _lib as L
from convert_to_quant_quip_int8_b200 import ops
from convert_to_quant_quip_int8_b200.comfy import fused_quant_kernels as FQ
from convert_to_quant_quip_int8_b200.comfy.quant_ops import QuantizedTensor
from test_gpu_fused_quant import check_codes, exact_gated, randn

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _status():
    yield
    ops.device_status(reset=True)


# --------------------------------------------------------------- read-back
@pytest.mark.parametrize("rows,n", [(1, 1), (5, 1), (1000, 3), (7, 8), (301, 31), (33, 32), (40, 33), (30, 47), (30, 49), (3, 255), (9, 264)])
@pytest.mark.parametrize("out", [BF, HF, F32])
def test_short_rows_read_back(rows, n, out):
    g = torch.Generator().manual_seed(rows + n)
    q = torch.randint(-128, 128, (rows, n), dtype=torch.int8, generator=g).cuda()
    s = torch.rand(rows, 1, generator=g).cuda()
    assert torch.equal(ops.dequant(q, s, L.QI8_S_ROW, out_dtype=out), (q.float() * s).to(out))
    assert torch.equal(ops.dequant(q, s[:1], L.QI8_S_SCALAR, out_dtype=out), (q.float() * s[0]).to(out))
    off = torch.empty(rows * n + 1, dtype=torch.int8, device="cuda")[1:].view(rows, n).copy_(q)  # off any boundary
    assert torch.equal(ops.dequant(off, s, L.QI8_S_ROW, out_dtype=out), (q.float() * s).to(out))
    assert torch.equal(ops.dequant(off, s[:1], L.QI8_S_SCALAR, out_dtype=out), (q.float() * s[0]).to(out))


def _us(f):
    """The fastest of a few runs: other work on the machine only adds to it."""
    times = []
    for _ in range(8):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        f()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b) * 1e3)
    return min(times)


@pytest.mark.parametrize("n", [1, 4, 16])
def test_short_rows_are_not_slow(n):
    # one scale per row as one block per row is the element-wise kernel; a warp for each row took 2 to 25 times as long
    rows = 4000000
    q = torch.ones(rows, n, dtype=torch.int8, device="cuda")
    s = torch.ones(rows, 1, device="cuda")
    elements = _us(lambda: ops.dequant(q, s, L.QI8_S_ROW_KBLOCK, n, BF))
    assert _us(lambda: ops.dequant(q, s, L.QI8_S_ROW, out_dtype=BF)) < 1.5 * elements
    assert _us(lambda: ops.dequant(q, s[:1], L.QI8_S_SCALAR, out_dtype=BF)) < 1.5 * elements


def test_one_scale_for_more_than_32_bits_of_values():
    q = torch.ones(1 << 16, (1 << 15) + 1, dtype=torch.int8, device="cuda")
    q[-1, -3:] = torch.tensor([5, -6, 7], dtype=torch.int8)
    s = torch.full((1,), 0.5, device="cuda")
    v = ops.dequant(q, s, L.QI8_S_SCALAR, out_dtype=BF)
    assert v[-1, -4:].tolist() == [0.5, 2.5, -3.0, 3.5] and v[0, 0] == 0.5 and (v[1234] == 0.5).all()


# ------------------------------------------------------------- far gates
def far_gated(g, u, act):
    """exact_gated, where act itself may be small.  Up to t = 92.1 the quotient is taken, and its rounding off by 2^-149
    at most, which counts |u| times; from there on act is under 2^-126 and may be 0."""
    y, _ = exact_gated(g, u, act)
    g, u = g.double(), u.double().abs()
    t = -g if act == "silu" else -2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)
    near = t < 92.1
    # the argument's rounding counts |t| times, that of u in the tanh form four units
    rel = 4 * (4 + t.abs() * (1 if act == "silu" else 4)) * 2.0 ** -24
    return y, rel * y.abs() + torch.where(near, 2.0 ** -148, 2.0 ** -126) * u


@pytest.mark.parametrize("output", ["fp8", "int8", "int8_block"])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_gates_as_far_as_results_are_normal_numbers(act, output):
    # 1 + exp(t) passes 2^126 from t = 87.3 on, where act is a normal number down to t = 91.9 (silu) and 89.7 (tanh)
    if act == "silu":
        g = -torch.cat([torch.linspace(80, 91.8, 60), torch.tensor([87.5, 88.0, 88.5, 95.0, 300.0])])
    else:
        g = -torch.cat([torch.linspace(9.7, 10.1, 60), torch.tensor([10.02, 10.05, 10.4, 11.0, 300.0])])
    g = g.cuda()[:, None].expand(-1, 256).contiguous()
    u = randn(*g.shape, seed=1) * 1e30
    q, s = FQ.gated_act_quant(g, u, activation=act, output=output)
    check_codes(q, s, *far_gated(g, u, act), output)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("output", ["fp8", "int8", "int8_block"])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("sign", [-1, 1])
def test_gates_of_one_size(act, output, dtype, sign):
    # each row's gates are near one value, so that its scale follows them into the tail
    centre = torch.tensor([0.02, 0.3, 1.0, 2.0, 3.0, 4.0, 5.0, 6.0, 8.0, 10.0, 12.0])
    g = sign * (centre.cuda()[:, None] * (1 + 0.02 * randn(11, 384, seed=2))).to(dtype)
    u = randn(11, 384, seed=3, dtype=dtype) * (1.0 if dtype == HF else 2.0 ** 60)
    q, s = FQ.gated_act_quant(g, u, activation=act, output=output)
    check_codes(q, s, *far_gated(g, u, act), output)


# The error of x Phi(x) = max(x, 0) - |x| h, h = exp(-x^2 / 2) t p(t), t = 1 / (1 + 0.27 |x|), in units of 2^-24: of
# x^2 / 2 three (square, constant, product), which count x^2 / 2 times; exp2 four; t five, which count up to three
# times in t p(t); p's steps five, the fit one, three products and the difference: under 32 + 2 x^2 of |x| h, and two
# of the result.
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("output", ["fp8", "int8", "int8_block"])
@pytest.mark.parametrize("sign", [-1, 1])
def test_gelu_of_gates_of_one_size(output, dtype, sign):
    centre = torch.tensor([0.02, 0.3, 1.0, 2.0, 3.0, 4.0, 5.0, 6.0, 8.0, 10.0, 12.0])
    g = sign * (centre.cuda()[:, None] * (1 + 0.02 * randn(11, 384, seed=2))).to(dtype)
    u = randn(11, 384, seed=3, dtype=dtype) * (1.0 if dtype == HF else 2.0 ** 60)
    q, s = FQ.gated_act_quant(g, u, activation="gelu", output=output)
    y, _ = exact_gated(g, u, "gelu")
    x = g.double().abs()
    h = 0.5 * torch.special.erfc(x / math.sqrt(2))
    check_codes(q, s, y, 2.0 ** -24 * ((32 + 2 * x * x) * x * h * u.double().abs() + 2 * y.abs()), output)


# ------------------------------------------------- outputs into int8 layouts
@pytest.mark.parametrize("rows", [1, 130])
def test_block_outputs_go_into_linear_layers(rows):
    x, w = randn(rows, 512, dtype=BF), randn(256, 512, seed=1, scale=0.05, dtype=BF)
    bias = randn(256, seed=2, dtype=BF)
    for layout, output in (("BlockWiseINT8Layout", "int8_block"), ("BlockWiseFP8Layout", "fp8")):
        wq = QuantizedTensor.from_float(w, layout, is_weight=True)
        q, s = FQ.rms_norm_quant(x, output=output)
        a = QuantizedTensor(q, layout, {"scale": s, "block_size": 128, "is_weight": False, "orig_dtype": x.dtype})
        y = torch.nn.functional.linear(a, wq, bias)
        va, vw = a.dequantize().double(), wq.dequantize().double()
        # a and w are rounded to bf16 where they are read back, y once; the sums are fp32
        total = va.abs() @ vw.abs().T + bias.double().abs()
        assert y.dtype == BF
        assert ((y.double() - va @ vw.T - bias.double()).abs() <= (3 * 2.0 ** -8 + 2.0 ** -14) * total).all()
