"""GPU tests of the quantized norm and gated activation against plain forms in 64 bits.

y is computed in fp32, so that a code may differ from the exact one's next to a
border.  What is checked: the scale is that of a maximum within DELTA of the exact
one, and code * scale is at most half a step, plus the error of y, off the exact
value.

The error of y, in units of 2^-24 of it: the sum of squares adds at most 128 values
in a row per thread and 15 in two trees, each addition one unit, which the root
halves; the root and its use two roundings, the weight one more: under 80.  The
gate: exp 2 units in the last place and its argument's rounding, which counts
|t| times; sum, division, product.  4 (4 + |t|) 2^-24 covers them, with t = g or
the tanh form's 2 u, whose own rounding (4 units) is |t| times that.  erf is off by
2 units of 1, which counts absolutely: |g| 2^-22.
"""

import math

import numpy as np
import pytest
import torch

import oracle as O
from convert_to_quant_quip_int8_b200 import _lib as L
from convert_to_quant_quip_int8_b200 import ops
from convert_to_quant_quip_int8_b200.comfy import fp8_kernels as F8
from convert_to_quant_quip_int8_b200.comfy import fused_quant_kernels as FQ
from convert_to_quant_quip_int8_b200.comfy import int8_kernels as I8

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
DELTA = 80 * 2.0 ** -24


def randn(*shape, seed=0, scale=1.0, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def blocks_of(v):
    """[rows, n] -> [rows, blocks, 128] with zeros behind the end."""
    return torch.nn.functional.pad(v, (0, -v.shape[1] % 128)).unflatten(1, (-1, 128))


def check_codes(q, s, y, tol, output):
    """Codes and scales [rows, n] against fp64 values y with error at most tol (elementwise)."""
    rows, n = y.shape
    assert q.shape == y.shape
    one = y.abs().unsqueeze(1) if output == "int8" else blocks_of(y).abs()
    slack = tol.unsqueeze(1) if output == "int8" else blocks_of(tol)
    lo, hi = (one - slack).amax(-1).clamp_min(0), (one + slack).amax(-1)
    sd = s.double().reshape(rows, -1)
    if output == "fp8":
        a, b = (torch.from_numpy(O.f8_scale(t.cpu().numpy())).cuda() for t in (lo, hi))
        assert ((sd == a) | (sd == b)).all()
    else:
        floor = 1e-30 if output == "int8" else 1e-8
        eps = 2.0 ** -23
        assert (sd >= (lo / 127).clamp_min(floor) * (1 - eps)).all() and (sd <= (hi / 127).clamp_min(floor) * (1 + eps)).all()
    full = sd.expand(rows, n) if output == "int8" else sd.repeat_interleave(128, 1)[:, :n]
    v = y / full
    if output == "fp8":
        _, exp = torch.frexp(v)
        half = torch.ldexp(torch.ones_like(v), (exp - 1).clamp_min(-6) - 4)
    else:
        assert q.dtype == torch.int8 and (q >= -127).all()
        half = 0.5 + 127 * 2.0 ** -23  # the reciprocal of the scale and the product with it are rounded
    worst = ((q.double() - v).abs() - half - tol / full).max().item()
    assert worst <= 1e-12, worst


def exact_norm(x, w, eps, residual=None):
    h = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    d = h.double()
    y = d / torch.sqrt(d.square().mean(-1, keepdim=True) + eps)
    return h, y if w is None else y * w.double()


# -------------------------------------------------------------------- norm
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("rows,n", [(1, 1), (1, 4096), (3, 127), (7, 128), (5, 129), (2, 1000), (33, 1451), (300, 256),
                                    (4, 8192), (9, 2560), (2, 16384), (3, 20000), (1, 32768), (2, 40000)])
@pytest.mark.parametrize("output", ["fp8", "int8", "int8_block"])
def test_norm(rows, n, dtype, output):
    if output == "int8_block" and n % 128:
        n = -(-n // 128) * 128
    x = randn(rows, n, seed=n, scale=1.5, dtype=dtype) * torch.exp2(torch.arange(rows, device="cuda") % 7.0 - 3).to(dtype)[:, None]
    w = randn(n, seed=1, dtype=F32 if n % 3 == 0 else dtype)
    r = randn(rows, n, seed=2, scale=3.0, dtype=dtype) if n % 2 == 0 else None
    got = FQ.rms_norm_quant(x, w, eps=1e-5, residual=r, output=output)
    h, y = exact_norm(x, w, 1e-5, r)
    assert len(got) == (2 if r is None else 3)
    if r is not None:
        assert torch.equal(got[2], h)
    check_codes(got[0], got[1], y, DELTA * y.abs(), output)


def test_norm_without_weight_and_with_leading_dimensions():
    x = randn(2, 3, 5, 200, dtype=BF)
    q, s, h = FQ.rms_norm_quant(x, residual=x)
    assert q.shape == x.shape == h.shape and s.shape == (2, 3, 5, 2) and torch.equal(h, x + x)
    _, y = exact_norm((x + x).view(-1, 200), None, 1e-6)
    check_codes(q.reshape(-1, 200), s.view(-1, 2), y, DELTA * y.abs(), "fp8")
    q, s = FQ.rms_norm_quant(x, output="int8")
    assert s.shape == (2, 3, 5, 1) and s.dtype == F32
    for e in (x[:0], x[..., :0]):
        q, s, h = FQ.rms_norm_quant(e, residual=e)
        assert q.shape == e.shape == h.shape
        q, s = FQ.gated_act_quant(e, e, output="int8")
        assert q.shape == e.shape


@pytest.mark.parametrize("dtype", [BF, F32])
def test_norm_takes_strides(dtype):
    big, res = randn(20, 700, dtype=dtype), randn(30, 650, seed=1, dtype=dtype)
    w = randn(1400, seed=2, dtype=dtype)
    for x, r, ww in ((big[:, 3:603], res[:20, :600], w[1:601]), (big[::2, :640], res[10:20, 5:645], w[::2][:640]),
                     (big.t()[:600, :16], None, w[:16]), (big[:1].expand(4, 700), None, w[:700]),
                     (big[:, :600], res[:20, :600], w[:600])):
        got = FQ.rms_norm_quant(x, ww, residual=r)
        _, y = exact_norm(x, ww, 1e-6, r)
        check_codes(got[0], got[1], y, DELTA * y.abs(), "fp8")
        if r is not None:
            assert torch.equal(got[2], (x.double() + r.double()).to(dtype))


def test_norm_of_many_rows_and_broadcast_ones():
    # more rows than resident blocks, several rows per block and one
    for rows, n in ((5000, 256), (2777, 1536), (1500, 4096), (700, 12288), (900, 4099)):
        x, r = randn(rows, n, seed=rows, dtype=BF), randn(rows, n, seed=n, scale=2.0, dtype=BF)
        x[rows // 2] *= 2.0 ** 70
        for output in ("fp8", "int8"):
            q, s, h = FQ.rms_norm_quant(x, residual=r, output=output)
            want, y = exact_norm(x, None, 1e-6, r)
            assert torch.equal(h, want)
            check_codes(q, s, y, DELTA * y.abs(), output)
    x = randn(6, 256, dtype=BF)
    for v in (x[:, None].expand(6, 3, 256), x[None].expand(4, 6, 256), x[:1].expand(5, 256)):
        q, s, h = FQ.rms_norm_quant(v, residual=v)
        e = FQ.rms_norm_quant(v.contiguous(), residual=v.contiguous())
        assert all(torch.equal(a.double(), b.double()) for a, b in zip((q, s, h), e))
        q, s = FQ.gated_act_quant(v, v)
        e = FQ.gated_act_quant(v.contiguous(), v.contiguous())
        assert torch.equal(q.double(), e[0].double()) and torch.equal(s.double(), e[1].double())


@pytest.mark.parametrize("output", ["fp8", "int8", "int8_block"])
@pytest.mark.parametrize("n", [256, 40064])
def test_norm_of_rows_out_of_the_ordinary(output, n):
    x = randn(7, n, dtype=BF)
    x[0] = 0.0
    x[1, 5] = float("nan")
    x[2, 9] = float("inf")
    x[3] *= 2.0 ** 100     # squares beyond fp32
    x[4] *= 2.0 ** -60     # squares below it: eps decides
    x[5] = 0.0
    x[5, 17] = 3e38
    q, s = FQ.rms_norm_quant(x, None, output=output)
    v = (F8.act_dequant_fp8(q, s, output_dtype=F32) if output == "fp8"
         else ops.dequant(q, s, L.QI8_S_ROW if output == "int8" else L.QI8_S_ROW_KBLOCK))
    assert torch.isnan(v[1]).all() and (v[0] == 0).all()
    # the infinity's own block (its row, where that has one scale); elsewhere h / inf = 0
    assert torch.isnan(v[2, :128]).all() and (output == "int8" or (v[2, 128:] == 0).all())
    rest = torch.tensor([0, 3, 4, 5, 6])
    _, y = exact_norm(x[rest], None, 1e-6)
    check_codes(q[rest], s[rest], y, DELTA * y.abs(), output)


@pytest.mark.parametrize("output", ["fp8", "int8"])
@pytest.mark.parametrize("n", [256, 12288, 40064])
@pytest.mark.parametrize("eps", [0.0, 1e-37, 1e-30, 1e-12])
def test_norm_of_small_rows_with_small_eps(n, eps, output):
    x = randn(6, n, seed=n, dtype=F32)
    for i, e in enumerate((-40, -60, -75, -100, -118, 50)):
        x[i] *= 2.0 ** e
    r = randn(6, n, seed=1, dtype=F32) * x.abs()
    for res in (None, r):
        got = FQ.rms_norm_quant(x, eps=eps, residual=res, output=output)
        _, y = exact_norm(x, None, eps, res)
        check_codes(got[0], got[1], y, DELTA * y.abs(), output)
    q, s = FQ.rms_norm_quant(torch.zeros(2, n, device="cuda"), eps=eps, output=output)
    v = F8.act_dequant_fp8(q, s, output_dtype=F32) if output == "fp8" else ops.dequant(q, s, L.QI8_S_ROW)
    assert torch.isnan(v).all() if eps == 0 else (v == 0).all()


def test_views_of_conjugates():
    # the imaginary part of a conjugate is the stored one with a sign that is not in memory
    z = torch.complex(randn(6, 256), randn(6, 256, seed=1))
    v = z.conj().imag
    assert v.is_neg()
    c = torch.empty(6, 256, device="cuda").copy_(v)
    for f in (lambda t: F8.act_quant_fp8(t), lambda t: F8.weight_quant_fp8(t),
              lambda t: FQ.rms_norm_quant(t, t[0], residual=t), lambda t: FQ.gated_act_quant(t, t)):
        assert all(torch.equal(a.double(), b.double()) for a, b in zip(f(v), f(c)))
    w = F8.weight_quant_fp8(randn(32, 256))
    assert torch.equal(F8.fp8_linear(v, *w, bias=v[0, :32]), F8.fp8_linear(c, *w, bias=c[0, :32]))


def test_rows_far_apart():
    # offsets beyond 32 bits: 5 rows 2^29 elements apart
    ld, n = 1 << 29, 300
    big = torch.empty(4 * ld + n, dtype=BF, device="cuda")
    x = big.as_strided((5, n), (ld, 1))
    x.copy_(randn(5, n, dtype=BF))
    c = x.contiguous()
    for a, b in ((FQ.rms_norm_quant(x, residual=x), FQ.rms_norm_quant(c, residual=c)),
                 (FQ.gated_act_quant(x, x, output="int8"), FQ.gated_act_quant(c, c, output="int8")),
                 (F8.act_quant_fp8(x), F8.act_quant_fp8(c)), (F8.weight_quant_fp8(x), F8.weight_quant_fp8(c))):
        assert all(torch.equal(u.double(), v.double()) for u, v in zip(a, b))
    w = F8.weight_quant_fp8(randn(40, n))
    assert torch.equal(F8.fp8_linear(x, *w), F8.fp8_linear(c, *w))


def test_more_than_32_bits_of_elements():
    rows, n = 530000, 4224
    x = torch.empty(rows, n, dtype=BF, device="cuda")
    x[:4], x[-300:] = randn(4, n, dtype=BF), randn(300, n, seed=1, dtype=BF)
    x[4:-300] = 1.0
    tail = x[-300:].clone()
    for f in (lambda t: FQ.rms_norm_quant(t, residual=t), lambda t: FQ.gated_act_quant(t, t),
              lambda t: FQ.gated_act_quant(t, t, output="int8"), lambda t: F8.act_quant_fp8(t)):
        got, want = f(x), f(tail)
        assert all(torch.equal(u[-300:].double(), v.double()) for u, v in zip(got, want))


def test_residual_sum_rounds_like_torch():
    x, r = randn(64, 512, scale=100.0, dtype=BF), randn(64, 512, seed=1, dtype=BF)
    assert torch.equal(FQ.rms_norm_quant(x, residual=r)[2], x + r)
    x, r = randn(64, 512, scale=6e4, dtype=HF), randn(64, 512, seed=1, scale=6e4, dtype=HF)
    h = FQ.rms_norm_quant(x, residual=r)[2]
    # infinities of both signs meet: NaN in the same places
    torch.testing.assert_close(h, x + r, rtol=0, atol=0, equal_nan=True)
    assert torch.isinf(h).any()


# ------------------------------------------------------------------- gated
def exact_gated(g, u, act):
    g, u = g.double(), u.double()
    if act == "gelu":
        y = 0.5 * g * torch.special.erfc(-g / math.sqrt(2)) * u
        return y, 16 * 2.0 ** -24 * y.abs() + g.abs() * u.abs() * 2.0 ** -22
    t = g if act == "silu" else 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)
    y = g / (1 + torch.exp(-t)) * u
    return y, 4 * (4 + t.abs() * (1 if act == "silu" else 4)) * 2.0 ** -24 * y.abs() + 2.0 ** -126


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("output", ["fp8", "int8", "int8_block"])
@pytest.mark.parametrize("rows,n", [(1, 1), (1, 10240), (3, 127), (16, 384), (5, 1000), (515, 273), (64, 2048),
                                    (2, 20000), (2, 40000)])
def test_gated(rows, n, act, dtype, output):
    if output == "int8_block" and n % 128:
        n = -(-n // 128) * 128
    g, u = randn(rows, n, seed=n, scale=3.0, dtype=dtype), randn(rows, n, seed=1, scale=2.0, dtype=dtype)
    q, s = FQ.gated_act_quant(g, u, activation=act, output=output)
    y, tol = exact_gated(g, u, act)
    check_codes(q, s, y, tol, output)


@pytest.mark.parametrize("n", [300, 1280])
def test_gated_halves_of_one_tensor(n):
    both = randn(4, 9, 2 * n, dtype=BF)
    for g, u in (both.chunk(2, -1), (both[..., n:], both[..., :n])):
        for output in ("fp8", "int8"):
            q, s = FQ.gated_act_quant(g, u, output=output)
            q2, s2 = FQ.gated_act_quant(g.contiguous(), u.contiguous(), output=output)
            assert torch.equal(q.double(), q2.double()) and torch.equal(s.double(), s2.double())


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_gated_far_values(act):
    # far gates: act is 0 or the gate itself; products beyond fp32 and NaN spoil their block only
    g = torch.zeros(2, 512, device="cuda")
    g[0, :8] = torch.tensor([-200.0, 200.0, -1e30, 1e30, -88.0, 88.0, -1e-30, 1e-30])
    u = torch.ones_like(g)
    g[1, 3], u[1, 3] = 3e38, 3e38
    g[1, 140] = float("nan")
    g[1, 300] = float("inf")
    q, s = FQ.gated_act_quant(g, u, activation=act)
    v = F8.act_dequant_fp8(q, s, output_dtype=F32)
    assert v[0, 3] == F8.act_dequant_fp8(*F8.act_quant_fp8(g[:1]), output_dtype=F32)[0, 3] and (v[0, 128:] == 0).all()
    assert torch.isnan(v[1, :384]).all() and (v[1, 384:] == 0).all()


# ------------------------------------------------------- behind one another
def test_feed_forward_chain_in_fp8():
    t, d, f = 150, 512, 1100
    x, r = randn(t, d, dtype=BF), randn(t, d, seed=1, dtype=BF)
    w, w13, w2 = randn(d, seed=2, dtype=BF), randn(2 * f, d, seed=3, scale=0.04), randn(d, f, seed=4, scale=0.03)
    w13q, w2q = F8.weight_quant_fp8(w13), F8.weight_quant_fp8(w2)
    q, s, h = FQ.rms_norm_quant(x, w, residual=r)
    gu = F8.fp8_gemm(q, s, *w13q)
    q2, s2 = FQ.gated_act_quant(gu[:, :f], gu[:, f:])
    y = F8.fp8_gemm(q2, s2, *w2q)
    # the same steps in fp64 on the codes' values
    def rows(q, s):
        return q.double() * s.double().repeat_interleave(128, 1)[:, :q.shape[1]]
    v13, v2 = (F8.weight_dequant_fp8(*p, output_dtype=F32).double() for p in (w13q, w2q))
    gu64 = rows(q, s) @ v13.T
    assert ((gu.double() - gu64).abs() <= 2.0 ** -8 * gu64.abs() + 1e-4 * (rows(q, s).abs() @ v13.abs().T)).all()
    yg, tol = exact_gated(gu[:, :f], gu[:, f:], "silu")
    check_codes(q2, s2, yg, tol, "fp8")
    y64 = rows(q2, s2) @ v2.T
    assert ((y.double() - y64).abs() <= 2.0 ** -8 * y64.abs() + 2e-4 * (rows(q2, s2).abs() @ v2.abs().T)).all()
    # and against no quantization at all: e4m3 is off by 2^-4 per operand at most, so two operands by under 0.13
    hd = h.double()
    n64 = hd / torch.sqrt(hd.square().mean(-1, keepdim=True) + 1e-6) * w.double()
    assert ((gu64 - n64 @ w13.double().T).abs() <= 0.13 * (n64.abs() @ w13.double().abs().T)).all()


def test_int8_outputs_feed_the_int8_products():
    t, d, n = 130, 512, 256
    x, w = randn(t, d, dtype=BF), randn(n, d, seed=1, scale=0.05)
    q, s = FQ.rms_norm_quant(x, output="int8_block")
    wq, ws = I8.weight_quant(w)
    y = I8.int8_gemm(q, s, wq, ws)
    vw = I8.weight_dequant(wq, ws, output_dtype=F32).double()
    va = q.double() * s.double().repeat_interleave(128, 1)
    ref, total = va @ vw.T, va.abs() @ vw.abs().T
    # fp16 output; sums of K / 128 exact blocks
    assert ((y.double() - ref).abs() <= 2.0 ** -11 * ref.abs() + 2.0 ** -20 * total + 2.0 ** -24).all()
    q, s = FQ.rms_norm_quant(x, output="int8")
    qr, sr = ops.quant_weight(w, L.QI8_S_ROW)
    y = ops.gemm_i8(q, qr, s, L.QI8_S_ROW, sr, L.QI8_S_ROW, None, F32)
    ref = (q.double() @ qr.double().T) * s.double() * sr.double().view(1, -1)
    assert ((y.double() - ref).abs() <= 2.0 ** -22 * ref.abs()).all()


@pytest.mark.parametrize("rows,n", [(3, 64), (5, 2731), (77, 300), (16, 4096)])
@pytest.mark.parametrize("out", [BF, HF, F32])
def test_int8_read_back(rows, n, out):
    q = torch.randint(-127, 128, (rows, n), dtype=torch.int8, device="cuda")
    s = randn(rows, 1).abs()
    assert torch.equal(ops.dequant(q, s, L.QI8_S_ROW, out_dtype=out), (q.float() * s).to(out))
    assert torch.equal(ops.dequant(q, s[:1, 0], L.QI8_S_SCALAR, out_dtype=out), (q.float() * s[0]).to(out))
    assert torch.equal(ops.dequant(q[:, 1:], s, L.QI8_S_ROW, out_dtype=out), (q[:, 1:].float() * s).to(out))


def test_refusals():
    x = randn(4, 200, dtype=BF)
    with pytest.raises(AssertionError, match="divisible"):
        FQ.rms_norm_quant(x, output="int8_block")
    with pytest.raises(AssertionError):
        FQ.rms_norm_quant(x, x[0, :100])
    with pytest.raises(AssertionError):
        FQ.rms_norm_quant(x, residual=x[:2])
    with pytest.raises(TypeError):
        FQ.rms_norm_quant(x, residual=x.half())
    with pytest.raises(TypeError):
        FQ.gated_act_quant(x, x.float())
    with pytest.raises(AssertionError):
        FQ.gated_act_quant(x, x[:, :100])
    for eps in (-1.0, 1e-40, float("nan"), float("inf")):
        with pytest.raises(AssertionError, match="eps"):
            FQ.rms_norm_quant(x, eps=eps)
    with pytest.raises(TypeError):
        FQ.rms_norm_quant(x.double())
    with pytest.raises(RuntimeError, match="backward"):
        FQ.rms_norm_quant(x, torch.nn.Parameter(x[0].clone()))
    with pytest.raises(RuntimeError, match="backward"):
        FQ.gated_act_quant(x, x.clone().requires_grad_())
    with pytest.raises(RuntimeError):
        FQ.gated_act_quant(x, x.cpu())
    assert L.load().qi8_gated_quant(x.data_ptr(), 200, x.data_ptr(), 200, 0, 4, 200, 0, 2, x.data_ptr(), 200,
                                    x.data_ptr(), None) == L.QI8_EINVAL


@pytest.mark.parametrize("output", ["fp8", "int8"])
def test_graph_and_stream(output):
    x, r, w = randn(40, 1000, dtype=BF), randn(40, 1000, seed=1, dtype=BF), randn(1000, seed=2, dtype=BF)
    FQ.rms_norm_quant(x, w, residual=r, output=output)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        q, s, h = FQ.rms_norm_quant(x, w, residual=r, output=output)
        q2, s2 = FQ.gated_act_quant(h, r, output=output)
    x.copy_(randn(40, 1000, seed=9, dtype=BF))
    g.replay()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eq, es, eh = FQ.rms_norm_quant(x, w, residual=r, output=output)
        eq2, es2 = FQ.gated_act_quant(eh, r, output=output)
    torch.cuda.synchronize()
    for a, b in ((q, eq), (s, es), (h, eh), (q2, eq2), (s2, es2)):
        assert torch.equal(a.double(), b.double())
