"""GPU tests of the 4-bit weight operators against plain forms in 64 bits.

Tolerances, from the arithmetic: products of codes and activations are exact
in fp32.  A tensor-core step sums 16 of them and the accumulator; with 24 bits
kept relative to the largest term it is off by at most 17 * 2^-23 of the sum of
absolute values S.  At most 8 such steps follow each other inside a group, then
one fma per group and one addition per warp or split, each 2^-24 of S.  With
up to 512 groups in a row that is (8 * 17 + 256 + 8) * 2^-23 S < 5e-5 S; ACC is
that bound.  The output is rounded once: half a step, eps / 2 of the value.
"""

import numpy as np
import pytest
import torch
import torch.nn.functional as F

import oracle as O
from convert_to_quant_quip_int8_b200 import _lib as L
from convert_to_quant_quip_int8_b200 import ops
from convert_to_quant_quip_int8_b200.comfy import int4_kernels as I4
from convert_to_quant_quip_int8_b200.comfy.quant_ops import QuantizedTensor

pytestmark = pytest.mark.gpu

ACC = 5e-5
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _status():
    yield
    ops.device_status(reset=True)


def randn(*shape, seed=0, scale=1.0, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def weight(n, k, group, seed=0, lead=()):
    """A packed random weight and its fp64 values."""
    rows = int(np.prod(lead, dtype=int)) * n
    codes, scale = O.i4_quantize(np.random.default_rng(seed).standard_normal((rows, k)) * 0.02, group)
    q = O.i4_pack(codes)
    v = torch.from_numpy(O.i4_values(q, scale, k, group)).cuda().view(*lead, n, k)
    q = torch.from_numpy(q).cuda().view(*lead, n, -1)
    return q, torch.from_numpy(scale).to(BF).cuda().view(*lead, n, -1), v


def close(y, ref, bound):
    """|y - ref| <= bound + half a step of y's type (subnormal steps of fp16 included)."""
    info = torch.finfo(y.dtype)
    tol = bound + info.eps / 2 * (ref.abs() + bound) + info.smallest_normal * info.eps
    off = (y.double() - ref).abs()
    assert torch.isfinite(y).all()
    worst = (off / tol).max().item() if y.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3g} times the tolerance"


# ------------------------------------------------------------ quantization
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,k", [(1, 1), (3, 31), (7, 128), (5, 1100), (33, 257), (64, 4096), (2, 20000)])
def test_quant_matches_definition(n, k, group, dtype):
    w = randn(n, k, seed=n * k, scale=0.02, dtype=dtype)
    q, s = I4.weight_quant_int4(w, group)
    codes, scale = O.i4_quantize(w.double().cpu().numpy(), group)
    assert np.array_equal(s.double().cpu().numpy(), scale)
    assert np.array_equal(O.i4_unpack(q.cpu().numpy()), codes)
    assert np.array_equal(q.cpu().numpy(), O.i4_pack(codes))
    for out in (BF, HF, F32):
        v = I4.weight_dequant_int4(q, s, k, group, out)
        ref = torch.from_numpy(O.i4_values(q.cpu().numpy(), scale, k, group))
        assert torch.equal(v.cpu(), ref.to(out))


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_quant_ties_go_to_even(dtype):
    # halves of a step are exact ties (in bf16 not all of those of 31 / 16: 403 has nine bits)
    rows = []
    for s in (1.0, 17 / 16, 31 / 16, 2.0 ** -10):
        steps = torch.arange(-13, 14).double() / 2 * s
        rows.append(torch.cat([torch.tensor([7 * s], dtype=torch.float64), steps,
                               torch.zeros(4, dtype=torch.float64)]))
    w = torch.stack(rows).to(dtype).cuda()
    q, s = I4.weight_quant_int4(w, 32)
    codes, scale = O.i4_quantize(w.double().cpu().numpy(), 32)
    assert np.array_equal(s.double().cpu().numpy(), scale)
    assert np.array_equal(O.i4_unpack(q.cpu().numpy()), codes)
    assert codes[0, 1:28].tolist() == [round(v / 2) for v in range(-13, 14)]


def test_quant_fp32_next_to_ties():
    # one step of fp32 on either side of every tie
    for s in (1.0, 19 / 16):
        tie = (torch.arange(-13, 14, 2).float() / 2 * s)
        w = torch.zeros(3, 32)
        w[:, 0] = 7 * s
        w[0, 1:15], w[1, 1:15], w[2, 1:15] = tie, torch.nextafter(tie, tie + 1), torch.nextafter(tie, tie - 1)
        q, sc = I4.weight_quant_int4(w.cuda(), 32)
        codes, scale = O.i4_quantize(w.double().numpy(), 32)
        assert np.array_equal(sc.double().cpu().numpy(), scale)
        assert np.array_equal(O.i4_unpack(q.cpu().numpy()), codes)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_quant_extremes(dtype):
    w = torch.zeros(6, 160, dtype=torch.float64)
    w[0, 5] = float("inf")
    w[1, 40] = float("nan")
    w[2, :32] = torch.finfo(dtype).max
    w[3, :32] = 2.0 ** -126
    w[4, 64:96] = -2.0 ** -98
    w = w.to(dtype)
    q, s = I4.weight_quant_int4(w.cuda(), 32)
    codes, scale = O.i4_quantize(w.double().numpy(), 32)
    assert np.array_equal(s.double().cpu().numpy(), scale, equal_nan=True)
    assert np.array_equal(O.i4_unpack(q.cpu().numpy()), codes)
    v = I4.weight_dequant_int4(q, s, 160, 32, F32).cpu()
    assert torch.isnan(v[0, :32]).all() and torch.isnan(v[1, 32:64]).all()
    assert torch.isnan(v).sum() == 64


@pytest.mark.parametrize("dtype", [BF, F32])
def test_quant_views_and_lead_dimensions(dtype):
    big = randn(40, 300, seed=3, dtype=dtype)
    for view in (big[:, 1:258], big[::2, :256], big.t(), big[5:6]):
        q, s = I4.weight_quant_int4(view, 64)
        qc, sc = I4.weight_quant_int4(view.clone(memory_format=torch.contiguous_format), 64)
        assert torch.equal(q, qc) and torch.equal(s, sc)
    q, s = I4.weight_quant_int4(big.view(4, 10, 300), 64)
    qf, sf = I4.weight_quant_int4(big, 64)
    assert q.shape == (4, 10, 192) and torch.equal(q.view_as(qf), qf) and torch.equal(s.view_as(sf), sf)
    assert I4.weight_dequant_int4(q, s, 300, 64, dtype).shape == (4, 10, 300)
    q, s = I4.weight_quant_int4(big[:0], 64)
    assert q.shape == (0, 192) and I4.weight_dequant_int4(q, s, 300, 64, dtype).shape == (0, 300)


def test_dequant_writes_its_rows_alone():
    q, s, v = weight(5, 77, 32, seed=9)
    out = torch.full((7, 90), 3.0, device="cuda")
    L.check(L.load().qi8_dequant_i4(q.data_ptr(), s.data_ptr(), 5, 77, 32, out.data_ptr(), L.QI8_F32, 90,
                                    L.stream_ptr()))
    assert torch.equal(out[:5, :77].double(), v) and (out[5:] == 3).all() and (out[:, 77:] == 3).all()


# ----------------------------------------------------------------- linear
def check_linear(m, n, k, group, dtype, bias, seed=0, x=None):
    q, s, v = weight(n, k, group, seed=seed)
    if x is None:
        x = randn(m, k, seed=seed + 1, dtype=dtype)
    b = randn(n, seed=seed + 2, scale=0.1, dtype=bias) if bias else None
    y = I4.int4_linear(x, q, s, group, b)
    assert y.shape == (m, n) and y.dtype == dtype
    ref = x.double() @ v.T
    bound = ACC * (x.double().abs() @ v.abs().T)
    if b is not None:
        ref = ref + b.double()
        bound = bound + 2.0 ** -23 * ref.abs()
    close(y, ref, bound)
    return y


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("m,n,k,group", [
    (1, 1, 1, 32), (1, 16, 128, 128), (1, 17, 129, 32), (2, 100, 1000, 64), (1, 4096, 4096, 128),
    (7, 503, 2989, 32), (8, 64, 8192, 64), (9, 33, 640, 128), (16, 1000, 1088, 64), (17, 48, 512, 32),
    (32, 130, 264, 128), (33, 129, 130, 64), (64, 256, 2048, 128), (65, 300, 300, 32), (100, 640, 1024, 128),
    (127, 257, 1032, 64), (128, 128, 128, 32), (200, 384, 4096, 128), (300, 1000, 777, 32), (1, 5, 20000, 128),
    (513, 515, 520, 64), (1000, 256, 256, 128)])
def test_linear(m, n, k, group, dtype):
    check_linear(m, n, k, group, dtype, None, seed=m + n)
    check_linear(m, n, k, group, dtype, dtype, seed=m + n + 1)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("m,n,k,group", [
    (17, 48, 8320, 32), (32, 130, 8328, 128), (33, 129, 8194, 64), (64, 1, 9000, 128), (65, 300, 8448, 32),
    (100, 640, 8320, 128), (127, 257, 8320, 64), (128, 128, 16384, 32), (129, 7, 8200, 64), (200, 384, 8704, 128),
    (257, 1000, 8321, 32), (40, 4104, 4096, 128), (300, 2100, 1024, 64), (520, 4096, 520, 32), (1100, 4112, 136, 128),
    (24, 10240, 4096, 64)])
def test_linear_beyond_the_small_products(m, n, k, group, dtype):
    """More than 2^29 multiply-adds or 8192 features: tensor-core tiles, split over clusters where they are few."""
    check_linear(m, n, k, group, dtype, None, seed=m + n)
    check_linear(m, n, k, group, dtype, F32, seed=m + n + 1)


@pytest.mark.parametrize("m", [20, 300])
def test_linear_tiles_hold_what_the_small_products_hold(m):
    """Non-finite values, scales of eight bits, wide scale ranges, strided rows, untouched columns, graphs at 8320
    features."""
    n, k, group = 72, 8320, 32
    q, s, _ = weight(n, k, group, seed=11)
    x = randn(m, k, seed=12, dtype=BF)
    good = I4.int4_linear(x, q, s, group)
    x2, s2 = x.clone(), s.clone()
    x2[1, 7], x2[2, k - 1], s2[5, 1] = float("nan"), float("inf"), float("nan")
    y = I4.int4_linear(x2, q, s2, group)
    assert torch.isnan(y[1]).all() and torch.isnan(y[:, 5]).all() and not torch.isfinite(y[2]).any()
    keep_m, keep_n = [i for i in range(m) if i not in (1, 2)], [i for i in range(n) if i != 5]
    assert torch.equal(y[keep_m][:, keep_n], good[keep_m][:, keep_n])

    big = randn(2 * m, k + 24, seed=5, dtype=BF)
    for v in (big[:m, :k], big[:m, 1:k + 1], big[::2, 8:k + 8]):
        assert torch.equal(I4.int4_linear(v, q, s, group), I4.int4_linear(v.contiguous(), q, s, group))

    rng = np.random.default_rng(1)
    codes = rng.integers(-8, 8, (n, k)).astype(np.int8)
    qa = torch.from_numpy(O.i4_pack(codes)).cuda()
    sa = (torch.rand(n, k // group, generator=torch.Generator().manual_seed(2)) * 0.01 + 1e-3).to(BF).cuda()
    va = torch.from_numpy(O.i4_values(qa.cpu().numpy(), sa.double().cpu().numpy(), k, group)).cuda()
    for dtype in (BF, HF):
        xa = randn(m, k, seed=8, dtype=dtype)
        mag = xa.double().abs() @ va.abs().T
        close(I4.int4_linear(xa, qa, sa, group), xa.double() @ va.T, (ACC + torch.finfo(dtype).eps / 2) * mag)
    codes = rng.integers(-7, 8, (n, k)).astype(np.int8)
    scale = np.ldexp(rng.integers(16, 32, (n, k // group)) / 16.0, rng.integers(-20, -8, (n, k // group)))
    qr = torch.from_numpy(O.i4_pack(codes)).cuda()
    vr = torch.from_numpy(codes * np.repeat(scale, group, 1)).cuda()
    xr = randn(m, k, seed=9, dtype=HF)
    close(ops.gemm_w4(xr, qr, torch.from_numpy(scale).to(BF).cuda(), group, out_dtype=F32), xr.double() @ vr.T,
          ACC * (xr.double().abs() @ vr.abs().T))

    out = torch.full((m + 2, n + 9), 3.0, dtype=BF, device="cuda")
    L.check(L.load().qi8_gemm_w4(x.data_ptr(), L.QI8_BF16, m, k, k, q.data_ptr(), s.data_ptr(), n, group, None, 0,
                                 out.data_ptr(), L.QI8_BF16, n + 9, None, 0, L.stream_ptr()))
    assert torch.equal(out[:m, :n], good) and (out[m:] == 3).all() and (out[:, n:] == 3).all()

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z = I4.int4_linear(x, q, s, group)
    for _ in range(2):
        z.zero_()
        graph.replay()
        assert torch.equal(z, good)


@pytest.mark.parametrize("m", [3, 40, 300])
def test_linear_bias_and_output_types(m):
    q, s, v = weight(96, 256, 64)
    x = randn(m, 256, dtype=BF)
    for bt in (BF, HF, F32):
        b = randn(96, seed=4, dtype=bt)
        ref = x.double() @ v.T + b.double()
        bound = ACC * (x.double().abs() @ v.abs().T) + 2.0 ** -23 * ref.abs()
        close(ops.gemm_w4(x, q, s, 64, b), ref, bound)
        y = ops.gemm_w4(x, q, s, 64, b, out_dtype=F32)
        assert y.dtype == F32
        close(y, ref, bound)


@pytest.mark.parametrize("m", [5, 70, 260])
@pytest.mark.parametrize("k", [256, 250])
def test_linear_views(m, k):
    big = randn(2 * m, k + 24, seed=5, dtype=BF)
    for x in (big[:m, :k], big[:m, 1:k + 1], big[::2, 8:k + 8], randn(k, m, seed=6, dtype=BF).t(),
              big[:1, :k].expand(m, k)):
        y = check_linear(m, 40, k, 64, BF, None, x=x)
        q, s, _ = weight(40, k, 64)
        assert torch.equal(y, I4.int4_linear(x.contiguous(), q, s, 64))
    q, s, _ = weight(40, k, 64)
    x = randn(2, 3, k, seed=7, dtype=HF)
    y = I4.int4_linear(x, q, s, 64)
    assert y.shape == (2, 3, 40) and torch.equal(y.view(6, 40), I4.int4_linear(x.view(6, k), q, s, 64))
    assert I4.int4_linear(x[0, 0], q, s, 64).shape == (40,)
    assert I4.int4_linear(x[:, :0], q, s, 64).shape == (2, 0, 40)


@pytest.mark.parametrize("m", [4, 30, 300])
def test_linear_arbitrary_scales_and_codes(m):
    """Scales of eight significant bits, code -8, garbage codes behind the row's end.  From 17 tokens on the weight
    may be rounded to 16 bits on its way to the tensor cores: half a step of x's type on every product."""
    n, k, group = 70, 200, 32
    rng = np.random.default_rng(1)
    codes = rng.integers(-8, 8, (n, 256)).astype(np.int8)
    q = torch.from_numpy(O.i4_pack(codes)).cuda()
    s = (torch.rand(n, 8, generator=torch.Generator().manual_seed(2)) * 0.01 + 1e-3).to(BF).cuda()
    v = torch.from_numpy(O.i4_values(q.cpu().numpy(), s.double().cpu().numpy(), k, group)).cuda()
    for dtype in (BF, HF):
        x = randn(m, k, seed=8, dtype=dtype)
        y = I4.int4_linear(x, q, s, group)
        ref, mag = x.double() @ v.T, x.double().abs() @ v.abs().T
        close(y, ref, (ACC + (torch.finfo(dtype).eps / 2 if m > 16 else 0.0)) * mag)


@pytest.mark.parametrize("m", [2, 20, 260])
@pytest.mark.parametrize("dtype,exps", [(HF, (-20, -8)), (HF, (-2, 3)), (BF, (-60, -40))])
def test_linear_scale_range(m, dtype, exps):
    """Scales far from 1, mixed within a row, stay exact in fp16 layers too (results within fp16's range)."""
    n, k, group = 48, 384, 32
    rng = np.random.default_rng(3)
    codes = rng.integers(-7, 8, (n, k)).astype(np.int8)
    scale = np.ldexp(rng.integers(16, 32, (n, k // group)) / 16.0, rng.integers(*exps, (n, k // group)))
    q = torch.from_numpy(O.i4_pack(codes)).cuda()
    v = torch.from_numpy(codes * np.repeat(scale, group, 1)).cuda()
    x = randn(m, k, seed=9, dtype=dtype)
    y = ops.gemm_w4(x, q, torch.from_numpy(scale).to(BF).cuda(), group, out_dtype=F32)
    close(y, x.double() @ v.T, ACC * (x.double().abs() @ v.abs().T))


@pytest.mark.parametrize("m", [3, 40, 300])
def test_linear_non_finite_stays_in_its_row_and_column(m):
    q, s, _ = weight(40, 300, 64, seed=11)
    x = randn(m, 300, seed=12, dtype=BF)
    good = I4.int4_linear(x, q, s, 64)
    x2, s2 = x.clone(), s.clone()
    x2[1, 7] = float("nan")
    x2[2, 299] = float("inf")
    s2[5, 1] = float("nan")
    y = I4.int4_linear(x2, q, s2, 64)
    assert torch.isnan(y[1]).all() and torch.isnan(y[:, 5]).all() and not torch.isfinite(y[2]).any()
    keep_m = [i for i in range(m) if i not in (1, 2)]
    keep_n = [i for i in range(40) if i != 5]
    assert torch.equal(y[keep_m][:, keep_n], good[keep_m][:, keep_n])


@pytest.mark.parametrize("m", [3, 40, 300])
def test_linear_writes_its_columns_alone(m):
    q, s, _ = weight(33, 100, 32, seed=13)
    x = randn(m, 100, seed=14, dtype=BF)
    out = torch.full((m + 2, 50), 3.0, dtype=BF, device="cuda")
    ws = torch.empty(m * 208, dtype=torch.uint8, device="cuda")  # 100 features: rows are copied to 104
    L.check(L.load().qi8_gemm_w4(x.data_ptr(), L.QI8_BF16, m, 100, 100, q.data_ptr(), s.data_ptr(), 33, 32, None, 0,
                                 out.data_ptr(), L.QI8_BF16, 50, ws.data_ptr(), ws.numel(), L.stream_ptr()))
    assert torch.equal(out[:m, :33], I4.int4_linear(x, q, s, 32))
    assert (out[m:] == 3).all() and (out[:, 33:] == 3).all()


@pytest.mark.parametrize("m", [1, 12, 60, 300])
def test_linear_repeats_and_graphs(m):
    q, s, _ = weight(520, 1024, 128, seed=15)
    x = randn(m, 1024, seed=16, dtype=BF)
    y = I4.int4_linear(x, q, s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = I4.int4_linear(x, q, s)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, z)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z = I4.int4_linear(x, q, s)
    x2 = randn(m, 1024, seed=17, dtype=BF)
    y2 = I4.int4_linear(x2, q, s)
    x.copy_(x2)
    for _ in range(2):
        z.zero_()
        graph.replay()
        assert torch.equal(z, y2)


def test_linear_large_offsets():
    """A weight of more than 2^31 codes: row offsets pass 32 bits."""
    n, k = 70000, 32768
    q = torch.full((n, k // 2), 0x88, dtype=torch.uint8, device="cuda")
    s = torch.ones(n, k // 128, dtype=BF, device="cuda")
    q[-1] = 0x99  # code 1
    q[1] = 0x77  # code -1
    x = torch.ones(2, k, dtype=BF, device="cuda")
    x[1] = 2
    y = I4.int4_linear(x, q, s)
    assert y[:, -1].tolist() == [k, 2 * k] and y[:, 1].tolist() == [-k, -2 * k]
    assert int((y != 0).sum()) == 4
    v = I4.weight_dequant_int4(q, s, k, 128, BF)
    assert (v[-1] == 1).all() and (v[1] == -1).all() and int((v != 0).sum()) == 2 * k
    q2, s2 = I4.weight_quant_int4(v * 7)
    assert (q2[-1] == 0xFF).all() and (q2[1] == 0x11).all()
    assert (q2[2:-1] == 0x88).all() and (s2[-1] == 1).all()


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_other_device():
    q, s, v = weight(64, 256, 64)
    x = randn(3, 256, dtype=BF)
    y = I4.int4_linear(x, q, s, 64)
    y1 = I4.int4_linear(x.to("cuda:1"), q.to("cuda:1"), s.to("cuda:1"), 64)
    assert y1.device.index == 1 and torch.equal(y.cpu(), y1.cpu())


def test_layout_through_flinear():
    w = randn(200, 300, scale=0.02, dtype=BF)
    wq = QuantizedTensor.from_float(w, "GroupWiseINT4Layout", group_size=32)
    b = randn(200, seed=1, dtype=BF)
    x = randn(2, 5, 300, seed=2, dtype=BF)
    y = F.linear(x, wq, b)
    p = wq._layout_params
    assert torch.equal(y, I4.int4_linear(x, wq._qdata, p["scale"], 32, b))
    d = wq.dequantize()
    assert d.dtype == BF and d.shape == (200, 300)
    assert torch.equal(d, I4.weight_dequant_int4(wq._qdata, p["scale"], 300, 32, BF))
    moved = wq.detach().clone()
    assert torch.equal(F.linear(x, moved, b), y)
    with pytest.raises(AssertionError, match="features"):
        F.linear(x[..., :299], wq)
    with pytest.raises(RuntimeError, match="backward"):
        F.linear(x.clone().requires_grad_(), wq)
    with torch.no_grad():
        assert torch.equal(F.linear(x.clone().requires_grad_(), wq, b), y)


def test_a_models_parameter_quantizes():
    w = torch.nn.Parameter(randn(40, 300, scale=0.02, dtype=BF))
    a = QuantizedTensor.from_float(w, "GroupWiseINT4Layout")
    b = QuantizedTensor.from_float(w.detach(), "GroupWiseINT4Layout")
    assert torch.equal(a._qdata, b._qdata) and not a._layout_params["scale"].requires_grad


def test_linear_refusals():
    q, s, _ = weight(40, 256, 64)
    x = randn(3, 256, dtype=BF)
    with pytest.raises(TypeError):
        I4.int4_linear(x.float(), q, s, 64)
    with pytest.raises(TypeError):
        I4.int4_linear(x, q, s.float(), 64)
    with pytest.raises(TypeError):
        ops.gemm_w4(x, q, s, 64, out_dtype=HF)
    for bad in (lambda: I4.int4_linear(x[:, :100], q, s, 64), lambda: I4.int4_linear(x, q, s, 128),
                lambda: I4.int4_linear(x, q, s, 64, randn(39, dtype=BF)),
                lambda: I4.int4_linear(x, torch.cat([q.flatten(), q.flatten()])[1:1 + q.numel()].view_as(q), s, 64),
                lambda: I4.weight_quant_int4(randn(4, 4), 16), lambda: I4.weight_quant_int4(randn(4)),
                lambda: I4.weight_dequant_int4(q, s, 300, 64)):
        with pytest.raises(AssertionError):
            bad()
    with pytest.raises(TypeError):
        I4.weight_quant_int4(torch.zeros(4, 128, dtype=torch.int32, device="cuda"))
    with pytest.raises(TypeError):
        I4.weight_dequant_int4(q, s, 256, 64, torch.int8)


# -------------------------------------------------------------------- moe
def moe_reference(x, router, v13, v2, top_k, renorm, act):
    """fp64 layer and a bound of the kernels' error: fp32 sums (ACC of their magnitudes), activation functions to
    2^-20, h to 16 bits (2^-16), the weights p to 2^-20."""
    x, r = x.double(), router.double()
    p = torch.from_numpy(O.moe_route((x @ r.T).cpu().numpy(), top_k, renorm)).cuda()
    y, bound = torch.zeros_like(x), torch.zeros_like(x)
    i = v2.shape[-1]
    for e in range(r.shape[0]):
        at = p[:, e].nonzero().flatten()
        if not len(at):
            continue
        gu, mag = x[at] @ v13[e].T, ACC * (x[at].abs() @ v13[e].abs().T)
        g, u = gu[:, :i], gu[:, i:]
        a = g * torch.sigmoid(g) if act == "silu" else 0.5 * g * (1 + torch.erf(g / 2 ** 0.5))
        h = a * u
        # both functions have slopes of at most 1.13
        dh = 1.13 * mag[:, :i] * (u.abs() + mag[:, i:]) + a.abs() * mag[:, i:] + (2.0 ** -16 + 2.0 ** -20) * h.abs() \
            + 2.0 ** -20 * (g * u).abs()
        out = h @ v2[e].T
        db = dh @ v2[e].abs().T + ACC * (h.abs() @ v2[e].abs().T) + 2.0 ** -20 * out.abs()
        y[at] += p[at, e:e + 1] * out
        bound[at] += p[at, e:e + 1] * db
    return y, bound


def moe_case(t, e, top_k, h, i, group, dtype, seed=0):
    q13, s13, v13 = weight(2 * i, h, group, seed=seed, lead=(e,))
    q2, s2, v2 = weight(h, i, group, seed=seed + 1, lead=(e,))
    x = randn(t, h, seed=seed + 2, dtype=dtype)
    router = randn(e, h, seed=seed + 3, scale=h ** -0.5, dtype=dtype)
    return x, router, q13, s13, v13, q2, s2, v2


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("t,e,top_k,h,i,group", [
    (1, 1, 1, 1, 1, 32), (1, 64, 8, 256, 128, 128), (2, 3, 3, 130, 17, 32), (5, 23, 3, 1090, 701, 32),
    (16, 64, 8, 512, 192, 64), (9, 4, 1, 264, 1024, 128), (33, 8, 2, 300, 100, 64), (64, 8, 2, 256, 640, 128),
    (64, 2, 2, 128, 128, 32), (65, 16, 4, 128, 96, 64), (150, 5, 2, 200, 72, 128), (3, 300, 40, 64, 64, 32)])
def test_moe(t, e, top_k, h, i, group, dtype):
    x, router, q13, s13, v13, q2, s2, v2 = moe_case(t, e, top_k, h, i, group, dtype, seed=t + e)
    for act, renorm, r in (("silu", True, router), ("gelu", False, router.float())):
        y = I4.moe_int4(x, r, q13, s13, q2, s2, top_k, group, renorm, act)
        assert y.shape == (t, h) and y.dtype == dtype
        close(y, *moe_reference(x, r, v13, v2, top_k, renorm, act))


def test_moe_ties_take_the_lowest_experts():
    x, router, q13, s13, v13, q2, s2, v2 = moe_case(6, 12, 3, 128, 64, 64, BF, seed=5)
    router[:] = router[4]  # all logits equal
    y = I4.moe_int4(x, router, q13, s13, q2, s2, 3, 64)
    close(y, *moe_reference(x, router, v13, v2, 3, True, "silu"))
    only = I4.moe_int4(x, router[:3].contiguous(), q13[:3], s13[:3], q2[:3], s2[:3], 3, 64)
    assert torch.equal(y, only)
    x.zero_()  # logits of 0 and -0
    assert not I4.moe_int4(x, router, q13, s13, q2, s2, 3, 64).any()


def test_moe_near_ties_follow_the_exact_logits():
    """Two experts whose logits differ by less than fp32 sums resolve."""
    h, e = 4096, 8
    x, router, q13, s13, v13, q2, s2, v2 = moe_case(4, e, 1, h, 32, 128, BF, seed=6)
    router = router.float()
    router[:] = router[0]
    router[5] = router[0] * (1 + 2.0 ** -22)
    y = I4.moe_int4(x, router, q13, s13, q2, s2, 1, 128)
    close(y, *moe_reference(x, router, v13, v2, 1, True, "silu"))


def test_moe_all_tokens_in_one_expert_and_unused_experts():
    x, router, q13, s13, v13, q2, s2, v2 = moe_case(64, 9, 1, 256, 200, 64, BF, seed=7)
    x[:, 0] = 3.0
    router[:, 0] = 0
    router[6, 0] = 100.0
    s13 = s13.clone()
    for other in (0, 1, 8):  # experts that no token chooses may hold anything
        s13[other] = float("nan")
    y = I4.moe_int4(x, router, q13, s13, q2, s2, 1, 64)
    close(y, *moe_reference(x, router, v13, v2, 1, True, "silu"))


def test_moe_non_finite_token_stays_alone():
    x, router, q13, s13, v13, q2, s2, v2 = moe_case(12, 6, 2, 256, 96, 64, BF, seed=8)
    good = I4.moe_int4(x, router, q13, s13, q2, s2, 2, 64)
    x2 = x.clone()
    x2[3, 17] = float("nan")
    x2[7, 0] = float("inf")
    y = I4.moe_int4(x2, router, q13, s13, q2, s2, 2, 64)
    assert torch.isnan(y[3]).all() and not torch.isfinite(y[7]).any()
    keep = [i for i in range(12) if i not in (3, 7)]
    assert torch.equal(y[keep], good[keep])


def test_moe_fp16_intermediate_passes_fp16_range():
    """h = act(g) * u beyond 65504 while the output fits."""
    x, router, q13, s13, v13, q2, s2, v2 = moe_case(3, 4, 2, 256, 64, 64, HF, seed=9)
    s13, v13 = s13 * 2048, v13 * 2048
    s2, v2 = s2 * 2.0 ** -16, v2 * 2.0 ** -16
    y = I4.moe_int4(x, router, q13, s13, q2, s2, 2, 64)
    ref, bound = moe_reference(x, router, v13, v2, 2, True, "silu")
    gu = x.double() @ v13[0].T
    assert (gu[:, :64] * gu[:, 64:]).abs().max() > 65504
    close(y, ref, bound)


def test_moe_views_and_empty():
    x, router, q13, s13, v13, q2, s2, v2 = moe_case(10, 6, 2, 250, 60, 32, BF, seed=10)
    y = I4.moe_int4(x, router, q13, s13, q2, s2, 2, 32)
    wide = torch.zeros(10, 300, dtype=BF, device="cuda")
    wide[:, 7:257] = x
    assert torch.equal(I4.moe_int4(wide[:, 7:257], router, q13, s13, q2, s2, 2, 32), y)
    assert torch.equal(I4.moe_int4(x.view(2, 5, 250), router, q13, s13, q2, s2, 2, 32), y.view(2, 5, 250))
    assert torch.equal(I4.moe_int4(x.t().contiguous().t(), router, q13, s13, q2, s2, 2, 32), y)
    assert I4.moe_int4(x[:0], router, q13, s13, q2, s2, 2, 32).shape == (0, 250)


@pytest.mark.parametrize("t", [1, 20])
def test_moe_repeats_streams_and_graphs(t):
    x, router, q13, s13, v13, q2, s2, v2 = moe_case(t, 16, 4, 512, 256, 128, BF, seed=11)
    args = (router, q13, s13, q2, s2, 4)
    y = I4.moe_int4(x, *args)
    for _ in range(3):
        assert torch.equal(I4.moe_int4(x, *args), y)
    xs = [randn(t, 512, seed=20 + j, dtype=BF) for j in range(4)]
    ref = [I4.moe_int4(v, *args) for v in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    out = [None] * 4
    for j, st in enumerate(streams):  # four at a time, a workspace each
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            for _ in range(5):
                out[j] = I4.moe_int4(xs[j], *args)
    torch.cuda.synchronize()
    for a, b in zip(out, ref):
        assert torch.equal(a, b)
    graphs, outs = [], []
    for v in xs[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(I4.moe_int4(v, *args))
        graphs.append(g)
    for j in (0, 1, 0):
        outs[j].zero_()
        graphs[j].replay()
        assert torch.equal(outs[j], ref[j])
    xs[0].copy_(xs[3])
    graphs[0].replay()
    assert torch.equal(outs[0], ref[3])


def test_moe_refusals():
    x, router, q13, s13, v13, q2, s2, v2 = moe_case(3, 6, 2, 256, 64, 64, BF, seed=12)
    for bad in (lambda: I4.moe_int4(x, router, q13, s13, q2, s2, 7, 64),
                lambda: I4.moe_int4(x, router, q13, s13, q2, s2, 0, 64),
                lambda: I4.moe_int4(x, router[:5], q13, s13, q2, s2, 2, 64),
                lambda: I4.moe_int4(x, router, q13[:5], s13[:5], q2, s2, 2, 64),
                lambda: I4.moe_int4(x, router, q13[:, :127].contiguous(), s13[:, :127].contiguous(), q2, s2, 2, 64),
                lambda: I4.moe_int4(x[:, :100], router, q13, s13, q2, s2, 2, 64),
                lambda: I4.moe_int4(x, router, q13, s13, q2, s2, 2, 128),
                lambda: I4.moe_int4(x, router.t().contiguous().t(), q13, s13, q2, s2, 2, 64)):
        with pytest.raises(AssertionError):
            bad()
    for bad in (lambda: I4.moe_int4(x.float(), router, q13, s13, q2, s2, 2, 64),
                lambda: I4.moe_int4(x, router.half(), q13, s13, q2, s2, 2, 64)):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(RuntimeError, match="backward"):
        I4.moe_int4(x.clone().requires_grad_(), router, q13, s13, q2, s2, 2, 64)


# --------------------------------------------------------- a run of them
@pytest.mark.parametrize("t", [1, 6])
def test_decode_step_of_a_quantized_block(t):
    """What a block does for new tokens: quantise float weights, project, experts, project back."""
    h, e, i, group = 384, 5, 160, 64
    w_in, w_out = randn(h, 256, seed=1, scale=0.05, dtype=BF), randn(256, h, seed=2, scale=0.05, dtype=BF)
    wi, wo = (QuantizedTensor.from_float(w, "GroupWiseINT4Layout", group_size=group) for w in (w_in, w_out))
    q13, s13 = I4.weight_quant_int4(randn(e, 2 * i, h, seed=3, scale=0.05, dtype=BF), group)
    q2, s2 = I4.weight_quant_int4(randn(e, h, i, seed=4, scale=0.05, dtype=BF), group)
    router = randn(e, h, seed=5, scale=h ** -0.5)
    x = randn(t, 256, seed=6, dtype=BF)

    a = F.linear(x, wi)
    m = I4.moe_int4(a, router, q13, s13, q2, s2, 2, group)
    y = F.linear(m, wo)

    # each step against 64 bits on the previous step's own output
    vi, vo = wi.dequantize().double(), wo.dequantize().double()
    close(a, x.double() @ vi.T, ACC * (x.double().abs() @ vi.abs().T))
    v13 = I4.weight_dequant_int4(q13, s13, h, group, F32).double()
    v2 = I4.weight_dequant_int4(q2, s2, i, group, F32).double()
    close(m, *moe_reference(a, router, v13, v2, 2, True, "silu"))
    close(y, m.double() @ vo.T, ACC * (m.double().abs() @ vo.abs().T))


def test_shortcut_and_python_path_agree(monkeypatch):
    """The wrappers' host-side shortcut computes what they compute without it, and leaves the rest to them."""
    assert L.fast_call() is not None, "csrc/call.cpp is not built"
    w = randn(3, 40, 300, seed=1, dtype=BF)
    x, b = randn(2, 5, 300, seed=2, dtype=BF), randn(40, seed=3)
    mx, router, q13, s13, _, q2, s2, _ = moe_case(7, 6, 2, 256, 64, 64, BF, seed=4)

    def calls():
        q, s = I4.weight_quant_int4(w, 64)
        return [q, s, I4.weight_dequant_int4(q, s, 300, 64, BF), I4.int4_linear(x, q[0], s[0], 64, b),
                I4.int4_linear(x[0], q[0], s[0], 64), I4.moe_int4(mx, router, q13, s13, q2, s2, 2, 64, False, "gelu"),
                I4.moe_int4(mx.view(1, 7, 256), router.float(), q13, s13, q2, s2, 2, 64)]

    fast = calls()
    f = L.fast_call()
    q, s = fast[0][0].contiguous(), fast[1][0].contiguous()
    xg = x.clone().requires_grad_()
    for args in ((x[..., ::2], q, s, 64, None), (x, q, s, 128, None), (x.float(), q, s, 64, None),
                 (xg, q, s, 64, None), (x, q, s, 64, b[:39]), (x.cpu(), q, s, 64, None), (x, q.cpu(), s, 64, None),
                 (x, q, s, 64, b.double()), (x[0, 0], q, s, 64, None), (x[:, :0], q, s, 64, None)):
        assert f.gemm_w4(*args) is None
    monkeypatch.setattr(L, "_call", False)
    for a, c in zip(fast, calls()):
        assert a.shape == c.shape and a.dtype == c.dtype and torch.equal(a, c)
