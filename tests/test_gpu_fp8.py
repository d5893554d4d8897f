"""GPU tests of the fp8 operators against plain forms in 64 bits.

Quantization is exact arithmetic and one rounding: codes and scales are equal to
the oracle's.  Products: a product of two codes is exact in fp32, as are the
scales' factors; a tensor-core step adds at most 32 products to the accumulator.
With 24 bits kept relative to the largest of those 33 terms each step is off by
33 * 2^-23 of S, the sum of the absolute values, and there are K / 32 of them, plus
one addition per split: at most (33 K / 32 + 64) * 2^-23 S.  The output is rounded
once: half a step, eps / 2 of the value.
"""

import numpy as np
import pytest
import torch
import torch.nn.functional as F

import oracle as O
from convert_to_quant_quip_int8_b200 import _lib as L
from convert_to_quant_quip_int8_b200 import ops
from convert_to_quant_quip_int8_b200.comfy import fp8_kernels as F8
from convert_to_quant_quip_int8_b200.comfy.quant_ops import QuantizedTensor

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
E4, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


@pytest.fixture(autouse=True)
def _status():
    yield
    ops.device_status(reset=True)


def randn(*shape, seed=0, scale=1.0, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def wide(*shape, seed=0, dtype=F32):
    """Values of very different sizes from block to block and row to row."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * torch.exp2(torch.randint(-9, 9, shape[:-1] + (1,), generator=g).float())
    n = shape[-1]
    f = torch.exp2(torch.randint(-6, 4, (-(-n // 128),), generator=g).float()).repeat_interleave(128)[:n]
    return (x * f).to(dtype).cuda()


def same_codes(q, s, v, tile):
    qo, so = O.f8_quantize(v.double().cpu().numpy(), tile)
    assert np.array_equal(s.double().cpu().numpy(), so, equal_nan=True)
    assert np.array_equal(q.double().cpu().numpy(), qo, equal_nan=True)
    return qo, so


def values(q, s, tile):
    """fp64 values on the GPU."""
    s = s.double()
    if tile > 1:
        s = s.repeat_interleave(tile, -2)[..., :q.shape[-2], :]
    return q.double() * s.repeat_interleave(128, -1)[..., :q.shape[-1]]


def check_product(y, a, b, bias=None):
    """y against a b^T + bias for fp64 values a and b."""
    k = a.shape[-1]
    ref = a @ b.T
    total = a.abs() @ b.abs().T
    if bias is not None:
        ref, total = ref + bias.double(), total + bias.double().abs()
    bound = (33 * k / 32 + 64) * 2.0 ** -23 * total
    info = torch.finfo(y.dtype)
    tol = bound + info.eps / 2 * (ref.abs() + bound) + info.smallest_normal * info.eps
    assert torch.isfinite(y).all()
    worst = ((y.double() - ref).abs() / tol).max().item()
    assert worst <= 1.0, f"{worst:.3g} times the tolerance"


# ------------------------------------------------------------ quantization
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("n,k", [(1, 1), (3, 31), (7, 128), (129, 129), (5, 1100), (128, 256), (300, 2989), (2, 20000)])
def test_quantizers_match_the_definition(n, k, dtype):
    x = wide(n, k, seed=n + k, dtype=dtype)
    for quant, dequant, tile in ((F8.act_quant_fp8, F8.act_dequant_fp8, 1),
                                 (F8.weight_quant_fp8, F8.weight_dequant_fp8, 128)):
        q, s = quant(x)
        assert q.dtype == E4 and s.dtype == E8 and q.shape == x.shape
        qo, so = same_codes(q, s, x, tile)
        v = torch.from_numpy(O.f8_values(qo, so, tile))
        for out in (BF, HF, F32):
            assert torch.equal(dequant(q, s, output_dtype=out).cpu(), v.to(out))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_quantizers_at_borders(dtype):
    # ties between codes, amax on and beside 448 * 2^e, zeros, the smallest and largest numbers
    codes = torch.arange(0, 127, dtype=torch.uint8).view(E4).double()
    mid = (codes[1:] + codes[:-1]) / 2
    rows = []
    for top in (448.0, 449.0, 447.0, 224.0):
        row = torch.zeros(256, dtype=torch.float64)
        row[0], row[128] = top, -top
        row[1:127], row[129:255] = mid, -mid * (1 + 2.0 ** -7)
        rows.append(row)
    rows += [torch.zeros(256, dtype=torch.float64), torch.full((256,), torch.finfo(dtype).max, dtype=torch.float64),
             torch.full((256,), 2.0 ** -126, dtype=torch.float64), torch.linspace(0, 2.0 ** -92, 256, dtype=torch.float64)]
    x = torch.stack(rows).to(dtype).cuda()
    same_codes(*F8.act_quant_fp8(x), x, 1)
    for r in range(x.shape[0]):
        same_codes(*F8.weight_quant_fp8(x[r:r + 1]), x[r:r + 1], 128)


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_blocks_that_are_not_finite(bad):
    x = randn(260, 300, dtype=BF)
    x[1, 130] = bad
    for quant, dequant, tile, hurt in ((F8.act_quant_fp8, F8.act_dequant_fp8, 1, np.s_[1:2, 128:256]),
                                       (F8.weight_quant_fp8, F8.weight_dequant_fp8, 128, np.s_[0:128, 128:256])):
        q, s = quant(x)
        same_codes(q, s, x, tile)
        v = dequant(q, s, output_dtype=F32)
        expected = torch.zeros(260, 300, dtype=torch.bool)
        expected[hurt] = True
        assert torch.equal(torch.isnan(v).cpu(), expected) and torch.isfinite(v.cpu()[~expected]).all()


def test_quantizers_take_strides_and_leading_dimensions():
    big = wide(6, 10, 300, dtype=BF)
    for x in (big[:, 1:7, 3:260], big.transpose(0, 1), big[::2], big[:, :, ::3], big[0, 0], big[:, :0], big[..., :0],
              big[:1, :1].expand(3, 4, 300), big[:, :1].expand(6, 4, 300), big[:1].expand(5, 10, 300), big[0, :3, None].expand(
                  3, 4, 300), big[:, 0].unsqueeze(1), big[:, 2:3, 8:], big.view(-1)[1:1 + 59 * 300].view(59, 300)):
        q, s = F8.act_quant_fp8(x)
        assert q.shape == x.shape and s.shape == (*x.shape[:-1], -(-x.shape[-1] // 128))
        if x.numel():
            same_codes(q.reshape(-1, x.shape[-1]), s.reshape(-1, s.shape[-1]), x.reshape(-1, x.shape[-1]), 1)
    w = big.view(60, 300)
    for x in (w[:, 5:], w.t(), w[::3], w[:0], w[:, :0], w.view(-1)[1:1 + 59 * 300].view(59, 300)):
        q, s = F8.weight_quant_fp8(x)
        assert q.shape == x.shape
        if x.numel():
            same_codes(q, s, x, 128)


# ----------------------------------------------------------------- product
SHAPES = [(1, 1, 1), (1, 128, 128), (1, 4096, 512), (2, 130, 129), (5, 257, 1000), (8, 64, 4096), (9, 5003, 301),
          (16, 300, 2048), (17, 128, 256), (31, 999, 130), (33, 640, 640), (64, 129, 1280), (65, 1000, 200),
          (127, 384, 3000), (129, 257, 1024), (200, 513, 2176), (256, 256, 128), (257, 1300, 640), (512, 2000, 96),
          (1000, 777, 333), (700, 2048, 512)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("out", [BF, HF, F32])
def test_gemm(m, n, k, out):
    a, a_s = F8.act_quant_fp8(wide(m, k, seed=m))
    b, b_s = F8.weight_quant_fp8(randn(n, k, seed=n, scale=2.0 ** -12 if out == HF else 0.02))
    bias = randn(n, seed=k, dtype=BF) if (m + n) % 2 else None
    y = F8.fp8_gemm(a, a_s, b, b_s, bias=bias, out_dtype=out)
    assert y.dtype == out and y.shape == (m, n)
    check_product(y, values(a, a_s, 1), values(b, b_s, 128), bias)


# more tiles than blocks: the rings, scales and accumulators go round
@pytest.mark.parametrize("m,n,k", [(17, 20000, 300), (32, 40000, 1100), (50, 20100, 640), (64, 30000, 129),
                                   (100, 20000, 640), (100, 33000, 4096), (128, 24000, 130), (300, 20000, 384),
                                   (2000, 5000, 640), (4100, 2600, 1300)])
def test_gemm_with_many_tiles(m, n, k):
    a, a_s = F8.act_quant_fp8(wide(m, k, seed=m))
    b, b_s = F8.weight_quant_fp8(wide(n, k, seed=n))
    va, vb = values(a, a_s, 1), values(b, b_s, 128)
    for _ in range(3):
        check_product(F8.fp8_gemm(a, a_s, b, b_s, out_dtype=F32), va, vb)


# few tiles of many columns: blocks that share them
@pytest.mark.parametrize("m", [1, 16, 17, 40, 65, 100, 128, 200])
@pytest.mark.parametrize("n,k", [(100, 16384), (520, 8200), (2050, 4000), (4096, 4096), (4000, 10240)])
def test_gemm_with_split_columns(m, n, k):
    a, a_s = F8.act_quant_fp8(wide(m, k, seed=m))
    b, b_s = F8.weight_quant_fp8(wide(n, k, seed=n))
    y = F8.fp8_gemm(a, a_s, b, b_s, out_dtype=F32)
    check_product(y, values(a, a_s, 1), values(b, b_s, 128))
    assert all(torch.equal(y, F8.fp8_gemm(a, a_s, b, b_s, out_dtype=F32)) for _ in range(3))


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_linear(m, n, k, dtype):
    x = randn(m, k, seed=m + 1, dtype=dtype)
    w, w_s = F8.weight_quant_fp8(randn(n, k, seed=n, scale=0.02))
    bias = randn(n, seed=k, dtype=dtype) if (m + k) % 2 else None
    y = F8.fp8_linear(x, w, w_s, bias)
    assert y.dtype == dtype and y.shape == (m, n)
    a, a_s = F8.act_quant_fp8(x)
    check_product(y, values(a, a_s, 1), values(w, w_s, 128), bias)


@pytest.mark.parametrize("m,n,k", [(1, 300, 200), (16, 300, 256), (40, 300, 200), (300, 300, 200), (300, 512, 512)])
def test_scales_reach_their_own_blocks(m, n, k):
    # every block of either operand has a scale of its own: a misplaced one changes the result by factors
    g = torch.Generator().manual_seed(m)
    a = torch.randint(-3, 4, (m, k), generator=g).float().to(E4).cuda()
    b = torch.randint(-3, 4, (n, k), generator=g).float().to(E4).cuda()
    a_s = torch.randint(120, 135, (m, -(-k // 128)), generator=g, dtype=torch.uint8).cuda().view(E8)
    b_s = torch.randint(120, 135, (-(-n // 128), -(-k // 128)), generator=g, dtype=torch.uint8).cuda().view(E8)
    check_product(F8.fp8_gemm(a, a_s, b, b_s, out_dtype=F32), values(a, a_s, 1), values(b, b_s, 128))


@pytest.mark.parametrize("m", [1, 20, 300])
def test_extreme_scales(m):
    n, k = 200, 384
    a = torch.ones(m, k).to(E4).cuda()
    b = torch.ones(n, k).to(E4).cuda()
    a_s = torch.full((m, 3), 27, dtype=torch.uint8).cuda()
    b_s = torch.full((2, 3), 227, dtype=torch.uint8).cuda()
    y = F8.fp8_gemm(a, a_s.view(E8), b, b_s.view(E8), out_dtype=F32)  # 2^-100 * 2^100
    assert (y == k).all()
    a_s[0, 1] = 255
    y = F8.fp8_gemm(a, a_s.view(E8), b, b_s.view(E8), out_dtype=F32)
    assert torch.isnan(y[0]).all() and (y[1:] == k).all()
    a_s[0, 1] = 27
    b_s[1, 2] = 255
    y = F8.fp8_gemm(a, a_s.view(E8), b, b_s.view(E8), out_dtype=F32)
    assert torch.isnan(y[:, 128:]).all() and (y[:, :128] == k).all()


@pytest.mark.parametrize("m", [1, 20, 300, 2000])
@pytest.mark.parametrize("a_code,b_code", [(0, 254), (254, 0), (1, 253), (0, 0), (200, 200)])
def test_scales_at_the_ends(m, a_code, b_code):
    n, k = 2600, 130
    a, b = torch.ones(m, k).to(E4).cuda(), torch.ones(n, k).to(E4).cuda()
    a_s = torch.full((m, 2), a_code, dtype=torch.uint8).cuda().view(E8)
    b_s = torch.full((21, 2), b_code, dtype=torch.uint8).cuda().view(E8)
    y = F8.fp8_gemm(a, a_s, b, b_s, out_dtype=F32)
    # 2^(a + b - 254) k, or what fp32 makes of it
    assert (y == torch.tensor(float(k) * 2.0 ** (a_code + b_code - 254), dtype=torch.float64).float().item()).all()


@pytest.mark.parametrize("m", [1, 12, 40, 300])
def test_nan_stays_in_its_row_and_tile(m):
    x, w = randn(m, 300, dtype=BF), randn(260, 300, seed=1, dtype=BF)
    x[m // 2, 7] = float("nan")
    w[130, 290] = float("inf")
    wq = F8.weight_quant_fp8(w)
    for y in (F8.fp8_linear(x, *wq), F8.fp8_gemm(*F8.act_quant_fp8(x), *wq)):
        expected = torch.zeros(m, 260, dtype=torch.bool)
        expected[m // 2] = True
        expected[:, 128:256] = True
        assert torch.equal(torch.isnan(y).cpu(), expected)


@pytest.mark.parametrize("m", [3, 40, 300])
def test_operands_with_strides_and_odd_alignment(m):
    n, k = 300, 333
    x, w = randn(m, k, dtype=BF), randn(n, k, seed=2, scale=0.02, dtype=BF)
    a, a_s = F8.act_quant_fp8(x)
    b, b_s = F8.weight_quant_fp8(w)
    va, vb = values(a, a_s, 1), values(b, b_s, 128)

    def off_by(t, d):  # the same rows, contiguous, starting d bytes off a 16-byte boundary
        r = torch.empty(t.numel() + 16, dtype=torch.uint8, device="cuda")[d:d + t.numel()].view(t.shape)
        return r.copy_(t.contiguous().view(torch.uint8)).view(E4)
    for a2 in (a, a.contiguous(), off_by(a, 1), a.t().contiguous().t()):
        for b2 in (b, b.contiguous(), off_by(b, 8), b.t().contiguous().t()):
            check_product(F8.fp8_gemm(a2, a_s, b2, b_s), va, vb)
    both = torch.cat([x, x], 1)
    for x2 in (both[:, k:], both[:, :k], x.t().contiguous().t()):
        check_product(F8.fp8_linear(x2, b.contiguous(), b_s), va, vb)


def test_leading_dimensions_and_empty_operands():
    x, w = randn(2, 3, 200, dtype=BF), randn(130, 200, seed=3, dtype=BF)
    wq = F8.weight_quant_fp8(w)
    y = F8.fp8_linear(x, *wq)
    assert y.shape == (2, 3, 130)
    assert torch.equal(y.view(6, 130), F8.fp8_linear(x.view(6, 200), *wq))
    assert torch.equal(y, F8.fp8_gemm(*F8.act_quant_fp8(x), *wq))
    assert F8.fp8_linear(x[0, 0], *wq).shape == (130,)
    assert F8.fp8_linear(x[:, :0], *wq).shape == (2, 0, 130)
    none = F8.weight_quant_fp8(w[:0])
    assert F8.fp8_linear(x, *none).shape == (2, 3, 0)
    bias = randn(130, dtype=BF)
    empty = F8.weight_quant_fp8(w[:, :0])
    assert torch.equal(F8.fp8_linear(x[..., :0], *empty, bias), bias.expand(2, 3, 130))
    assert torch.equal(F8.fp8_gemm(*F8.act_quant_fp8(x[..., :0]), *empty), torch.zeros(2, 3, 130, dtype=BF, device="cuda"))


def test_refusals():
    x, w = randn(4, 256, dtype=BF), randn(128, 256, dtype=BF)
    a, a_s = F8.act_quant_fp8(x)
    b, b_s = F8.weight_quant_fp8(w)
    with pytest.raises(AssertionError):
        F8.fp8_linear(x[:, :200], b, b_s)
    with pytest.raises(AssertionError):
        F8.fp8_gemm(a[:, :128], a_s[:, :1].contiguous(), b, b_s)
    with pytest.raises(AssertionError, match="Bias"):
        F8.fp8_linear(x, b, b_s, bias=x[0])
    with pytest.raises(TypeError):
        F8.fp8_linear(x.double(), b, b_s)
    with pytest.raises(TypeError):
        F8.fp8_gemm(a, a_s, b, b_s, out_dtype=torch.int32)
    with pytest.raises(TypeError):
        F8.act_quant_fp8(x.to(torch.int8))
    with pytest.raises(RuntimeError, match="backward"):
        F8.fp8_linear(x.clone().requires_grad_(), b, b_s)
    with pytest.raises(RuntimeError, match="backward"):
        F8.act_quant_fp8(x.clone().requires_grad_())
    with pytest.raises(RuntimeError):
        F8.fp8_linear(x.cpu(), b, b_s)
    with torch.no_grad():
        F8.fp8_linear(x.clone().requires_grad_(), b, b_s)
    F8.weight_quant_fp8(torch.nn.Parameter(w))


# -------------------------------------------------- streams, graphs, layout
@pytest.mark.parametrize("m", [1, 16, 40, 130, 600])
def test_same_bits_every_time_and_on_another_stream(m):
    x, w = randn(m, 1100, dtype=BF), randn(1000, 1100, seed=4, scale=0.02, dtype=BF)
    wq = F8.weight_quant_fp8(w)
    first = F8.fp8_linear(x, *wq)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        others = [F8.fp8_linear(x, *wq) for _ in range(8)]
    here = [F8.fp8_linear(x, *wq) for _ in range(8)]
    torch.cuda.synchronize()
    assert all(torch.equal(first, y) for y in others + here)


@pytest.mark.parametrize("m", [1, 16, 130, 600])
def test_captured_graphs_replay_with_new_inputs(m):
    x, w = randn(m, 512, dtype=BF), randn(700, 512, seed=5, scale=0.02, dtype=BF)
    wq = F8.weight_quant_fp8(w)
    F8.fp8_linear(x, *wq)
    graphs, outs = [], []
    for _ in range(2):  # each has a workspace of its own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(F8.fp8_linear(x, *wq))
        graphs.append(g)
    for seed in (6, 7):
        x.copy_(randn(m, 512, seed=seed, dtype=BF))
        streams = [torch.cuda.Stream() for _ in graphs]
        for g, s in zip(graphs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        expected = F8.fp8_linear(x, *wq)
        assert all(torch.equal(expected, o) for o in outs)


@pytest.mark.parametrize("m", [1, 5, 16, 40, 300])
def test_two_streams_at_once(m):
    x = [randn(m, 2100, seed=s, dtype=BF) for s in (1, 2)]
    w = [F8.weight_quant_fp8(randn(1900, 2100, seed=s, scale=0.02, dtype=BF)) for s in (3, 4)]
    expected = [F8.fp8_linear(*p) for p in ((x[0], *w[0]), (x[1], *w[1]))]
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(F8.fp8_linear(x[i], *w[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, expected[i]) for y in outs[i])


@pytest.mark.parametrize("m", [1, 9, 40, 600])
def test_operands_written_just_before(m):
    # kernels that start while the one before ends must not read what it still writes
    n, k = 1500, 2048
    xs, ws = [randn(m, k, seed=s, dtype=BF) for s in range(6)], [randn(n, k, seed=s, scale=0.05, dtype=BF) for s in range(6)]
    expected = [F8.fp8_linear(x, *F8.weight_quant_fp8(w)) for x, w in zip(xs, ws)]
    torch.cuda.synchronize()
    x, w = torch.empty_like(xs[0]), torch.empty_like(ws[0])
    q, s = F8.weight_quant_fp8(ws[0])
    got = []
    for i in list(range(6)) * 5:
        x.copy_(xs[i])
        w.copy_(ws[i])
        q2, s2 = F8.weight_quant_fp8(w)
        q.copy_(q2)
        s.copy_(s2)
        got.append(F8.fp8_linear(x, q, s))
        got.append(F8.fp8_linear(x, *F8.weight_quant_fp8(w)))
    for j, y in enumerate(got):
        assert torch.equal(y, expected[j // 2 % 6])


def test_rows_behind_the_result_are_left_alone():
    lib, m, n, k = L.load(), 5, 70, 256
    for m in (5, 40, 300):
        a, a_s = F8.act_quant_fp8(randn(m, k, dtype=BF))
        b, b_s = F8.weight_quant_fp8(randn(n, k, seed=1, dtype=BF))
        out = torch.full((m + 3, n + 9), 7.0, dtype=BF, device="cuda")
        rc = lib.qi8_gemm_f8(a.data_ptr(), a_s.data_ptr(), m, k, k, b.data_ptr(), b_s.data_ptr(), n, k, None, 0,
                             out.data_ptr(), L.QI8_BF16, n + 9, None, 0, torch.cuda.current_stream().cuda_stream)
        L.check(rc)
        assert (out[m:] == 7).all() and (out[:, n:] == 7).all()
        assert torch.equal(out[:m, :n], F8.fp8_gemm(a, a_s, b, b_s))


def test_layout_linear():
    x, w, bias = randn(2, 40, 300, dtype=BF), randn(260, 300, seed=8, scale=0.02, dtype=BF), randn(260, dtype=BF)
    wq = QuantizedTensor.from_float(w, "BlockWiseFP8Layout", is_weight=True)
    xq = QuantizedTensor.from_float(x, "BlockWiseFP8Layout")
    q, s = F8.weight_quant_fp8(w)
    expected = F8.fp8_linear(x, q, s, bias)
    assert torch.equal(F.linear(x, wq, bias), expected)
    assert torch.equal(F.linear(xq, wq, bias), expected)
    assert torch.equal(F.linear(input=x, weight=wq, bias=bias), expected)
    assert wq.shape == w.shape and torch.equal(wq.dequantize(), F8.weight_dequant_fp8(q, s, output_dtype=BF))
    # a plain weight: the activations' values
    assert torch.equal(F.linear(xq, w, bias), F.linear(xq.dequantize(), w, bias))
    c = wq.clone()
    assert torch.equal(F.linear(x, c, bias), expected)
    back = wq.cpu().cuda()
    assert torch.equal(F.linear(x, back, bias), expected)
    c.copy_(QuantizedTensor.from_float(w * 2, "BlockWiseFP8Layout", is_weight=True))
    assert torch.equal(F.linear(x, c), F8.fp8_linear(x, *F8.weight_quant_fp8(w * 2)))


@pytest.mark.parametrize("m,ld", [(5, 1 << 30), (20, 1 << 28), (300, 1 << 24)])
def test_codes_far_apart(m, ld):
    # offsets beyond 32 bits in either operand
    k, n = 400, 1000
    a, a_s = F8.act_quant_fp8(randn(m, k, dtype=BF))
    b, b_s = F8.weight_quant_fp8(randn(n, k, seed=1, dtype=BF))
    far = torch.empty((m - 1) * ld + k, dtype=E4, device="cuda").as_strided((m, k), (ld, 1))
    far.view(torch.uint8).copy_(a.view(torch.uint8))
    assert torch.equal(F8.fp8_gemm(far, a_s, b, b_s), F8.fp8_gemm(a, a_s, b, b_s))
    a2, a2_s = F8.act_quant_fp8(randn(n, k, seed=1, dtype=BF))
    b2, b2_s = F8.weight_quant_fp8(randn(m, k, dtype=BF))
    far.view(torch.uint8).copy_(b2.view(torch.uint8))
    for t in (9, 100, n):
        assert torch.equal(F8.fp8_gemm(a2[:t], a2_s[:t], far, b2_s), F8.fp8_gemm(a2[:t], a2_s[:t], b2, b2_s))


@pytest.mark.parametrize("m,n,out", [(70000, 32768, BF), (128, 8388480, F32)])
def test_results_beyond_32_bits(m, n, out):
    k = 128 if m > 1000 else 16
    a, a_s = F8.act_quant_fp8(randn(m, k, dtype=BF))
    b, b_s = F8.weight_quant_fp8(randn(n, k, seed=1, dtype=BF))
    y = F8.fp8_gemm(a, a_s, b, b_s, out_dtype=out)
    rows, cols = slice(max(0, m - 300), m), slice(n - n % 128 - 128, n)
    va, vb = values(a[rows], a_s[rows], 1), values(b[cols], b_s[cols.start // 128:], 128)
    check_product(y[rows, cols], va, vb)


@pytest.mark.parametrize("k", [31, 300, 2989])
def test_a_single_row_has_no_stride(k):
    lib = L.load()
    for m, n in ((1, 70), (1, 1), (12, 1), (1, 5003)):
        a, a_s = F8.act_quant_fp8(randn(m, k, dtype=BF))
        b, b_s = F8.weight_quant_fp8(randn(n, k, seed=1, dtype=BF))
        y = F8.fp8_gemm(a, a_s, b, b_s, out_dtype=F32)
        check_product(y, values(a, a_s, 1), values(b, b_s, 128))
        assert torch.equal(F8.fp8_gemm(a.contiguous(), a_s, b, b_s, out_dtype=F32), y)
        assert torch.equal(F8.fp8_gemm(a, a_s, b.contiguous(), b_s, out_dtype=F32), y)
    one, many = torch.empty(k, dtype=E4, device="cuda"), torch.empty(2, k, dtype=E4, device="cuda")
    assert lib.qi8_gemm_f8_workspace_bytes(one.data_ptr(), 1, k, k, one.data_ptr(), 1, k) == 0
    assert lib.qi8_gemm_f8_workspace_bytes(many.data_ptr(), 2, k, k, one.data_ptr(), 1, k) == 2 * (-(-k // 16) * 16)


@pytest.mark.parametrize("m,n,k", [(1, 6144, 4096), (2, 6144, 4096), (3, 4096, 5120), (5, 2560, 2560), (8, 4096, 2560),
                                   (9, 2560, 2560), (4, 8192, 1024), (4, 8208, 1024), (1, 500, 5248), (7, 1000, 2600),
                                   (33, 700, 2560), (100, 4096, 10240), (60, 2048, 1300), (128, 1024, 8192)])
def test_gemm_beside_the_borders_of_its_kernels(m, n, k):
    a, b = wide(m, k, seed=m), wide(n, k, seed=n)
    bias = randn(n, seed=5, dtype=HF)
    (aq, a_s), (bq, b_s) = F8.act_quant_fp8(a), F8.weight_quant_fp8(b)
    for out in (BF, F32):
        check_product(F8.fp8_gemm(aq, a_s, bq, b_s, bias, out), values(aq, a_s, 1), values(bq, b_s, 128), bias)
    assert torch.equal(F8.fp8_linear(a.to(BF), bq, b_s), F8.fp8_gemm(*F8.act_quant_fp8(a.to(BF)), bq, b_s))


@pytest.mark.parametrize("m", [1, 60, 700])
def test_beside_the_other_products_on_another_stream(m):
    # both kinds of kernels hold tensor memory and most of an SM's shared memory
    k, n = 1024, 2048
    x = randn(m, k, dtype=BF)
    w, w_s = F8.weight_quant_fp8(randn(n, k, seed=1, dtype=BF))
    a, b = (torch.randint(-127, 128, s, dtype=torch.int8, device="cuda") for s in ((600, k), (n, k)))
    w4, s4 = ops.quant_weight_i4(randn(n, k, seed=2, dtype=BF))
    y8, y32, y4 = F8.fp8_linear(x, w, w_s), ops.gemm_i8(a, b, out_dtype=torch.int32), ops.gemm_w4(x, w4, s4)
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(20):
        with torch.cuda.stream(one):
            got.append((F8.fp8_linear(x, w, w_s), y8))
        with torch.cuda.stream(two):
            got.append((ops.gemm_i8(a, b, out_dtype=torch.int32), y32))
            got.append((ops.gemm_w4(x, w4, s4), y4))
            got.append((F8.fp8_linear(x, w, w_s), y8))
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for u, v in got)
