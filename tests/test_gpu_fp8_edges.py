"""GPU tests of the fp8 operators where their kernels, layouts and launches change over."""

import pytest
import torch
import torch.nn.functional as F

from convert_to_quant_quip_int8_b200 import _lib as L
from convert_to_quant_quip_int8_b200 import ops
from convert_to_quant_quip_int8_b200.comfy import fp8_kernels as F8
from convert_to_quant_quip_int8_b200.comfy.quant_ops import QuantizedTensor
from test_gpu_fp8 import check_product, randn, values, wide

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


# as many tiles as clusters of four, or of two and eight, run at once, and one more
@pytest.mark.parametrize("m", [9, 64, 100])
@pytest.mark.parametrize("n,k", [(4224, 4096), (4225, 4096), (4160, 10240), (1920, 10240), (1921, 10240), (9472, 2048),
                                 (9473, 2048)])
def test_gemm_with_as_many_clusters_as_run_at_once(m, n, k):
    a, a_s = F8.act_quant_fp8(wide(m, k, seed=m))
    b, b_s = F8.weight_quant_fp8(wide(n, k, seed=n))
    y = F8.fp8_gemm(a, a_s, b, b_s, out_dtype=F32)
    check_product(y, values(a, a_s, 1), values(b, b_s, 128))
    assert all(torch.equal(y, F8.fp8_gemm(a, a_s, b, b_s, out_dtype=F32)) for _ in range(3))


# ------------------------------------------------------- kernels in a chain
# The one read before the wait for the last kernel: gemm_f8_rows_kernel copies its weight while the tokens' quantizer
# runs.  Cases that get there (at most 8 tokens, more than 8192 values of x): 5 and 8 x 2048, 3 x 4096.  5 and 8 x 2100
# with contiguous codes too, behind a kernel that brings the weight to rows of 16 bytes.  2 x 2048 quantizes in each
# block and waits first, 9 x 2048 goes to the tcgen05 kernel.
@pytest.mark.parametrize("m,k,contiguous", [(2, 2048, False), (5, 2048, False), (8, 2048, False), (3, 4096, False),
                                            (5, 2100, True), (8, 2100, True), (3, 4090, True), (9, 2048, False),
                                            (9, 2100, True)])
def test_weights_written_just_before(m, k, contiguous):
    n = 1500
    xs, ws = [randn(m, k, seed=s, dtype=BF) for s in range(4)], [randn(n, k, seed=s, scale=0.05, dtype=BF) for s in range(4)]
    ready = [F8.weight_quant_fp8(w) for w in ws]
    if contiguous:
        ready = [(q.contiguous(), s) for q, s in ready]
    expected = [F8.fp8_linear(x, *w) for x, w in zip(xs, ready)]
    torch.cuda.synchronize()
    x, q, s = torch.empty_like(xs[0]), ready[0][0].clone(), ready[0][1].clone()
    assert not contiguous or q.stride(0) % 16
    got = []
    for i in list(range(4)) * 6:
        x.copy_(xs[i])
        s.view(torch.uint8).copy_(ready[i][1].view(torch.uint8))
        q.copy_(ready[i][0])  # the kernel before the product's first
        got.append((F8.fp8_linear(x, q, s), expected[i]))
        w, w_s = F8.weight_quant_fp8(ws[i])  # one that lets the next start early
        got.append((F8.fp8_linear(x, w.contiguous() if contiguous else w, w_s), expected[i]))
    # the same in a graph, where launches follow one another at once
    g, outs = torch.cuda.CUDAGraph(), []
    with torch.cuda.graph(g):
        for i in list(range(4)) * 3:
            w, w_s = F8.weight_quant_fp8(ws[i])
            q.view(torch.uint8).copy_(w.view(torch.uint8))
            s.view(torch.uint8).copy_(w_s.view(torch.uint8))
            outs.append((F8.fp8_linear(xs[i], w, w_s), expected[i]))
            outs.append((F8.fp8_linear(xs[i], q, s), expected[i]))
    for _ in range(5):
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(y, e) for y, e in got + outs)


# ------------------------------------------------------------------- sums
@pytest.mark.parametrize("m,n,k", [(1, 300, 5120), (4, 300, 5120), (8, 300, 2560), (16, 300, 16384), (100, 520, 16384),
                                   (128, 5000, 16384), (300, 5000, 16384)])
def test_sums_keep_24_bits(m, n, k):
    # odd codes from 9 to 15: products of 81 to 225 are whole numbers, as are sums of any order, which stay under 2^22
    # and so are exact in fp32, and in nothing with fewer than 22 bits
    g = torch.Generator().manual_seed(m)
    a, b = (torch.randint(4, 8, s, generator=g).mul(2).add(1).float().cuda() for s in ((m, k), (n, k)))
    one = [torch.full(s, 127, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
           for s in ((m, -(-k // 128)), (-(-n // 128), -(-k // 128)))]
    y = F8.fp8_gemm(a.to(torch.float8_e4m3fn), one[0], b.to(torch.float8_e4m3fn), one[1], out_dtype=F32)
    want = a.double() @ b.double().T
    assert want.max() < 2 ** 22 and torch.equal(y.double(), want)
    # and beside a product 2^17 times as large as the others' sum: the accumulator's last bits count
    a[:, 0], b[:, 0] = 448.0, 448.0
    for side, t in ((0, a), (1, b)):
        one[side].view(torch.uint8)[:, 0] = 127 + 2
    a[:, 1:128], b[:, 1:128] = 0.0, 0.0
    y = F8.fp8_gemm(a.to(torch.float8_e4m3fn), one[0], b.to(torch.float8_e4m3fn), one[1], out_dtype=F32)
    want = 448.0 * 448.0 * 16 + a[:, 128:].double() @ b[:, 128:].double().T
    assert want.max() < 2 ** 24 and torch.equal(y.double(), want)
