"""More GPU tests of the 4-bit operators: the ends of their types, their variants for large layers, what they refuse.

Weights are random codes in [-8, 7] and random scales, unpacked on the GPU by the
oracle's table of positions.  Tolerances: a tensor-core step sums 16 products
(exact in fp32) and its accumulator and is off by at most 17 * 2^-23 of the sum of
absolute values S.  ``steps`` of them in one accumulator, and the few additions
that join warps, groups or splits, are off by at most (17 steps + 264) * 2^-23 S:
8 steps per group and up to 256 groups of a warp in the rows kernel, all steps
of K in the tiles kernel.  The output is rounded once, half a step.
"""

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fwAD
import torch.nn.functional as F

import oracle as O
from convert_to_quant_quip_int8_b200 import ops
from convert_to_quant_quip_int8_b200.comfy import int4_kernels as I4
from convert_to_quant_quip_int8_b200.comfy.quant_ops import QuantizedTensor
from test_gpu_int4 import close, moe_reference, randn

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _status():
    yield
    ops.device_status(reset=True)


def bound_of(steps):
    return (17 * steps + 264) * 2.0 ** -23


def weight(n, k, group, seed=0, lead=(), exps=(-8, -5), bits=5):
    """A packed random weight, scales of ``bits`` significant bits, and its fp64 values [*lead, n, k]."""
    kp = O.i4_padded(k)
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randint(0, 256, (*lead, n, kp // 2), dtype=torch.uint8, device="cuda", generator=g)
    shape = (*lead, n, kp // group)
    mant = torch.randint(1 << (bits - 1), 1 << bits, shape, device="cuda", generator=g).double() / 2 ** (bits - 1)
    s = torch.ldexp(mant, torch.randint(*exps, shape, device="cuda", generator=g)).to(BF)
    byte, shift = (torch.from_numpy(a).cuda() for a in O.i4_positions(k))
    v = ((q[..., byte] >> shift.to(torch.uint8)) & 15).double() - 8
    v *= s.double().repeat_interleave(group, -1)
    return q, s, v[..., :k]


def check_linear(m, n, k, group, dtype, steps, seed=0, bias=False, **how):
    q, s, v = weight(n, k, group, seed=seed, **how)
    x = randn(m, k, seed=seed + 1, dtype=dtype)
    b = randn(n, seed=seed + 2, scale=0.1, dtype=dtype) if bias else None
    y = I4.int4_linear(x, q, s, group, b)
    ref, mag = x.double() @ v.T, x.double().abs() @ v.abs().T
    if b is not None:
        ref += b.double()
        mag += b.double().abs()
    close(y, ref, bound_of(steps) * mag)
    assert torch.equal(y, I4.int4_linear(x, q, s, group, b))


# ------------------------------------------------------ the ends of the types
@pytest.mark.parametrize("m,k", [(1, 384), (3, 384), (12, 384), (40, 384), (20, 8320), (300, 8320)])
@pytest.mark.parametrize("group", [32, 128])
def test_linear_of_the_largest_activations(m, k, group):
    """bf16 activations up to the type's largest: a group's sum of code * x may pass fp32's range, the result does
    not."""
    q, s, v = weight(72, k, group, seed=m, exps=(-44, -40))
    x = randn(m, k, seed=1, scale=1e38).clamp(-3.38e38, 3.38e38).to(BF)
    x[0, :128] = torch.finfo(BF).max
    y = I4.int4_linear(x, q, s, group)
    close(y, x.double() @ v.T, bound_of(-(-k // 128) * 8) * (x.double().abs() @ v.abs().T))


@pytest.mark.parametrize("m,k", [(1, 384), (12, 384), (40, 384), (20, 8320)])
def test_linear_of_the_smallest_activations(m, k):
    """Normal bf16 activations down to 2^-126: products stay exact.  The output's own rounding near its smallest
    numbers is half of bf16's smallest step."""
    q, s, v = weight(72, k, 32, seed=m, exps=(-4, 4))
    x = torch.ldexp(randn(m, k, seed=1).clamp(-4, 4), torch.tensor(-123, device="cuda")).to(BF)
    x[x.abs() < 2.0 ** -126] = 2.0 ** -126
    y = I4.int4_linear(x, q, s, 32)
    ref = x.double() @ v.T
    steps = -(-k // 128) * 8
    off = (y.double() - ref).abs()
    mag = x.double().abs() @ v.abs().T
    # sums held in units of 2^10 lose no more than fp32's smallest step, 2^-149, an addition: 17 to a tensor-core
    # step, times a scale of up to 2^4
    small = (17 * steps * 2 ** 4 + 264) * 2.0 ** -139
    bound = bound_of(steps) * mag + small
    # the output's half step: eps / 2 = 2^-8 of a normal number, 2^-134 of the smallest ones
    assert (off <= bound + torch.finfo(BF).eps / 2 * (ref.abs() + bound) + 2.0 ** -134).all()


@pytest.mark.parametrize("t", [1, 9, 40])
def test_moe_of_the_largest_values(t):
    """Activations up to bf16's largest, and h = act(g) * u near fp32's largest, against small scales."""
    e, top_k, h, i, group = 6, 2, 256, 200, 128
    q13, s13, v13 = weight(2 * i, h, group, seed=1, lead=(e,), exps=(-8, -7))
    q2, s2, v2 = weight(h, i, group, seed=2, lead=(e,), exps=(-44, -42))
    x = randn(t, h, seed=3, scale=1e38).clamp(-3.38e38, 3.38e38).to(BF)
    router = randn(e, h, seed=4, scale=h ** -0.5) * 2.0 ** -126
    # codes of rms 4.6, 256 of them with x of 1e38: g and u of rms 2^15 with scales of 1.5 * 2^-118, 2^61 with 2^-72
    for exp in (-110, -64):
        sc, vc = torch.ldexp(s13, torch.tensor(exp, device="cuda")), torch.ldexp(v13, torch.tensor(exp, device="cuda"))
        y = I4.moe_int4(x, router, q13, sc, q2, s2, top_k, group)
        ref, bound = moe_reference(x, router, vc, v2, top_k, True, "silu")
        assert torch.isfinite(ref.to(BF)).all()
        close(y, ref, bound)


def test_moe_intermediate_next_to_the_end_of_fp32():
    """h = 7.875 * 2^62 * 8.125 * 2^60 is less than half a step of bf16 below 2^128."""
    q13 = torch.from_numpy(O.i4_pack(np.array([[7] + [0] * 127, [5] + [0] * 127], np.int8))).cuda()[None]
    q2 = torch.from_numpy(O.i4_pack(np.array([[1] + [0] * 127], np.int8))).cuda()[None]
    s13 = torch.tensor([1.125 * 2.0 ** 62, 1.625 * 2.0 ** 60], dtype=BF).view(1, 2, 1).expand(1, 2, 4).contiguous().cuda()
    s2 = torch.full((1, 1, 4), 2.0 ** -20, dtype=BF, device="cuda")
    x = torch.ones(1, 1, dtype=BF, device="cuda")
    y = I4.moe_int4(x, x, q13, s13, q2, s2, 1, 32)
    ref = torch.full((1, 1), 7.875 * 8.125 * 2.0 ** 102, dtype=torch.float64, device="cuda")
    close(y, ref, 2.0 ** -16 * ref)


# ------------------------------------------------------------------ gradients
def test_no_gradient_is_dropped():
    """Scales are numbers too: whoever wants their gradient, or a tangent, is told that there is none."""
    q, s, _ = weight(40, 256, 64)
    q13, s13, _ = weight(128, 256, 64, lead=(6,))
    q2, s2, _ = weight(256, 64, 64, lead=(6,))
    x, router, b = randn(3, 256, dtype=BF), randn(6, 256, dtype=BF), randn(40, dtype=BF)
    grad = lambda t: t.clone().requires_grad_()  # noqa: E731

    def calls(f):
        """Each call with f of one of its arguments."""
        return [lambda: I4.int4_linear(f(x), q, s, 64, b), lambda: I4.int4_linear(x, q, f(s), 64, b),
                lambda: I4.int4_linear(x, q, s, 64, f(b)), lambda: I4.weight_dequant_int4(q, f(s), 256, 64, BF),
                lambda: I4.moe_int4(f(x), router, q13, s13, q2, s2, 2, 64),
                lambda: I4.moe_int4(x, f(router), q13, s13, q2, s2, 2, 64),
                lambda: I4.moe_int4(x, router, q13, f(s13), q2, s2, 2, 64),
                lambda: I4.moe_int4(x, router, q13, s13, q2, f(s2), 2, 64)]

    for call in calls(grad):
        with pytest.raises(RuntimeError, match="backward"):
            call()
        with torch.no_grad():
            call()
    with fwAD.dual_level():
        for call in calls(lambda t: fwAD.make_dual(t, torch.ones_like(t))):
            for no_grad in (False, True):  # forward mode goes on under no_grad
                with torch.set_grad_enabled(not no_grad), pytest.raises(RuntimeError, match="backward"):
                    call()
        for call in calls(lambda t: t):
            call()


# ----------------------------------------------------------- the layout's shape
def test_layout_has_the_weights_shape():
    w = randn(40, 300, scale=0.02, dtype=BF)
    wq = QuantizedTensor.from_float(w, "GroupWiseINT4Layout", group_size=32)
    d = wq.dequantize()
    assert wq.shape == w.shape == d.shape and wq.numel() == w.numel() and wq.size(1) == 300
    # what torch works out from the shape before it reaches the tensor
    assert torch.equal(wq.reshape(-1), d.reshape(-1)) and torch.equal(wq.flatten(), d.flatten())
    for a, b in zip(wq.split(100, 1), d.split(100, 1)):
        assert torch.equal(a, b)
    for a, b in zip(wq.chunk(2, 1), d.chunk(2, 1)):
        assert torch.equal(a, b)
    assert torch.equal(wq[:, -7:], d[:, -7:]) and torch.equal(wq.t(), d.t())
    for v in (wq.detach(), wq.clone(), wq.to("cuda"), torch.empty_like(wq)):
        assert isinstance(v, QuantizedTensor) and v.shape == w.shape
    x = randn(3, 300, seed=1, dtype=BF)
    assert torch.equal(F.linear(x, torch.nn.Parameter(wq, requires_grad=False)), F.linear(x, wq))
    w3 = randn(4, 10, 200, scale=0.02, dtype=BF)
    q3 = QuantizedTensor.from_float(w3, "GroupWiseINT4Layout", group_size=64)
    assert q3.shape == w3.shape and torch.equal(q3.flatten(), q3.dequantize().flatten())


@pytest.mark.parametrize("layout", ["GroupWiseINT4Layout", "TensorWiseINT8Layout"])
def test_layout_records_a_stream_for_its_memory(layout):
    """The memory of a tensor that another stream still uses is not handed out again."""
    wq = QuantizedTensor.from_float(randn(2048, 8192, scale=0.02, dtype=BF), layout)
    torch.cuda.synchronize()
    at, n = wq._qdata.data_ptr(), wq._qdata.numel()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)  # about 0.1 s
    wq.record_stream(side)
    del wq
    new = [torch.empty(n, dtype=torch.uint8, device="cuda").data_ptr() for _ in range(3)]
    busy = not side.query()
    torch.cuda.synchronize()
    assert busy and at not in new


def test_layout_is_not_changed_behind_its_back():
    """Writing to a 4-bit tensor: raw codes or a tensor of the same format, or an error; never nothing or half of
    it."""
    w, w2 = randn(40, 300, scale=0.02, dtype=BF), randn(40, 300, seed=1, scale=0.02, dtype=BF)
    wq, other = (QuantizedTensor.from_float(v, "GroupWiseINT4Layout", group_size=32) for v in (w, w2))
    before = wq.dequantize()
    for bad in (lambda: wq.add_(1), lambda: wq.mul_(2), lambda: wq.zero_(), lambda: torch.add(w, w, out=wq),
                lambda: wq.copy_(w2), lambda: wq.copy_(w2[:, :192].to(torch.uint8).t().contiguous()),
                lambda: wq.copy_(QuantizedTensor.from_float(w2, "GroupWiseINT4Layout", group_size=64)),
                lambda: wq.copy_(QuantizedTensor.from_float(w2[:, :290], "GroupWiseINT4Layout", group_size=32)),
                lambda: wq.copy_(QuantizedTensor.from_float(w2, "TensorWiseINT8Layout")),
                lambda: QuantizedTensor.from_float(w2, "TensorWiseINT8Layout").copy_(wq)):
        with pytest.raises((RuntimeError, TypeError)):
            bad()
        assert torch.equal(wq.dequantize(), before)
    assert torch.equal(wq + 1, before + 1)
    x = before.clone()
    assert torch.equal(x.add_(wq), before + before)  # reading it is no writing
    assert torch.equal(wq.copy_(other).dequantize(), other.dequantize())
    same = QuantizedTensor.from_float(w, "GroupWiseINT4Layout", group_size=32)
    assert torch.equal(same.copy_(other._qdata)._qdata, other._qdata)


def test_linear_takes_keywords():
    w = randn(48, 256, scale=0.02, dtype=BF)  # int8 layers have outputs in sixteens
    x, b = randn(3, 256, seed=1, dtype=BF), randn(48, seed=2, dtype=BF)
    for layout in ("GroupWiseINT4Layout", "TensorWiseINT8Layout", "AxisWiseINT8Layout"):
        wq = QuantizedTensor.from_float(w, layout)
        y = F.linear(x, wq, b)
        assert not torch.equal(y, F.linear(x, wq))
        assert torch.equal(F.linear(x, wq, bias=b), y)
    wq = QuantizedTensor.from_float(w, "GroupWiseINT4Layout", group_size=64)
    assert torch.equal(F.linear(x.half(), weight=wq, bias=b), F.linear(x.half(), wq, b))
    assert torch.equal(F.linear(input=x, weight=wq), F.linear(x, wq))


# ------------------------------------------------------------------- refusals
def test_integers_beyond_the_c_types_are_refused():
    q, s, _ = weight(40, 256, 64)
    q13, s13, _ = weight(128, 256, 64, lead=(6,))
    q2, s2, _ = weight(256, 64, 64, lead=(6,))
    x, router = randn(3, 256, dtype=BF), randn(6, 256, dtype=BF)
    for big in (1 << 70, -(1 << 70), (1 << 32) + 64, -1):
        for bad in (lambda: I4.int4_linear(x, q, s, big), lambda: I4.weight_quant_int4(x, big),
                    lambda: I4.weight_dequant_int4(q, s, 256, big, BF),
                    lambda: I4.weight_dequant_int4(q, s, big, 64, BF),
                    lambda: I4.moe_int4(x, router, q13, s13, q2, s2, big, 64),
                    lambda: I4.moe_int4(x, router, q13, s13, q2, s2, 2, big)):
            with pytest.raises(AssertionError):
                bad()
    for top_k in ((1 << 32) + 2, 2 - (1 << 32)):  # 2 in their lowest 32 bits
        with pytest.raises(AssertionError):
            I4.moe_int4(x, router, q13, s13, q2, s2, top_k, 64)


# ------------------------------------- variants for large layers, many tiles
def sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("m,over,k,group,bias", [
    (1, 1, 264, 32, False), (7, 267, 2989, 32, True), (8, 16, 1000, 64, False), (2, 17, 9000, 128, True),
    (9, 9, 264, 128, False), (12, 267, 1000, 64, True), (16, 1, 2989, 32, False), (10, 17, 640, 64, False),
    (13, 31, 1100, 128, True), (16, 32, 9000, 32, False)])
def test_linear_of_few_tokens_and_many_rows(m, over, k, group, bias, dtype):
    """More than 32 rows per SM: one block of codes ahead and, from 9 tokens on, two tiles of rows per warp."""
    check_linear(m, 32 * sms() + over, k, group, dtype, 8, seed=m, bias=bias)


def experts_variant(t, e, top_k, h, i):
    """(pairs per chunk, rows over the warps in gate/up, in down), by the launch's rules."""
    pairs = t * top_k
    cap = 4 if t <= 4 or pairs <= 3 * e else 8 if t <= 8 or pairs <= 10 * e else 16
    used = min(pairs, e)
    return (cap, *(used * (-(-rows // tile) // 8) >= 2 * sms() for rows, tile in ((O.i4_padded(i), 16), (h, 32))))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("t,e,top_k,h,i,group,cap", [
    (16, 64, 8, 1349, 601, 32, 4), (16, 64, 8, 1352, 600, 128, 4), (10, 300, 30, 250, 100, 64, 4),
    (40, 64, 8, 1352, 513, 64, 8), (40, 64, 8, 1281, 640, 32, 8), (64, 150, 24, 550, 250, 128, 16),
    (64, 150, 24, 552, 129, 32, 16), (64, 150, 24, 512, 256, 64, 16)])
def test_moe_of_wide_layers(t, e, top_k, h, i, group, cap, dtype):
    """Eight warps side by side over an expert's rows, in gate/up and in down."""
    assert experts_variant(t, e, top_k, h, i) == (cap, True, True)
    q13, s13, v13 = weight(2 * i, h, group, seed=1, lead=(e,))
    q2, s2, v2 = weight(h, i, group, seed=2, lead=(e,))
    x, router = randn(t, h, seed=3, dtype=dtype), randn(e, h, seed=4, scale=h ** -0.5, dtype=dtype)
    s13, v13 = s13 * 0.25, v13 * 0.25  # g and u of a few units
    s2, v2 = s2 * 0.25, v2 * 0.25
    for act, renorm in (("silu", True), ("gelu", False)):
        y = I4.moe_int4(x, router, q13, s13, q2, s2, top_k, group, renorm, act)
        close(y, *moe_reference(x, router, v13, v2, top_k, renorm, act))
        assert torch.equal(y, I4.moe_int4(x, router, q13, s13, q2, s2, top_k, group, renorm, act))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("m,n,k,group", [
    (32, 140000, 128, 64), (24, 60000, 384, 32), (24, 60001, 1150, 128),
    (64, 90000, 100, 32), (48, 60000, 384, 128), (40, 57001, 1152, 64),
    (128, 60000, 104, 128), (100, 60000, 384, 64), (100, 60000, 1147, 32),
    (1100, 12000, 100, 32), (1100, 12000, 384, 128), (700, 30001, 1152, 64)])
def test_linear_of_several_tiles_per_block(m, n, k, group, dtype):
    """At least three tiles on some block for every width of the tensor-core tile, an odd number of 128-feature blocks
    each: rings, accumulators and their phases carry over from tile to tile."""
    width = next(b for b in (32, 64, 128, 256) if m <= b or b == 256)
    blocks = O.i4_padded(k) // 128
    assert blocks % 2 and -(-n // 128) * -(-m // width) > 2 * sms() and m * n * k > 1 << 29
    check_linear(m, n, k, group, dtype, 8 * blocks, seed=m + k, bias=bool(k & 128))


@pytest.mark.parametrize("m", [4, 30, 300])
def test_small_products_keep_scales_of_eight_bits(m):
    """Up to 2^29 multiply-adds and 8192 features the scale multiplies the fp32 sum: nothing is rounded but the
    result."""
    for dtype in (BF, HF):
        for group in (32, 64, 128):
            check_linear(m, 70, 200, group, dtype, 8, seed=m, bits=8)


def test_linear_weight_of_more_than_4_gb():
    """Row offsets in bytes pass 32 bits, in the rows kernel and in the tensor-core tiles."""
    n, k = 66000, 131072
    q = torch.full((n, k // 2), 0x88, dtype=torch.uint8, device="cuda")
    s = torch.ones(n, k // 128, dtype=BF, device="cuda")
    q[1], q[65537], q[-1] = 0x77, 0xAA, 0x99  # codes -1, 2 (4 GB behind row 1) and 1
    for m in (2, 20):
        x = torch.ones(m, k, dtype=BF, device="cuda")
        x[1] = 2
        y = I4.int4_linear(x, q, s)
        for col, code in ((1, -1), (65537, 2), (-1, 1)):
            assert y[:2, col].tolist() == [code * k, 2 * code * k]
        assert int((y != 0).sum()) == 3 * m
