"""GPU tests of the int8 read-back at the sizes where it goes another way."""

import pytest
import torch

from convert_to_quant_quip_int8_b200 import _lib as L
from convert_to_quant_quip_int8_b200 import ops

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
