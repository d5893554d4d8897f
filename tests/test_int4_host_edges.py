"""CPU tests of the 4-bit operators' host side: what they refuse before a kernel runs, the layout tensor, the build."""

import os
import subprocess
import sysconfig

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from convert_to_quant_quip_int8_b200 import _lib as L
from convert_to_quant_quip_int8_b200 import build as B
from convert_to_quant_quip_int8_b200 import ops
from convert_to_quant_quip_int8_b200.comfy import quant_ops as Q


def _weight(n=16, k=256, group=128):
    return (torch.zeros(n, k // 2, dtype=torch.uint8), torch.ones(n, k // group, dtype=torch.bfloat16))


def test_no_gradient_of_a_scale_is_dropped(monkeypatch):
    monkeypatch.setattr(ops, "_one_device", lambda x, *t: x.device)
    q, s = _weight()
    x = torch.zeros(2, 256, dtype=torch.bfloat16)
    q13, s13, q2, s2 = q.expand(4, 16, 128), s.expand(4, 16, 2), *(t.expand(4, -1, -1) for t in _weight(256, 128))

    def calls(f):
        return (lambda: ops.gemm_w4(x, q, f(s)), lambda: ops.dequant_i4(q, f(s), 256),
                lambda: ops.moe_w4(x, torch.zeros(4, 256), q13, f(s13), q2, s2, 2),
                lambda: ops.moe_w4(x, torch.zeros(4, 256), q13, s13, q2, f(s2), 2))

    for call in calls(lambda t: t.clone().requires_grad_()):
        with pytest.raises(RuntimeError, match="backward"):
            call()


def test_tangents_are_refused():
    x = torch.zeros(2, 2)
    with fwAD.dual_level():
        d = fwAD.make_dual(x, torch.ones(2, 2))
        for no_grad in (False, True):
            with torch.set_grad_enabled(not no_grad), pytest.raises(RuntimeError, match="backward"):
                ops._no_grad(None, x, d)
        ops._no_grad(x, None)
    ops._no_grad(d, x)


def _layout(n=16, k=250, group=64, lead=()):
    q, s = _weight(n, -(-k // 128) * 128, group)
    return Q.QuantizedTensor(q.expand(*lead, *q.shape), "GroupWiseINT4Layout",
                             {"scale": s.expand(*lead, *s.shape), "group_size": group, "in_features": k,
                              "orig_dtype": torch.bfloat16})


def test_layout_shows_the_weights_shape():
    wq = _layout()
    assert wq.shape == (16, 250) and wq.numel() == 4000 and wq._qdata.shape == (16, 128)
    for v in (wq.detach(), wq.clone(), torch.empty_like(wq), torch.nn.Parameter(wq, requires_grad=False), wq.to("cpu")):
        assert isinstance(v, Q.QuantizedTensor) and v.shape == (16, 250)
    assert _layout(lead=(3,)).shape == (3, 16, 250)
    inner, ctx = wq.__tensor_flatten__()
    again = Q.QuantizedTensor.__tensor_unflatten__({k: getattr(wq, k) for k in inner}, ctx, None, None)
    assert again.shape == (16, 250)
    w8 = Q.QuantizedTensor(torch.zeros(16, 128, dtype=torch.int8), "TensorWiseINT8Layout",
                           {"scale": torch.ones(()), "orig_dtype": torch.bfloat16})
    assert w8.shape == (16, 128)


def test_a_checkpoint_entry_needs_what_rebuilds_the_weight():
    wq = _layout(k=250)
    needs = Q.QUANT_ALGOS["int4_groupwise"]["required_parameters"]
    assert needs == {"weight_scale", "in_features"}
    assert {k for k in wq._layout_params if k not in ("scale", "orig_dtype", "group_size")} <= needs


def test_writes_to_a_packed_tensor_are_refused():
    wq, before = _layout(), _layout()._qdata.clone()
    plain = torch.ones(16, 250, dtype=torch.bfloat16)
    w8 = Q.QuantizedTensor(torch.zeros(16, 250, dtype=torch.int8), "TensorWiseINT8Layout",
                           {"scale": torch.ones(()), "orig_dtype": torch.bfloat16})
    for bad in (lambda: wq.add_(1), lambda: wq.zero_(), lambda: wq.fill_(3), lambda: torch.mul(plain, 2, out=wq),
                lambda: torch._foreach_add_([wq], 1.0), lambda: wq.copy_(plain), lambda: wq.copy_(plain.byte()),
                lambda: wq.copy_(before.to(torch.int16)), lambda: wq.copy_(before[:1]), lambda: wq.copy_(w8),
                lambda: w8.copy_(wq), lambda: wq.copy_(_layout(k=249)), lambda: wq.copy_(_layout(group=32))):
        with pytest.raises((RuntimeError, TypeError)) as e:
            bad()
        assert not isinstance(e.value, RecursionError)
        assert torch.equal(wq._qdata, before) and wq._layout_params["group_size"] == 64
    other = _layout()
    other._qdata.fill_(0x9A)
    other._layout_params["scale"].fill_(0.5)
    assert wq.copy_(other) is wq
    assert torch.equal(wq._qdata, other._qdata) and (wq._layout_params["scale"] == 0.5).all()
    wq.copy_(before)
    assert torch.equal(wq._qdata, before)


def test_copy_into_a_plain_tensor_dequantizes(monkeypatch):
    wq = _layout()
    value = torch.arange(4000.0).view(16, 250)
    monkeypatch.setattr(Q.GroupWiseINT4Layout, "dequantize", staticmethod(lambda *a, **k: value))
    buf = torch.zeros(16, 250)
    assert buf.copy_(wq) is buf and torch.equal(buf, value)


def test_linear_passes_keywords_on(monkeypatch):
    seen = []
    linear = torch.nn.functional.linear
    for layout in ("GroupWiseINT4Layout", "TensorWiseINT8Layout"):
        monkeypatch.setitem(Q._LAYOUT_REGISTRY[torch.ops.aten.linear.default], layout,
                            lambda func, args, kwargs: seen.append((*args, None)[:3]) or torch.zeros(()))
    wq, x, b = _layout(), torch.zeros(2, 250), torch.zeros(16)
    w8 = Q.QuantizedTensor(torch.zeros(16, 250, dtype=torch.int8), "TensorWiseINT8Layout",
                           {"scale": torch.ones(()), "orig_dtype": torch.bfloat16})
    for w in (wq, w8):
        linear(x, w, bias=b)
        assert seen[-1][0] is x and seen[-1][1] is w and seen[-1][2] is b
        linear(x, w)
        assert seen[-1][1] is w and seen[-1][2] is None
    linear(x, weight=wq, bias=b)
    assert seen[-1][0] is x and seen[-1][1] is wq and seen[-1][2] is b
    linear(input=x, weight=wq)
    assert seen[-1][0] is x and seen[-1][1] is wq and seen[-1][2] is None
    out = torch.ones(())
    assert linear(x, wq, out=out) is out and out == 0
    with pytest.raises(RuntimeError, match="shape"):
        linear(x, w8, b, out=torch.ones(3))
    with pytest.raises(TypeError):
        linear(x, wq, b, bias=b)


def test_integers_are_not_cut_to_c_integers(monkeypatch):
    monkeypatch.setattr(ops, "_one_device", lambda x, *t: x.device)
    q13, s13, q2, s2 = (t.expand(6, -1, -1).contiguous() for t in (*_weight(128, 256, 64), *_weight(256, 128, 64)))
    x, router = torch.zeros(3, 256, dtype=torch.bfloat16), torch.zeros(6, 256, dtype=torch.bfloat16)
    for top_k in ((1 << 32) + 2, 2 - (1 << 32), 1 << 70, 0, 7, -1):
        with pytest.raises(AssertionError, match="top_k"):
            ops.moe_w4(x, router, q13, s13, q2, s2, top_k, 64)
    with pytest.raises(AssertionError, match="activation"):
        ops.moe_w4(x, router, q13, s13, q2, s2, 2, 64, True, (1 << 32) + 1)


@pytest.mark.parametrize("k", [0, -5])
def test_weights_without_features_are_refused(monkeypatch, k):
    monkeypatch.setattr(ops, "_one_device", lambda x, *t: x.device)
    q, s = torch.empty(4, 0, dtype=torch.uint8), torch.empty(4, 0, dtype=torch.bfloat16)
    with pytest.raises(AssertionError, match="features"):
        ops.dequant_i4(q, s, k)
    with pytest.raises(AssertionError, match="features"):
        ops._check_i4(q, s, k, 128, 2)


def test_shortcut_belongs_to_one_torch_and_one_python(monkeypatch):
    """csrc/call.cpp holds layouts of torch's and Python's objects: the file for another of either is not loaded."""
    here = B.call_path()
    assert torch.__version__ in here and here.endswith(sysconfig.get_config_var("EXT_SUFFIX"))
    assert os.path.exists(B.build_call())
    monkeypatch.setattr(L, "_call", None)
    assert L.fast_call() is not None
    monkeypatch.setattr(L, "_call", None)
    monkeypatch.setattr(torch, "__version__", "0.0.1+other")
    assert B.call_path() != here and not os.path.exists(B.call_path())
    assert L.fast_call() is None


def test_build_without_a_host_compiler_still_builds_the_library(monkeypatch, capsys):
    done = []
    monkeypatch.setattr(B, "build", lambda **k: done.append("lib"))

    def no_compiler(**k):
        raise subprocess.CalledProcessError(1, "g++")

    monkeypatch.setattr(B, "build_call", no_compiler)
    B.main(["build"])
    assert done == ["lib"] and "warning" in capsys.readouterr().err


def test_layouts_of_others_work_as_before(monkeypatch):
    """A registered class without the base class, and a type that nobody registered: shape and copies are the data's."""
    class Bare:
        pass

    monkeypatch.setitem(Q.LAYOUTS, "Bare", Bare)
    for name in ("Bare", "Unknown"):
        def make(v):
            return Q.QuantizedTensor(torch.full((4, 6), v, dtype=torch.int8), name,
                                     {"scale": torch.ones(()) * v, "orig_dtype": torch.float32})
        a, b = make(1), make(2)
        assert a.shape == (4, 6) and a.clone().shape == (4, 6)
        assert a.copy_(b) is a and (a._qdata == 2).all() and a._layout_params["scale"] == 2
        a.copy_(torch.full((4, 6), 3.0))
        assert (a._qdata == 3).all()
