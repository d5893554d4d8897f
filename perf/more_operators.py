"""Operators of 8-bit activations: what they compute, in plain torch and by the framework.

* ``quant``   a weight into fp8 codes with one scale for each tile of 128 x 128
* ``linear``  ``y = x W^T + b`` on an fp8 weight: the activations are quantized
              to fp8 with one scale for each token and 128 features, or arrive so
* ``norm``    root-mean-square norm of ``x + residual`` with an 8-bit output
* ``gated``   ``act(gate) * up`` of a gated feed-forward with an 8-bit output

fp8: e4m3 codes, ``value = code * 2^e`` with ``e`` the smallest whole number
from -100 on for which the block's largest value is at most 448 * 2^e.  Blocks are
128 columns of one row (activations) or 128 rows by 128 columns (weights); the
last ones may be smaller.  Rows of codes lie whole 16 bytes apart.  int8: one scale ``amax / 127`` for each row, codes
rounded to nearest.  The norm and the gate round nowhere between the residual's
sum (held in x's type) and the codes.
"""

import math

import torch

own = False

_BLOCK = 128
_E_MIN = -100  # exponent of a block of zeros


# ------------------------------------------------------------------ cases
def listed():
    bf, hf, f32 = "bfloat16", "float16", "float32"
    return [
        # a feed-forward weight of a text encoder layer (4096 -> 10240) on its way into a checkpoint
        dict(name="quant 10240x4096", op="quant", n=10240, k=4096, dtype=bf),
        # a small fp32 weight that ends inside a tile both ways
        dict(name="quant 1531x1100 f32", op="quant", n=1531, k=1100, dtype=f32),
        # one new token through an attention projection: the call whose latency counts
        dict(name="linear 1x4096x4096", op="linear", t=1, n=4096, k=4096, dtype=bf, bias=False, codes=False),
        # a few tokens, sizes that fit no tile, fp16 with bias
        dict(name="linear 9x5003x2989", op="linear", t=9, n=5003, k=2989, dtype=hf, bias=True, codes=False),
        # a batch of single tokens, or a short prompt, whose activations the norm left in fp8
        dict(name="gemm 100x10240x4096", op="linear", t=100, n=10240, k=4096, dtype=bf, bias=False, codes=True),
        # a batch of 8 x 512 prompt tokens through the feed-forward's first weight
        dict(name="linear 4096x10240x4096", op="linear", t=4096, n=10240, k=4096, dtype=bf, bias=True, codes=False),
        # one new token before its attention projection
        dict(name="norm 1x4096", op="norm", t=1, n=4096, dtype=bf, residual=True, out="fp8"),
        # odd sizes, fp16, no residual, int8 for a weight with a scale for each row
        dict(name="norm 77x1451 int8", op="norm", t=77, n=1451, dtype=hf, residual=False, out="int8"),
        # a batch of prompts between two layers
        dict(name="norm 4096x4096", op="norm", t=4096, n=4096, dtype=bf, residual=True, out="fp8"),
        # a few tokens, one product that holds gate and up side by side
        dict(name="gated 16x10240", op="gated", t=16, n=10240, dtype=bf, joined=True, act="silu", out="fp8"),
        # the gated feed-forward of the text encoder on a batch of prompts
        dict(name="gated 4096x10240", op="gated", t=4096, n=10240, dtype=bf, joined=False, act="gelu_tanh", out="fp8"),
        # odd sizes in int8
        dict(name="gated 515x2731 int8", op="gated", t=515, n=2731, dtype=hf, joined=False, act="gelu", out="int8"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _sizes(rng, *sizes):
    """Most layers have sizes of whole 64s, some have not."""
    return [-(-s // 64) * 64 for s in sizes] if rng.random() < 0.6 else list(sizes)


def draw(rng):
    op = rng.choice(["quant", "linear", "linear", "norm", "gated"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
    if op == "quant":
        while True:
            n, k = _sizes(rng, _log(rng, 32, 32768), _log(rng, 32, 32768))
            if n * k <= 10240 * 4096:
                break
        return dict(op=op, n=n, k=k, dtype=rng.choice(["bfloat16", "float16", "float32"]))
    if op == "linear":
        while True:
            t = _log(rng, 1, 4096)
            n, k = _sizes(rng, _log(rng, 64, 32768), _log(rng, 64, 16384))
            if n * k <= 32768 * 4096 and t * n * k <= 4096 * 10240 * 4096 and t * n <= 4096 * 10240:
                break
        return dict(op=op, t=t, n=n, k=k, dtype=dtype, bias=rng.random() < 0.5, codes=rng.random() < 0.3)
    while True:
        t = _log(rng, 1, 8192)
        n, = _sizes(rng, _log(rng, 64, 16384))
        if t * n <= 4096 * 4096:
            break
    out = rng.choice(["fp8", "fp8", "int8"])
    if op == "norm":
        return dict(op=op, t=t, n=n, dtype=dtype, residual=rng.random() < 0.7, out=out)
    return dict(op=op, t=t, n=n, dtype=dtype, joined=rng.random() < 0.5, act=rng.choice(["silu", "gelu", "gelu_tanh"]),
                out=out)


# ------------------------------------------------------ the formats, plainly
def _exponents(amax):
    m, x = torch.frexp(amax)  # amax = m 2^x, 0.5 <= m < 1; 448 = 0.875 * 2^9
    return torch.where(m > 0, (x - 9 + (m > 0.875).int()).clamp_min(_E_MIN), _E_MIN)


def _scales(e):
    return (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _columns(v):
    """[rows, n] -> [rows, blocks, 128], zeros behind the end."""
    n = v.shape[1]
    return torch.nn.functional.pad(v, (0, -n % _BLOCK)).unflatten(1, (-1, _BLOCK))


def _rows_of_16(q):
    """The same codes, rows whole 16 bytes apart."""
    n = q.shape[1]
    return torch.nn.functional.pad(q.view(torch.uint8), (0, -n % 16)).view(q.dtype)[:, :n]


def _fp8_rows(v):
    """Codes [rows, n] and scales [rows, blocks] of activations."""
    g = _columns(v)
    e = _exponents(g.abs().amax(-1))
    q = torch.ldexp(g, -e.unsqueeze(-1)).to(torch.float8_e4m3fn)
    return _rows_of_16(q.flatten(1)[:, : v.shape[1]]), _scales(e)


def _fp8_tiles(w):
    """Codes [n, k] and scales [tiles, tiles] of a weight."""
    n, k = w.shape
    g = torch.nn.functional.pad(w, (0, -k % _BLOCK, 0, -n % _BLOCK)).unflatten(1, (-1, _BLOCK)).unflatten(0, (-1, _BLOCK))
    e = _exponents(g.abs().amax((1, 3)))
    q = torch.ldexp(g, -e[:, None, :, None]).to(torch.float8_e4m3fn)
    return _rows_of_16(q.flatten(2).flatten(0, 1)[:n, :k]), _scales(e)


def _weight_values(q, s):
    n, k = q.shape
    f = s.float().repeat_interleave(_BLOCK, 0)[:n].repeat_interleave(_BLOCK, 1)[:, :k]
    return q.float() * f


def _row_values(q, s):
    return q.float() * s.float().repeat_interleave(_BLOCK, 1)[:, : q.shape[1]]


def _int8_rows(v, dtype):
    """What the int8 codes of each row stand for."""
    s = (v.abs().amax(-1, keepdim=True) / 127).clamp_min(1e-30)
    return (torch.round(v * (1 / s)).clamp(-127, 127) * s).to(dtype)


# ----------------------------------------------------------------- inputs
def _activations(gen, t, n, dtype):
    """Bell-shaped activations with a few large channels."""
    x = torch.randn(t, n, generator=gen, device="cuda")
    far = torch.randperm(n, generator=gen, device="cuda")[: max(1, n // 200)]
    x[:, far] *= 8.0
    return x.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = getattr(torch, case["dtype"])
    state = dict(case=case)
    op, n = case["op"], case["n"]
    if op in ("quant", "linear"):
        k = case["k"]
        w = torch.randn(n, k, generator=gen, device="cuda") * (0.02 * (0.5 + torch.rand(n, 1, generator=gen, device="cuda")))
        if op == "quant":
            state["w"] = w.to(dtype)
            return state
        state["q"], state["s"] = _fp8_tiles(w)
        x = _activations(gen, case["t"], k, dtype)
        state["x"] = _fp8_rows(x.float()) if case["codes"] else x
        state["bias"] = (torch.randn(n, generator=gen, device="cuda") * 0.1).to(dtype) if case["bias"] else None
        return state
    t = case["t"]
    if op == "norm":
        state["x"] = _activations(gen, t, n, dtype)
        state["residual"] = (_activations(gen, t, n, torch.float32) * 3.0).to(dtype) if case["residual"] else None
        state["weight"] = (1.0 + 0.2 * torch.randn(n, generator=gen, device="cuda")).to(dtype)
    elif case["joined"]:
        both = (torch.randn(t, 2 * n, generator=gen, device="cuda") * 1.5).to(dtype)
        state["gate"], state["up"] = both[:, :n], both[:, n:]
    else:
        state["gate"], state["up"] = ((torch.randn(t, n, generator=gen, device="cuda") * 1.5).to(dtype) for _ in range(2))
    return state


# -------------------------------------------------------------- plain forms
def _plain_quant(st):
    q, s = _fp8_tiles(st["w"].float())
    return dict(q=q, scale=s)


def _plain_linear(st):
    if st["case"]["codes"]:
        q, s = st["x"]
    else:
        q, s = _fp8_rows(st["x"].float())
    y = _row_values(q, s) @ _weight_values(st["q"], st["s"]).T
    if st["bias"] is not None:
        y = y + st["bias"].float()
    return y.to(getattr(torch, st["case"]["dtype"]))


def _out(v, case):
    if case["out"] == "int8":
        return dict(values=_int8_rows(v, getattr(torch, case["dtype"])))
    q, s = _fp8_rows(v)
    return dict(q=q, scale=s)


def _plain_norm(st):
    h = st["x"]
    if st["residual"] is not None:
        h = (h.float() + st["residual"].float()).to(h.dtype)
    f = h.float()
    y = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + 1e-6) * st["weight"].float()
    out = _out(y, st["case"])
    return out if st["residual"] is None else dict(out, sum=h)


def _gate(g, act):
    if act == "silu":
        return g * torch.sigmoid(g)
    if act == "gelu":
        return 0.5 * g * (1 + torch.erf(g * 0.5 ** 0.5))
    return 0.5 * g * (1 + torch.tanh((2 / math.pi) ** 0.5 * (g + 0.044715 * g * g * g)))


def _plain_gated(st):
    return _out(_gate(st["gate"].float(), st["case"]["act"]) * st["up"].float(), st["case"])


# ------------------------------------------------------ the framework's calls
def _own_quant(st):
    from convert_to_quant_quip_int8_b200.comfy import fp8_kernels
    q, s = fp8_kernels.weight_quant_fp8(st["w"])
    return dict(q=q, scale=s)


def _own_linear(st):
    from convert_to_quant_quip_int8_b200.comfy import fp8_kernels
    if st["case"]["codes"]:
        return fp8_kernels.fp8_gemm(*st["x"], st["q"], st["s"], bias=st["bias"],
                                    out_dtype=getattr(torch, st["case"]["dtype"]))
    return fp8_kernels.fp8_linear(st["x"], st["q"], st["s"], bias=st["bias"])


def _own_out(q, s, case):
    if case["out"] == "fp8":
        return dict(q=q, scale=s)
    from convert_to_quant_quip_int8_b200 import _lib, ops
    return dict(values=ops.dequant(q, s, _lib.QI8_S_ROW, out_dtype=getattr(torch, case["dtype"])))


def _own_norm(st):
    from convert_to_quant_quip_int8_b200.comfy import fused_quant_kernels
    case = st["case"]
    got = fused_quant_kernels.rms_norm_quant(st["x"], st["weight"], eps=1e-6, residual=st["residual"], output=case["out"])
    out = _own_out(got[0], got[1], case)
    return out if st["residual"] is None else dict(out, sum=got[2])


def _own_gated(st):
    from convert_to_quant_quip_int8_b200.comfy import fused_quant_kernels
    case = st["case"]
    q, s = fused_quant_kernels.gated_act_quant(st["gate"], st["up"], activation=case["act"], output=case["out"])
    return _own_out(q, s, case)


_PLAIN = dict(quant=_plain_quant, linear=_plain_linear, norm=_plain_norm, gated=_plain_gated)
_OWN = dict(quant=_own_quant, linear=_own_linear, norm=_own_norm, gated=_own_gated)


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


# ------------------------------------------------------------------- work
def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    op, n = case["op"], case["n"]
    blocks = lambda m: -(-m // _BLOCK)  # noqa: E731
    if op == "quant":
        k = case["k"]
        return dict(bytes=n * k * (size + 1) + blocks(n) * blocks(k), flops=2 * n * k)
    t = case["t"]
    if op == "linear":
        k = case["k"]
        x = t * (k + blocks(k)) if case["codes"] else t * k * size
        return dict(bytes=n * k + blocks(n) * blocks(k) + x + size * (t * n + (n if case["bias"] else 0)),
                    flops=2 * t * n * k)
    reads = 2 if op == "gated" or case["residual"] else 1
    writes = size if op == "norm" and case["residual"] else 0
    # int8: the values that the codes stand for are written too
    out = t * (n + blocks(n)) if case["out"] == "fp8" else t * n * size
    return dict(bytes=t * n * (reads * size + writes) + out + (n * size if op == "norm" else 0), flops=8 * t * n)


# ------------------------------------------------------------------ exact
def _e4m3(v):
    """The nearest e4m3 number of each value of at most 448 in fp64, ties to the even one."""
    top = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -30)))
    top = torch.where(torch.exp2(top) > v.abs(), top - 1, top)
    top = torch.where(torch.exp2(top + 1) <= v.abs(), top + 1, top)
    step = torch.exp2(top.clamp_min(-6.0) - 3.0)
    return torch.round(v / step) * step


def _exact_scale(amax):
    e = torch.ceil(torch.log2(amax.clamp_min(2.0 ** -140) / 448.0))
    e = torch.where(448.0 * torch.exp2(e - 1) >= amax, e - 1, e)  # log2 may be off next to a power of two
    e = torch.where(448.0 * torch.exp2(e) < amax, e + 1, e)
    return torch.exp2(e.clamp_min(float(_E_MIN)))


def _exact_rows(v):
    q, s = torch.empty_like(v), []
    for at in range(0, v.shape[1], _BLOCK):
        part = v[:, at:at + _BLOCK]
        s.append(_exact_scale(part.abs().amax(1)))
        q[:, at:at + _BLOCK] = _e4m3(part / s[-1].unsqueeze(1))
    return q, torch.stack(s, 1)


def _exact_out(v, case):
    if case["out"] == "fp8":
        q, s = _exact_rows(v)
        return dict(q=q, scale=s)
    s = (v.abs().amax(1, keepdim=True) / 127.0).clamp_min(1e-30)
    return dict(values=torch.round(v / s) * s)


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "quant":
        w = st["w"].double()
        q, s = torch.empty_like(w), []
        for at in range(0, case["n"], _BLOCK):
            rows = w[at:at + _BLOCK]
            s.append(torch.stack([_exact_scale(part.abs().amax()) for part in rows.split(_BLOCK, 1)]))
            q[at:at + _BLOCK] = _e4m3(rows / s[-1].repeat_interleave(_BLOCK)[: case["k"]])
        return dict(q=q, scale=torch.stack(s))
    if op == "linear":
        if case["codes"]:
            q, s = st["x"][0].double(), st["x"][1].double()
        else:
            q, s = _exact_rows(st["x"].double())
        y = torch.zeros(case["t"], case["n"], dtype=torch.float64, device=q.device)
        tile = st["s"].double()
        for j, at in enumerate(range(0, case["k"], _BLOCK)):
            part = (q[:, at:at + _BLOCK] * s[:, j:j + 1]) @ st["q"][:, at:at + _BLOCK].double().T
            y += part * tile[:, j].repeat_interleave(_BLOCK)[: case["n"]]
        return y if st["bias"] is None else y + st["bias"].double()
    if op == "norm":
        h = st["x"].double()
        if st["residual"] is not None:
            h = (h + st["residual"].double()).to(st["x"].dtype).double()
        y = h / torch.sqrt(h.square().sum(1, keepdim=True) / case["n"] + 1e-6) * st["weight"].double()
        out = _exact_out(y, case)
        return out if st["residual"] is None else dict(out, sum=h)
    g, u = st["gate"].double(), st["up"].double()
    if case["act"] == "silu":
        a = g / (1.0 + torch.exp(-g))
    elif case["act"] == "gelu":
        a = 0.5 * g * torch.special.erfc(-g / math.sqrt(2.0))
    else:
        a = g / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3)))
    return _exact_out(a * u, case)
