"""The 4-bit weight operators: what they compute, in plain torch and by the framework.

Three operators share one weight format (codes of 4 bits, one scale for each
group of consecutive input features):

* ``quant``   a weight into 4-bit codes and group scales, and read back
* ``linear``  ``y = x W^T + b`` with the 4-bit weight, from one token to a prompt
* ``moe``     a mixture-of-experts layer for a few tokens: router, the k best
              experts of each token, their gated feed-forward, weighted sum

The format: ``W[n, k] = code[n, k] * scale[n, k // group]``; a row is padded with
zeros to a multiple of 128 features.  A code is held as ``code + 8`` in 4 bits,
eight in a 32-bit word in the order of features 0, 2, 4, 6, 1, 3, 5, 7 from the
lowest bits.  Of the 16 words of 128 features, word 4 a + b holds the eight
features from 32 b + 8 a on.  Scales are bf16 with at most five significant
bits, so that ``code * scale`` is a bf16 number.
"""

import math

import torch

own = False

_SCALE_MIN = 2.0 ** -100  # the scale of a group of zeros


# ------------------------------------------------------------------ cases
def listed():
    bf, hf, f32 = "bfloat16", "float16", "float32"
    return [
        # one feed-forward weight of a text encoder layer (4096 -> 10240) on its way into a 4-bit checkpoint
        dict(name="quant 10240x4096", op="quant", n=10240, k=4096, group=128, dtype=bf),
        # a small adapter-sized fp32 weight whose rows end inside a group
        dict(name="quant ragged f32", op="quant", n=1531, k=1100, group=32, dtype=f32),
        # one new token through an attention projection: the call whose latency counts
        dict(name="linear 1x4096x4096", op="linear", t=1, n=4096, k=4096, group=128, dtype=bf, bias=False),
        # one new token through an output head: far larger than the L2
        dict(name="linear 1x65536x8192", op="linear", t=1, n=65536, k=8192, group=128, dtype=bf, bias=False),
        # a few tokens, sizes that fit no tile, small groups, fp16 with bias
        dict(name="linear 7x5003x2989", op="linear", t=7, n=5003, k=2989, group=32, dtype=hf, bias=True),
        # a small batch of sequences, one token each, through the feed-forward's way back
        dict(name="linear 16x4096x10240", op="linear", t=16, n=4096, k=10240, group=64, dtype=bf, bias=True),
        # a large batch of single tokens, or a short prompt
        dict(name="linear 100x10240x4096", op="linear", t=100, n=10240, k=4096, group=128, dtype=bf, bias=True),
        # a batch of 8 x 512 prompt tokens
        dict(name="linear 4096x10240x4096", op="linear", t=4096, n=10240, k=4096, group=128, dtype=bf, bias=False),
        # one new token through a layer of many small experts
        dict(name="moe 1 of 64x1024", op="moe", t=1, e=64, top=8, h=2048, i=1024, group=128, dtype=bf, renorm=True, act="silu"),
        # a batch of single tokens: about every expert has work, one to five tokens each
        dict(name="moe 16 of 64x1536", op="moe", t=16, e=64, top=8, h=4096, i=1536, group=128, dtype=bf, renorm=True, act="silu"),
        # few experts as wide as a dense feed-forward, many tokens each
        dict(name="moe 48 of 8x10240", op="moe", t=48, e=8, top=2, h=4096, i=10240, group=64, dtype=bf, renorm=True, act="silu"),
        # odd sizes, fp16, probabilities used as they are, GELU gates
        dict(name="moe 5 of 23x701", op="moe", t=5, e=23, top=3, h=1090, i=701, group=32, dtype=hf, renorm=False, act="gelu"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quant", "linear", "linear", "moe", "moe"])
    group = rng.choice([32, 64, 128])
    if op == "quant":
        while True:
            n, k = _log(rng, 32, 32768), _log(rng, 32, 32768)
            if n * k <= 10240 * 4096:
                break
        return dict(op=op, n=n, k=k, group=group, dtype=rng.choice(["bfloat16", "float16", "float32"]))
    dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
    if op == "linear":
        while True:
            t, n, k = _log(rng, 1, 4096), _log(rng, 64, 65536), _log(rng, 64, 16384)
            if rng.random() < 0.6:  # most layers have sizes of whole 64s, some have not
                n, k = -(-n // 64) * 64, -(-k // 64) * 64
            if n * k <= 65536 * 8192 and t * n * k <= 4096 * 10240 * 4096 and t * n <= 4096 * 10240:
                break
        return dict(op=op, t=t, n=n, k=k, group=group, dtype=dtype, bias=rng.random() < 0.5)
    while True:
        t, e = _log(rng, 1, 64), _log(rng, 2, 256)
        h, i = _log(rng, 128, 8192), _log(rng, 64, 10240)
        if rng.random() < 0.7:
            h, i = -(-h // 64) * 64, -(-i // 64) * 64
        top = rng.randint(1, min(8, e))
        if e * h * i <= 8 * 4096 * 10240 and min(e, t * top) * t * h * i <= 8 * 48 * 4096 * 10240:
            break
    return dict(op=op, t=t, e=e, top=top, h=h, i=i, group=group, dtype=dtype, renorm=rng.random() < 0.5,
                act=rng.choice(["silu", "silu", "gelu"]))


# ------------------------------------------------------- the format, plainly
def _round5(s):
    """Positive fp32 numbers to five significant bits, ties to even."""
    b = s.view(torch.int32)
    b = (b + 0x3FFFF + ((b >> 19) & 1)) & ~0x7FFFF
    return b.view(torch.float32)


def _padded(k):
    return -(-k // 128) * 128


def _groups(w, group):
    """[..., k] -> [..., padded k / group, group], zeros behind the end."""
    k = w.shape[-1]
    if k % 128:
        w = torch.nn.functional.pad(w, (0, _padded(k) - k))
    return w.unflatten(-1, (-1, group))


def _quantise(w, group, wide=torch.float64):
    """fp32 weight -> codes as whole numbers [..., padded k] and fp32 scales; the quotients in `wide`."""
    g = _groups(w, group)
    amax = g.abs().amax(-1)
    s = _round5(amax / 7).clamp_min(_SCALE_MIN)
    c = torch.round(g.to(wide) / s.unsqueeze(-1).to(wide)).clamp(-7, 7)
    return c.to(torch.int8).flatten(-2), s


def _pack(codes):
    u = codes.add(8).to(torch.uint8).unflatten(-1, (-1, 4, 4, 4, 2))  # [block, b, a, pair, odd]
    u = u.transpose(-4, -3).transpose(-2, -1).flatten(-5)  # [block, a, b, odd, pair]: nibbles, lowest first
    return u[..., 0::2] | (u[..., 1::2] << 4)


def _unpack(q):
    nib = torch.stack((q & 15, q >> 4), -1).flatten(-2).unflatten(-1, (-1, 4, 4, 2, 4))
    return nib.transpose(-4, -3).transpose(-2, -1).flatten(-5).to(torch.int8) - 8


def _values(q, s, k, group, dtype):
    """The weight that codes and scales stand for, as `dtype`."""
    g = _unpack(q).to(dtype).unflatten(-1, (-1, group)) * s.to(dtype).unsqueeze(-1)
    return g.flatten(-2)[..., :k]


# ----------------------------------------------------------------- inputs
def _weight(gen, shape, group):
    """A packed weight as a converter would have left it: bell-shaped rows of different sizes."""
    q, s = [], []
    *lead, n, k = shape
    rows = math.prod(lead) * n
    step = max(1, (1 << 26) // k)
    for at in range(0, rows, step):
        m = min(step, rows - at)
        size = 0.02 * (0.5 + torch.rand(m, 1, generator=gen, device="cuda"))
        c, sc = _quantise(torch.randn(m, k, generator=gen, device="cuda") * size, group, torch.float32)
        q.append(_pack(c))
        s.append(sc.to(torch.bfloat16))
    return torch.cat(q).view(*lead, n, -1), torch.cat(s).view(*lead, n, -1)


def _activations(gen, t, k, dtype):
    """Normal activations with a few large channels."""
    x = torch.randn(t, k, generator=gen, device="cuda")
    far = torch.randperm(k, generator=gen, device="cuda")[: max(1, k // 200)]
    x[:, far] *= 8.0
    return x.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = getattr(torch, case["dtype"])
    state = dict(case=case)
    if case["op"] == "quant":
        n, k = case["n"], case["k"]
        w = torch.randn(n, k, generator=gen, device="cuda") * (0.02 * (0.5 + torch.rand(n, 1, generator=gen, device="cuda")))
        state["w"] = w.to(dtype)
    elif case["op"] == "linear":
        t, n, k = case["t"], case["n"], case["k"]
        state["q"], state["s"] = _weight(gen, (n, k), case["group"])
        state["x"] = _activations(gen, t, k, dtype)
        state["bias"] = (torch.randn(n, generator=gen, device="cuda") * 0.1).to(dtype) if case["bias"] else None
    else:
        t, e, h, i = case["t"], case["e"], case["h"], case["i"]
        state["q13"], state["s13"] = _weight(gen, (e, 2 * i, h), case["group"])
        state["q2"], state["s2"] = _weight(gen, (e, h, i), case["group"])
        state["x"] = torch.randn(t, h, generator=gen, device="cuda").to(dtype)
        state["router"] = (torch.randn(e, h, generator=gen, device="cuda") * h ** -0.5).to(dtype)
    return state


# -------------------------------------------------------------- plain forms
def _plain_quant(st):
    c = st["case"]
    codes, s = _quantise(st["w"].float(), c["group"])
    g = codes.float().unflatten(-1, (-1, c["group"])) * s.unsqueeze(-1)
    return dict(scale=s.to(torch.bfloat16), values=g.flatten(-2)[..., : c["k"]].to(st["w"].dtype))


def _plain_linear(st):
    c = st["case"]
    y = st["x"].float() @ _values(st["q"], st["s"], c["k"], c["group"], torch.float32).T
    if st["bias"] is not None:
        y = y + st["bias"].float()
    return y.to(st["x"].dtype)


def _route(logits, top, renorm):
    """The k largest of each row (the lowest index first among equals) and their weights in fp32."""
    ids = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :top]
    p = torch.softmax(logits, -1).gather(1, ids)
    if renorm:
        p = p / p.sum(-1, keepdim=True)
    return ids, p


def _gate(g, act):
    if act == "silu":
        return g * torch.sigmoid(g)
    return 0.5 * g * (1 + torch.erf(g * 0.5 ** 0.5))


def _plain_moe(st):
    c = st["case"]
    x = st["x"].float()
    ids, p = _route(st["x"].double() @ st["router"].double().T, c["top"], c["renorm"])
    used, slot = torch.unique(ids, return_inverse=True)
    w13 = _values(st["q13"][used], st["s13"][used], c["h"], c["group"], torch.float32)
    gu = torch.matmul(x, w13.transpose(1, 2))  # [used, t, 2 i]
    h = _gate(gu[..., : c["i"]], c["act"]) * gu[..., c["i"]:]
    del w13, gu
    w2 = _values(st["q2"][used], st["s2"][used], c["i"], c["group"], torch.float32)
    y = torch.matmul(h, w2.transpose(1, 2))  # [used, t, h]
    rows = torch.arange(c["t"], device=y.device).unsqueeze(1)
    return (y[slot, rows] * p.float().unsqueeze(-1)).sum(1).to(st["x"].dtype)


def _own_quant(st):
    from convert_to_quant_quip_int8_b200.comfy import int4_kernels
    c = st["case"]
    q, s = int4_kernels.weight_quant_int4(st["w"], group_size=c["group"])
    values = int4_kernels.weight_dequant_int4(q, s, c["k"], group_size=c["group"], output_dtype=st["w"].dtype)
    return dict(scale=s, values=values)


def _own_linear(st):
    from convert_to_quant_quip_int8_b200.comfy import int4_kernels
    return int4_kernels.int4_linear(st["x"], st["q"], st["s"], group_size=st["case"]["group"], bias=st["bias"])


def _own_moe(st):
    from convert_to_quant_quip_int8_b200.comfy import int4_kernels
    c = st["case"]
    return int4_kernels.moe_int4(st["x"], st["router"], st["q13"], st["s13"], st["q2"], st["s2"], top_k=c["top"],
                                 group_size=c["group"], renormalize=c["renorm"], activation=c["act"])


_PLAIN = dict(quant=_plain_quant, linear=_plain_linear, moe=_plain_moe)
_OWN = dict(quant=_own_quant, linear=_own_linear, moe=_own_moe)


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


# ------------------------------------------------------------------- work
def _weight_bytes(rows, k, group):
    return rows * _padded(k) // 2 + rows * 2 * (_padded(k) // group)


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "quant":
        n, k = case["n"], case["k"]
        return dict(bytes=2 * n * k * size + _weight_bytes(n, k, case["group"]), flops=4 * n * k)
    if case["op"] == "linear":
        t, n, k = case["t"], case["n"], case["k"]
        return dict(bytes=_weight_bytes(n, k, case["group"]) + size * (t * k + t * n + (n if case["bias"] else 0)),
                    flops=2 * t * n * k)
    t, e, top, h, i = (case[x] for x in ("t", "e", "top", "h", "i"))
    used = e * (1 - (1 - top / e) ** t)  # experts that get a token when all are equally likely
    one = _weight_bytes(2 * i, h, case["group"]) + _weight_bytes(h, i, case["group"])
    return dict(bytes=int(used * one) + size * (2 * t * h + e * h), flops=2 * t * e * h + 2 * t * top * 3 * h * i)


# ------------------------------------------------------------------ exact
def _exact_values(q, s, k, group):
    """The weight in fp64, from the format's definition: one nibble of one word of each block at a time."""
    words = q.contiguous().view(torch.int32).unflatten(-1, (-1, 16))
    w = torch.empty(*words.shape[:-1], 128, dtype=torch.float64, device=q.device)
    for word in range(16):
        first = 32 * (word % 4) + 8 * (word // 4)
        for nibble, feature in enumerate((0, 2, 4, 6, 1, 3, 5, 7)):
            w[..., first + feature] = ((words[..., word] >> (4 * nibble)) & 15).double() - 8.0
    return (w.flatten(-2) * s.double().repeat_interleave(group, dim=-1))[..., :k]


def exact(case, seed):
    st = prepare(case, seed)
    group = case["group"]
    if case["op"] == "quant":
        w = st["w"].double()
        n, k = w.shape
        scale = torch.zeros(n, _padded(k) // group, dtype=torch.float64, device=w.device)
        for j in range(-(-k // group)):
            scale[:, j] = w[:, j * group:(j + 1) * group].abs().amax(1) / 7.0
        mant, exp = torch.frexp(scale)
        scale = torch.ldexp(torch.round(mant * 32.0) / 32.0, exp).clamp_min(_SCALE_MIN)  # torch.round: ties to even
        full = scale.repeat_interleave(group, dim=1)[:, :k]
        return dict(scale=scale, values=torch.round(w / full).clamp(-7.0, 7.0) * full)
    x = st["x"].double()
    if case["op"] == "linear":
        y = torch.empty(case["t"], case["n"], dtype=torch.float64, device=x.device)
        step = max(1, (1 << 27) // case["k"])
        for at in range(0, case["n"], step):
            y[:, at:at + step] = x @ _exact_values(st["q"][at:at + step], st["s"][at:at + step], case["k"], group).T
        return y if st["bias"] is None else y + st["bias"].double()
    weight = torch.zeros(case["t"], case["e"], dtype=torch.float64)
    for t, row in enumerate((x @ st["router"].double().T).tolist()):
        best = sorted(range(case["e"]), key=lambda j: (-row[j], j))[: case["top"]]
        p = [math.exp(v - max(row)) for v in row]
        total = math.fsum(p[j] for j in best) if case["renorm"] else math.fsum(p)
        for j in best:
            weight[t, j] = p[j] / total
    weight = weight.to(x.device)
    y = torch.zeros_like(x)
    for j in range(case["e"]):
        at = weight[:, j].nonzero().flatten()
        if not len(at):
            continue
        gu = x[at] @ _exact_values(st["q13"][j], st["s13"][j], case["h"], group).T
        g, u = gu[:, : case["i"]], gu[:, case["i"]:]
        if case["act"] == "silu":
            g = g / (1.0 + torch.exp(-g))
        else:
            g = g * 0.5 * torch.special.erfc(-g / math.sqrt(2.0))
        y[at] += weight[at, j:j + 1] * ((g * u) @ _exact_values(st["q2"][j], st["s2"][j], case["i"], group).T)
    return y
