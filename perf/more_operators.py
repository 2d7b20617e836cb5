"""Performance cases of a training step at small batches and in little memory: group norm with its activation, an AdamW step over
all tensors of a network with states in 32 or 8 bits, and the matrix product in 8-bit floating point with a scale for each block
of 128.

A case is a dict of plain values.  `prepare` makes what a training or answering program holds before the call, `run` makes one
pass, either through the framework's entry points (`own`) or in elementary torch operations in 32 bits, and `exact` gives the same
results from the definitions in 64 bits.

Group norm: rows are pixels, columns are channels; "bf16" is bf16 everywhere, "mixed" has x and dx in fp32 and y and dy in bf16.
z = ((x - mean) * rstd) * weight + bias is rounded to fp32 after each of its four operations, so that the border of a ReLU is the
same wherever it is computed.

AdamW: states are rounded to fp32 after each operation of m = m b1 + g (1 - b1) and v = v b2 + (g g) (1 - b2).  In 8 bits a value
is a float without subnormals beside an exponent for 128 neighbours: m has a sign and 7 bits, v 8 bits, of which the lowest three
are the mantissa; code 0 is zero, and a v above zero is never rounded to it.  With a seed the states and bf16 parameters are
rounded up or down at random, by bits that are a function of seed, step and place; without one to the nearest.  States of a tensor
begin at multiples of 128.

8-bit product: e4m3 values with a scale 2^e for 128 columns of a row (weights: 128 x 128), e the smallest with no value above 448.
"""
from __future__ import annotations

import math
import random

import torch

own = False

BF, F32, F64, I64 = torch.bfloat16, torch.float32, torch.float64, torch.int64
TYPES = {"bf16": (BF, BF), "mixed": (F32, BF), "fp32": (F32, F32)}      # input, output
EPS = 1e-5
LR, BETA1, BETA2, ADAM_EPS, DECAY, T0 = 1e-3, 0.9, 0.999, 1e-8, 0.05, 1000


def listed():
    return [
        # a new classifier on a frozen network: four small tensors, where latency counts
        dict(name="adamw_head", op="adamw", count=4, total=11_274, skew=1.0, row=128, p="fp32", g="fp32", bits=32, delta=False,
             clip=0.0, seed=-1),
        # a network of AlexNet's size and shares with states in 8 bits, its gradients clipped by their norm on the way
        dict(name="adamw_alexnet_8bit", op="adamw", count=16, total=60_965_224, skew=2.5, row=128, p="fp32", g="fp32", bits=8,
             delta=False, clip=3.0, seed=11),
        # parameters as many and as ragged as the 22K-class Inception's, all in bf16, which little memory is left beside
        dict(name="adamw_ragged_bf16", op="adamw", count=331, total=33_554_467, skew=2.0, row=128, p="bf16", g="bf16", bits=8,
             delta=False, clip=0.0, seed=12),
        # a large model, packed without gaps, its gradients in bf16, states in 32 bits
        dict(name="adamw_large", op="adamw", count=75, total=134_217_695, skew=1.5, row=1, p="fp32", g="bf16", bits=32, delta=False,
             clip=0.0, seed=-1),
        # one image of 14 x 14 pixels, as a service answers; training batches of 56 x 56 and 14 x 14 pixels, forward and backward;
        # odd widths with the input in fp32
        dict(name="group_norm_image", op="group", bwd=False, images=1, pixels=196, c=576, groups=32, act="silu", types="bf16"),
        dict(name="group_norm_batch", op="group", bwd=False, images=32, pixels=3136, c=192, groups=32, act="relu", types="bf16"),
        dict(name="group_norm_backward", op="group", bwd=True, images=256, pixels=196, c=576, groups=32, act="relu", types="bf16"),
        dict(name="group_norm_odd", op="group", bwd=True, images=37, pixels=113, c=1003, groups=17, act="silu", types="mixed"),
        # a fully-connected layer: a few rows as a service answers; AlexNet's first at its training batch; its two gradients for a
        # larger batch; a large one
        dict(name="fp8_few_rows", op="fp8", bwd=False, m=7, k=4096, n=4096, bias=True, relu=False),
        dict(name="fp8_batch", op="fp8", bwd=False, m=256, k=9216, n=4096, bias=True, relu=True),
        dict(name="fp8_backward", op="fp8", bwd=True, m=1024, k=9216, n=4096, bias=False, relu=False),
        dict(name="fp8_large", op="fp8", bwd=False, m=8192, k=4096, n=16384, bias=True, relu=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["adamw", "group", "fp8"])
    if op == "adamw":
        p = rng.choice(["fp32", "fp32", "bf16"])
        return dict(op="adamw", count=_log(rng, 1, 331), total=_log(rng, 700, 1.2e8), skew=rng.choice([0.0, 1.0, 2.0, 2.5]),
                    row=rng.choice([1, 128, 128]), p=p, g=rng.choice(["fp32", "bf16"]), bits=rng.choice([8, 8, 32]),
                    delta=p == "fp32" and rng.random() < 0.3, clip=rng.choice([0.0, 0.5, 4.0]), seed=rng.choice([-1, 3, 4]))
    if op == "group":
        groups = _log(rng, 1, 64)
        c = groups * _log(rng, 1, 64)
        if rng.random() < 0.6:
            c = _up(c, math.lcm(groups, 8))
        rows = max(1, min(_log(rng, 1, 400_000), 30_000_000 // c))
        images = min(rows, _log(rng, 1, 512))
        return dict(op="group", bwd=rng.random() < 0.6, images=images, pixels=rows // images, c=c, groups=groups,
                    act=rng.choice(["", "relu", "silu"]), types=rng.choice(["bf16", "bf16", "mixed", "fp32"]))
    bwd = rng.random() < 0.5
    m, k, n = _log(rng, 1, 8192), _log(rng, 64, 9216), _log(rng, 64, 9216)
    if rng.random() < 0.6:
        k, n = (k + 127) // 128 * 128, (n + 127) // 128 * 128
    while m * k * n > 3e11:
        m = (m + 1) // 2
    return dict(op="fp8", bwd=bwd, m=m, k=k, n=n, bias=not bwd and rng.random() < 0.6, relu=not bwd and rng.random() < 0.4)


def _sizes(case):
    """Element counts of an AdamW case's tensors: shares whose logarithm spreads by `skew`, odd ones among them."""
    rng = random.Random(case["count"] * 1_000_003 + case["total"])
    share = [math.exp(rng.gauss(0.0, case["skew"])) for _ in range(case["count"])]
    whole = sum(share)
    sizes = [max(1, int(case["total"] * s / whole)) for s in share]
    sizes[sizes.index(max(sizes))] += max(0, case["total"] - sum(sizes))
    return sizes


def _type(name):
    return BF if name == "bf16" else F32


def _up(n, to):
    return (n + to - 1) // to * to


def work(case):
    if case["op"] == "adamw":
        n = sum(_sizes(case))
        p, g = _type(case["p"]).itemsize, _type(case["g"]).itemsize
        # in 8 bits the new states are also given as the values they stand for, in 16 bits each
        states = 16 if case["bits"] == 32 else 4 + 4
        return {"bytes": n * (2 * p + g + states), "flops": n * 16}
    if case["op"] == "group":
        p, c = case["images"] * case["pixels"], case["c"]
        x, y = (t.itemsize for t in TYPES[case["types"]])
        if not case["bwd"]:
            return {"bytes": p * c * (x + y) + 8 * case["images"] * case["groups"] + 8 * c, "flops": 10 * p * c}
        return {"bytes": p * c * (2 * x + y) + 8 * case["images"] * case["groups"] + 16 * c, "flops": 20 * p * c}
    m, k, n = case["m"], case["k"], case["n"]
    if not case["bwd"]:
        return {"bytes": 2 * m * k + n * k + 2 * m * n, "flops": 2 * m * n * k}
    return {"bytes": 2 * m * n + n * k + m * k + 2 * m * k + 2 * n * k, "flops": 4 * m * n * k}


# ---- states in 8 bits ----

def _signed(c):
    return c - (1 << 64) if c >> 63 else c


_GAMMA, _MIX1, _MIX2 = _signed(0x9E3779B97F4A7C15), _signed(0xBF58476D1CE4E5B9), _signed(0x94D049BB133111EB)


def _shift(z, n):
    return (z >> n) & ((1 << (64 - n)) - 1)


def _mix(z):
    """64 bits in which every bit of z shows (the finaliser of the splittable generator of Steele, Lea and Flood)."""
    z = z + _GAMMA
    z = (z ^ _shift(z, 30)) * _MIX1
    z = (z ^ _shift(z, 27)) * _MIX2
    return z ^ _shift(z, 31)


def _bits(key, n):
    """32 random bits for each of n places: two neighbours share 64."""
    z = _mix(key + torch.arange((n + 1) // 2, dtype=I64, device=key.device))
    return torch.stack([z & 0xFFFFFFFF, _shift(z, 32)], 1).view(-1)[:n]


def _encode(x, top, r):
    """Codes of x (one row for each 128 values) and the rows' exponents.  top: the largest code, 127 beside a sign or 255."""
    raw = x.view(torch.int32)
    mag = torch.clamp(raw & 0x7FFFFFFF, max=0x7FC00000)
    exp = torch.clamp(((mag.max(1, keepdim=True).values + 0xFFFFF) >> 20) >> 3, min=32)
    up = 0x7FFFF + ((mag >> 20) & 1) if r is None else r
    code = torch.clamp(((mag + up) >> 20) - (8 * exp - (top - 7)), min=0)
    if top == 255:
        return torch.where(mag > 0, torch.clamp(code, min=1), code).to(torch.uint8), exp.to(torch.uint8)
    return torch.where((raw < 0) & (code > 0), code + 128, code).to(torch.uint8), exp.to(torch.uint8)


def _decode(code, exp, top):
    c = code.to(torch.int32)
    mag = c if top == 255 else c & 127
    x = torch.where(mag > 0, (mag + 8 * exp.to(torch.int32) - (top - 7)) << 20, mag).view(F32)
    return x if top == 255 else torch.where(c > 127, -x, x)


# ---- inputs ----

def _adamw_prepare(case, gen):
    dev, sizes = gen.device, _sizes(case)
    places = [_up(n, 128) for n in sizes]                      # of the states
    spans = [_up(n, case["row"]) for n in sizes]               # of the tensors
    total, flat = sum(places), sum(spans)
    width = torch.tensor(sizes, device=dev)
    first = torch.tensor(places, device=dev).cumsum(0) - torch.tensor(places, device=dev)
    start = torch.tensor(spans, device=dev).cumsum(0) - torch.tensor(spans, device=dev)
    which = torch.repeat_interleave(torch.arange(len(sizes), device=dev), width)
    inner = torch.arange(sum(sizes), device=dev) - (width.cumsum(0) - width)[which]
    at, of = first[which] + inner, start[which] + inner        # a value's place among the states, and among the tensors
    scale = 10.0 ** (-2.0 - 2.0 * ((torch.arange(len(sizes), device=dev) * 7 + 3) % 11) / 10.0)
    size = torch.zeros(total, device=dev)
    size[at] = scale[which]
    decays = (torch.arange(len(sizes), device=dev) % 2 == 0)   # every other tensor, as weights and biases
    decay = torch.zeros(total, device=dev)
    decay[at] = decays[which].float() * DECAY
    s = dict(case=case, sizes=sizes, places=places, total=total, decay=decay, at=at, of=of)
    if case["row"] == 128:
        s["at"] = s["of"] = None
    # what a run has behind it: gradients of a size each, their mean and mean square
    g = torch.randn(total, generator=gen, device=dev) * size
    m = (0.3 * torch.randn(total, generator=gen, device=dev) * size).view(-1, 128)
    v = (torch.exp(0.7 * torch.randn(total, generator=gen, device=dev)) * size * size).view(-1, 128)

    def tensors(dtype, values):
        t = torch.zeros(flat, dtype=dtype, device=dev)
        if s["at"] is None:
            t.copy_(values)
        else:
            t[of] = values[at].to(dtype)
        return t, list(t.split(spans))

    p = 0.02 * torch.randn(total, generator=gen, device=dev) * (size > 0)
    s["p"], params = tensors(_type(case["p"]), p)
    s["g"], grads = tensors(_type(case["g"]), g)
    params, grads = [t[:n] for t, n in zip(params, sizes)], [t[:n] for t, n in zip(grads, sizes)]
    norm = s["g"].float().square().sum(dtype=F64).sqrt()
    s["norm"] = torch.stack([norm, torch.ones_like(norm)]).float()
    s["max_norm"] = norm.item() / case["clip"] if case["clip"] else 0.0
    s["out"] = torch.zeros(flat, device=dev) if case["delta"] else None
    if case["bits"] == 8:
        m8, v8 = _encode(m, 127, None), _encode(v, 255, None)
    if own:
        from geeps_b200.ops import functional as F
        s["params"], s["grads"] = F.GradList(params), F.GradList(grads)
        s["outs"] = F.GradList([t[:n] for t, n in zip(s["out"].split(spans), sizes)]) if case["delta"] else None
        state = s["state"] = F.AdamWState(params, bits=case["bits"], decay=decays.tolist(), steps=T0)
        if case["bits"] == 8:
            state.m.copy_(m8[0].view(-1))
            state.v.copy_(v8[0].view(-1))
            state.exponents.copy_(torch.cat([m8[1], v8[1]], 1))
            s["values"] = (torch.empty(total, dtype=BF, device=dev), torch.empty(total, dtype=BF, device=dev))
        else:
            state.m.copy_(m.view(-1))
            state.v.copy_(v.view(-1))
        return s
    s["steps"] = torch.full((1,), T0, dtype=I64, device=dev)
    if case["bits"] == 8:
        s["m"], s["m_exp"] = m8
        s["v"], s["v_exp"] = v8
    else:
        s["m"], s["v"] = m, v
    return s


def _normalise(x, images, groups):
    """[images, pixels, groups, channels] of (x - mean) * rstd, and [mean, rstd] as the forward pass keeps them."""
    x = x.float().view(images, -1, groups, x.shape[1] // groups)
    mean = x.mean((1, 3), keepdim=True)
    d = x - mean
    rstd = 1.0 / torch.sqrt((d * d).mean((1, 3), keepdim=True) + EPS)
    return d * rstd, torch.stack([mean.view(images, groups), rstd.view(images, groups)], 2)


def _group_prepare(case, gen):
    dev, c = gen.device, case["c"]
    p = case["images"] * case["pixels"]
    xt, yt = TYPES[case["types"]]
    # channels of different size and centre, as a convolution leaves them
    x = torch.randn(p, c, generator=gen, device=dev) * (0.5 + torch.rand(c, generator=gen, device=dev))
    x = (x + 0.5 * torch.randn(c, generator=gen, device=dev)).to(xt)
    s = dict(case=case, x=x, weight=1.0 + 0.2 * torch.randn(c, generator=gen, device=dev), bias=0.2 * torch.randn(c, generator=gen, device=dev))
    if case["bwd"]:
        s.update(dy=(1e-2 * torch.randn(p, c, generator=gen, device=dev)).to(yt), stats=_normalise(x, case["images"], case["groups"])[1],
                 dx=torch.empty(p, c, dtype=xt, device=dev), dweight=torch.empty(c, device=dev), dbias=torch.empty(c, device=dev))
    else:
        s.update(y=torch.empty(p, c, dtype=yt, device=dev), stats=torch.empty(case["images"], case["groups"], 2, device=dev))
    return s


def _quantise(x, tile):
    """e4m3 values of x [rows, columns] and the exponents of their scales, one for 128 columns of a row or for 128 x 128."""
    rows, cols = x.shape
    h = 128 if tile else 1
    x = torch.nn.functional.pad(x.float(), (0, _up(cols, 128) - cols, 0, _up(rows, h) - rows))
    x = x.view(-1, h, x.shape[1] // 128, 128)
    top = x.abs().amax((1, 3), keepdim=True)
    bits = top.view(torch.int32)
    # the exponent of top, less 8 where its fraction is at most 1.75 and less 7 where it is more
    e = torch.clamp((bits >> 23) - 127 - 8 + ((bits & 0x7FFFFF) > 0x600000).int(), min=-127)
    q = (x * ((127 - e) << 23).view(F32)).to(torch.float8_e4m3fn)
    return q.view(-1, q.shape[2] * 128)[:rows, :cols].contiguous(), e.view(e.shape[0], -1)


def _values(q, e, rows, cols):
    """What such a matrix stands for, in 32 bits."""
    scale = ((e + 127) << 23).view(F32)
    if e.shape[0] != rows:
        scale = scale.repeat_interleave(128, 0)[:rows]
    return q.float() * scale.repeat_interleave(128, 1)[:, :cols]


def _fp8_prepare(case, gen):
    dev = gen.device
    m, k, n = case["m"], case["k"], case["n"]
    x = (torch.randn(m, k, generator=gen, device=dev) * (0.2 + torch.rand(k, generator=gen, device=dev))).to(BF)
    w = (torch.randn(n, k, generator=gen, device=dev) / math.sqrt(k)).to(BF)
    s = dict(case=case, bias=0.1 * torch.randn(n, generator=gen, device=dev) if case["bias"] else None)
    if case["bwd"]:
        # kept from the forward pass: the input and the weights as their columns are multiplied
        s.update(dy=(1e-2 * torch.randn(m, n, generator=gen, device=dev)).to(BF), dx=torch.empty(m, k, dtype=BF, device=dev),
                 dw=torch.empty(n, k, dtype=BF, device=dev))
        if own:
            from geeps_b200.ops import functional as F
            s.update(wt=F.Fp8Matrix(k, n, dev), xt=F.Fp8Matrix(k, m, dev), dyq=F.Fp8Matrix(m, n, dev), dyt=F.Fp8Matrix(n, m, dev))
            F.quantize_fp8(w, None, transposed=s["wt"], tile=True)
            F.quantize_fp8(x, None, transposed=s["xt"])
        else:
            s.update(wt=_quantise(w.T.contiguous(), True), xt=_quantise(x.T.contiguous(), False))
        return s
    s.update(x=x, y=torch.empty(m, n, dtype=BF, device=dev))
    if own:
        from geeps_b200.ops import functional as F
        s.update(xq=F.Fp8Matrix(m, k, dev), w=F.Fp8Matrix(n, k, dev))
        F.quantize_fp8(w, s["w"], tile=True)
    else:
        s["w"] = _quantise(w, True)
    return s


def prepare(case, seed):
    gen = torch.Generator(device=torch.device("cuda", torch.cuda.current_device())).manual_seed(seed)
    return {"adamw": _adamw_prepare, "group": _group_prepare, "fp8": _fp8_prepare}[case["op"]](case, gen)


# ---- plain forms ----

def _adamw_plain(s):
    case, dev = s["case"], s["p"].device
    s["steps"] += 1
    key = _mix(case["seed"] * 0x100000001B3 + s["steps"])

    def among_states(t):
        if s["at"] is None:
            return t.float()
        return torch.zeros(s["total"], device=dev).index_copy_(0, s["at"], t[s["of"]].float())

    p, g = among_states(s["p"]), among_states(s["g"])
    if case["clip"]:
        norm, bound = s["norm"][0], torch.full_like(s["norm"][0], s["max_norm"])
        g = g * torch.where(norm > bound, bound / norm, torch.ones_like(norm))
    m, v = (s["m"], s["v"]) if case["bits"] == 32 else (_decode(s["m"], s["m_exp"], 127), _decode(s["v"], s["v_exp"], 255))
    g = g.view(-1, 128)
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + (g * g) * (1 - BETA2)
    c1, c2 = (1.0 / (1.0 - b ** s["steps"].to(F64)) for b in (BETA1, BETA2))
    change = -LR * ((m * c1.float()) / (torch.sqrt(v * c2.float()) + ADAM_EPS) + s["decay"].view(-1, 128) * p.view(-1, 128))
    if case["bits"] == 8:
        r = None, None
        if case["seed"] >= 0:
            b = _bits(key, s["total"]).view(-1, 128)
            r = (((b & 0xFFFF) << 4) + 8).int(), ((b >> 16 << 4) + 8).int()
        s["m"], s["m_exp"] = _encode(m, 127, r[0])
        s["v"], s["v_exp"] = _encode(v, 255, r[1])
        values = [_decode(s["m"], s["m_exp"], 127).view(-1).to(BF), _decode(s["v"], s["v_exp"], 255).view(-1).to(BF)]
    else:
        s["m"], s["v"] = m, v
        values = [m.view(-1), v.view(-1)]
    new = change.view(-1) if case["delta"] else p + change.view(-1)
    if case["p"] == "bf16" and case["seed"] >= 0:
        up = (_bits(_mix(key), s["total"]) & 0xFFFF).int()
        new = ((new.view(torch.int32) + up) & -65536).view(F32)
    t = s["out"] if case["delta"] else s["p"]
    if s["at"] is None:
        t.copy_(new)
    else:
        t[s["of"]] = new[s["at"]].to(t.dtype)
    return [t] + values


def _slope(z, act):
    """The activation's slope at z."""
    if act == "relu":
        return (z > 0).float()
    g = 1.0 / (1.0 + torch.exp(-z))
    return g * (1.0 + z * (1.0 - g))


def _group_plain(s):
    case = s["case"]
    images, groups, c = case["images"], case["groups"], case["c"]
    w, b = s["weight"].view(groups, -1), s["bias"].view(groups, -1)
    if not case["bwd"]:
        n, stats = _normalise(s["x"], images, groups)
        z = n * w + b
        if case["act"] == "relu":
            z = torch.clamp(z, min=0)
        elif case["act"] == "silu":
            z = z / (1.0 + torch.exp(-z))
        return z.view(-1, c).to(s["y"].dtype), stats
    mean, rstd = s["stats"].view(images, 1, groups, 1, 2).unbind(-1)
    n = (s["x"].float().view(images, -1, groups, c // groups) - mean) * rstd
    dz = s["dy"].float().view_as(n)
    if case["act"]:
        dz = dz * _slope(n * w + b, case["act"])
    a = dz * w
    dx = rstd * (a - a.mean((1, 3), keepdim=True) - n * (a * n).mean((1, 3), keepdim=True))
    return dx.view(-1, c).to(s["dx"].dtype), (dz * n).sum((0, 1)).view(-1), dz.sum((0, 1)).view(-1)


def _fp8_plain(s):
    case = s["case"]
    m, k, n = case["m"], case["k"], case["n"]
    if case["bwd"]:
        dx = _values(*_quantise(s["dy"], False), m, n) @ _values(*s["wt"], k, n).T
        dw = _values(*_quantise(s["dy"].T, False), n, m) @ _values(*s["xt"], k, m).T
        return dx.to(BF), dw.to(BF)
    y = _values(*_quantise(s["x"], False), m, k) @ _values(*s["w"], n, k).T
    if case["bias"]:
        y = y + s["bias"]
    if case["relu"]:
        y = torch.clamp(y, min=0)
    return y.to(BF)


# ---- one pass ----

def run(state):
    s, case = state, state["case"]
    if not own:
        return {"adamw": _adamw_plain, "group": _group_plain, "fp8": _fp8_plain}[case["op"]](s)
    from geeps_b200.ops import functional as F
    if case["op"] == "adamw":
        F.adamw_step(s["params"], s["grads"], s["state"], LR, betas=(BETA1, BETA2), eps=ADAM_EPS, weight_decay=DECAY, out=s["outs"],
                     clip=(s["norm"], s["max_norm"]) if case["clip"] else None, seed=case["seed"] if case["seed"] >= 0 else None)
        m, v = (s["state"].m, s["state"].v) if case["bits"] == 32 else F.adamw_moments(s["state"], *s["values"])
        return [s["out"] if case["delta"] else s["p"], m, v]
    if case["op"] == "group":
        norm = F.GroupNorm(case["groups"], s["weight"], s["bias"], s["stats"], eps=EPS, act=case["act"] or None, dweight=s.get("dweight"),
                           dbias=s.get("dbias"))
        if not case["bwd"]:
            F.group_norm_forward(s["x"], s["y"], case["images"], norm)
            return s["y"], s["stats"]
        F.group_norm_backward(s["x"], s["dy"], s["dx"], case["images"], norm)
        return s["dx"], s["dweight"], s["dbias"]
    if case["bwd"]:
        F.quantize_fp8(s["dy"], s["dyq"], transposed=s["dyt"])
        F.matmul_fp8(s["dyq"], s["wt"], s["dx"])
        F.matmul_fp8(s["dyt"], s["xt"], s["dw"])
        return s["dx"], s["dw"]
    F.quantize_fp8(s["x"], s["xq"])
    return F.matmul_fp8(s["xq"], s["w"], s["y"], bias=s["bias"], relu=case["relu"])


# ---- definitions in 64 bits ----

def _step64(x, mantissa):
    """The distance of neighbouring values with so many bits of mantissa around x."""
    return torch.exp2((torch.frexp(x).exponent - 1 - mantissa).to(F64))


def _state64(x, bits, r):
    """x [blocks, 128] as a state in 8 bits stands for it, by the random bits r in 20 (or to the nearest)."""
    step = _step64(x, 3)
    mag = x.abs() / step
    mag = (torch.round(mag) if r is None else torch.floor(mag + r.to(F64) / 2 ** 20)) * step
    # the largest value's binade, the next one where it may be rounded up to that
    high = x.abs().amax(1, keepdim=True)
    top = (torch.frexp(torch.clamp(high, min=2.0 ** -95)).exponent - 1).to(F64)
    top = top + (high > 1.875 * torch.exp2(top)).to(F64)
    bits -= 3                                             # of the exponent
    low = torch.exp2(top - 2 ** bits + 1)                 # code 0 would be this value: the codes from 1 on lie above
    if bits == 5:
        return torch.where(x > 0, torch.maximum(mag, low * 1.125), mag)
    return torch.where(mag <= low, torch.zeros_like(mag), mag) * torch.sign(x)


def _adamw_exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    dev, total = s["p"].device, s["total"]
    at = torch.arange(total, device=dev) if s["at"] is None else s["at"]
    of = at if s["of"] is None else s["of"]

    def wide(t):
        w = torch.zeros(total, dtype=F64, device=dev)
        w[at] = t[of].to(F64)
        return w.view(-1, 128)

    p, g = wide(s["p"]), wide(s["g"])
    if case["clip"]:
        g = g * min(1.0, s["max_norm"] / s["norm"][0].item())
    m, v = (s["m"], s["v"]) if case["bits"] == 32 else (_decode(s["m"], s["m_exp"], 127), _decode(s["v"], s["v_exp"], 255))
    m = torch.lerp(g, m.to(F64), BETA1)
    v = torch.lerp(g ** 2, v.to(F64), BETA2)
    t = T0 + 1
    change = -LR * (m / (1 - BETA1 ** t) / ((v / (1 - BETA2 ** t)) ** 0.5 + ADAM_EPS) + s["decay"].to(F64).view(-1, 128) * p)
    if case["bits"] == 8:
        r = None, None
        if case["seed"] >= 0:
            b = _bits(_mix(torch.tensor([case["seed"] * 0x100000001B3 + t], dtype=I64, device=dev)), total).view(-1, 128)
            r = (b % 65536) * 16 + 8, (b // 65536) * 16 + 8
        m, v = _state64(m, 7, r[0]), _state64(v, 8, r[1])
    new = torch.zeros(s["p"].numel(), dtype=F64, device=dev)
    new[of] = (change if case["delta"] else p + change).view(-1)[at]
    return [new, m.view(-1), v.view(-1)]


def _group_exact(case, seed):
    s = prepare(case, seed)
    images, groups, c = case["images"], case["groups"], case["c"]
    x, w, b = (s[k].to(F64).requires_grad_(True) for k in ("x", "weight", "bias"))
    var, mean = torch.var_mean(x.view(images, -1, groups, c // groups), (1, 3), unbiased=False, keepdim=True)
    rstd = (var + EPS) ** -0.5
    z = torch.addcmul(b, ((x.view(images, -1, groups, c // groups) - mean) * rstd).view(-1, c), w)
    y = torch.relu(z) if case["act"] == "relu" else z * torch.sigmoid(z) if case["act"] else z
    if not case["bwd"]:
        return y.detach(), torch.stack([mean.view(images, groups), rstd.view(images, groups)], 2).detach()
    return torch.autograd.grad(y, (x, w, b), s["dy"].to(F64))


def _round64(x, tile):
    """x as its e4m3 values and scales stand for it."""
    rows, cols = x.shape
    h = 128 if tile else 1
    full = torch.zeros(_up(rows, h), _up(cols, 128), dtype=F64, device=x.device)
    full[:rows, :cols] = x
    blocks = full.unflatten(1, (-1, 128)).unflatten(0, (-1, h))
    scale = torch.exp2(torch.ceil(torch.log2(torch.clamp(blocks.abs().amax((1, 3), keepdim=True), min=1e-300) / 448.0)))
    v = blocks / scale
    step = torch.clamp(_step64(v, 3), min=2.0 ** -9)
    return (torch.round(v / step) * step * scale).reshape(full.shape)[:rows, :cols]


def _fp8_exact(case, seed):
    gen = torch.Generator(device=torch.device("cuda", torch.cuda.current_device())).manual_seed(seed)
    m, k, n = case["m"], case["k"], case["n"]
    # the inputs as `prepare` makes them, before anything of them is rounded to 8 bits
    x = (torch.randn(m, k, generator=gen, device=gen.device) * (0.2 + torch.rand(k, generator=gen, device=gen.device))).to(BF)
    w = (torch.randn(n, k, generator=gen, device=gen.device) / math.sqrt(k)).to(BF)
    bias = 0.1 * torch.randn(n, generator=gen, device=gen.device) if case["bias"] else None
    if case["bwd"]:
        dy = (1e-2 * torch.randn(m, n, generator=gen, device=gen.device)).to(BF)
        return _round64(dy, False) @ _round64(w, True), _round64(dy.T, False) @ _round64(x.T, False).T
    y = _round64(x, False) @ _round64(w, True).T
    if bias is not None:
        y += bias
    return y.clamp_(min=0) if case["relu"] else y


def exact(case, seed):
    return {"adamw": _adamw_exact, "group": _group_exact, "fp8": _fp8_exact}[case["op"]](case, seed)
