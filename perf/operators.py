"""Performance cases of the operators that keep a deep network's training stable: normalisation before and after a
residual block, the block's gate and residual scale, and clipping of the gradients by their global norm.

A case is a dict of plain values.  `prepare` makes what a training program holds before the call, `run` makes one pass,
either through the framework's entry points (`own`) or in elementary torch operations in 32 bits, and `exact` gives the
same results from the definitions in 64 bits.

Rows are pixels (or tokens), columns are channels, as in every layer of this framework.  Types: "bf16" is bf16 everywhere,
"mixed" a residual stream in fp32 around blocks in bf16, "fp32" fp32 everywhere.  Parameters and statistics are fp32.
"""
from __future__ import annotations

import math
import random

import torch

own = False

BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
TYPES = {"bf16": (BF, BF), "mixed": (F32, BF), "fp32": (F32, F32)}      # residual stream, inside a block
EPS = 1e-5


def listed():
    return [
        # gradient clipping from a program's own gradient buffers into the buffers that the tables' updates leave from, where
        # every parameter starts on a row of 128 values: a new classifier on a frozen network (four small tables, where
        # latency counts); a network whose parameters are as many and as ragged as the 22K-class Inception's, with gradients
        # in bf16; a network of AlexNet's size and shares; a large model in bf16, packed without gaps
        dict(name="clip_head", op="clip", count=4, total=11_274, skew=1.0, row=128, src="fp32", dst="fp32", ratio=3.0),
        dict(name="clip_ragged_bf16", op="clip", count=331, total=33_554_467, skew=2.0, row=128, src="bf16", dst="fp32", ratio=1.7),
        dict(name="clip_alexnet", op="clip", count=16, total=60_965_224, skew=2.5, row=128, src="fp32", dst="fp32", ratio=12.0),
        dict(name="clip_large_bf16", op="clip", count=75, total=268_435_391, skew=1.5, row=1, src="bf16", dst="bf16", ratio=1.2),
        # ... and the step that most steps are: in place, with a norm below the bound
        dict(name="clip_quiet", op="clip", count=16, total=60_965_224, skew=2.5, row=128, src="fp32", dst="", ratio=0.4),
        # a norm in front of a block: one row at a time as a service answers, and a training batch of 14 x 14 pixels, forward
        # and backward with the gradient of the connection that goes round the block
        dict(name="norm_one_row", op="norm", bwd=False, images=1, pixels=1, c=4096, kind="rms", types="bf16"),
        dict(name="norm_batch", op="norm", bwd=False, images=256, pixels=196, c=576, kind="layer", types="bf16"),
        dict(name="norm_batch_backward", op="norm", bwd=True, images=256, pixels=196, c=576, kind="layer", types="bf16"),
        # the end of a block with the norm in front of the next: a few rows with a gate for each; a training batch with a gate
        # per image, forward and backward; odd widths with the residual stream in fp32
        dict(name="join_few_rows", op="join", bwd=False, images=1, pixels=7, c=2048, post="rms", next="rms", scale=True,
             gate="pixel", sigmoid=False, types="bf16"),
        dict(name="join_batch", op="join", bwd=False, images=256, pixels=196, c=1024, post="layer", next="layer", scale=True,
             gate="image", sigmoid=True, types="bf16"),
        dict(name="join_batch_backward", op="join", bwd=True, images=256, pixels=196, c=1024, post="layer", next="layer",
             scale=True, gate="image", sigmoid=True, types="bf16"),
        dict(name="join_odd_backward", op="join", bwd=True, images=37, pixels=113, c=1003, post="rms", next="", scale=True,
             gate="pixel", sigmoid=True, types="mixed"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.35:
        dst = rng.choice(["fp32", "bf16", ""])
        return dict(op="clip", count=_log(rng, 1, 331), total=_log(rng, 700, 1.2e8), skew=rng.choice([0.0, 1.0, 2.0, 2.5]),
                    row=rng.choice([1, 128, 128]), src=rng.choice(["fp32", "bf16"]), dst=dst, ratio=0.5 if dst == "" else rng.choice([0.7, 1.5, 9.0]))
    c = _log(rng, 1, 16384)
    if rng.random() < 0.6:
        c = (c + 7) // 8 * 8
    rows = max(1, min(_log(rng, 1, 400_000), 30_000_000 // c))
    images = min(rows, _log(rng, 1, 512))
    case = dict(images=images, pixels=rows // images, c=c, types=rng.choice(["bf16", "bf16", "mixed", "fp32"]), bwd=rng.random() < 0.6)
    if rng.random() < 0.4:
        return dict(op="norm", kind=rng.choice(["layer", "rms"]), **case)
    return dict(op="join", post=rng.choice(["layer", "rms", ""]), next=rng.choice(["layer", "rms", ""]), scale=rng.random() < 0.7,
                gate=rng.choice(["pixel", "image", ""]), sigmoid=rng.random() < 0.5, **case)


def _sizes(case):
    """Element counts of the tensors of a clipping case: shares whose logarithm spreads by `skew`, odd ones among them."""
    rng = random.Random(case["count"] * 1_000_003 + case["total"])
    share = [math.exp(rng.gauss(0.0, case["skew"])) for _ in range(case["count"])]
    whole = sum(share)
    sizes = [max(1, int(case["total"] * s / whole)) for s in share]
    sizes[sizes.index(max(sizes))] += max(0, case["total"] - sum(sizes))
    return sizes


def _flat(sizes, row, dtype, dev):
    """One buffer for all tensors of a clipping case, each of which starts at a multiple of `row` values, and its views."""
    starts, at = [], 0
    for n in sizes:
        starts.append(at)
        at += (n + row - 1) // row * row
    flat = torch.zeros(at, dtype=dtype, device=dev)
    return flat, [flat[a:a + n] for a, n in zip(starts, sizes)]


def _type(name):
    return BF if name == "bf16" else F32


def work(case):
    if case["op"] == "clip":
        n = sum(_sizes(case))
        src, dst = 2 if case["src"] == "bf16" else 4, {"bf16": 2, "fp32": 4, "": 0}[case["dst"]]
        return {"bytes": n * (src + dst), "flops": n * (3 if dst else 2)}
    p, c = case["images"] * case["pixels"], case["c"]
    r, b = (t.itemsize for t in TYPES[case["types"]])
    if case["op"] == "norm":
        if not case["bwd"]:
            return {"bytes": p * c * (r + b) + 8 * p + 8 * c, "flops": 8 * p * c}
        return {"bytes": p * c * (3 * r + b) + 8 * p + 12 * c, "flops": 16 * p * c}
    gates = {"pixel": p, "image": case["images"], "": 0}[case["gate"]] * c * b
    if not case["bwd"]:
        return {"bytes": p * c * (2 * r + b + (b if case["next"] else 0)) + gates, "flops": 20 * p * c}
    return {"bytes": p * c * (2 * r + 2 * b + (r + b if case["next"] else 0)) + 2 * gates, "flops": 40 * p * c}


# ---- inputs ----

def _normalise(x, kind):
    """n = (x - mean) * rstd over the columns, and [mean, rstd] as the forward pass keeps them."""
    x = x.float()
    mean = x.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(x[:, :1])
    d = x - mean
    rstd = 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
    return d * rstd, torch.cat([mean, rstd], 1)


def _parameters(gen, c):
    dev = gen.device
    return (1.0 + 0.2 * torch.randn(c, generator=gen, device=dev), 0.1 * torch.randn(c, generator=gen, device=dev))


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    if case["op"] == "clip":
        sizes = _sizes(case)
        flat, grads = _flat(sizes, case["row"], _type(case["src"]), dev)
        for i, g in enumerate(grads):       # layers whose gradients differ in size by some orders of magnitude
            scale = 10.0 ** (-1.0 - 3.0 * ((i * 7 + 3) % 11) / 10.0)
            g.copy_(torch.randn(g.numel(), generator=gen, device=dev) * scale)
        norm = math.sqrt((flat.float() ** 2).sum(dtype=F64).item())
        s = dict(case=case, grads=grads, max_norm=norm / case["ratio"], result=torch.zeros(2, device=dev), flat=flat, out=None)
        if case["dst"]:
            s["flat"], s["out"] = _flat(sizes, case["row"], _type(case["dst"]), dev)
        if own:
            from geeps_b200.ops import functional as F
            s["grad_list"] = F.GradList(grads)
            s["out_list"] = F.GradList(s["out"]) if s["out"] is not None else None
        return s
    p, c = case["images"] * case["pixels"], case["c"]
    stream, block = TYPES[case["types"]]

    def rows(dtype, size, centre=0.0):
        return (torch.randn(p, c, generator=gen, device=dev) * size + centre).to(dtype)

    def empty(dtype, like=p):
        return torch.empty(like, c, dtype=dtype, device=dev)

    def sums():
        return torch.empty(c, device=dev)

    s = dict(case=case)
    if case["op"] == "norm":
        w, b = _parameters(gen, c)
        s.update(x=rows(stream, 2.0, 0.5), weight=w, bias=b)
        if case["bwd"]:
            s.update(dy=rows(block, 1e-2), dres=rows(stream, 1e-2), stats=_normalise(s["x"], case["kind"])[1],
                     dx=empty(stream), dweight=sums(), dbias=sums())
        else:
            s.update(y=empty(block), stats=torch.empty(p, 2, device=dev))
        return s
    s.update(x=rows(block, 1.5, -0.25), weight=None, bias=None, scale=None, gate=None, next_weight=None, next_bias=None)
    if case["post"]:
        s["weight"], s["bias"] = _parameters(gen, c)
    if case["next"]:
        s["next_weight"], s["next_bias"] = _parameters(gen, c)
    if case["scale"]:
        s["scale"] = 0.3 + 0.1 * torch.randn(c, generator=gen, device=dev)
    if case["gate"]:
        g = p if case["gate"] == "pixel" else case["images"]
        s["gate"] = torch.randn(g, c, generator=gen, device=dev).to(block)
    if not case["bwd"]:
        s.update(res=rows(stream, 2.0), out=empty(stream), y=empty(block) if case["next"] else None,
                 stats=torch.empty(p, 2, device=dev) if case["post"] else None,
                 next_stats=torch.empty(p, 2, device=dev) if case["next"] else None)
        return s
    s.update(dout=rows(stream, 1e-2), dx=empty(block), dres=empty(stream), stats=None, out=None, dy=None, next_stats=None)
    s["dgate"] = torch.empty_like(s["gate"]) if case["gate"] else None
    for name, there in (("dweight", case["post"]), ("dbias", case["post"]), ("dscale", case["scale"]),
                        ("dnext_weight", case["next"]), ("dnext_bias", case["next"])):
        s[name] = sums() if there else None
    if case["post"]:
        s["stats"] = _normalise(s["x"], case["post"])[1]
    if case["next"]:
        s.update(out=rows(stream, 2.0), dy=rows(block, 1e-2))
        s["next_stats"] = _normalise(s["out"], case["next"])[1]
    return s


# ---- plain forms ----

def _clip_plain(s):
    total = sum((g.float() * g.float()).sum(dtype=F64) for g in s["grads"])
    norm = torch.sqrt(total)
    c = torch.where(norm > s["max_norm"], s["max_norm"] / norm, torch.ones_like(norm)).float()
    for g, o in zip(s["grads"], s["grads"] if s["out"] is None else s["out"]):
        o.copy_(g.float() * c)
    return torch.stack([norm.float(), c]), s["flat"]


def _affine(n, w, b):
    return n if w is None else n * w + b


def _norm_gradient(dz, n, rstd, w, kind):
    a = dz if w is None else dz * w
    centre = a.mean(1, keepdim=True) if kind == "layer" else 0.0
    return rstd * (a - centre - n * (a * n).mean(1, keepdim=True))


def _saved(x, stats):
    return (x.float() - stats[:, :1]) * stats[:, 1:]


def _norm_plain(s):
    case = s["case"]
    if not case["bwd"]:
        n, stats = _normalise(s["x"], case["kind"])
        return _affine(n, s["weight"], s["bias"]).to(s["y"].dtype), stats
    n, dy = _saved(s["x"], s["stats"]), s["dy"].float()
    dx = _norm_gradient(dy, n, s["stats"][:, 1:], s["weight"], case["kind"]) + s["dres"].float()
    return dx.to(s["dx"].dtype), (dy * n).sum(0), dy.sum(0)


def _gate_rows(s):
    """The gate's factor for every row, or None."""
    if s["gate"] is None:
        return None
    g = s["gate"].float()
    if s["case"]["sigmoid"]:
        g = 1.0 / (1.0 + torch.exp(-g))
    return g.repeat_interleave(s["x"].shape[0] // g.shape[0], 0)


def _join_plain(s):
    case = s["case"]
    if not case["bwd"]:
        z, stats = _normalise(s["x"], case["post"]) if case["post"] else (s["x"].float(), None)
        z = _affine(z, s["weight"], s["bias"])
        g = _gate_rows(s)
        if g is not None:
            z = z * g
        if s["scale"] is not None:
            z = z * s["scale"]
        h = s["res"].float() + z
        outs = [h.to(s["out"].dtype)]
        if stats is not None:
            outs.append(stats)
        if case["next"]:
            n, stats = _normalise(h, case["next"])
            outs += [_affine(n, s["next_weight"], s["next_bias"]).to(s["y"].dtype), stats]
        return outs
    dh, after = s["dout"].float(), []
    if case["next"]:
        n, dy = _saved(s["out"], s["next_stats"]), s["dy"].float()
        dh = dh + _norm_gradient(dy, n, s["next_stats"][:, 1:], s["next_weight"], case["next"])
        after = [(dy * n).sum(0), dy.sum(0)]
    n = _saved(s["x"], s["stats"]) if case["post"] else s["x"].float()
    z = _affine(n, s["weight"], s["bias"])
    g, outs = _gate_rows(s), []
    dz = dh if g is None else dh * g
    if s["scale"] is not None:
        outs.append((dz * z).sum(0))
        dz = dz * s["scale"]
    if g is not None:
        dg = dh * z if s["scale"] is None else dh * z * s["scale"]
        if case["sigmoid"]:
            dg = dg * g * (1.0 - g)
        outs.append(dg.view(s["gate"].shape[0], -1, case["c"]).sum(1).to(s["dgate"].dtype))
    if case["post"]:
        outs += [(dz * n).sum(0), dz.sum(0)]
        dz = _norm_gradient(dz, n, s["stats"][:, 1:], s["weight"], case["post"])
    return [dz.to(s["dx"].dtype), dh.to(s["dres"].dtype)] + outs + after


# ---- one pass ----

def _norms(F, s):
    case = s["case"]
    post = F.Norm(case["post"], s["weight"], s["bias"], s["stats"], eps=EPS, dweight=s.get("dweight"),
                  dbias=s.get("dbias")) if case["post"] else None
    pre = F.Norm(case["next"], s["next_weight"], s["next_bias"], s["next_stats"], eps=EPS, dweight=s.get("dnext_weight"),
                 dbias=s.get("dnext_bias")) if case["next"] else None
    return post, pre


def run(state):
    s, case = state, state["case"]
    if not own:
        return {"clip": _clip_plain, "norm": _norm_plain, "join": _join_plain}[case["op"]](s)
    from geeps_b200.ops import functional as F
    if case["op"] == "clip":
        F.clip_gradients(s["grad_list"], s["max_norm"], s["result"], out=s["out_list"])
        return s["result"], s["flat"]
    if case["op"] == "norm":
        norm = F.Norm(case["kind"], s["weight"], s["bias"], s["stats"], eps=EPS, dweight=s.get("dweight"), dbias=s.get("dbias"))
        if not case["bwd"]:
            F.norm_forward(s["x"], s["y"], norm)
            return s["y"], s["stats"]
        F.norm_backward(s["x"], s["dy"], s["dx"], norm, dres=s["dres"])
        return s["dx"], s["dweight"], s["dbias"]
    post, pre = _norms(F, s)
    if not case["bwd"]:
        F.residual_forward(s["x"], s["res"], s["out"], post=post, scale=s["scale"], gate=s["gate"], sigmoid=case["sigmoid"],
                           y=s["y"], pre=pre)
        return [s[k] for k in ("out", "stats", "y", "next_stats") if s[k] is not None]
    F.residual_backward(s["x"], s["dout"], s["dx"], s["dres"], post=post, scale=s["scale"], dscale=s["dscale"], gate=s["gate"],
                        dgate=s["dgate"], sigmoid=case["sigmoid"], out=s["out"], dy=s["dy"], pre=pre)
    return [s[k] for k in ("dx", "dres", "dscale", "dgate", "dweight", "dbias", "dnext_weight", "dnext_bias") if s[k] is not None]


# ---- definitions in 64 bits: gradients by differentiation of the forward pass ----

def _norm64(x, kind, w, b):
    if kind == "layer":
        var, mean = torch.var_mean(x, 1, unbiased=False, keepdim=True)
    else:
        var, mean = x.square().mean(1, keepdim=True), torch.zeros_like(x[:, :1])
    rstd = (var + EPS) ** -0.5
    return torch.addcmul(b, (x - mean) * rstd, w), torch.cat([mean, rstd], 1)


def _leaf(t):
    return None if t is None else t.detach().to(F64).requires_grad_(True)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "clip":
        norm = math.sqrt(math.fsum(torch.linalg.vector_norm(g.to(F64)).item() ** 2 for g in s["grads"]))
        c = min(1.0, s["max_norm"] / norm)
        flat = torch.zeros(s["flat"].numel(), dtype=F64, device=s["flat"].device)
        for g, o in zip(s["grads"], s["grads"] if s["out"] is None else s["out"]):
            flat[o.storage_offset():o.storage_offset() + o.numel()] = g.to(F64) * c
        return torch.tensor([norm, c], dtype=F64), flat
    if case["op"] == "norm":
        x, w, b = _leaf(s["x"]), _leaf(s["weight"]), _leaf(s["bias"])
        y, stats = _norm64(x, case["kind"], w, b)
        if not case["bwd"]:
            return y.detach(), stats.detach()
        dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"].to(F64))
        return dx + s["dres"].to(F64), dw, db
    leaves = {k: _leaf(s[k]) for k in ("x", "weight", "bias", "scale", "gate", "next_weight", "next_bias")}
    z, stats = _norm64(leaves["x"], case["post"], leaves["weight"], leaves["bias"]) if case["post"] else (leaves["x"], None)
    branch = z.view(case["images"], case["pixels"], case["c"])
    if leaves["gate"] is not None:
        g = torch.sigmoid(leaves["gate"]) if case["sigmoid"] else leaves["gate"]
        branch = branch * g.view(case["images"], -1, case["c"])
    if leaves["scale"] is not None:
        branch = branch * leaves["scale"]
    branch = branch.reshape(-1, case["c"])
    if not case["bwd"]:
        with torch.no_grad():
            h = s["res"].to(F64) + branch
            outs = [h] + ([stats] if stats is not None else [])
            if case["next"]:
                outs += list(_norm64(h, case["next"], leaves["next_weight"], leaves["next_bias"]))
        return [t.detach() for t in outs]
    dh, after = s["dout"].to(F64), []
    if case["next"]:
        h = _leaf(s["out"])
        y, _ = _norm64(h, case["next"], leaves["next_weight"], leaves["next_bias"])
        d, dw, db = torch.autograd.grad(y, (h, leaves["next_weight"], leaves["next_bias"]), s["dy"].to(F64))
        dh, after = dh + d, [dw, db]
    names = [k for k in ("x", "scale", "gate", "weight", "bias") if leaves[k] is not None]
    grads = torch.autograd.grad(branch, [leaves[k] for k in names], dh)
    return [grads[0], dh] + list(grads[1:]) + after
