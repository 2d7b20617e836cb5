"""Norms before and after a residual block, its gate and residual scale: kernels against the definitions in 64 bits.

Tolerances: an output is rounded once to its type (half a step, finfo.eps / 2 of its value), and what it is computed from in
fp32 is off by a number of roundings of 2^-24 of the magnitudes that enter.  A row's sum is a tree of at most 32 + 5 + 16
additions, so 64 of them bound a row's sums and the operations round them (`STEPS`); a column sum adds the rows of a slot one
after the other, which adds their number.
"""
import itertools

import pytest
import torch

from geeps_b200.ops import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
TYPES = {"bf16": (BF, BF), "mixed": (F32, BF), "fp32": (F32, F32)}
U, STEPS = 2.0 ** -24, 64


def close(got, ref, mag, steps=STEPS, what=""):
    half = torch.finfo(got.dtype).eps / 2 if got.dtype != F32 else U
    tol = half * ref.abs() + (1 + half) * steps * U * mag
    off = (got.double() - ref).abs()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    worst = (off - tol).max().item() if off.numel() else 0.0
    assert worst <= 0, f"{what}: {worst} beyond the tolerance, {off.max().item()} off"


def norm64(x, kind, w, b, eps):
    """Value, n, mean, rstd and the magnitude that the roundings of n are relative to."""
    mean = x.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(x[:, :1])
    rstd = ((x - mean).square().mean(1, keepdim=True) + eps) ** -0.5
    n = (x - mean) * rstd
    return (n if w is None else n * w) + (0 if b is None else b), n, mean, rstd, (x.abs() + mean.abs()) * rstd


def rand(gen, shape, dtype, size=1.0, centre=0.0):
    return (torch.randn(shape, generator=gen, device=DEV) * size + centre).to(dtype)


def param(gen, c, on=True):
    return 1.0 + 0.3 * torch.randn(c, generator=gen, device=DEV) if on else None


def d(t):
    return None if t is None else t.double()


def check_norm(gen, rows, c, kind, types, affine=True, make=None, eps=1e-5):
    rt, bt = TYPES[types]
    make = make or (lambda dtype: torch.empty(rows, c, dtype=dtype, device=DEV))
    x = make(rt).copy_(rand(gen, (rows, c), rt, 2.0, 0.5))
    w, b = param(gen, c, affine), param(gen, c, affine)
    stats = torch.full((rows, 2), -7.0, device=DEV)
    y = make(bt)
    F.norm_forward(x, y, F.Norm(kind, w, b, stats, eps))
    y64, n, mean, rstd, mag = norm64(d(x), kind, d(w), d(b), eps)
    wa, ba = (1.0 if w is None else d(w).abs()), (0.0 if b is None else d(b).abs())
    # the variance is a sum of squares of differences that are off by their own rounding: STEPS covers it twice
    close(y, y64, mag * wa * (1 + n.abs()) + ba, what="y")
    assert (stats[:, 0].double() - mean[:, 0]).abs().max() <= STEPS * U * (d(x).abs().mean(1).max() + 1e-30)
    assert ((stats[:, 1].double() / rstd[:, 0]) - 1).abs().max() <= STEPS * U * (1 + mag.square().mean(1).max())
    dy, dres = make(bt).copy_(rand(gen, (rows, c), bt)), make(rt).copy_(rand(gen, (rows, c), rt))
    dx, dw, db = make(rt), torch.full((c,), 7.0, device=DEV), torch.full((c,), 7.0, device=DEV)
    F.norm_backward(x, dy, dx, F.Norm(kind, w, b, stats, eps, dw, db), dres=dres)
    a = d(dy) * (1.0 if w is None else d(w))
    m0 = a.mean(1, keepdim=True) if kind == "layer" else 0.0
    ref = rstd * (a - m0 - n * (a * n).mean(1, keepdim=True)) + d(dres)
    m = rstd * (a.abs() + a.abs().mean(1, keepdim=True) + (1 + mag) * (1 + n.abs()) * (a.abs() * (1 + mag)).mean(1, keepdim=True)) + d(dres).abs()
    close(dx, ref, m * (1 + n.abs()), what="dx")
    steps = STEPS + rows
    close(dw, (d(dy) * n).sum(0), (d(dy).abs() * (1 + mag) * (1 + n.abs())).sum(0), steps, "dweight")
    close(db, d(dy).sum(0), d(dy).abs().sum(0), steps, "dbias")


SHAPES = [(1, 1), (3, 1), (5, 7), (64, 8), (33, 64), (1, 96), (130, 200), (17, 257), (9, 1000), (50, 1024), (700, 576), (7, 4096),
          (3, 4104), (5, 8192), (2, 8193), (3, 16384), (2, 16383), (5000, 16)]


@pytest.mark.parametrize("rows,c", SHAPES)
@pytest.mark.parametrize("types", list(TYPES))
def test_norm_forward_and_backward(rows, c, types):
    gen = torch.Generator(device=DEV).manual_seed(rows * 31 + c)
    for kind in ("layer", "rms"):
        check_norm(gen, rows, c, kind, types, affine=(rows + c) % 3 != 0)


@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("pitch,offset", [(1, 0), (8, 0), (3, 1), (8, 8), (0, 1)])
def test_rows_of_wider_matrices_and_odd_addresses(types, pitch, offset):
    gen = torch.Generator(device=DEV).manual_seed(pitch * 10 + offset)
    rows, c, held = 37, 328, []

    def make(dtype):
        flat = torch.full((rows * (c + pitch) + offset + 5,), -3.0, dtype=dtype, device=DEV)
        v = flat[offset:offset + rows * (c + pitch)].view(rows, c + pitch)[:, :c]
        held.append((flat, v))
        return v
    check_norm(gen, rows, c, "layer", types, make=make)
    for flat, v in held:                       # nothing beside the rows was touched
        rest = torch.ones_like(flat, dtype=torch.bool)
        rest[offset:offset + rows * (c + pitch)].view(rows, c + pitch)[:, :c] = False
        assert (flat[rest] == -3.0).all()


class Join:
    """One join with its reference in 64 bits: gradients by differentiation."""

    def __init__(self, seed, rows, c, post, pre, scale, gate, sigmoid, types, dout=True, eps=1e-5):
        g = torch.Generator(device=DEV).manual_seed(seed)
        rt, bt = TYPES[types]
        self.__dict__.update(rows=rows, c=c, post=post, pre=pre, sigmoid=sigmoid, rt=rt, bt=bt, eps=eps)
        self.x, self.res = rand(g, (rows, c), bt, 1.5, -0.25), rand(g, (rows, c), rt, 2.0)
        self.w, self.b = param(g, c, bool(post)), param(g, c, bool(post))
        self.w2, self.b2 = param(g, c, bool(pre)), param(g, c, bool(pre))
        self.scale = param(g, c) if scale else None
        self.gate = rand(g, (gate, c), bt) if gate else None
        self.dout = rand(g, (rows, c), rt) if dout or not pre else None
        self.dy = rand(g, (rows, c), bt) if pre else None
        e = lambda t, n=rows: torch.full((n, c), 7.0, dtype=t, device=DEV)
        f = lambda on: torch.full((c,), 7.0, device=DEV) if on else None
        self.out, self.y = e(rt), e(bt) if pre else None
        self.stats = torch.full((rows, 2), 7.0, device=DEV) if post else None
        self.stats2 = torch.full((rows, 2), 7.0, device=DEV) if pre else None
        self.dx, self.dres, self.dgate = e(bt), e(rt), e(bt, gate) if gate else None
        self.dw, self.db, self.dscale, self.dw2, self.db2 = f(post), f(post), f(scale), f(pre), f(pre)

    def norms(self):
        return (F.Norm(self.post, self.w, self.b, self.stats, self.eps, self.dw, self.db) if self.post else None,
                F.Norm(self.pre, self.w2, self.b2, self.stats2, self.eps, self.dw2, self.db2) if self.pre else None)

    def forward(self):
        post, pre = self.norms()
        F.residual_forward(self.x, self.res, self.out, post=post, scale=self.scale, gate=self.gate, sigmoid=self.sigmoid, y=self.y, pre=pre)

    def backward(self, **kw):
        post, pre = self.norms()
        F.residual_backward(self.x, self.dout, self.dx, self.dres, post=post, scale=self.scale, dscale=self.dscale, gate=self.gate,
                            dgate=self.dgate, sigmoid=self.sigmoid, out=self.out, dy=self.dy, pre=pre, **kw)

    def check(self):
        self.forward()
        x, res = d(self.x), d(self.res)
        per = self.rows // self.gate.shape[0] if self.gate is not None else 1
        z, n, mean, rstd, mag = norm64(x, self.post, d(self.w), d(self.b), self.eps) if self.post else (x, x, None, 1.0, x.abs())
        g = torch.ones_like(x)
        if self.gate is not None:
            g = (torch.sigmoid(d(self.gate)) if self.sigmoid else d(self.gate)).repeat_interleave(per, 0)
        s = 1.0 if self.scale is None else d(self.scale)
        w = 1.0 if self.w is None else d(self.w)
        h = res + s * g * z
        zmag = mag * (1 + n.abs()) * abs(w) + z.abs()
        hmag = res.abs() + (s * g).abs() * zmag
        close(self.out, h, hmag, what="out")
        if self.pre:
            y, n2, _, rstd2, _ = norm64(h, self.pre, d(self.w2), d(self.b2), self.eps)
            m = hmag * rstd2
            m = m + m.mean(1, keepdim=True) + n2.abs() * (m * (1 + n2.abs())).mean(1, keepdim=True)
            close(self.y, y, m * d(self.w2).abs() + d(self.b2).abs(), 2 * STEPS, "y")
        self.backward()
        # backward from what the forward pass left: the stored out and stats
        dh, mdh = (torch.zeros_like(x), torch.zeros_like(x)) if self.dout is None else (d(self.dout), d(self.dout).abs())
        rowsteps = STEPS + self.rows
        if self.pre:
            st = d(self.stats2)
            o, dy = d(self.out), d(self.dy)
            n2, rs = (o - st[:, :1]) * st[:, 1:], st[:, 1:]
            m2 = (o.abs() + st[:, :1].abs()) * rs
            a = dy * d(self.w2)
            m0 = a.mean(1, keepdim=True) if self.pre == "layer" else 0.0
            dh = dh + rs * (a - m0 - n2 * (a * n2).mean(1, keepdim=True))
            mdh = mdh + rs * (a.abs() + a.abs().mean(1, keepdim=True) + (1 + m2) * (a.abs() * (1 + m2)).mean(1, keepdim=True))
            close(self.dw2, (dy * n2).sum(0), (dy.abs() * m2).sum(0), rowsteps, "dnext_weight")
            close(self.db2, dy.sum(0), dy.abs().sum(0), rowsteps, "dnext_bias")
        close(self.dres, dh, mdh, what="dres")
        if self.post:
            st = d(self.stats)
            n, rs = (x - st[:, :1]) * st[:, 1:], st[:, 1:]
            m1 = (x.abs() + st[:, :1].abs()) * rs
        else:
            n, rs, m1 = x, 1.0, x.abs()
        b = 0.0 if self.b is None else d(self.b)
        z, zm = n * w + b, m1 * abs(w) + abs(b)
        gm = g.abs()
        if self.scale is not None:
            close(self.dscale, (dh * g * z).sum(0), (mdh * gm * zm).sum(0), rowsteps, "dscale")
        if self.gate is not None:
            f = g * (1 - g) if self.sigmoid else 1.0
            dg = (dh * s * z * f).view(-1, per, self.c).sum(1)
            close(self.dgate, dg, (mdh * abs(s) * zm * abs(f)).view(-1, per, self.c).sum(1) , STEPS + per, "dgate")
        e, em = dh * g * s * w, mdh * gm * abs(s) * abs(w)
        if self.post:
            close(self.dw, (dh * g * s * n).sum(0), (mdh * gm * abs(s) * m1).sum(0), rowsteps, "dweight")
            close(self.db, (dh * g * s).sum(0), (mdh * gm * abs(s)).sum(0), rowsteps, "dbias")
            m0 = e.mean(1, keepdim=True) if self.post == "layer" else 0.0
            ref = rs * (e - m0 - n * (e * n).mean(1, keepdim=True))
            close(self.dx, ref, rs * (em + em.mean(1, keepdim=True) + (1 + m1) * (em * (1 + m1)).mean(1, keepdim=True)), 2 * STEPS, "dx")
        else:
            close(self.dx, e, em, what="dx")


COMBOS = list(itertools.product(("layer", "rms", ""), ("layer", "rms", ""), (True, False), ("pixel", "image", ""), (True, False)))


@pytest.mark.parametrize("i", range(0, len(COMBOS), 2))
def test_join_variants(i):
    post, pre, scale, gate, sigmoid = COMBOS[i]
    images, pixels = (6, 11)
    c = (72, 520, 33)[i % 3]
    rows = images * pixels
    Join(i, rows, c, post, pre, scale, {"pixel": rows, "image": images, "": 0}[gate], sigmoid, ("bf16", "mixed", "fp32")[i // 2 % 3]).check()


@pytest.mark.parametrize("rows,c,images", [(1, 1, 1), (1, 2048, 1), (2, 1, 1), (7, 2048, 7), (300, 1024, 3), (4096, 64, 512), (4096, 64, 4096),
                                           (4099, 24, 1), (1000, 16, 500), (40, 4100, 5), (6, 9000, 2), (5, 16384, 1), (4, 16384, 2),
                                           (3000, 8, 1000), (12000, 16, 40)])
@pytest.mark.parametrize("types", ["bf16", "fp32"])
def test_join_sizes_and_images_cut_by_blocks(rows, c, images, types):
    Join(rows + c, rows, c, "layer", "rms", True, images, True, types).check()


# Many rows a slot, so that every ring goes round, for every number of vectors a thread, slots of lanes, warps and several warps,
# blocks of 512 and rows too wide for a ring; whole vectors and single columns
TURNS = [(9000, 8), (9001, 24), (14000, 64), (9001, 192), (6000, 256), (9000, 576), (6001, 1024), (3000, 2048), (1500, 4096), (1300, 4104),
         (900, 6144), (700, 8192), (450, 12288), (450, 16384), (60000, 1), (40000, 3), (9000, 33), (5000, 257), (3001, 1001), (2000, 2050), (900, 4099),
         (500, 8195), (450, 16383)]


@pytest.mark.parametrize("rows,c", TURNS)
@pytest.mark.parametrize("types", list(TYPES))
def test_norm_with_many_rows_a_slot(rows, c, types):
    gen = torch.Generator(device=DEV).manual_seed(rows * 31 + c)
    check_norm(gen, rows, c, ("layer", "rms")[(rows + c) % 2], types)


@pytest.mark.parametrize("rows,c", TURNS)
@pytest.mark.parametrize("gate", ["pixel", "image", ""])
def test_join_with_many_rows_a_slot(rows, c, gate):
    images = next(n for n in (7, 5, 4, 3, 1) if rows % n == 0)
    g = {"pixel": rows, "image": images, "": 0}[gate]
    i = (rows + c) % 3
    Join(rows + c, rows, c, ("layer", "rms", "layer")[i], ("rms", "", "layer")[i], True, g, i != 1, ("bf16", "mixed", "fp32")[(rows // 100 + c) % 3]).check()


@pytest.mark.parametrize("images,pixels,c", [(1, 60000, 8), (1, 50001, 24), (2, 20000, 32), (3, 11111, 64), (7, 4000, 5), (1, 9000, 130), (5, 700, 16),
                                             (900, 40, 8), (2, 37, 16), (11, 333, 100)])
@pytest.mark.parametrize("types", ["bf16", "fp32"])
def test_join_with_images_of_many_slots(images, pixels, c, types):
    Join(images + c, images * pixels, c, "layer", "rms", True, images, True, types).check()
    Join(images + c, images * pixels, c, "", "", False, images, False, types).check()


def test_join_without_dout():
    Join(5, 90, 136, "rms", "layer", True, 9, False, "bf16", dout=False).check()


def test_results_repeat_bit_for_bit():
    j = Join(3, 3000, 248, "layer", "layer", True, 30, True, "bf16")
    names = ("out", "y", "dx", "dres", "dgate", "dscale", "dw", "db", "dw2", "db2")
    first = None
    for _ in range(3):
        j.forward()
        j.backward()
        now = [getattr(j, k).clone() for k in names]
        assert first is None or all(torch.equal(a, b) for a, b in zip(first, now))
        first = now


@pytest.mark.parametrize("types", list(TYPES))
def test_outputs_in_the_place_of_inputs(types):
    a, b = Join(11, 77, 264, "layer", "rms", True, 77, True, types), Join(11, 77, 264, "layer", "rms", True, 77, True, types)
    a.forward()
    a.backward()
    b.out = b.res
    b.forward()
    b.dres, b.dgate, b.dx = b.dout, b.gate, b.dy
    b.backward()
    for k in ("out", "y", "dres", "dx", "dgate", "dscale", "dw", "db", "dw2", "db2"):
        assert torch.equal(getattr(a, k), getattr(b, k)), k
    if types != "mixed":                       # every pairing of an output with an input of its type
        c = Join(11, 77, 264, "layer", "rms", True, 77, True, types)
        c.forward()
        c.dres, c.dx, c.dgate = c.x, c.dout, c.out
        c.backward()
        for k in ("dres", "dx", "dgate", "dscale", "dw", "db", "dw2", "db2"):
            assert torch.equal(getattr(a, k), getattr(c, k)), k


@pytest.mark.parametrize("c", [4101, 8021, 8968, 12289, 16384])
@pytest.mark.parametrize("types,gate", [("bf16", 20), ("mixed", 160), ("fp32", 160), ("fp32", 0)])
def test_outputs_in_the_place_of_inputs_of_wide_rows(c, types, gate):
    a, b = Join(c, 160, c, "layer", "rms", True, gate, True, types), Join(c, 160, c, "layer", "rms", True, gate, True, types)
    a.forward()
    a.backward()
    b.out = b.res
    b.forward()
    b.dres, b.dgate, b.dx = b.dout, b.gate, b.dy
    b.backward()
    for k in ("out", "y", "dres", "dx", "dgate", "dscale", "dw", "db", "dw2", "db2"):
        assert (getattr(a, k) is None and getattr(b, k) is None) or torch.equal(getattr(a, k), getattr(b, k)), k


@pytest.mark.parametrize("c", [9000, 9001])
def test_wide_rows_repeat_in_a_captured_graph(c):
    j = Join(c, 300, c, "layer", "layer", True, 30, True, "bf16")
    j.forward()
    j.backward()
    names = ("out", "y", "dx", "dres", "dgate", "dscale", "dw", "db", "dw2", "db2")
    first = {k: getattr(j, k).clone() for k in names}
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        j.forward()
        j.backward()
    for k in names:
        getattr(j, k).zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(first[k], getattr(j, k)) for k in names)


def test_large_means_small_spreads_and_constant_rows():
    for kind in ("layer", "rms"):
        x = torch.randn(8, 640, device=DEV) * 1e-2 + 100.0
        x[3] = 5.0
        x[4] = 0.0
        y, st = torch.empty_like(x), torch.empty(8, 2, device=DEV)
        F.norm_forward(x, y, F.Norm(kind, None, None, st, 1e-5))
        ref, n, mean, rstd, mag = norm64(x.double(), kind, None, None, 1e-5)
        close(y, ref, mag * (1 + n.abs()), what=kind)
        assert (y[4] == 0).all()


def test_a_row_that_is_not_finite_stays_alone():
    j = Join(2, 40, 96, "layer", "layer", True, 40, True, "fp32")
    j.x[7, 5], j.res[9, 0] = float("inf"), float("nan")
    j.forward()
    ok = torch.ones(40, dtype=torch.bool, device=DEV)
    ok[[7, 9]] = False
    assert torch.isfinite(j.out[ok]).all() and torch.isfinite(j.y[ok]).all()
    assert torch.isnan(j.y[7]).all() and torch.isnan(j.y[9]).all() and torch.isnan(j.out[7]).all()
    assert torch.isfinite(j.out[9, 1:]).all()
    j.backward()
    assert torch.isfinite(j.dres[ok]).all() and torch.isfinite(j.dx[ok]).all() and torch.isfinite(j.dgate[ok]).all()


def test_gates_far_out():
    j = Join(4, 12, 64, "rms", "", False, 12, True, "fp32")
    j.gate[:, ::2], j.gate[:, 1::2] = -2e4, 2e4
    j.check()


@pytest.mark.parametrize("gate", [60, 12])
@pytest.mark.parametrize("types", ["mixed", "fp32"])
def test_slope_of_gates_that_are_nearly_open(gate, types):
    j = Join(8, 60, 200, "layer", "rms", True, gate, True, types)
    j.gate.copy_(torch.linspace(-24, 24, gate * 200, device=DEV).view(gate, 200))
    j.check()


def test_no_rows():
    j = Join(1, 0, 48, "layer", "layer", True, 0, True, "bf16")
    j.forward()
    j.backward()
    for k in ("dscale", "dw", "db", "dw2", "db2"):
        assert (getattr(j, k) == 0).all(), k


def test_gradients_against_differences():
    """Along a random direction of all inputs: (L(+t) - L(-t)) / 2t in fp32.  The difference's own error is t^2 times third
    derivatives (bounded by the halved step) plus the roundings of L over t."""
    j = Join(21, 30, 40, "layer", "rms", True, 6, True, "fp32")
    keys = ("x", "res", "w", "b", "scale", "gate", "w2", "b2")
    gen = torch.Generator(device=DEV).manual_seed(9)
    dirs = {k: torch.randn(getattr(j, k).shape, generator=gen, device=DEV) for k in keys}
    base = {k: getattr(j, k).clone() for k in keys}

    def loss(t):
        for k in keys:
            getattr(j, k).copy_(base[k] + t * dirs[k])
        j.forward()
        return (j.out.double() * j.dout.double()).sum().item() + (j.y.double() * j.dy.double()).sum().item()
    diffs = [(loss(t) - loss(-t)) / (2 * t) for t in (8e-3, 4e-3)]
    loss(0.0)
    j.backward()
    grads = dict(x=j.dx, res=j.dres, w=j.dw, b=j.db, scale=j.dscale, gate=j.dgate, w2=j.dw2, b2=j.db2)
    slope = sum((grads[k].double() * dirs[k].double()).sum().item() for k in keys)
    size = (j.out.double() * j.dout.double()).abs().sum().item() + (j.y.double() * j.dy.double()).abs().sum().item()
    tol = 2 * abs(diffs[0] - diffs[1]) + 2 * STEPS * U * size / 4e-3
    assert abs(slope - diffs[1]) <= tol, (slope, diffs, tol)


def test_calls_in_a_graph_and_on_another_stream_with_their_own_workspaces():
    a, b = Join(31, 2000, 136, "layer", "rms", True, 20, True, "bf16"), Join(32, 2000, 136, "layer", "rms", True, 20, True, "bf16")
    want = []
    for j in (a, b):
        j.forward()
        j.backward()
        want.append([t.clone() for t in (j.dx, j.dres, j.dgate, j.dscale, j.dw, j.db, j.dw2, j.db2)])
    graphs = []
    for j in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            j.forward()
            j.backward()
        graphs.append(g)
        for t in (j.dx, j.dres, j.dgate, j.dscale, j.dw, j.db, j.dw2, j.db2):
            t.fill_(7.0)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for j, w in zip((a, b), want):
        assert all(torch.equal(t, v) for t, v in zip((j.dx, j.dres, j.dgate, j.dscale, j.dw, j.db, j.dw2, j.db2), w))


def test_a_workspace_of_the_callers_own():
    j = Join(8, 1500, 64, "layer", "layer", True, 15, True, "bf16")
    j.forward()
    j.backward()
    want = [t.clone() for t in (j.dx, j.dgate, j.dscale, j.dw2)]
    n = F.norm_work(1500, 64, 15, join=True, pre=True)
    assert n > 0
    work = torch.full((n + 8,), 7.0, device=DEV)
    j.backward(work=work[:n])
    assert all(torch.equal(t, v) for t, v in zip((j.dx, j.dgate, j.dscale, j.dw2), want)) and (work[n:] == 7.0).all()
    with pytest.raises(ValueError, match="work"):
        j.backward(work=work[:n - 1])


def test_refusals():
    x, y = torch.zeros(6, 16, dtype=BF, device=DEV), torch.zeros(6, 16, dtype=BF, device=DEV)
    st, v = torch.zeros(6, 2, device=DEV), torch.zeros(16, device=DEV)
    norm = F.Norm("layer", v, v, st)
    with pytest.raises(ValueError, match="unknown norm"):
        F.Norm("batch")
    with pytest.raises(ValueError, match="eps"):
        F.Norm("rms", eps=-1.0)
    with pytest.raises(ValueError, match="types"):
        F.norm_forward(x, y.float(), norm)
    with pytest.raises(ValueError, match="types"):
        F.norm_forward(x.half(), y.half(), norm)
    with pytest.raises(ValueError, match="\\[6, 16\\]"):
        F.norm_forward(x, y[:5], norm)
    with pytest.raises(ValueError, match="contiguous"):
        F.norm_forward(x.t().contiguous().t(), y, norm)
    with pytest.raises(ValueError, match="weight"):
        F.norm_forward(x, y, F.Norm("layer", v[:8], v, st))
    with pytest.raises(ValueError, match="stats"):
        F.norm_forward(x, y, F.Norm("layer", v, v, st[:3]))
    with pytest.raises(ValueError, match="stats"):
        F.norm_backward(x, y, y.clone(), F.Norm("layer", v, v))
    with pytest.raises(ValueError, match="16384"):
        F.norm_forward(torch.zeros(1, 16385, dtype=BF, device=DEV), torch.zeros(1, 16385, dtype=BF, device=DEV), F.Norm("rms"))
    with pytest.raises(ValueError, match="16384"):
        F.norm_forward(torch.zeros(3, 0, dtype=BF, device=DEV), torch.zeros(3, 0, dtype=BF, device=DEV), F.Norm("rms"))
    with pytest.raises(ValueError, match="overlaps"):
        wide = torch.zeros(7, 16, dtype=BF, device=DEV)
        F.norm_forward(wide[:6], wide[1:], norm)
    with pytest.raises(ValueError, match="overlaps"):
        F.residual_forward(x, x, y, y=y, pre=norm)
    with pytest.raises(ValueError, match="overlaps"):      # a gate per image cannot be written over by the rows
        F.residual_forward(x, y.clone(), y, gate=y[:2])
    with pytest.raises(ValueError, match="divide"):
        F.residual_forward(x, x, y, gate=torch.zeros(4, 16, dtype=BF, device=DEV))
    with pytest.raises(ValueError, match="pre"):
        F.residual_forward(x, x, y, pre=norm)
    with pytest.raises(ValueError, match="gate"):
        F.residual_backward(x, x, y, y.clone(), dgate=y.clone())
    with pytest.raises(RuntimeError):                       # rows of an output on top of one another
        F.norm_forward(x, y[:1].expand(6, 16), norm)
    with pytest.raises(ValueError, match="cpu"):
        F.norm_forward(x, y.cpu(), norm)
    with pytest.raises(ValueError, match="cpu"):
        F.norm_forward(x.cpu(), y.cpu(), norm)
    wide = torch.zeros(6, 32, dtype=BF, device=DEV)         # two ranges of columns of one matrix share nothing
    F.norm_forward(wide[:, :16], wide[:, 16:], F.Norm("layer"))


def test_refused_statistics_workspaces_and_gradients():
    x, y = torch.zeros(6, 16, dtype=BF, device=DEV), torch.zeros(6, 16, dtype=BF, device=DEV)
    st, v = torch.zeros(13, device=DEV), torch.zeros(40, device=DEV)
    with pytest.raises(ValueError, match="8 bytes"):
        F.norm_forward(x, y, F.Norm("layer", stats=st[1:].view(6, 2)))
    good = st[:12].view(6, 2)
    with pytest.raises(ValueError, match="overlaps"):
        F.norm_backward(x, y, x.clone(), F.Norm("layer", None, None, good, dweight=v[:16], dbias=v[8:24]))
    with pytest.raises(ValueError, match="overlaps"):
        F.norm_backward(x, y, x.clone(), F.Norm("layer", v[4:20], None, good, dweight=v[:16]))
    rows = torch.zeros(3000, 16, dtype=BF, device=DEV)
    n = F.norm_work(3000, 16)
    with pytest.raises(ValueError, match="8 bytes"):
        F.norm_backward(rows, rows.clone(), rows.clone(), F.Norm("layer", stats=torch.zeros(3000, 2, device=DEV)),
                        work=torch.zeros(n + 1, device=DEV)[1:])
    with pytest.raises(ValueError, match="work"):
        F.norm_backward(rows, rows.clone(), rows.clone(), F.Norm("layer", stats=torch.zeros(3000, 2, device=DEV)),
                        work=torch.zeros(n - 1, device=DEV))
    a, b = torch.full((48,), 3.0, device=DEV), torch.randn(6, 16, device=DEV).to(BF)      # gradients side by side in one buffer
    F.norm_forward(b, y, F.Norm("layer", stats=good))
    F.norm_backward(b, b, x, F.Norm("layer", stats=good, dweight=a[:16], dbias=a[16:32]))
    assert (a[32:] == 3.0).all() and torch.isfinite(a).all() and (a[:16] != 3.0).all()
