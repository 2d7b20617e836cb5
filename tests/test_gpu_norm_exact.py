"""Sums of the norms' and joins' backward pass on whole numbers, where fp32 adds without rounding: every sum is compared for
equality, so a row, a slot's share or an image's share that is lost or counted twice shows in any of them.

Values are whole numbers up to 3, statistics are given as they are (means are whole, 1/std is 1/2, 1 or 2), parameters are powers of two.
A term of a sum is then a multiple of 1/4 below 2^7 of a random sign: a sum of the 600000 at the most has a standard deviation below
2^14 and stays a multiple of 1/4 below 2^17 with all of its parts, where fp32 has bits down to 2^-7."""
import pytest
import torch

from geeps_b200.ops import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
TYPES = {"bf16": (BF, BF), "mixed": (F32, BF), "fp32": (F32, F32)}


def whole(gen, shape, dtype, most=3):
    return torch.randint(-most, most + 1, shape, generator=gen, device=DEV).to(dtype)


def power(gen, n):
    return 2.0 ** torch.randint(-1, 2, (n,), generator=gen, device=DEV).float()


def some_stats(gen, rows):
    return torch.stack([torch.randint(-1, 2, (rows,), generator=gen, device=DEV).float(), power(gen, rows)], 1)


def normalised(x, stats):
    return (x.double() - stats[:, :1].double()) * stats[:, 1:].double()


def same(got, want, what):
    """Equal, where `got` is rounded once to its type."""
    bad = got != want.to(got.dtype)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} differ, by up to {(got.double() - want).abs().max().item()}"


def check_norm(rows, c, types, kind="rms"):
    gen = torch.Generator(device=DEV).manual_seed(rows * 31 + c)
    rt, bt = TYPES[types]
    x, dy, stats = whole(gen, (rows, c), rt), whole(gen, (rows, c), bt), some_stats(gen, rows)
    dx, dw, db = torch.empty(rows, c, dtype=rt, device=DEV), torch.full((c,), 7.0, device=DEV), torch.full((c,), 7.0, device=DEV)
    F.norm_backward(x, dy, dx, F.Norm(kind, power(gen, c), None, stats, dweight=dw, dbias=db))
    same(dw, (dy.double() * normalised(x, stats)).sum(0), "dweight")
    same(db, dy.double().sum(0), "dbias")


def check_join(images, pixels, c, types, gate="image", post="rms", pre="", most=3):
    """Without `pre` the gradient of the sum is dout itself, so the branch's sums are exact; with it only the sums of the norm
    behind are.  dgate in bf16 is the exact sum rounded once."""
    rows = images * pixels
    gen = torch.Generator(device=DEV).manual_seed(rows * 31 + c)
    rt, bt = TYPES[types]
    x, dout = whole(gen, (rows, c), bt, most), whole(gen, (rows, c), rt, most)
    stats = some_stats(gen, rows)
    w, s = power(gen, c), power(gen, c)
    gate = whole(gen, ({"image": images, "pixel": rows}[gate], c), bt, 2) if gate else None
    e, f = (lambda t, n=rows: torch.full((n, c), 7.0, dtype=t, device=DEV)), (lambda: torch.full((c,), 7.0, device=DEV))
    dx, dres, dgate = e(bt), e(rt), None if gate is None else e(bt, gate.shape[0])
    dscale, dw, db, dw2, db2 = f(), f(), f(), f(), f()
    kw = {}
    if pre:
        out, dy, stats2 = whole(gen, (rows, c), rt), whole(gen, (rows, c), bt), some_stats(gen, rows)
        kw = dict(out=out, dy=dy, pre=F.Norm(pre, power(gen, c), None, stats2, dweight=dw2, dbias=db2))
    F.residual_backward(x, dout, dx, dres, post=F.Norm(post, w, None, stats, dweight=dw, dbias=db) if post else None, scale=s, dscale=dscale,
                        gate=gate, dgate=dgate, **kw)
    if pre:
        same(dw2, (dy.double() * normalised(out, stats2)).sum(0), "dnext_weight")
        same(db2, dy.double().sum(0), "dnext_bias")
        return
    n = normalised(x, stats) if post else x.double()
    z = n * w.double() if post else n
    g = 1.0 if gate is None else gate.double().repeat_interleave(rows // gate.shape[0], 0)
    dh = dout.double()
    same(dres, dh, "dres")
    same(dscale, (dh * g * z).sum(0), "dscale")
    if post:
        same(dw, (dh * g * s.double() * n).sum(0), "dweight")
        same(db, (dh * g * s.double()).sum(0), "dbias")
    else:
        same(dx, dh * g * s.double(), "dx")
    if gate is not None:
        same(dgate, (dh * s.double() * z).view(gate.shape[0], -1, c).sum(1), "dgate")


# more images than slots, and more slots than a grid has blocks along an axis: narrow rows of single columns have 75776 slots
@pytest.mark.parametrize("images,pixels,c", [(70000, 2, 4), (100000, 2, 3), (75776, 2, 1), (75775, 3, 7), (65532, 5, 5), (200000, 3, 1)])
@pytest.mark.parametrize("types", list(TYPES))
def test_gates_of_many_images_of_narrow_rows(images, pixels, c, types):
    check_join(images, pixels, c, types)


IMAGES = [(1, 60000, 8), (1, 50001, 24), (2, 20000, 32), (3, 11111, 64), (7, 4000, 5), (1, 9000, 130), (5, 700, 16), (900, 40, 8), (2, 37, 16),
          (11, 333, 100), (512, 8, 64), (3000, 4, 8), (300, 40, 16), (5, 8, 4100), (3, 2, 9000), (2, 2, 16384), (1, 1, 8), (1, 30000, 1), (60, 100, 520)]


@pytest.mark.parametrize("images,pixels,c", IMAGES)
@pytest.mark.parametrize("types", list(TYPES))
def test_gates_of_images(images, pixels, c, types):
    check_join(images, pixels, c, types, post="rms" if c % 3 else "")


ROWS = [(9000, 8), (9001, 24), (14000, 64), (9001, 192), (6000, 256), (9000, 576), (6001, 1024), (3000, 2048), (1500, 4096), (1300, 4104), (900, 6144), (700, 8192),
        (450, 12288), (450, 16384), (60000, 1), (40000, 3), (9000, 33), (5000, 257), (3001, 1001), (2000, 2050), (900, 4099), (500, 8195), (450, 16383), (1, 1), (3, 40)]


@pytest.mark.parametrize("rows,c", ROWS)
@pytest.mark.parametrize("types", list(TYPES))
def test_column_sums(rows, c, types):
    check_norm(rows, c, types)
    check_join(rows, 1, c, types, gate="")
    check_join(rows, 1, c, types, gate="pixel", pre="rms")


@pytest.mark.parametrize("rows,c", ROWS[::2])
def test_column_sums_with_a_gate_for_every_pixel(rows, c):
    check_join(rows, 1, c, "bf16", gate="pixel")
    check_join(rows, 1, c, "fp32", gate="pixel", post="layer")
    check_join(rows, 1, c, "mixed", gate="", pre="layer")


def no_rows(types, gate_rows, dgate, c=40):
    rt, bt = TYPES[types]
    e = lambda t, n=0: torch.empty(n, c, dtype=t, device=DEV)
    f = lambda: torch.full((c,), 7.0, device=DEV)
    gate = torch.ones(gate_rows, c, dtype=bt, device=DEV)
    sums = [f() for _ in range(5)]
    stats = torch.empty(0, 2, device=DEV)
    F.residual_forward(e(bt), e(rt), e(rt), post=F.Norm("layer", stats=stats), gate=gate, y=e(bt), pre=F.Norm("rms", stats=stats))
    F.residual_backward(e(bt), e(rt), e(bt), e(rt), post=F.Norm("layer", stats=stats, dweight=sums[0], dbias=sums[1]), scale=f(), dscale=sums[2], gate=gate,
                        dgate=dgate, sigmoid=True, out=e(rt), dy=e(bt), pre=F.Norm("rms", stats=stats, dweight=sums[3], dbias=sums[4]))
    assert all((s == 0).all() for s in sums)


@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("gate_rows", [1, 4, 1000])
def test_images_without_rows_have_a_gradient_of_zero(types, gate_rows):
    bt = TYPES[types][1]
    dgate = torch.full((gate_rows, 40), 7.0, dtype=bt, device=DEV)
    no_rows(types, gate_rows, dgate)
    assert (dgate == 0).all()
    no_rows(types, gate_rows, None)
    wide = torch.full((gate_rows + 1, 61), 7.0, dtype=bt, device=DEV)      # rows of a wider matrix, and nothing beside them
    no_rows(types, gate_rows, wide[:gate_rows, 3:43])
    assert (wide[:gate_rows, 3:43] == 0).all()
    wide[:gate_rows, 3:43] = 7.0
    assert (wide == 7.0).all()


@pytest.mark.parametrize("types", ["bf16", "fp32"])
@pytest.mark.parametrize("c,images", [(64, 2), (32, 5), (16, 3), (64, 40)])
def test_a_row_that_is_not_finite_leaves_other_images_alone(types, c, images):
    """Slots that share a warp take the same number of turns, and some have no row in the last: what they compute there must not
    come from a row of an image before.  A row without a finite value in every tenth place of all images but the last; only the last's
    gradient is compared, and all of it."""
    pixels = 2000
    for shift in range(0, 8):
        rows = images * pixels + shift * images
        per = rows // images
        gen = torch.Generator(device=DEV).manual_seed(shift)
        rt, bt = TYPES[types]
        x, dout, stats, gate = whole(gen, (rows, c), bt), whole(gen, (rows, c), rt), some_stats(gen, rows), whole(gen, (images, c), bt, 2)
        last = rows - per
        x[:last:10], stats[:last:10] = float("nan"), float("nan")
        x[5:last:10], stats[5:last:10] = float("inf"), float("inf")
        s, dgate = power(gen, c), torch.full((images, c), 7.0, dtype=bt, device=DEV)
        dx, dres = torch.empty_like(x), torch.empty_like(dout)
        F.residual_backward(x, dout, dx, dres, post=F.Norm("layer", None, None, stats), scale=s, gate=gate, dgate=dgate)
        same(dres, dout.double(), "dres")
        same(dgate[-1], (dout.double() * s.double() * normalised(x, stats))[last:].sum(0), f"dgate of the last image, {rows} rows")
