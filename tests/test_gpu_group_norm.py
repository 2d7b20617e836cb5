"""Group norm with its activation, forward and backward, against 64-bit arithmetic."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
EPS = 1e-5
BF, F32 = torch.bfloat16, torch.float32
TYPES = {"bf16": (BF, BF), "mixed": (F32, BF), "fp32": (F32, F32)}

# images, pixels, channels, groups: single values, odd widths, groups across vectors, wide groups, many small images, images cut over
# many blocks in two launches
SIZES = [(1, 1, 1, 1), (3, 1, 8, 2), (2, 5, 7, 7), (2, 3, 24, 8), (1, 196, 576, 32), (5, 49, 1003, 17), (4, 64, 96, 32), (3, 100, 256, 1),
         (700, 2, 16, 4), (1, 20000, 32, 4), (2, 3000, 136, 17), (1, 33, 4096, 1), (1, 9, 16384, 1), (2, 7, 16383, 3), (9, 3136, 64, 32),
         (1, 1, 16384, 16384), (1, 5000, 9, 3)]


def made(images, pixels, c, groups, types, seed, offset=0.0, wider=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    xt, yt = TYPES[types]
    p = images * pixels
    x = (torch.randn(p, c, generator=gen, device=DEV) * (0.5 + torch.rand(c, generator=gen, device=DEV)) + offset).to(xt)
    dy = torch.randn(p, c, generator=gen, device=DEV).to(yt)
    if wider:
        x, dy = (torch.nn.functional.pad(t, (0, wider))[:, :c] for t in (x, dy))
    return x, dy, 1 + 0.3 * torch.randn(c, generator=gen, device=DEV), 0.3 * torch.randn(c, generator=gen, device=DEV)


def statistics(x, images, groups):
    v = x.double().view(images, -1, groups, x.shape[1] // groups)
    var, mean = torch.var_mean(v, (1, 3), unbiased=False)
    return torch.stack([mean, (var + EPS) ** -0.5], 2)


def spread(s, images, groups, c):
    """[images, groups] as [images, 1, C]."""
    return s.repeat_interleave(c // groups, 1).view(images, 1, c)


def act64(z, act):
    return torch.relu(z) if act == "relu" else z * torch.sigmoid(z) if act else z


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("act", [None, "relu", "silu"])
def test_forward(size, types, act):
    from geeps_b200.ops import functional as F
    images, pixels, c, groups = size
    x, _, w, b = made(*size, types, 1, offset=3.0)
    y = torch.full(x.shape, float("nan"), dtype=TYPES[types][1], device=DEV)
    stats = torch.full((images, groups, 2), float("nan"), device=DEV)
    F.group_norm_forward(x, y, images, F.GroupNorm(groups, w, b, stats, EPS, act))
    want = statistics(x, images, groups)
    check_forward(x, y, stats, want, w, b, images, groups, act)


def check_forward(x, y, stats, want, w, b, images, groups, act):
    c = x.shape[1]
    # a mean: at most 32 additions of differences in a part, then joins of parts, threads and blocks, 64 roundings in all of what is
    # at most the largest value; squared differences likewise, of the standard deviation
    top = x.double().abs().max()
    std = 1 / want[..., 1]
    dmean = 64 * 2.0 ** -24 * top + 1e-30
    drel = 128 * 2.0 ** -24 + dmean / std
    assert ((stats[..., 0].double() - want[..., 0]).abs() <= dmean).all()
    assert ((stats[..., 1].double() / want[..., 1] - 1).abs() <= drel).all()
    n = (x.double().view(images, -1, c) - spread(want[..., 0], images, groups, c)) * spread(want[..., 1], images, groups, c)
    z = n * w.double() + b.double()
    out = act64(z, act).view_as(x)
    # z: the statistics' errors and three roundings; an activation's slope is at most 1.1, SiLU's exponential and quotient 2^-20 of it
    dz = w.double().abs() * (n.abs() * (spread(drel, images, groups, c) + 2.0 ** -22) + spread(dmean / std, images, groups, c)) + 2.0 ** -23 * (z.abs() + b.double().abs())
    tol = 1.1 * dz.view_as(x) + (2.0 ** -20 if act == "silu" else 0.0) * out.abs() + torch.finfo(y.dtype).eps / 2 * out.abs() + 1e-30
    assert ((y.double() - out).abs() <= tol * 1.01).all()


def gradients(x, dy, stats, w, b, images, groups, act):
    """From the statistics that the kernel is given.  ReLU: where z, rounded to fp32 after each operation, is above zero."""
    c = x.shape[1]
    mean, rstd = (spread(stats[..., i], images, groups, c) for i in range(2))
    z32 = (x.float().view(images, -1, c) - mean) * rstd * w + b
    n = (x.double().view(images, -1, c) - mean.double()) * rstd.double()
    dz = dy.double().view_as(n)
    if act == "relu":
        dz = dz * (z32 > 0)
    elif act == "silu":
        z = n * w.double() + b.double()
        g = torch.sigmoid(z)
        dz = dz * g * (1 + z * (1 - g))
    a = (dz * w.double()).view(images, -1, groups, c // groups)
    ng = n.view_as(a)
    ca, cb = a.mean((1, 3), keepdim=True), (a * ng).mean((1, 3), keepdim=True)
    dx = (a - ca - ng * cb).view_as(n) * rstd.double()
    return n, dz, dx, (dz * n).sum((0, 1)), dz.sum((0, 1))


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("act", [None, "relu", "silu"])
def test_backward(size, types, act):
    from geeps_b200.ops import functional as F
    images, pixels, c, groups = size
    x, dy, w, b = made(*size, types, 2)
    stats = statistics(x, images, groups).float()
    dx = torch.full_like(x, float("nan"))
    dw, db = torch.full((c,), float("nan"), device=DEV), torch.full((c,), float("nan"), device=DEV)
    F.group_norm_backward(x, dy, dx, images, F.GroupNorm(groups, w, b, stats, EPS, act, dw, db))
    check_backward(x, dy, dx, dw, db, stats, w, b, images, groups, act)


def check_backward(x, dy, dx, dw, db, stats, w, b, images, groups, act):
    c, pixels = x.shape[1], x.shape[0] // images
    n, dz, want, want_w, want_b = gradients(x, dy, stats, w, b, images, groups, act)
    # dz and n: 2^-22 each (SiLU's slope 2^-19).  A sum of k values: k + 300 additions of 2^-24 of the magnitudes, where k is a
    # thread's pixels and the rest threads, channels and blocks
    slope = 2.0 ** -19 if act == "silu" else 2.0 ** -22
    adds = (min(pixels, 512) + 300 + c // groups / 32) * 2.0 ** -24 + slope + 2.0 ** -22
    mags = dz.abs() if act != "silu" else dy.double().abs().view_as(dz) * 1.1
    assert ((db.double() - want_b).abs() <= (adds + images * 2.0 ** -24) * mags.sum((0, 1)) + 1e-30).all()
    assert ((dw.double() - want_w).abs() <= (adds + images * 2.0 ** -24) * (mags * n.abs()).sum((0, 1)) + 1e-30).all()
    a = (mags * w.double().abs()).view(images, -1, groups, c // groups)
    ng = n.abs().view_as(a)
    rstd = spread(stats[..., 1].double(), images, groups, c)
    size = (a + a.mean((1, 3), keepdim=True) + ng * (a * ng).mean((1, 3), keepdim=True)).view_as(n) * rstd
    tol = (adds + 2.0 ** -20) * size.view_as(x) + torch.finfo(dx.dtype).eps / 2 * want.view_as(x).abs() + 1e-30
    assert ((dx.double() - want.view_as(x)).abs() <= tol * 1.01).all()
