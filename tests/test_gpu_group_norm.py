"""Group norm with its activation, forward and backward, against 64-bit arithmetic."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
EPS = 1e-5
BF, F32 = torch.bfloat16, torch.float32
TYPES = {"bf16": (BF, BF), "mixed": (F32, BF), "fp32": (F32, F32)}

# images, pixels, channels, groups: single values, odd widths, groups across vectors, wide groups, many small images, images cut over
# many blocks in two launches, many images with some pixels in registers (bf16, backward)
SIZES = [(1, 1, 1, 1), (3, 1, 8, 2), (2, 5, 7, 7), (2, 3, 24, 8), (1, 196, 576, 32), (5, 49, 1003, 17), (4, 64, 96, 32), (3, 100, 256, 1),
         (700, 2, 16, 4), (1, 20000, 32, 4), (2, 3000, 136, 17), (1, 33, 4096, 1), (1, 9, 16384, 1), (2, 7, 16383, 3), (9, 3136, 64, 32),
         (1, 1, 16384, 16384), (1, 5000, 9, 3), (460, 196, 72, 4), (500, 190, 72, 4)]


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


@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("wider,shift", [(8, 0), (3, 0), (5, 3)])
def test_rows_of_wider_matrices_at_any_address(types, wider, shift):
    """Pitches and addresses that allow vectors and such that do not; what lies beside the rows stays as it was."""
    from geeps_b200.ops import functional as F
    images, pixels, c, groups = 3, 50, 64, 8
    x, dy, w, b = made(images, pixels, c, groups, types, 3)

    def inside(t):
        full = torch.full((t.shape[0], c + wider + 3), 9.0, dtype=t.dtype, device=DEV).view(-1)
        full = full[shift:shift + t.shape[0] * (c + wider)].view(t.shape[0], c + wider)
        full[:, :c] = t
        return full
    xf, dyf = inside(x), inside(dy)
    yf, dxf = inside(torch.zeros_like(dy)), inside(torch.zeros_like(x))
    stats = torch.empty(images, groups, 2, device=DEV)
    F.group_norm_forward(xf[:, :c], yf[:, :c], images, F.GroupNorm(groups, w, b, stats, EPS, "silu"))
    check_forward(x, yf[:, :c], stats, statistics(x, images, groups), w, b, images, groups, "silu")
    dw, db = torch.empty(c, device=DEV), torch.empty(c, device=DEV)
    F.group_norm_backward(xf[:, :c], dyf[:, :c], dxf[:, :c], images, F.GroupNorm(groups, w, b, stats, EPS, "relu", dw, db))
    check_backward(x, dy, dxf[:, :c], dw, db, stats, w, b, images, groups, "relu")
    for t in (xf, dyf, yf, dxf):
        assert (t[:, c:] == 9.0).all()


def test_in_place_without_parameters_and_into_a_slice_of_the_same_rows():
    from geeps_b200.ops import functional as F
    images, pixels, c, groups = 4, 30, 48, 6
    x, dy, _, _ = made(images, pixels, c, groups, "bf16", 4)
    one, zero = torch.ones(c, device=DEV), torch.zeros(c, device=DEV)
    stats = statistics(x, images, groups).float()
    y, dx = x.clone(), dy.clone()
    F.group_norm_forward(y, y, images, F.GroupNorm(groups, act="relu"))
    check_forward(x, y, stats, statistics(x, images, groups), one, zero, images, groups, "relu")
    F.group_norm_backward(x, dx, dx, images, F.GroupNorm(groups, stats=stats, act="silu"))
    dw, db = torch.empty(c, device=DEV), torch.empty(c, device=DEV)
    other = torch.empty_like(x)
    F.group_norm_backward(x, dy, other, images, F.GroupNorm(groups, stats=stats, act="silu", dweight=dw, dbias=db))
    check_backward(x, dy, other, dw, db, stats, one, zero, images, groups, "silu")
    assert torch.equal(dx, other)
    wide = torch.cat([x, torch.full_like(x, 5.0)], 1)
    F.group_norm_forward(wide[:, :c], wide[:, c:], images, F.GroupNorm(groups, act="relu"))
    assert torch.equal(wide[:, :c], x) and torch.equal(wide[:, c:], y)


@pytest.mark.parametrize("size", [(2, 40, 64, 8), (1, 20000, 32, 4), (3, 11, 21, 3)], ids=str)
def test_a_mean_far_from_zero_and_groups_without_spread(size):
    """The variance does not lose what the mean has: 1000 standard deviations from zero in fp32 (a value then has 14 bits below the
    deviation: the bound of check_forward goes by the largest value)."""
    from geeps_b200.ops import functional as F
    images, pixels, c, groups = size
    x, _, w, b = made(*size, "fp32", 5)
    x = x + 1000.0
    x[:pixels, : c // groups] = 3.25                                   # a group that is all one value
    y, stats = torch.empty_like(x), torch.empty(images, groups, 2, device=DEV)
    F.group_norm_forward(x, y, images, F.GroupNorm(groups, w, b, stats, EPS, None))
    want = statistics(x, images, groups)
    assert stats[0, 0].tolist() == [3.25, torch.tensor(EPS).rsqrt().item()] or abs(stats[0, 0, 1].item() * EPS ** 0.5 - 1) < 1e-6
    check_forward(x, y, stats, want, w, b, images, groups, None)


def test_values_that_are_not_finite_stay_in_their_group():
    from geeps_b200.ops import functional as F
    images, pixels, c, groups = 2, 9, 32, 4
    x, dy, w, b = made(images, pixels, c, groups, "bf16", 6)
    clean, stats = torch.empty_like(x), torch.empty(images, groups, 2, device=DEV)
    F.group_norm_forward(x, clean, images, F.GroupNorm(groups, w, b, stats, EPS, "relu"))
    for bad in (float("nan"), float("inf"), -float("inf")):
        z = x.clone()
        z[pixels + 2, 9] = bad                                           # image 1, group 1
        y = torch.empty_like(x)
        F.group_norm_forward(z, y, images, F.GroupNorm(groups, w, b, None, EPS, "relu"))
        hit = torch.zeros_like(x, dtype=torch.bool)
        hit[pixels:, 8:16] = True
        assert y[pixels:, 8:16].isnan().all() and torch.equal(y[~hit], clean[~hit])
        d = dy.clone()
        d[pixels + 2, 9] = bad
        dx = torch.empty_like(x)
        F.group_norm_backward(x, d, dx, images, F.GroupNorm(groups, w, b, stats, EPS, None))
        assert not dx[pixels:, 8:16].isfinite().any() and dx[~hit].isfinite().all()


@pytest.mark.parametrize("size", [(5, 400, 96, 32), (460, 196, 72, 4), (2, 20000, 64, 8), (3, 300, 51, 3)], ids=str)
def test_repeats_bit_for_bit_on_other_streams_and_in_two_graphs_at_once(size):
    from geeps_b200.ops import functional as F
    images, pixels, c, groups = size
    x, dy, w, b = made(images, pixels, c, groups, "bf16", 7)

    def buffers():
        return dict(y=torch.empty_like(x), dx=torch.empty_like(x), stats=torch.empty(images, groups, 2, device=DEV), dw=torch.empty(c, device=DEV), db=torch.empty(c, device=DEV))

    def both(o):
        n = F.GroupNorm(groups, w, b, o["stats"], EPS, "relu", o["dw"], o["db"])
        F.group_norm_forward(x, o["y"], images, n)
        F.group_norm_backward(x, dy, o["dx"], images, n)
    first = buffers()
    both(first)
    outs, graphs, streams = [buffers() for _ in range(2)], [], [torch.cuda.Stream() for _ in range(2)]
    for o in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            both(o)
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(o[k], first[k]) for k in first)


def test_offsets_that_pass_32_bits():
    """More than 2^31 values: the last image is normalised as by itself."""
    from geeps_b200.ops import functional as F
    images, pixels, c, groups = 33, 1 << 20, 64, 8
    gen = torch.Generator(device=DEV).manual_seed(8)
    x = torch.randn(images * pixels, c, dtype=BF, device=DEV, generator=gen)
    w, b = 1 + 0.3 * torch.randn(c, device=DEV, generator=gen), 0.3 * torch.randn(c, device=DEV, generator=gen)
    y, stats = torch.empty_like(x), torch.empty(images, groups, 2, device=DEV)
    F.group_norm_forward(x, y, images, F.GroupNorm(groups, w, b, stats, EPS, "relu"))
    last = x[-pixels:]
    check_forward(last, y[-pixels:], stats[-1:], statistics(last, 1, groups), w, b, 1, groups, "relu")
    del y
    dx, alone = torch.empty_like(x), torch.empty_like(last)
    F.group_norm_backward(x, x, dx, images, F.GroupNorm(groups, w, b, stats, EPS, "relu"))
    F.group_norm_backward(last, last, alone, 1, F.GroupNorm(groups, w, b, stats[-1:].clone(), EPS, "relu"))
    # two cuts of the same sums: 2^20 terms of random signs in parts of 2^12 at the most, whose means are off by 2^-12 of a term's size at
    # the worst; then a rounding on either side
    assert ((dx[-pixels:].double() - alone.double()).abs() <= 2.0 ** -7 * alone.double().abs() + 2.0 ** -10).all()


def test_gradients_match_differences():
    """Of the sum of dy y, in fp32: a central difference with step h is off by h^2 of a third derivative and 2^-22 / h of the sum."""
    from geeps_b200.ops import functional as F
    images, pixels, c, groups = 2, 6, 12, 3
    x, dy, w, b = made(images, pixels, c, groups, "fp32", 8)
    stats, dx = torch.empty(images, groups, 2, device=DEV), torch.empty_like(x)
    dw, db = torch.empty(c, device=DEV), torch.empty(c, device=DEV)
    y = torch.empty_like(x)

    def total(x, w, b):
        F.group_norm_forward(x, y, images, F.GroupNorm(groups, w, b, stats, EPS, "silu"))
        return (y.double() * dy.double()).sum().item()
    total(x, w, b)
    F.group_norm_backward(x, dy, dx, images, F.GroupNorm(groups, w, b, stats.clone(), EPS, "silu", dw, db))
    h = 2.0 ** -7
    size = (y.double().abs() * dy.double().abs()).sum().item()
    for t, grad in ((x, dx), (w, dw), (b, db)):
        for i in range(0, t.numel(), 5):
            v = t.view(-1)[i].item()
            t.view(-1)[i] = v + h
            up, high = total(x, w, b), t.view(-1)[i].item()
            t.view(-1)[i] = v - h
            down, low = total(x, w, b), t.view(-1)[i].item()
            t.view(-1)[i] = v
            assert abs((up - down) / (high - low) - grad.view(-1)[i].item()) <= 40 * h * h + 2.0 ** -22 / h * size


@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("size", [(2, 64, 64, 8), (1, 30000, 64, 8), (2, 50, 21, 3)], ids=str)
def test_the_border_of_the_relu_is_that_of_rounded_operations(size, types):
    """A bias that is minus the product to the last bit: z is zero there, and no gradient passes, while a fused multiply-add leaves the
    product's rounding error, above zero as often as below."""
    from geeps_b200.ops import functional as F
    images, pixels, c, groups = size
    x, dy, w, _ = made(*size, types, 9)
    x = x.view(images, pixels, c)
    x[:, ::2] = x[:1, :1]                                                # half of the pixels of a channel have one value ...
    x = x.view(-1, c)
    stats = statistics(x, images, groups).float()
    stats[1:] = stats[:1]                                                # ... and z, in all images
    mean, rstd = (spread(stats[:1, :, i], 1, groups, c)[0] for i in range(2))
    b = -(((x[:1].float() - mean) * rstd) * w)[0]
    dx, dw, db = torch.empty_like(x), torch.empty(c, device=DEV), torch.empty(c, device=DEV)
    F.group_norm_backward(x, dy, dx, images, F.GroupNorm(groups, w, b, stats, EPS, "relu", dw, db))
    z = ((x.float().view(images, pixels, c) - mean) * rstd) * w + b
    assert (z[:, ::2] == 0).all()
    check_backward(x, dy, dx, dw, db, stats, w, b, images, groups, "relu")
    kept = (dy.float().view(images, pixels, c) * (z > 0)).double().sum((0, 1))
    assert ((db.double() - kept).abs() <= 2.0 ** -14 * dy.double().abs().sum(0) * 2.0 ** -4).all()


def test_without_rows_the_parameters_have_gradients_of_zero():
    from geeps_b200.ops import functional as F
    x = torch.empty(0, 16, dtype=BF, device=DEV)
    dw, db = torch.full((16,), 7.0, device=DEV), torch.full((16,), 7.0, device=DEV)
    for images in (0, 4):
        F.group_norm_forward(x, x.clone(), images, F.GroupNorm(4))
        dw.fill_(7.0), db.fill_(7.0)
        F.group_norm_backward(x, x.clone(), x.clone(), images, F.GroupNorm(4, stats=torch.empty(images, 4, 2, device=DEV), dweight=dw, dbias=db))
        assert (dw == 0).all() and (db == 0).all()


def test_refusals():
    from geeps_b200.ops import functional as F
    x = torch.zeros(12, 16, dtype=BF, device=DEV)
    stats = torch.zeros(3, 4, 2, device=DEV)
    ok = F.GroupNorm(4, stats=stats)
    for match, call in (
            ("whole pixels", lambda: F.group_norm_forward(x, x.clone(), 5, F.GroupNorm(4))),
            ("divide", lambda: F.group_norm_forward(x, x.clone(), 3, F.GroupNorm(5))),
            ("activation", lambda: F.GroupNorm(4, act="tanh")),
            ("groups", lambda: F.GroupNorm(0)),
            ("eps", lambda: F.GroupNorm(4, eps=-1.0)),
            ("types", lambda: F.group_norm_forward(x, x.float(), 3, ok)),
            ("types", lambda: F.group_norm_forward(x.half(), x.half(), 3, ok)),
            ("rows, channels", lambda: F.group_norm_forward(x.view(3, 4, 16), x, 3, ok)),
            ("stats", lambda: F.group_norm_forward(x, x.clone(), 3, F.GroupNorm(4, stats=stats[:2]))),
            ("stats", lambda: F.group_norm_backward(x, x.clone(), x.clone(), 3, F.GroupNorm(4))),
            ("fp32", lambda: F.group_norm_forward(x, x.clone(), 3, F.GroupNorm(4, weight=torch.zeros(15, device=DEV)))),
            ("work", lambda: F.group_norm_backward(x, x.clone(), x.clone(), 3, ok, work=torch.zeros(1, device=DEV))),
            ("y", lambda: F.group_norm_forward(x, x[:6].clone(), 3, ok)),
            ("contiguous", lambda: F.group_norm_forward(x.t().contiguous().t(), x.clone(), 3, ok)),
            ("overlaps", lambda: F.group_norm_forward(x[:9], x[3:], 3, F.GroupNorm(4))),
            ("on cpu", lambda: F.group_norm_forward(x, x.cpu(), 3, ok))):
        with pytest.raises((ValueError, RuntimeError), match=match):
            call()


@pytest.mark.parametrize("c", [16385, 25600, 40000])
def test_too_many_channels_are_refused(c):
    from geeps_b200.ops import functional as F
    x = torch.zeros(4, c, dtype=BF, device=DEV)
    stats = torch.zeros(2, 1, 2, device=DEV)
    for call in (lambda: F.group_norm_forward(x, torch.empty_like(x), 2, F.GroupNorm(1)),
                 lambda: F.group_norm_backward(x, x.clone(), torch.empty_like(x), 2, F.GroupNorm(1, stats=stats))):
        with pytest.raises(ValueError, match="16384"):
            call()


@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("size", [(1, 64, 64, 8), (1, 30000, 64, 8), (1, 9, 16384, 1), (1, 50, 21, 3), (1, 20000, 21, 3)], ids=str)
def test_the_border_of_the_relu_is_the_same_forward_and_backward(size, types):
    """A bias that is minus the product to the last bit, as above: what the forward pass lets through is what the backward pass lets
    through, and z of rounded operations says what that is."""
    from geeps_b200.ops import functional as F
    images, pixels, c, groups = size
    x, _, w, _ = made(*size, types, 9)
    x[::2] = x[:1]                                                       # half of the pixels of a channel have one value, and z
    stats, y = torch.empty(1, groups, 2, device=DEV), torch.empty(x.shape, dtype=TYPES[types][1], device=DEV)
    F.group_norm_forward(x, y, 1, F.GroupNorm(groups, w, None, stats, EPS))
    mean, rstd = (spread(stats[:, :, i], 1, groups, c)[0] for i in range(2))
    b = -(((x[:1].float() - mean) * rstd) * w)[0]
    norm = F.GroupNorm(groups, w, b, stats, EPS, "relu", torch.empty(c, device=DEV), torch.empty(c, device=DEV))
    F.group_norm_forward(x, y, 1, norm)
    z = ((x.float() - mean) * rstd) * w + b
    assert (z[::2] == 0).all() and torch.equal(y > 0, z > 0)
    for r in (0, 1, pixels // 2, pixels - 1):                            # the gradient of the bias, from a row at a time
        dy = torch.zeros_like(y)
        dy[r] = 1.0
        F.group_norm_backward(x, dy, torch.empty_like(x), 1, norm)
        assert torch.equal(norm.dbias, (y[r] > 0).float())


@pytest.mark.parametrize("types", ["bf16", "fp32"])
@pytest.mark.parametrize("size", [(64, 119, 2, 2), (64, 119, 8, 8), (64, 64, 64, 64), (20, 100, 21, 7)], ids=str)
def test_a_first_pixel_far_from_the_others(size, types):
    """As the corner of an image may be.  A thread has one or two of these pixels, and the first one is what the threads' means are taken
    from: the squares about it, at most 128 times those about the mean, are rounded four times each (2^-24) before the latter come of them, and
    these are added, 128 of them at most: 640 roundings in all, half of that of 1/std.  The mean: 160 of differences, at most the outlier's."""
    from geeps_b200.ops import functional as F
    images, pixels, c, groups = size
    for far in (30.0, 1000.0):
        x, _, _, _ = made(*size, types, 11)
        first = x.view(images, pixels, c)[:, 0]
        first.copy_(far * torch.where(first > 0, 1.0, -1.0))
        stats = torch.empty(images, groups, 2, device=DEV)
        F.group_norm_forward(x, torch.empty_like(x), images, F.GroupNorm(groups, stats=stats, eps=EPS))
        want = statistics(x, images, groups)
        print("largest error of 1/std", (stats[..., 1].double() / want[..., 1] - 1).abs().max().item() * 2 ** 24)
        assert ((stats[..., 1].double() / want[..., 1] - 1).abs() <= 320 * 2.0 ** -24).all()
        assert ((stats[..., 0].double() - want[..., 0]).abs() <= 160 * 2.0 ** -24 * far).all()
