"""Bits that the norms' backward pass keeps: n = (x - mean) rstd from the statistics at hand is a difference and a product, each
rounded once, so it is off by at most 2 * 2^-24 of itself (and their product), whatever the mean is.  Against the formula in 64 bits
of the very x, mean and rstd that the call is given.

With one row and dy = 1 the weight's gradient is n, which shows every bit of it."""
import pytest
import torch

from geeps_b200.ops import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
TYPES = {"bf16": (BF, BF), "mixed": (F32, BF), "fp32": (F32, F32)}
U = 2.0 ** -24
CHANNELS = [1, 2, 5, 8, 64, 200, 576, 1001, 1024, 2050, 4096, 4104, 8192, 8193, 12296, 16383]


def far_rows(rows, c, dtype, centre, spread, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(rows, c, generator=gen, device=DEV) * spread + centre).to(dtype)


def stats_of(x, kind):
    """What the forward pass leaves."""
    st = torch.empty(x.shape[0], 2, device=DEV)
    F.norm_forward(x, torch.empty_like(x), F.Norm(kind, None, None, st))
    return st


def n_of(x, st):
    return (x.double() - st[:, :1].double()) * st[:, 1:].double()


def close(got, want, what):
    off = ((got.double() - want).abs() - (2 * U + U * U) * want.abs()).max().item()
    assert off <= 0, f"{what}: {off} beyond two roundings"


@pytest.mark.parametrize("c", CHANNELS)
@pytest.mark.parametrize("centre,spread", [(0.0, 1.0), (100.0, 0.01), (-7.0, 3.0)])
@pytest.mark.parametrize("types", list(TYPES))
def test_n_of_one_row(c, centre, spread, types):
    rt, bt = TYPES[types]
    one = torch.ones(1, c, device=DEV)
    dw, dw2 = torch.full((c,), 7.0, device=DEV), torch.full((c,), 7.0, device=DEV)
    x = far_rows(1, c, rt, centre, spread, c)
    st = stats_of(x, "layer")
    F.norm_backward(x, one.to(bt), torch.empty_like(x), F.Norm("layer", None, None, st, dweight=dw))
    close(dw, n_of(x, st)[0], "norm")
    b, h = far_rows(1, c, bt, centre, spread, c + 1), far_rows(1, c, rt, centre, spread, c + 2)
    st, st2 = stats_of(b, "layer"), stats_of(h, "layer")
    F.residual_backward(b, one.to(rt), torch.empty_like(b), torch.empty_like(h), post=F.Norm("layer", None, None, st, dweight=dw))
    close(dw, n_of(b, st)[0], "join")
    for gate in (None, torch.ones(1, c, device=DEV).to(bt)):
        F.residual_backward(b, None, torch.empty_like(b), torch.empty_like(h), post=F.Norm("layer", None, None, st), gate=gate, out=h, dy=one.to(bt),
                            pre=F.Norm("layer", None, None, st2, dweight=dw2))
        close(dw2, n_of(h, st2)[0], "norm behind a join")


@pytest.mark.parametrize("types", list(TYPES))
def test_one_channel_is_its_own_mean(types):
    """n is 0: no gradient for the weight, none through the norm."""
    rt, bt = TYPES[types]
    rows = 300
    x, dy, dres = far_rows(rows, 1, rt, 3.0, 2.0, 1), far_rows(rows, 1, bt, 0.0, 1.0, 2), far_rows(rows, 1, rt, 0.0, 1.0, 3)
    dw, dx = torch.full((1,), 7.0, device=DEV), torch.empty_like(x)
    F.norm_backward(x, dy, dx, F.Norm("layer", None, None, stats_of(x, "layer"), dweight=dw), dres=dres)
    assert dw.item() == 0.0 and torch.equal(dx, dres)
    b, db = far_rows(rows, 1, bt, 3.0, 2.0, 4), torch.empty(rows, 1, dtype=bt, device=DEV)
    F.residual_backward(b, dres, db, dx, post=F.Norm("layer", None, None, stats_of(b, "layer"), dweight=dw))
    assert dw.item() == 0.0 and (db == 0).all()


@pytest.mark.parametrize("c", [2, 3])
@pytest.mark.parametrize("centre,spread", [(0.0, 1.0), (50.0, 0.5)])
def test_gradients_of_few_channels(c, centre, spread):
    """dx = rstd (a - mean a - n mean(a n)) cancels where channels are few.  What is left is off by the roundings of its terms: with
    |n| <= sqrt(c) each of a, mean a and n mean(a n) is at most M = c max|a|, and the sums, products and n take 5 + c roundings."""
    rows = 4000
    x, dy = far_rows(rows, c, F32, centre, spread, 5), far_rows(rows, c, F32, 0.0, 1.0, 6)
    st, dx = stats_of(x, "layer"), torch.empty_like(x)
    F.norm_backward(x, dy, dx, F.Norm("layer", None, None, st))
    n, a, rs = n_of(x, st), dy.double(), st[:, 1:].double()
    want = rs * (a - a.mean(1, keepdim=True) - n * (a * n).mean(1, keepdim=True))
    most = rs * c * a.abs().max(1, keepdim=True)[0] * 3
    assert ((dx.double() - want).abs() <= (5 + c) * U * most + U * want.abs()).all()
