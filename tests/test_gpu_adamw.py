"""AdamW steps over many tensors against the formulas in 64 bits, with states in 32 and 8 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
B1, B2, EPS, WD, LR = 0.9, 0.999, 1e-8, 0.05, 1e-3


def flat(sizes, dtype, gen, gap=0, scale=1.0):
    """Tensors of the given sizes in one buffer, `gap` values apart (0: packed, so most begin anywhere)."""
    buf = torch.empty(sum(n + gap for n in sizes) + 8, dtype=dtype, device=DEV)
    buf.copy_(torch.randn(buf.numel(), generator=gen, device=DEV) * scale)
    out, at = [], 0
    for n in sizes:
        out.append(buf[at:at + n])
        at += n + gap
    return out


def states(state, bits):
    from geeps_b200.ops import functional as F
    if bits == 32:
        m, v = state.m.clone(), state.v.clone()
    else:
        m, v = F.adamw_moments(state, torch.empty_like(state.m, dtype=torch.float32), torch.empty_like(state.v, dtype=torch.float32))
    return [[x[o:o + n] for o, n in zip(state.offsets, state.params.numel)] for x in (m, v)]


def want(p, g, m, v, t, decay, c=1.0):
    """The formulas in 64 bits: new m, v and the change."""
    p, g, m, v = (x.double() for x in (p, g, m, v))
    g = g * c
    m, v = B1 * m + (1 - B1) * g, B2 * v + (1 - B2) * g * g
    return m, v, -LR * (m / (1 - B1 ** t) / (torch.sqrt(v / (1 - B2 ** t)) + EPS) + (WD * p if decay else 0.0))


SIZES = [[1], [128, 127, 129, 1, 513, 2048], [5000, 3, 0, 100_003], [300] * 700]


@pytest.mark.parametrize("sizes", SIZES, ids=len)
@pytest.mark.parametrize("pt,gt", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("gap", [0, 128])
def test_three_steps_follow_the_formulas(sizes, pt, gt, bits, gap):
    from geeps_b200.ops import functional as F
    gen = torch.Generator(device=DEV).manual_seed(len(sizes) + bits)
    sizes = [n if gap == 0 else (n + 127) // 128 * 128 for n in sizes]
    params = flat(sizes, pt, gen, gap, 0.1)
    decay = [i % 3 != 0 for i in range(len(sizes))]
    state = F.AdamWState(params, bits=bits, decay=decay)
    for t in (1, 2, 3):
        grads = flat(sizes, gt, gen, gap, 10.0 ** -t)
        before, (m0, v0) = [p.clone() for p in params], states(state, bits)
        F.adamw_step(params, grads, state, LR, betas=(B1, B2), eps=EPS, weight_decay=WD)
        m1, v1 = states(state, bits)
        assert state.steps.tolist() == [t, 0]
        for i in range(0, len(sizes), max(1, len(sizes) // 50)):
            m, v, change = want(before[i], grads[i], m0[i], v0[i], t, decay[i])
            # m and v: three roundings of 2^-24 of terms no larger than |b m| + |a g|; the change: 2^-19 (square root and quotient
            # 2^-21 each, the fp32 operations), and 2^-24 of p, before it is rounded to p's type
            top = B1 * m0[i].double().abs() + (1 - B1) * grads[i].double().abs()
            if bits == 32:
                assert ((m1[i].double() - m).abs() <= 3 * 2.0 ** -24 * top).all()
                assert ((v1[i].double() - v).abs() <= 5 * 2.0 ** -24 * v + 1e-44).all()
            else:
                # half a step of three bits of mantissa; below the block's range m vanishes and v stays above zero
                pad = -sizes[i] % 128
                for got, x, low in ((m1[i], m, 2.0 ** -14), (v1[i], v, 2.0 ** -30)):
                    high = torch.nn.functional.pad(x.abs(), (0, pad)).view(-1, 128).amax(1).repeat_interleave(128)[:sizes[i]]
                    assert ((got.double() - x).abs() <= x.abs() * (2.0 ** -4 + 2.0 ** -20) + low * high + 1e-28).all()
                assert (v1[i][v > 1e-30] > 0).all()
            off = (params[i].double() - before[i].double() - change).abs()
            half = torch.finfo(pt).eps / 2
            assert (off <= 2.0 ** -19 * change.abs() + (half + 2.0 ** -24) * (before[i].double().abs() + change.abs())).all()
