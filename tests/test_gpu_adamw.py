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


def test_out_receives_the_change_and_may_be_the_gradients():
    from geeps_b200.ops import functional as F
    gen = torch.Generator(device=DEV).manual_seed(3)
    sizes = [1000, 7, 4096]
    params = flat(sizes, torch.float32, gen, 3, 0.1)
    grads = flat(sizes, torch.float32, gen, 5, 0.01)
    plain, twin = [p.clone() for p in params], F.AdamWState([p.clone() for p in params])
    for out in ([torch.empty_like(g) for g in grads], [torch.empty_like(g, dtype=torch.bfloat16) for g in grads], grads):
        state = F.AdamWState(params)
        before, g0 = [p.clone() for p in params], [g.clone() for g in grads]
        F.adamw_step(params, grads, state, LR, weight_decay=WD, out=out)
        for p, b, g, o in zip(params, before, g0, out):
            assert torch.equal(p, b)
            _, _, change = want(b, g, torch.zeros_like(b), torch.zeros_like(b), 1, True)
            assert ((o.double() - change).abs() <= (2.0 ** -19 + torch.finfo(o.dtype).eps / 2) * change.abs()).all()
    F.adamw_step(plain, g0, twin, LR, weight_decay=WD)
    for p, b, o in zip(plain, params, grads):
        assert torch.equal(p, b + o)                       # what an additive table makes of it


def test_a_norm_above_its_bound_scales_the_gradients_on_their_way():
    from geeps_b200.ops import functional as F
    gen = torch.Generator(device=DEV).manual_seed(4)
    grads = flat([5000, 300], torch.bfloat16, gen, 0, 1.0)
    for ratio in (0.5, 4.0, float("inf")):
        params = [torch.zeros(5000, device=DEV), torch.zeros(300, device=DEV)]
        state, norm = F.AdamWState(params), torch.zeros(2, device=DEV)
        F.clip_gradients(grads, float("inf"), norm)
        bound = 0.0 if ratio == float("inf") else norm[0].item() / ratio
        F.adamw_step(params, grads, state, LR, clip=(norm, bound))
        c = min(1.0, bound / norm[0].item())
        for o, n, g in zip(state.offsets, state.params.numel, grads):
            m = (1 - B1) * c * g.double()
            assert ((state.m[o:o + n].double() - m).abs() <= 4 * 2.0 ** -24 * m.abs()).all()
    norm.fill_(float("inf"))                                # the factor is 0 then, and what is not finite goes on
    params[0].fill_(1.0)
    F.adamw_step(params, grads, state, LR, clip=(norm, 1.0))
    assert params[0].isfinite().all()


@pytest.mark.parametrize("pt", [torch.float32, torch.bfloat16])
def test_random_rounding_keeps_the_mean_and_depends_on_seed_step_and_place(pt):
    """States in 8 bits whose mean moves by less than half a code in a step: rounded at random they follow it on average.  The mean of
    n values that are each up or down with the right odds is off by at most 5 standard deviations of it, d / (2 sqrt(n)) each, where d
    is the distance of two codes (an eighth of the value)."""
    from geeps_b200.ops import functional as F
    n = 1 << 20
    params, grads = [torch.full((n,), 0.5, dtype=pt, device=DEV)], [torch.full((n,), 0.25, device=DEV)]

    def after(steps, seed):
        p = [params[0].clone()]
        state = F.AdamWState(p, bits=8)
        for _ in range(steps):
            F.adamw_step(p, grads, state, LR, seed=seed)
        m, v = F.adamw_moments(state, torch.empty(n, device=DEV), torch.empty(n, device=DEV))
        return m, v, p[0], state
    for steps in (1, 7):
        m, v, p, state = after(steps, 5)
        wm, wv = 0.25 * (1 - B1 ** steps), 0.0625 * (1 - B2 ** steps)
        for got, w in ((m, wm), (v, wv)):
            assert abs(got.double().mean().item() - w) <= 5 * steps * (w / 8) / (2 * math.sqrt(n)) + 2.0 ** -20 * w
        again = after(steps, 5)
        assert torch.equal(state.m, again[3].m) and torch.equal(state.v, again[3].v) and torch.equal(p, again[2])
        other = after(steps, 6)
        assert not torch.equal(state.m, other[3].m) and not torch.equal(state.v, other[3].v)
        if pt is torch.bfloat16:                            # a change below half a step of bf16 (0.5: 2^-9)
            off = p.double().mean().item() - 0.5
            assert abs(off + LR * steps) <= 5 * steps * 2.0 ** -9 / math.sqrt(n) + 0.1 * LR * steps and len(p.unique()) > 1
    nearest = after(7, None)
    assert len(nearest[0].unique()) == 1


@pytest.mark.parametrize("bits", [32, 8])
def test_values_that_are_not_finite(bits):
    from geeps_b200.ops import functional as F
    for bad in (float("nan"), float("inf"), -float("inf")):
        p, g = [torch.ones(400, device=DEV)], [torch.full((400,), 0.5, device=DEV)]
        state = F.AdamWState(p, bits=bits)
        F.adamw_step(p, g, state, LR, seed=1)
        g[0][130] = bad
        F.adamw_step(p, g, state, LR, seed=1)
        finite = p[0].isfinite()
        assert not finite[130] and finite[:130].all() and finite[131:].all()
        g[0][130] = 0.5
        F.adamw_step(p, g, state, LR, seed=1)
        assert not p[0][130].isfinite() and p[0][:128].isfinite().all() and p[0][256:].isfinite().all()


def test_replayed_steps_count_and_read_the_rate_from_the_device():
    from geeps_b200.ops import functional as F
    gen = torch.Generator(device=DEV).manual_seed(8)
    sizes = [3000, 50]
    start = flat(sizes, torch.float32, gen, 0, 0.1)
    grads = flat(sizes, torch.float32, gen, 0, 0.01)

    def run(replay):
        params = [p.clone() for p in start]
        state, lr = F.AdamWState(params, bits=8), torch.tensor([LR], device=DEV)
        args = (F.GradList(params), F.GradList(grads), state, lr)
        F.adamw_step(*args, weight_decay=WD, seed=2)
        if replay:
            stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                F.adamw_step(*args, weight_decay=WD, seed=2)
            torch.cuda.synchronize()
        for i in range(4):
            lr.fill_(LR / (i + 1))
            if replay:
                graph.replay()
            else:
                F.adamw_step(*args, weight_decay=WD, seed=2)
        torch.cuda.synchronize()
        return params, state
    (p, a), (q, b) = run(False), run(True)
    assert all(torch.equal(x, y) for x, y in zip(p, q)) and torch.equal(a.m, b.m) and torch.equal(a.v, b.v) and torch.equal(a.exponents, b.exponents)
    assert a.steps.tolist() == b.steps.tolist() == [5, 0]
    by_value = [x.clone() for x in start]
    state = F.AdamWState(by_value, bits=8)
    for i in range(5):
        F.adamw_step(by_value, grads, state, LR if i == 0 else torch.tensor(LR / i).item(), weight_decay=WD, seed=2)
    assert all(((x - y).abs() <= 2.0 ** -20 * (x.abs() + LR)).all() for x, y in zip(p, by_value))


def test_states_can_be_saved_and_restored():
    from geeps_b200.ops import functional as F
    p, g = [torch.ones(300, device=DEV)], [torch.full((300,), 0.1, device=DEV)]
    state = F.AdamWState(p, bits=8)
    F.adamw_step(p, g, state, LR, seed=1)
    saved = [t.clone() for t in (p[0], state.m, state.v, state.exponents, state.steps)]
    F.adamw_step(p, g, state, LR, seed=1)
    again = F.AdamWState([saved[0]], bits=8)
    again.m, again.v, again.exponents, again.steps = saved[1:]
    F.adamw_step([saved[0]], g, again, LR, seed=1)
    assert torch.equal(saved[0], p[0]) and torch.equal(again.m, state.m) and again.steps.tolist() == [2, 0]


def test_more_values_than_32_bits_of_bytes():
    from geeps_b200.ops import functional as F
    n = (1 << 30) + 12345                                   # fp32: more than 2^32 bytes
    p, g = torch.zeros(n, device=DEV), torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    g[0], g[n - 1], g[n // 2] = 1.0, -1.0, 2.0
    state = F.AdamWState([p], bits=8)
    F.adamw_step([p], [g], state, LR)
    hit = p.nonzero().view(-1).tolist()
    assert hit == [0, n // 2, n - 1]
    assert abs(p[0].item() + LR) < 1e-8 and abs(p[n - 1].item() - LR) < 1e-8


def test_refusals():
    from geeps_b200.ops import functional as F
    p, g = torch.zeros(100, device=DEV), torch.zeros(100, device=DEV)
    state = F.AdamWState([p])
    step = lambda **kw: F.adamw_step(kw.pop("params", [p]), kw.pop("grads", [g]), kw.pop("state", state), kw.pop("lr", LR), **kw)
    for match, call in (
            ("bits", lambda: F.AdamWState([p], bits=16)), ("parameter", lambda: F.AdamWState([])),
            ("decay", lambda: F.AdamWState([p], decay=[True, False])), ("steps", lambda: F.AdamWState([p], steps=-1)),
            ("counts", lambda: step(grads=[g[:50]])), ("counts", lambda: step(params=[p, g])), ("counts", lambda: step(out=[g[:3]])),
            ("betas", lambda: step(betas=(1.0, 0.9))), ("betas", lambda: step(eps=-1.0)), ("betas", lambda: step(weight_decay=-0.1)),
            ("lr", lambda: step(lr=torch.zeros(1, dtype=torch.float64, device=DEV))), ("lr", lambda: step(lr=torch.zeros(2, device=DEV))),
            ("clip", lambda: step(clip=(torch.zeros(2), 1.0))), ("clip", lambda: step(clip=(torch.zeros(2, device=DEV), -1.0))),
            ("overlap", lambda: step(grads=[p])), ("overlap", lambda: step(out=[p])), ("overlap", lambda: step(clip=(p, 1.0))),
            ("32 bits", lambda: F.adamw_moments(state, p, g)),
            ("moments|bf16", lambda: F.adamw_moments(F.AdamWState([p], bits=8), p, g))):
        with pytest.raises(ValueError, match=match):
            call()
    state.m = state.m[:64]
    with pytest.raises(ValueError, match="AdamWState"):
        step()


@pytest.mark.parametrize("eps", [0.0, 1e-40, 1e-30, 1e-20, 1e-15])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("n", [1024, 1001])
def test_small_gradients_beside_a_small_eps(eps, bits, n):
    """Second moments below the smallest normal number (1.2e-38) count, and a gradient of zero beside an eps above zero changes nothing.
    The change: 2^-19 of it as elsewhere, and what v's two roundings and eps' own leave, each half of 2^-149 at the most: of the root half
    of what v is off by, relative to v."""
    from geeps_b200.ops import functional as F
    gen = torch.Generator(device=DEV).manual_seed(6)
    g = torch.where(torch.rand(n, generator=gen, device=DEV) < 0.5, -1.0, 1.0) * 10.0 ** (-19.0 + 4 * torch.rand(n, generator=gen, device=DEV))
    g[3::5] = 1.0                                   # beside large ones
    if eps:
        g[4::5] = 0.0
    p, out = torch.zeros(n, device=DEV), torch.empty(n, device=DEV)
    state = F.AdamWState([p], bits=bits)
    F.adamw_step([p], [g], state, LR, betas=(B1, B2), eps=eps, out=[out])
    d = g.double()
    m, v, e = (1 - B1) * d, (1 - B2) * d * d, torch.tensor(eps).float().double().item()
    change = -LR * (m / (1 - B1)) / (torch.sqrt(v / (1 - B2)) + e)
    change[d == 0] = 0.0
    off = 2.0 ** -19 + torch.where(v > 0, 2.1 * 2.0 ** -150 / v, 0.0)
    assert ((out.double() - change).abs() <= off * change.abs()).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_without_values_take_their_steps(bits):
    """A worker whose share is empty: the steps count, and what is asked of no values gives none."""
    from geeps_b200.ops import functional as F
    p, g = [torch.empty(0, device=DEV), torch.empty(0, dtype=torch.bfloat16, device=DEV)], [torch.empty(0, device=DEV)] * 2
    state = F.AdamWState(p, bits=bits)
    for _ in range(2):
        F.adamw_step(p, g, state, LR, seed=1)
    F.adamw_step(p, g, state, LR, out=[torch.empty(0, device=DEV)] * 2)
    assert state.steps.tolist() == [3, 0]
    if bits == 8:
        F.adamw_moments(state, torch.empty(0, device=DEV), torch.empty(0, device=DEV))


def test_the_mean_of_first_moments_at_the_end_of_their_codes():
    """Beside a 1, whose code is 120: code 1 is 2^-15 x 9/8.  From there on the mean of what random rounding leaves is the value; from
    2^-15 to code 1 it is code 1 by the odds of the distance from 2^-15; below it is 0.  n values that are one of two, d apart: 5
    standard deviations of their mean, d / (2 sqrt(n)) each, and the 2^-16 that 16 random bits leave of d."""
    from geeps_b200.ops import functional as F
    blocks, least, step = 4096, 2.0 ** -15, 2.0 ** -18
    for x in (3.0e-5, 3.1e-5, 3.2e-5, 3.4e-5, 3.5e-5, 5.0e-5, 6.0e-5, 1.0e-3):
        g = torch.full((blocks, 128), 2 * x, device=DEV)
        g[:, 0] = 2.0                                       # m = g / 2
        p, out = torch.zeros(blocks * 128, device=DEV), torch.empty(blocks * 128, device=DEV)
        state = F.AdamWState([p], bits=8)
        F.adamw_step([p], [g.view(-1)], state, LR, betas=(0.5, B2), out=[out], seed=9)
        m, _ = F.adamw_moments(state, torch.empty_like(p), torch.empty_like(p))
        m = m.view(blocks, 128)
        assert (m[:, 0] == 1).all()
        mean = m[:, 1:].double().mean().item()
        want = x if x >= least + step else 0.0 if x < least else (x - least) / step * (least + step)
        d = least + step if x < least + step else 2.0 ** math.floor(math.log2(x)) / 8
        assert abs(mean - want) <= 5 * d / (2 * math.sqrt(blocks * 127)) + 2.0 ** -16 * d + 2.0 ** -23 * x
