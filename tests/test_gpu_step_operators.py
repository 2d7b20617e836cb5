"""Group norms, 8-bit products and AdamW steps as a network's training step uses them together."""
import pytest
import torch
import torch.nn.functional as TF

from geeps_b200.models.inception_bn import inception_bn_small
from geeps_b200.models.net import Concat, Net
from geeps_b200.ops.layers import Conv2d, GroupNorm, Input, Linear, Pool
from geeps_b200.parallel.ps_module import PSModule
from geeps_b200.utils.config import TABLE_ADDITIVE, TRANSPORT_NVLINK, TRANSPORT_TCP
from test_gpu_residual import bind, cfg

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, F64 = torch.bfloat16, torch.float64


def test_a_group_norm_layer_has_the_gradients_of_autograd():
    """Alone and as the end of a branch that writes into a slice of a wider tensor.  bf16 in and out: half a step (2^-8) of the
    result, and of an fp32 gradient 2^-12 of its terms (some 600 of them, random signs)."""
    x = torch.randn(3, 7, 5, 48, device=DEV).to(BF)
    dy = torch.randn(3, 7, 5, 96, device=DEV).to(BF)
    layers = [GroupNorm("a", 6, act="silu"), GroupNorm("b", 12)]
    cat = Concat("cat", [[layers[0]], [layers[1]]], concurrent=False)
    cat.setup(tuple(x.shape), DEV)
    bind([cat], 3)
    y = cat.forward(x).view(3, 7, 5, 96)
    dx = cat.backward(dy.view(-1, 96)).view_as(x)
    leaf = x.to(F64).requires_grad_(True)
    p = [{k: v.to(F64).requires_grad_(True) for k, v in l.p32.items()} for l in layers]
    parts = [TF.group_norm(leaf.permute(0, 3, 1, 2), l.groups, q["gamma"], q["beta"], l.eps).permute(0, 2, 3, 1) for l, q in zip(layers, p)]
    want = torch.cat([TF.silu(parts[0]), parts[1]], 3)
    assert ((y.to(F64) - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -14).all()
    grads = torch.autograd.grad(want, [leaf] + [q[k] for q in p for k in ("gamma", "beta")], dy.to(F64))
    # two branches' gradients, rounded, and their sum
    size = grads[0].abs().max()
    assert ((dx.to(F64) - grads[0]).abs() <= 3 * 2.0 ** -8 * size).all()
    for g, got in zip(grads[1:], [l.g32[k] for l in layers for k in ("gamma", "beta")]):
        assert ((got.to(F64) - g).abs() <= 2.0 ** -12 * dy.to(F64).abs().sum((0, 1, 2)).max()).all()
    with pytest.raises(ValueError, match="divide"):
        GroupNorm("c", 7).setup(tuple(x.shape), DEV)


@pytest.mark.parametrize("fp32_out", [False, True])
def test_an_fp8_layer_is_near_the_bf16_layer(fp32_out):
    """Each operand is off by half a step of e4m3, 2^-4 of a value at the most and evenly spread, so 2^-4 / sqrt(3) in the mean
    square; products of two such have sqrt(2) of that, whatever the number of terms: 0.051, with the outputs' own rounding below 0.06."""
    gen = torch.Generator().manual_seed(1)
    x, dy = torch.randn(96, 640, generator=gen).to(DEV).to(BF), torch.randn(96, 264, generator=gen).to(DEV).to(BF)
    got = []
    for fp8 in (False, True):
        l = Linear("fc", 264, std=0.05, fp32_out=fp32_out, fp8=fp8)
        l.setup((96, 640), DEV)
        bind([l], 2)
        y = l.forward(x).clone()
        dx = l.backward(dy).clone()
        got.append((y, dx, l.g32["weight"], l.g32["bias"]))
    # column sums of the same 96 rows, in any order: 96 roundings of 2^-24 of the magnitudes on either side
    assert ((got[0][3] - got[1][3]).abs() <= 96 * 2.0 ** -23 * dy.float().abs().sum(0)).all()
    for a, b in zip(got[0][:3], got[1][:3]):
        assert a.dtype == b.dtype and (a.double() - b.double()).norm() <= 0.06 * a.double().norm()


def net(fp8=True):
    return Net("n", Input(cpad=8), [Conv2d("c0", 24, 3, pad=1, bias=False, std=0.2, need_dx=False), GroupNorm("g0", 4, act="relu"),
                                    Conv2d("c1", 32, 3, pad=1, bias=False, std=0.1), GroupNorm("g1", 8, act="silu"), Pool("avg", 0, 1, ceil_mode=False),
                                    Linear("f1", 64, relu=True, std=0.2, fp8=fp8), Linear("fc", 10, std=0.3, fp32_out=True, fp8=fp8)])


def batch(n=16):
    gen = torch.Generator(device=DEV).manual_seed(5)
    return torch.randn(n, 3, 8, 8, generator=gen, device=DEV), torch.randint(0, 10, (n,), generator=gen, device=DEV)


def module(transport=TRANSPORT_NVLINK, adamw=None, make=net, shape=(16, 3, 8, 8), **kw):
    return PSModule(make(), shape, cfg(transport, table_mode=TABLE_ADDITIVE, learning_rate=0.01, weight_decay=0.1), device="cuda:0", seed=4,
                    adamw=adamw or {}, **kw)


@pytest.mark.parametrize("transport", [TRANSPORT_NVLINK, TRANSPORT_TCP])
@pytest.mark.parametrize("clip", [None, 0.05])
def test_a_step_moves_the_parameters_by_the_formula(transport, clip):
    """From the states that the first step leaves: m = (1 - b1) g and v = (1 - b2) g^2, so the change is that of m and v."""
    mod = module(transport, clip_gradients=clip)
    x, y = batch()
    mod.step(x, y, capture=True)
    before = {k: v.clone() for k, v in mod.captured.items()}
    state, specs = mod.adamw.state, [(t.layer, sp) for t in mod.tables for sp in t.specs]
    m = [state.m[o:o + n].double().clone() for o, n in zip(state.offsets, state.params.numel)]
    v = [state.v[o:o + n].double().clone() for o, n in zip(state.offsets, state.params.numel)]
    mod.step(x, y, capture=True)
    after = {k: v.clone() for k, v in mod.captured.items()}
    assert state.steps[0].item() == 2
    if clip is not None:
        assert mod.clip_result[0].item() > clip                # it does clip
        total = sum((a / 0.1).square().sum().item() for a in m) ** 0.5
        assert abs(total - clip) <= 1e-5 * clip
    for (l, sp), a, b in zip(specs, m, v):
        p = before[f"{l.name}.{sp.name}"].double().view(-1)
        change = -0.01 * (a / 0.1 / ((b / (1 - 0.999)).sqrt() + 1e-8) + (0.1 * p if sp.decay else 0.0))
        off = after[f"{l.name}.{sp.name}"].double().view(-1) - p - change
        # 2^-18 of the change; the sum is a rounding of the parameter, the states one each of m and v
        assert (off.abs() <= 2.0 ** -18 * change.abs() + 2.0 ** -23 * (p.abs() + change.abs())).all(), (l.name, sp.name)
    mod.close()


@pytest.mark.parametrize("bits,seed", [(32, None), (8, 7)])
def test_steps_with_graphs_recorded_steps_and_neither_train_alike(bits, seed):
    """A network without convolutions: none of its gradients is a sum in an order that changes (16 rows a column sum are one block's),
    so the parameters are the same to the last bit."""
    make = lambda: Net("n", Input(cpad=8), [GroupNorm("g0", 4, act="relu"), Linear("f1", 64, relu=True, std=0.2, fp8=True), GroupNorm("g1", 8, act="silu"),
                                            Linear("fc", 10, std=0.3, fp32_out=True, fp8=True)])
    x, y = batch()
    ends = []
    for kw in (dict(), dict(use_tape=True), dict(use_graph=True)):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            mod = module(adamw=dict(bits=bits, seed=seed), clip_gradients=5.0, make=make, **kw)
            for _ in range(10):
                mod.step(x, y)
            st.synchronize()
            assert not kw or mod.is_steady(x, y), mod.tape_mismatch
            assert mod.adamw.state.steps.tolist() == [10, 0] and mod.adamw.state.bits == bits
            mod.step(x, y, capture=True)
            ends.append({k: v.clone() for k, v in mod.captured.items()})
            mod.set_hyper_params(learning_rate=0.0, momentum=0.9)             # without a new capture
            assert not kw or mod.is_steady(x, y)
            st.synchronize()
            mod.close()
    for other in ends[1:]:
        assert other.keys() == ends[0].keys() and all(torch.equal(other[k], ends[0][k]) for k in other)


def test_a_rate_of_zero_holds_the_parameters():
    x, y = batch()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        mod = module(use_graph=True)

        def steps(n):
            for _ in range(n):
                mod.step(x, y)
            st.synchronize()
            return {k: v.clone() for k, v in mod.params_fp32().items()}
        steps(6)
        mod.set_hyper_params(learning_rate=0.0)
        held, later = steps(1), steps(3)
        assert all(torch.equal(later[k], held[k]) for k in held)
        mod.set_hyper_params(learning_rate=0.01, weight_decay=0.2)            # another decay: recorded again
        assert not mod.is_steady(x, y)
        moved = steps(6)
        assert mod.is_steady(x, y) and all(not torch.equal(moved[k], held[k]) for k in held)
        mod.close()


def test_an_inception_net_with_group_norms_trains_in_graphs_and_with_managed_activations():
    gen = torch.Generator(device=DEV).manual_seed(2)
    x, y = torch.randn(8, 3, 32, 32, generator=gen, device=DEV), torch.randint(0, 10, (8,), generator=gen, device=DEV)
    losses = []
    for kw in (dict(), dict(use_graph=True), dict(manage_activations=True)):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            mod = module(make=lambda: inception_bn_small(norm="group"), shape=(8, 3, 32, 32), **kw)
            losses.append([mod.step(x, y).clone() for _ in range(5)])
            st.synchronize()
            mod.close()
    losses = [[v.item() for v in out] for out in losses]
    assert all(v == v and v < 20 for out in losses for v in out)
    # one step's loss is a sum in any order; afterwards atomics of the weight gradients, which AdamW's quotient of m and v magnifies
    # where a gradient is near zero
    for other in losses[1:]:
        assert abs(other[0] - losses[0][0]) <= 64 * 2.0 ** -24 * abs(losses[0][0])


@pytest.mark.parametrize("bits,seed", [(32, None), (8, 3)])
def test_a_resumed_module_goes_on_with_its_states(bits, seed, tmp_path):
    x, y = batch()
    kw = dict(adamw=dict(bits=bits, seed=seed))
    mod = module(**kw)
    for _ in range(3):
        mod.step(x, y)
    mod.save_snapshot(str(tmp_path))
    kept = {k: None if getattr(mod.adamw.state, k) is None else getattr(mod.adamw.state, k).clone() for k in ("m", "v", "exponents", "steps")}
    mod.step(x, y)
    went = mod.adamw.state.m.float()
    mod.close()
    other = module(resume_from=str(tmp_path), **kw)
    assert other.steps == 3 and all(k is None or torch.equal(k, other.adamw._resumed[n]) for n, k in kept.items())
    other.step(x, y)
    state = other.adamw.state
    assert state.steps.tolist() == [4, 0]
    if bits == 32:            # the gradients of equal parameters: sums in any order, at worst another rounding (2^-8) of a layer's bf16 gradient
        for o, n in zip(state.offsets, state.params.numel):
            a, b = went[o:o + n], state.m[o:o + n]
            assert (a - b).abs().max() <= 2.0 ** -8 * a.abs().max()
    other.close()
    with pytest.raises(ValueError, match="AdamWState"):
        wrong = module(resume_from=str(tmp_path), adamw=dict(bits=40 - bits))
        try:
            wrong.step(x, y)
        finally:
            wrong.close()


def test_refusals():
    with pytest.raises(ValueError, match="additive"):
        PSModule(net(), (16, 3, 8, 8), cfg(TRANSPORT_NVLINK), device="cuda:0", adamw={})
    with pytest.raises(ValueError, match="fp32"):
        module(bf16_weights_only=True)


def exact_net():
    """A network whose gradients are sums in one order: the same steps end in the same bits."""
    return Net("n", Input(cpad=8), [GroupNorm("g0", 4, act="relu"), Linear("f1", 64, relu=True, std=0.2, fp8=True), GroupNorm("g1", 8, act="silu"),
                                    Linear("fc", 10, std=0.3, fp32_out=True, fp8=True)])


@pytest.mark.parametrize("how", ["plain", "tape", "graph"])
def test_periodic_snapshots_hold_the_states(how, tmp_path):
    kw = {"plain": {}, "tape": dict(use_tape=True), "graph": dict(use_graph=True)}[how]
    x, y = batch()

    def run(steps, every=0, **more):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            c = cfg(TRANSPORT_NVLINK, table_mode=TABLE_ADDITIVE, learning_rate=0.01, weight_decay=0.1, snapshot_interval=every, snapshot_dir=str(tmp_path))
            mod = PSModule(exact_net(), (16, 3, 8, 8), c, device="cuda:0", seed=4, adamw=dict(bits=8, seed=3), **kw, **more)
            for _ in range(steps):
                mod.step(x, y)
            st.synchronize()
            state = {k: getattr(mod.adamw.state, k).clone() for k in ("m", "v", "exponents", "steps")}
            mod.step(x, y, capture=True)
            end = {k: v.clone() for k, v in mod.captured.items()}
            assert mod.ps.clock_value == mod.steps + 1
            mod.close()
            return state, end
    want, end = run(12)
    for every in (5, 3):
        run(7 if every == 5 else 11, every)          # the initial values are clock 0, so step 12 ends clock 12
        clocks = [5] if every == 5 else [3, 5, 6, 9, 12]
        assert sorted(int(p.name.split(".")[1]) for p in tmp_path.glob("snapshot.*")) == clocks and (tmp_path / "LATEST").read_text() == str(clocks[-1])
        for c in clocks:
            kept = torch.load(tmp_path / f"snapshot.{c}" / "adamw.0")
            assert kept["steps"].tolist() == [c - 1, 0] and (kept["v"] != 0).any()
        state, other = run(12 - (clocks[-1] - 1), resume_from=str(tmp_path))
        assert all(torch.equal(state[k], want[k]) for k in want) and all(torch.equal(other[k], end[k]) for k in end)


def test_a_snapshot_taken_from_another_stream_has_the_last_step(tmp_path):
    """The step is still on its way on the stream that it was called on."""
    x, y = batch()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        mod = module(make=exact_net, adamw=dict(bits=32))
        for _ in range(3):
            mod.step(x, y)
        st.synchronize()
        torch.cuda._sleep(400_000_000)           # some 0.2 s
        mod.step(x, y)
    mod.save_snapshot(str(tmp_path))
    kept = torch.load(tmp_path / "snapshot.5" / "adamw.0")
    st.synchronize()
    assert kept["steps"].tolist() == [4, 0] and torch.equal(kept["m"], mod.adamw.state.m) and torch.equal(kept["v"], mod.adamw.state.v)
    mod.close()


def test_a_rate_set_from_another_stream_is_for_the_next_step():
    """A step that is still on its way keeps the rate that it was called with, the one called next has the new one."""
    x, y = batch()
    ends = []
    for apart in (False, True):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            mod = module(make=exact_net, adamw=dict(bits=32))
            for _ in range(3):
                mod.step(x, y)
            st.synchronize()
            if apart:
                torch.cuda._sleep(400_000_000)           # some 0.2 s
            mod.step(x, y)
            if not apart:
                mod.set_hyper_params(learning_rate=0.5)
        if apart:
            mod.set_hyper_params(learning_rate=0.5)
        with torch.cuda.stream(st):
            mod.step(x, y)
            mod.step(x, y, capture=True)
            st.synchronize()
            ends.append({k: v.clone() for k, v in mod.captured.items()})
            mod.close()
    assert all(torch.equal(ends[0][k], ends[1][k]) for k in ends[0])


def test_group_norms_whose_inputs_are_evicted_and_in_graphs_train_alike():
    """Parameters after ten steps to the last bit, of which the last ones are replays, or have their activations fetched back."""
    make = lambda: Net("n", Input(cpad=8), [GroupNorm("g0", 4, act="relu"), GroupNorm("g1", 2, act="silu"), GroupNorm("g2", 8), GroupNorm("g3", 4, act="relu"),
                                            Linear("f1", 32, relu=True, std=0.01, fp8=True), Linear("fc", 10, std=0.3, fp32_out=True, fp8=True)])
    gen = torch.Generator(device=DEV).manual_seed(5)
    x, y = torch.randn(16, 3, 64, 64, generator=gen, device=DEV), torch.randint(0, 10, (16,), generator=gen, device=DEV)
    ends = []
    for kw in (dict(), dict(use_graph=True), dict(manage_activations=True, cache_fraction=0.0)):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            mod = module(make=make, shape=(16, 3, 64, 64), adamw=dict(bits=8, seed=2), **kw)
            if "cache_fraction" in kw:
                assert len(mod.managed) == 4 and mod.budget_rows < mod.working_set_rows            # not all of them fit
            for _ in range(10):
                mod.step(x, y)
            assert "use_graph" not in kw or mod.is_steady(x, y), mod.tape_mismatch
            mod.step(x, y, capture=True)
            st.synchronize()
            ends.append({k: v.clone() for k, v in mod.captured.items()})
            mod.close()
    first = ends[0]
    assert all(v.isfinite().all() for v in first.values()) and (first["g0.gamma"] != 1).any() and (first["g3.beta"] != 0).any()
    for other in ends[1:]:
        assert other.keys() == first.keys() and all(torch.equal(other[k], first[k]) for k in first), [k for k in first if not torch.equal(other[k], first[k])]


def test_two_workers_give_half_of_their_own_steps_each():
    """The updates that an additive table gets from two workers with gradients of their own: the mean of their steps, each clipped by
    its own norm.  Each change is within 2^-18 of itself, and an fp32 rounding of the quantities that it is the sum of."""
    from types import SimpleNamespace as Space

    from geeps_b200.parallel.ps_module import _AdamW
    gen = torch.Generator(device=DEV).manual_seed(8)
    sizes, world = {"weight": 3000, "bias": 70}, 2
    p = {k: torch.randn(n, generator=gen, device=DEV) for k, n in sizes.items()}
    workers = [_AdamW(DEV, world, 0.02, 0.1, rank=r) for r in range(world)]
    state = [{k: (torch.zeros(n, device=DEV, dtype=F64), torch.zeros(n, device=DEV, dtype=F64)) for k, n in sizes.items()} for _ in workers]
    mods = [Space(steps=0, _period=2, clip_gradients=1.5, _clip_work=None, clip_result=torch.zeros(2, device=DEV), device=DEV) for _ in workers]
    for step in range(1, 4):
        total, want, size = ({k: torch.zeros(n, device=DEV, dtype=F64) for k, n in sizes.items()} for _ in range(3))
        for w, mod, s in zip(workers, mods, state):
            g = {k: 0.1 * torch.randn(n, generator=gen, device=DEV) for k, n in sizes.items()}
            norm = sum(v.to(F64).square().sum() for v in g.values()).sqrt()
            c = min(1.0, 1.5 / norm.item())
            assert c < 1.0
            for k in sizes:
                m, v = s[k]
                m.mul_(0.9).add_(0.1 * c * g[k].to(F64))
                v.mul_(0.999).add_(0.001 * (c * g[k].to(F64)).square())
                own = -0.02 * (m / (1 - 0.9 ** step) / ((v / (1 - 0.999 ** step)).sqrt() + 1e-8) + (0.1 * p[k].to(F64) if k == "weight" else 0.0))
                want[k] += own / world
                # m is a sum of signed terms: its roundings go by their sizes, of which a step's 0.1 g is the largest part
                size[k] += 0.02 / world * (0.9 * m.abs() + c * g[k].to(F64).abs()) / (v / (1 - 0.999 ** step)).sqrt() + own.abs() / world
            layer = Space(p32=p, g32=g)
            mod.tables, mod.steps = [Space(layer=layer, specs=[Space(name="weight", decay=True), Space(name="bias", decay=False)])], step - 1
            w.begin()
            w.step(mod)
            for k in sizes:
                total[k] += g[k].to(F64)
        for k in sizes:
            assert ((total[k] - want[k]).abs() <= 2.0 ** -18 * size[k]).all()
            p[k] += want[k].float()
