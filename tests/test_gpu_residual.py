"""Residual blocks as layers of a network, and clipping of a training step's gradients: what a program uses together.

Gradients of the layers are compared with those of torch autograd on the same bf16 values in fp64.  Every tensor between two
layers is rounded to bf16 (half a step, 2^-8 of its value), forward and backward; a path through a block has some ten of them, and
their errors are independent, so the relative error of a gradient as a whole (norm of the difference over the norm) stays
below 10 * 2^-8 by a wide margin.  A ReLU's mask is taken from the layer: its gradient jumps where a rounding carries a value
across zero, and a share q of such values alone is a relative error of sqrt(q) (2^-8 of the values: 6 %), whatever the kernels do."""
import pytest
import torch
import torch.nn.functional as TF

from geeps_b200.models.net import Net, Residual
from geeps_b200.ops.layers import Conv2d, Input, Linear, Norm, Pool
from geeps_b200.parallel.ps_module import PSModule
from geeps_b200.utils.config import DEVICE_CUDA, TABLE_SGD_MOMENTUM, TRANSPORT_NVLINK, TRANSPORT_TCP, GeePsConfig

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, F64 = torch.bfloat16, torch.float64
TOL = 10 * 2.0 ** -8
_port = [28400]


def cfg(transport=TRANSPORT_NVLINK, **kw):
    _port[0] += 20
    base = dict(device=DEVICE_CUDA, cuda_device=0, transport=transport, table_mode=TABLE_SGD_MOMENTUM, tcp_base_port=_port[0],
                bf16_compute_cache=1, learning_rate=0.05, momentum=0.0)
    base.update(kw)
    return GeePsConfig(**base)


def block(name, c, post=None, pre="layer", scale=None, gate=None):
    if gate == "image":
        gate = [Pool("avg", 0, 1, ceil_mode=False), Linear(name + "_g1", 16, relu=True, std=0.3), Linear(name + "_g2", c, std=0.3)]
    elif gate == "pixel":
        gate = [Conv2d(name + "_g", c, 1, std=0.2)]
    return Residual(name, [Conv2d(name + "_a", 2 * c, 3, pad=1, relu=True, std=0.08), Conv2d(name + "_b", c, 1, std=0.12)], pre=pre, post=post,
                    scale=scale, gate=gate)


def bind(layers, seed):
    """Parameters of their own for every layer, and buffers for their gradients."""
    gen = torch.Generator().manual_seed(seed)
    subs = [s for l in layers for s in (l.sublayers() if hasattr(l, "sublayers") else [l])]
    for l in subs:
        for sp in l.param_specs():
            v = sp.initial(gen)
            if sp.init.startswith("const"):
                v = v + 0.2 * torch.randn(v.shape, generator=gen)
            l.p32[sp.name] = v.to(DEV)
            l.p16[sp.name] = v.to(DEV).to(BF)
            l.g32[sp.name] = torch.full(sp.shape, 7.0, device=DEV)
    return subs


class Twin:
    """The same blocks in fp64 on leaves that hold the layers' values."""

    def __init__(self, layers):
        self.leaf = {}
        self.layers = layers

    def p(self, l, name):
        key = (id(l), name)
        if key not in self.leaf:
            v = l.p16[name] if isinstance(l, (Conv2d, Linear)) and name == "weight" else l.p32[name]
            self.leaf[key] = (l, name, v.double().requires_grad_(True))
        return self.leaf[key][2]

    def norm(self, x, layer, kind, prefix, eps):
        mean = x.mean(-1, keepdim=True) if kind == "layer" else 0.0
        n = (x - mean) * ((x - mean).square().mean(-1, keepdim=True) + eps) ** -0.5
        n = n * self.p(layer, prefix + "gamma")
        return n + self.p(layer, prefix + "beta") if prefix + "beta" in layer.p32 else n

    def run(self, l, x):
        if isinstance(l, Norm):
            return self.norm(x, l, l.kind, "", l.eps)
        if isinstance(l, Conv2d):
            w = self.p(l, "weight")[:, :l.kd].reshape(l.cout, l.k, l.k, l.cg).permute(0, 3, 1, 2)
            y = TF.conv2d(x.permute(0, 3, 1, 2), w, self.p(l, "bias"), l.stride, l.pad).permute(0, 2, 3, 1)
            return y * (l.y.view(y.shape) > 0) if l.relu else y
        if isinstance(l, Pool):
            return x.mean((1, 2), keepdim=True)
        if isinstance(l, Linear):
            y = x.flatten(1) @ self.p(l, "weight").t() + self.p(l, "bias")
            return y * (l.y.view(y.shape) > 0) if l.relu else y
        h = x
        if l.pre:
            owner = self.owner.get(id(l.pre))
            h = self.norm(h, owner or l.pre, l.pre.kind, "next_" if owner else "", l.pre.eps)
        for s in l.layers:
            h = self.run(s, h)
        b = h
        if l.join.post:
            b = self.norm(b, l.join, l.join.post.kind, "", l.join.post.eps)
        if l.gate:
            g = h
            for s in l.gate:
                g = self.run(s, g)
            g = torch.sigmoid(g) if l.join.sigmoid else g
            b = b * (g if g.dim() == 4 else g[:, None, None, :])
        if l.join.scale is not None:
            b = b * self.p(l.join, "scale")
        return x + b

    def forward(self, x):
        self.owner = {id(l.join.next): l.join for l in self.layers if isinstance(l, Residual) and l.join.next}
        for l in self.layers:
            x = self.run(l, x)
        return x


def off(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


@pytest.mark.parametrize("kinds", [
    [dict(pre="layer")], [dict(pre=None, post="layer")], [dict(pre="rms", post="rms", scale=0.5, gate="image")], [dict(pre="rms", gate="pixel", scale=0.7)],
    [dict(pre="layer", post="layer", gate="image"), dict(pre="rms", scale=0.3), dict(pre=None, gate="pixel"), dict(pre="layer", post="rms")],
])
def test_blocks_have_the_gradients_of_autograd(kinds):
    shape, c = (4, 6, 6, 24), 24          # global pooling is of square images; others are refused (below)
    net = Net("n", Input(), [block(f"b{i}", c, **k) for i, k in enumerate(kinds)] + [Norm("last", "layer"), Pool("avg", 0, 1, ceil_mode=False),
                                                                                     Linear("fc", 16, std=0.3, fp32_out=True)])
    s = shape
    for l in net.layers:
        s = l.setup(s, DEV)
    for a, b in zip(net.layers, net.layers[1:]):
        if isinstance(a, Residual) and isinstance(b, Residual):
            a.link(b)
    layers = net.layers[:-2]
    subs = bind(layers, 3)
    x = torch.randn(shape, generator=torch.Generator().manual_seed(1)).to(DEV).to(BF)
    h = x
    for l in layers:
        h = l.forward(h)
    dy = torch.randn(h.shape, generator=torch.Generator().manual_seed(2)).to(DEV).to(BF)
    d = dy
    for l in reversed(layers):
        d = l.backward(d)
    twin, x64 = Twin(layers), x.double().requires_grad_(True)
    y64 = twin.forward(x64)
    assert off(h.view(y64.shape), y64.detach()) <= TOL
    leaves = list(twin.leaf.values())
    assert {(id(l), n) for l, n, _ in leaves} == {(id(l), sp.name) for l in subs for sp in l.param_specs()}
    grads = torch.autograd.grad(y64, [x64] + [t for _, _, t in leaves], dy.double().view(y64.shape))
    assert off(d.view(shape), grads[0]) <= TOL
    for (l, name, _), g in zip(leaves, grads[1:]):
        assert off(l.g32[name], g) <= TOL, (l.name, name)


def small_net():
    return Net("small", Input(cpad=8), [Conv2d("c0", 24, 3, pad=1, std=0.2, need_dx=False), block("b1", 24, pre="layer", post="rms", scale=0.5, gate="image"),
                                        block("b2", 24, pre="rms", scale=0.5), Norm("n", "layer"), Pool("avg", 0, 1, ceil_mode=False),
                                        Linear("fc", 10, std=0.3, fp32_out=True)])


def test_a_net_links_blocks_and_counts_their_parameters():
    net = small_net()
    net.setup((4, 3, 8, 8), DEV)
    b1, b2 = net.layers[1], net.layers[2]
    assert b1.follower is b2 and b2.pre.joined and b2.pre.param_specs() == []
    assert [s.name for s in b1.join.param_specs()] == ["gamma", "scale", "next_gamma"]
    names = [l.name for l in net.param_layers()]
    assert "b1_join" in names and "b2_pre" not in names and "b1_g1" in names


def batch(n=8):
    gen = torch.Generator(device=DEV).manual_seed(5)
    return torch.randn(n, 3, 8, 8, generator=gen, device=DEV), torch.randint(0, 10, (n,), generator=gen, device=DEV)


def step_change(clip, transport, **kw):
    """Parameters before and after one step, and the step's {norm, factor}."""
    mod = PSModule(small_net(), (8, 3, 8, 8), cfg(transport), device="cuda:0", seed=4, clip_gradients=clip, **kw)
    x, y = batch()
    mod.step(x, y, capture=True)
    before = {k: v.clone() for k, v in mod.captured.items()}
    result = mod.clip_result.tolist() if clip is not None else None
    mod.step(x, y, capture=True)
    after = {k: v.clone() for k, v in mod.captured.items()}
    torch.cuda.synchronize()
    mod.close()
    return before, after, result


@pytest.mark.parametrize("transport", [TRANSPORT_NVLINK, TRANSPORT_TCP])
def test_a_clipped_step_changes_the_parameters_by_the_scaled_gradients(transport):
    b0, a0, _ = step_change(None, transport)
    b1, a1, r1 = step_change(float("inf"), transport)
    lr = 0.05
    norm = sum(((a0[k] - b0[k]).double() / lr).square().sum().item() for k in b0) ** 0.5
    # a difference of parameters is off by the rounding of the parameters themselves, 2^-24 of them over the rate
    size = sum(b0[k].double().square().sum().item() for k in b0) ** 0.5
    assert abs(r1[0] - norm) <= 2.0 ** -23 * size / lr + 1e-3 * norm and r1[1] == 1.0
    bound = norm / 4
    b2, a2, r2 = step_change(bound, transport)
    assert abs(r2[1] - bound / r2[0]) <= 2.0 ** -22
    for k in b0:
        assert torch.equal(b0[k], b1[k]) and torch.equal(b0[k], b2[k])
        full, cut = (a0[k] - b0[k]).double(), (a2[k] - b2[k]).double()
        assert ((cut - full * r2[1]).abs() <= 2.0 ** -22 * b0[k].double().abs() + 2.0 ** -22 * full.abs() + 2e-3 * full.abs().max()).all(), k


def same_training(losses):
    """The loss is a sum of a batch's terms in any order, which is all that may differ in the first step (64 of them at the most,
    a rounding each); from then on slices of weight gradients have met in fp32 atomics in any order, whose differences cross
    roundings of weights and activations to bf16 here and there: the bound is this suite's for runs that differ in that."""
    for other in losses[1:]:
        assert abs(other[0] - losses[0][0]) <= 64 * 2.0 ** -24 * abs(losses[0][0])
        assert torch.allclose(torch.tensor(other), torch.tensor(losses[0]), rtol=1e-3), losses


def test_blocks_and_clipping_train_alike_with_graphs_recorded_steps_and_neither():
    x, y = batch()
    losses = []
    for kw in (dict(), dict(use_tape=True), dict(use_graph=True)):
        torch.manual_seed(0)
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            mod = PSModule(small_net(), (8, 3, 8, 8), cfg(TRANSPORT_NVLINK, momentum=0.9), device="cuda:0", seed=4, clip_gradients=0.5, **kw)
            out = [mod.step(x, y).clone() for _ in range(10)]
            st.synchronize()
            assert not kw or mod.is_steady(x, y), mod.tape_mismatch
            assert mod.clip_result[0].item() > 0
            losses.append([v.item() for v in out])
            mod.close()
    same_training(losses)


def test_blocks_train_with_managed_activations():
    x, y = batch(64)

    def run(**kw):
        mod = PSModule(Net("m", Input(cpad=8), [Conv2d("c0", 24, 3, pad=1, std=0.2, need_dx=False), block("b1", 24, pre="layer", scale=0.5, gate="image"),
                                                block("b2", 24, pre="layer"), Pool("avg", 0, 1, ceil_mode=False), Linear("fc", 10, std=0.3, fp32_out=True)]),
                       (64, 3, 32, 32), cfg(), device="cuda:0", seed=4, **kw)
        xs = torch.randn(64, 3, 32, 32, generator=torch.Generator(device=DEV).manual_seed(6), device=DEV)
        out = [mod.step(xs, y).item() for _ in range(3)]
        n = len(mod.managed)
        mod.close()
        return out, n
    plain, none = run()
    capped, managed = run(manage_activations=True, cache_fraction=0.5, clip_gradients=float("inf"))
    assert none == 0 and managed >= 3
    same_training([plain, capped])


def test_refusals():
    with pytest.raises(ValueError, match="keeps the shape"):
        Residual("r", [Conv2d("c", 16, 3, pad=1)]).setup((2, 4, 4, 24), DEV)
    with pytest.raises(ValueError, match="square"):
        block("r", 24, gate="image").setup((2, 6, 5, 24), DEV)
    with pytest.raises(ValueError, match="gate"):
        Residual("r", [Conv2d("c", 24, 3, pad=1)], gate=[Conv2d("g", 16, 1)]).setup((2, 4, 4, 24), DEV)
    with pytest.raises(ValueError, match="clip_gradients"):
        PSModule(small_net(), (8, 3, 8, 8), cfg(), device="cuda:0", clip_gradients=-1.0)
