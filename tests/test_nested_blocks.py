"""Containers inside of containers: residual blocks in a branch, branches in a residual block."""
import pytest
import torch

from geeps_b200.models.net import Concat, Net, Residual
from geeps_b200.ops.layers import Conv2d, Input, Linear, Norm, Pool

BF = torch.bfloat16


def block(name, c):
    return Residual(name, [Conv2d(name + "_a", c, 3, pad=1, relu=True, std=0.1), Conv2d(name + "_b", c, 1, std=0.2)], pre="layer", post="rms", scale=0.5,
                    gate=[Conv2d(name + "_g", c, 1, std=0.2)])


def branches():
    """A block at the end of a branch (its output is a slice), one in front of a convolution, and branches inside of a block."""
    inner = Concat("in", [[Conv2d("i0", 8, 1, relu=True, std=0.2)], [block("r2", 16), Conv2d("i1", 8, 1, std=0.2)]])
    return Concat("m", [[Conv2d("c0", 24, 1, std=0.2), block("r0", 24)], [block("r1", 16), Conv2d("c1", 8, 3, pad=1, std=0.1)],
                        [Residual("r3", [inner], pre="rms")]])


def net():
    return Net("nested", Input(cpad=8), [Conv2d("first", 16, 3, pad=1, std=0.2, need_dx=False), branches(), Norm("n", "layer"), Pool("avg", 0, 1, ceil_mode=False),
                                         Linear("fc", 10, std=0.3, fp32_out=True)])


NAMES = {"first", "c0", "r0_pre", "r0_a", "r0_b", "r0_g", "r0_join", "r1_pre", "r1_a", "r1_b", "r1_g", "r1_join", "c1", "r3_pre", "i0", "r2_pre", "r2_a", "r2_b",
         "r2_g", "r2_join", "i1", "n", "fc"}


def test_every_layer_with_parameters_is_found():
    n = net()
    n.setup((2, 3, 6, 6), torch.device("cpu"))
    assert {l.name for l in n.param_layers()} == NAMES
    assert n.num_params() == sum(sp.num_valid() for l in n.all_layers() for sp in l.param_specs())
    assert not any(isinstance(l, (Concat, Residual)) for l in n.all_layers())


def test_the_mode_reaches_every_layer():
    n = net()
    n.setup((2, 3, 6, 6), torch.device("cpu"))
    n.train(False)
    assert not any(l.training for l in n.all_layers()) and {l.name for l in n.all_layers()} >= NAMES


def losses(steps=6, concurrent=True, **kw):
    from geeps_b200.parallel.ps_module import PSModule
    from test_gpu_residual import cfg
    n = net()
    for l in [m for m in n.layers if isinstance(m, Concat)]:
        l.concurrent = concurrent
    gen = torch.Generator(device="cuda:0").manual_seed(5)
    x, y = torch.randn(8, 3, 8, 8, generator=gen, device="cuda:0"), torch.randint(0, 10, (8,), generator=gen, device="cuda:0")
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        mod = PSModule(n, (8, 3, 8, 8), cfg(momentum=0.9), device="cuda:0", seed=4, **kw)
        first = None
        out = []
        for i in range(steps):
            out.append(mod.step(x, y, capture=i < 2).clone())
            if i < 2:
                now = {k: v.clone() for k, v in mod.captured.items()}
                first, moved = (now, None) if i == 0 else (first, {k for k in now if not torch.equal(first[k], now[k])})
        stream.synchronize()
        mod.close()
    assert {k.split(".")[0] for k in moved} == NAMES            # every layer's parameters are trained
    return [v.item() for v in out]


@pytest.mark.gpu
def test_nested_blocks_train_with_and_without_streams_and_graphs():
    from test_gpu_residual import same_training
    same_training([losses(steps=10), losses(steps=10, concurrent=False), losses(steps=10, use_graph=True), losses(steps=10, clip_gradients=float("inf"))])


@pytest.mark.gpu
def test_nested_blocks_have_the_gradients_of_autograd():
    """Tolerance: as for blocks in a row; the longest way through these has thirty roundings to bf16, whose errors are independent:
    sqrt(30) of half a step at the most is 5.5 * 2^-8."""
    from test_gpu_residual import TOL, Twin, bind, off

    class Nested(Twin):
        def run(self, l, x):
            if isinstance(l, Concat):
                outs = []
                for br in l.branches:
                    h = x
                    for s in br:
                        h = self.run(s, h)
                    outs.append(h)
                return torch.cat(outs, -1)
            return super().run(l, x)
    dev, shape = torch.device("cuda:0"), (4, 6, 6, 16)
    m = branches()
    m.setup(shape, dev)
    subs = bind([m], 3)
    x = torch.randn(shape, generator=torch.Generator().manual_seed(1)).to(dev).to(BF)
    y = m.forward(x)
    dy = torch.randn(y.shape, generator=torch.Generator().manual_seed(2)).to(dev).to(BF)
    dx = m.backward(dy.clone())
    twin, x64 = Nested([m]), x.double().requires_grad_(True)
    y64 = twin.forward(x64)
    assert off(y.view(y64.shape), y64.detach()) <= TOL
    leaves = list(twin.leaf.values())
    assert {(id(l), k) for l, k, _ in leaves} == {(id(l), sp.name) for l in subs for sp in l.param_specs()}
    grads = torch.autograd.grad(y64, [x64] + [t for _, _, t in leaves], dy.double().view(y64.shape))
    assert off(dx.view(shape), grads[0]) <= TOL
    for (l, k, _), g in zip(leaves, grads[1:]):
        assert off(l.g32[k], g) <= TOL, (l.name, k)
