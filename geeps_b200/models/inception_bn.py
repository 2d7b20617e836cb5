"""Inception-BN family: the small 32x32 variant (CIFAR-shaped) and the ImageNet-22K-shaped
GoogLeNet-BN with a 1024 x 21841 classifier.  norm="group" puts a group norm with its ReLU in the place of every BatchNorm."""
from __future__ import annotations

from ..ops.layers import BatchNorm, Conv2d, GroupNorm, Input, Linear, Pool
from .net import Concat, Net


def norm_groups(channels: int) -> int:
    """Groups of a group norm: 32, or the largest power of two below that divides the channels."""
    return next(g for g in (32, 16, 8, 4, 2, 1) if channels % g == 0)


class _Norms:
    """Convolutions with a norm and a ReLU behind them, and the modules made of them."""

    def __init__(self, norm: str):
        if norm not in ("batch", "group"):
            raise ValueError(f"unknown norm {norm!r}; batch or group")
        self.norm = norm

    def conv(self, name, cout, k, stride=1, pad=0, need_dx=True):
        behind = BatchNorm(name + "_bn", relu=True) if self.norm == "batch" else GroupNorm(name + "_gn", norm_groups(cout), act="relu")
        return [Conv2d(name, cout, k, stride=stride, pad=pad, bias=False, std=0.0, need_dx=need_dx), behind]


def _module(conv, name, c1, c3):
    return Concat(name, [conv(name + "_1x1", c1, 1), conv(name + "_3x3", c3, 3, pad=1)])


def _downsample(conv, name, c3):
    return Concat(name, [conv(name + "_3x3", c3, 3, stride=2, pad=1), [Pool("max", 3, 2, pad=1, ceil_mode=False)]])


def inception_bn_small(num_classes: int = 10, norm: str = "batch") -> Net:
    """conv3x3-96; modules (32|32), (32|48); downsample (80|pool); modules (112|48), (96|64),
    (80|80), (48|96); downsample (96|pool); modules (176|160) x2; global avgpool; FC."""
    conv = _Norms(norm).conv
    layers = conv("conv1", 96, 3, pad=1, need_dx=False)
    layers += [_module(conv, "in3a", 32, 32), _module(conv, "in3b", 32, 48), _downsample(conv, "in3c", 80)]
    layers += [_module(conv, "in4a", 112, 48), _module(conv, "in4b", 96, 64), _module(conv, "in4c", 80, 80), _module(conv, "in4d", 48, 96),
               _downsample(conv, "in4e", 96)]
    layers += [_module(conv, "in5a", 176, 160), _module(conv, "in5b", 176, 160)]
    layers += [Pool("avg", 0, 1, ceil_mode=False), Linear("fc", num_classes, std=0.01, fp32_out=True)]
    return Net("inception_bn_small", Input(cpad=8), layers)


def _inception(conv, name, c1, c3r, c3, cd3r, cd3, pool, cproj):
    """GoogLeNet-BN module: 1x1 | 1x1-3x3 | 1x1-3x3-3x3 | pool-1x1."""
    branches = []
    if c1:
        branches.append(conv(name + "_1x1", c1, 1))
    branches.append(conv(name + "_3x3r", c3r, 1) + conv(name + "_3x3", c3, 3, pad=1))
    branches.append(conv(name + "_d3r", cd3r, 1) + conv(name + "_d3a", cd3, 3, pad=1)
                    + conv(name + "_d3b", cd3, 3, pad=1))
    branches.append([Pool(pool, 3, 1, pad=1, ceil_mode=False)] + conv(name + "_proj", cproj, 1))
    return Concat(name, branches)


def _inception_down(conv, name, c3r, c3, cd3r, cd3):
    """Stride-2 module: 1x1-3x3/2 | 1x1-3x3-3x3/2 | maxpool/2."""
    return Concat(name, [
        conv(name + "_3x3r", c3r, 1) + conv(name + "_3x3", c3, 3, stride=2, pad=1),
        conv(name + "_d3r", cd3r, 1) + conv(name + "_d3a", cd3, 3, pad=1)
        + conv(name + "_d3b", cd3, 3, stride=2, pad=1),
        [Pool("max", 3, 2, pad=1, ceil_mode=False)],
    ])


def inception_bn_22k(num_classes: int = 21841, norm: str = "batch") -> Net:
    """GoogLeNet-BN trunk (224x224 input, 1024-wide final feature) + a 1024 x 21841 classifier."""
    conv = _Norms(norm).conv
    layers = conv("conv1", 64, 7, stride=2, pad=3, need_dx=False) + [Pool("max", 3, 2, ceil_mode=True)]
    layers += conv("conv2r", 64, 1) + conv("conv2", 192, 3, pad=1) + [Pool("max", 3, 2, ceil_mode=True)]
    layers += [
        _inception(conv, "in3a", 64, 64, 64, 64, 96, "avg", 32),
        _inception(conv, "in3b", 64, 64, 96, 64, 96, "avg", 64),
        _inception_down(conv, "in3c", 128, 160, 64, 96),
        _inception(conv, "in4a", 224, 64, 96, 96, 128, "avg", 128),
        _inception(conv, "in4b", 192, 96, 128, 96, 128, "avg", 128),
        _inception(conv, "in4c", 160, 128, 160, 128, 160, "avg", 128),
        _inception(conv, "in4d", 96, 128, 192, 160, 192, "avg", 128),
        _inception_down(conv, "in4e", 128, 192, 192, 256),
        _inception(conv, "in5a", 352, 192, 320, 160, 224, "avg", 128),
        _inception(conv, "in5b", 352, 192, 320, 192, 224, "max", 128),
        Pool("avg", 0, 1, ceil_mode=False),
        Linear("fc", num_classes, std=0.01, fp32_out=True),
    ]
    return Net("inception_bn_22k", Input(cpad=8), layers)
