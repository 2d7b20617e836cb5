"""Clipping of gradients by their global norm against the definition in 64 bits.

Tolerances: the squares are added in 64 bits, so the norm is off by its one rounding to fp32 (2^-24) and the coefficient by
its own; a gradient takes the coefficient's, the product's and, in bf16, its storage's rounding.
"""
import math

import pytest
import torch

from geeps_b200.ops import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24


def norm64(grads):
    return math.sqrt(math.fsum((g.double() ** 2).sum().item() for g in grads))


def check(grads, max_norm, out=None, lists=False):
    before = [g.clone() for g in grads]
    norm = norm64(before)
    c = max_norm / norm if norm > max_norm else 1.0
    result = torch.full((2,), -1.0, device=DEV)
    if lists:
        F.clip_gradients(F.GradList(grads), max_norm, result, out=None if out is None else F.GradList(out))
    else:
        F.clip_gradients(grads, max_norm, result, out=out)
    got = [float(v) for v in result.cpu()]
    assert abs(got[0] - norm) <= 2 * U * norm and abs(got[1] - c) <= 2 * U * c, (got, norm, c)
    for i, (g, b, o) in enumerate(zip(grads, before, grads if out is None else out)):
        if out is not None:
            assert torch.equal(g, b), i
        if c == 1.0 and o.dtype == b.dtype:
            assert torch.equal(o, b), i
            continue
        ref = b.double() * c
        half = torch.finfo(BF).eps / 2 if o.dtype == BF else 0.0
        assert ((o.double() - ref).abs() <= (half + 3 * U) * ref.abs() * (1 + half) + 2.0 ** -149).all(), i


def grads_of(sizes, dtype, seed=0, size=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return [(torch.randn(n, generator=gen, device=DEV) * size).to(dtype) for n in sizes]


@pytest.mark.parametrize("sizes", [[1], [7], [8], [9, 1, 17], [1024], [8191, 8192, 8193], [100003], [1, 2, 3, 0, 5, 70000, 33], [300001, 5, 2000000],
                                   [13] * 70, [257] * 1500, [0], [4194304]])
@pytest.mark.parametrize("src,dst", [(F32, None), (BF, None), (F32, F32), (BF, F32), (F32, BF), (BF, BF)])
def test_clips_like_the_definition(sizes, src, dst):
    grads = grads_of(sizes, src, len(sizes))
    norm = norm64(grads)
    for ratio in (4.0, 0.5):
        out = None if dst is None else [torch.full((n,), 7.0, dtype=dst, device=DEV) for n in sizes]
        check([g.clone() for g in grads], norm / ratio, out, lists=ratio > 1)


@pytest.mark.parametrize("a,b", [(1, 1), (1, 2), (3, 0), (0, 5), (8, 4)])
@pytest.mark.parametrize("src,dst", [(F32, F32), (BF, F32), (F32, BF), (BF, BF)])
def test_odd_addresses_and_nothing_beside_them(a, b, src, dst):
    n = 30011
    src_flat, dst_flat = grads_of([n + 16], src)[0], torch.full((n + 16,), 7.0, dtype=dst, device=DEV)
    check([src_flat[a:a + n]], 3.0, [dst_flat[b:b + n]])
    assert (dst_flat[:b] == 7).all() and (dst_flat[b + n:] == 7).all()
    keep = src_flat.clone()
    check([src_flat[a:a + n]], 2.0)
    assert torch.equal(src_flat[:a], keep[:a]) and torch.equal(src_flat[a + n:], keep[a + n:])


def test_types_mixed_in_one_list_and_shapes():
    g = [torch.randn(64, 3, 5, device=DEV), torch.randn(77, device=DEV).to(BF), torch.randn(1, device=DEV), torch.randn((), device=DEV)]
    check(g, 1.5)


def test_bounds_and_extremes():
    check(grads_of([1000], F32, 1, 1e30), 1.0)              # squares beyond fp32
    check(grads_of([1000], F32, 2, 1e-30), 1e-31)           # ... and below
    g = grads_of([999, 3], F32, 3)
    check(g, float("inf"))
    check(g, 0.0)
    assert all((t == 0).all() for t in g)
    check(g, 0.0)                                            # a norm of zero: nothing to clip
    check([torch.full((4,), 2.0, device=DEV)], 4.0)          # the bound itself


def test_no_tensors():
    r = torch.full((2,), 7.0, device=DEV)
    F.clip_gradients([], 1.0, r)
    assert r.tolist() == [0.0, 1.0]


def test_norms_that_are_not_finite():
    g = [torch.ones(100, device=DEV), torch.ones(50, device=DEV)]
    g[1][7] = float("inf")
    r = torch.zeros(2, device=DEV)
    F.clip_gradients(g, 1.0, r)
    assert math.isinf(r[0].item()) and r[1].item() == 0.0
    assert (g[0] == 0).all() and torch.isnan(g[1][7]) and (g[1][:7] == 0).all()
    g = [torch.ones(100, device=DEV)]
    g[0][3] = float("nan")
    F.clip_gradients(g, 1.0, r)
    assert math.isnan(r[0].item()) and r[1].item() == 1.0 and g[0][0].item() == 1.0 and torch.isnan(g[0][3])


def test_results_repeat_bit_for_bit_and_do_not_depend_on_addresses():
    flat = grads_of([3_000_000], F32, 5)[0]
    r = [torch.zeros(2, device=DEV) for _ in range(3)]
    F.clip_gradients([flat], float("inf"), r[0])
    F.clip_gradients([flat], float("inf"), r[1])
    F.clip_gradients([flat.clone()], float("inf"), r[2])
    assert torch.equal(r[0], r[1]) and torch.equal(r[0], r[2])


def test_a_list_reads_its_tensors_anew_and_replays_in_graphs():
    g = grads_of([5000, 300_000], F32, 6)
    glist, r, r2 = F.GradList(g), torch.zeros(2, device=DEV), torch.zeros(2, device=DEV)
    out, out2 = [torch.empty_like(t) for t in g], [torch.empty_like(t) for t in g]
    F.clip_gradients(glist, 1.0, r, out=out)
    graphs = []
    for res, o in ((r, out), (r2, out2)):           # two graphs of one list, at once
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            F.clip_gradients(glist, 2.0, res, out=o)
        graphs.append(graph)
    for t in g:
        t.mul_(3.0)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    norm = norm64(g)
    for res, o in ((r, out), (r2, out2)):
        assert abs(res[0].item() - norm) <= 2 * U * norm
        assert abs(norm64(o) - 2.0) <= 2.0 * 4 * U


def test_more_elements_than_32_bits_of_bytes():
    n = (1 << 31) // 2 + 12345                     # bf16: more than 2^31 bytes
    g = torch.zeros(n, dtype=BF, device=DEV)
    g[0], g[n - 1], g[n // 2] = 3.0, 4.0, 12.0
    r = torch.zeros(2, device=DEV)
    F.clip_gradients([g], 6.5, r)
    assert r.tolist() == [13.0, 0.5]
    assert g[0].item() == 1.5 and g[n - 1].item() == 2.0 and g[n // 2].item() == 6.0


def test_refusals():
    g, r = torch.zeros(100, device=DEV), torch.zeros(2, device=DEV)
    with pytest.raises(ValueError, match="shares memory"):
        F.clip_gradients([g, g], 1.0, r)
    with pytest.raises(ValueError, match="shares memory"):
        F.clip_gradients([g[:60], g[59:]], 1.0, r)
    with pytest.raises(ValueError, match="contiguous"):
        F.clip_gradients([g[::2]], 1.0, r)
    with pytest.raises(ValueError, match="bf16"):
        F.clip_gradients([g.half()], 1.0, r)
    with pytest.raises(ValueError, match="device"):
        F.clip_gradients([g.cpu()], 1.0, r)
    with pytest.raises(ValueError, match="max_norm"):
        F.clip_gradients([g], -1.0, r)
    with pytest.raises(ValueError, match="max_norm"):
        F.clip_gradients([g], float("nan"), r)
    with pytest.raises(ValueError, match="counts"):
        F.clip_gradients([g], 1.0, r, out=[g[:50]])
    with pytest.raises(ValueError, match="overlap"):
        F.clip_gradients([g[:50], g[50:]], 1.0, r, out=[g[50:], g[:50]])
    with pytest.raises(ValueError, match="overlap"):
        F.clip_gradients([g[:50]], 1.0, r, out=[g[25:75]])
    with pytest.raises(ValueError, match="result"):
        F.clip_gradients([g], 1.0, r[:1])
    with pytest.raises(ValueError, match="result"):
        F.clip_gradients([g], 1.0, r.double())
    g.fill_(1.0)                                    # out may be the gradients themselves
    F.clip_gradients([g], 5.0, r, out=[g])
    assert r.tolist() == [10.0, 0.5] and (g == 0.5).all()
