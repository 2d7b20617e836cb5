"""Host side of group norm, AdamW steps and 8-bit products: launch shapes, workspaces and refusals, which need no GPU."""
import copy
import ctypes as C
import os
import pickle
import subprocess
import sys

import pytest
import torch

from geeps_b200 import train
from geeps_b200.models.inception_bn import inception_bn_22k, inception_bn_small, norm_groups
from geeps_b200.ops import _lib as L
from geeps_b200.ops import functional as F
from geeps_b200.ops.layers import BatchNorm, GroupNorm

A, B, D = 1 << 32, 1 << 36, 1 << 40          # addresses that are never touched: every call here is refused


def shape(images, pixels, c, groups, backward, vec, types):
    out = (C.c_int * 9)()
    assert L.lib().geeps_group_norm_shape(C.c_longlong(images), C.c_longlong(pixels), c, groups, int(backward), int(vec), *types, out) == 0
    return list(out)


def work(images, pixels, c, groups, backward):
    return L.lib().geeps_group_norm_work(C.c_longlong(images), C.c_longlong(pixels), c, groups, int(backward))


@pytest.mark.parametrize("c,groups", [(1, 1), (8, 1), (8, 8), (24, 8), (96, 32), (192, 32), (576, 32), (1003, 17), (1024, 1), (2048, 1), (2056, 1), (4096, 32),
                                      (16384, 1), (16384, 16384), (16383, 3), (16381, 16381), (16376, 23)])
@pytest.mark.parametrize("images,pixels", [(1, 1), (1, 7), (3, 196), (256, 196), (32, 3136), (1, 1 << 30), (1 << 16, 4), (2, 50176)])
def test_group_norm_shapes_cover_the_pixels_within_the_launch_limits(images, pixels, c, groups):
    for backward in (False, True):
        for types in ((0, 0), (1, 0), (1, 1)):
            for vec in ((True, False) if c % 8 == 0 else (False,)):
                fused, width, chunks, rows, keep, blocks, smem, threads, held = shape(images, pixels, c, groups, backward, vec, types)
                assert c % width == 0 and width % (c // groups) == 0 and (not vec or width % 8 == 0)
                assert chunks * rows >= pixels and blocks == images * (c // width) * chunks < 1 << 31
                assert 1 <= chunks <= (8 if fused else 256) and smem <= 227 * 1024
                columns = width // (8 if vec else 1)
                if fused and vec:
                    assert columns <= threads and keep == max(0, -(-rows // max(1, threads // columns)) - held) and held in (0, 3)
                    assert not held or (backward and not types[0] and 3 * (smem + 1024) <= 228 * 1024)
                    # everything kept lies in shared memory
                    assert keep * threads * 16 * ((2 if types[0] else 1) + ((2 if types[1] else 1) if backward else 0)) < smem
                else:
                    assert keep == 0 and held == 0
                parts = images * (1 if fused else chunks)
                assert work(images, pixels, c, groups, backward) >= (0 if fused else parts * groups * 2) + (parts * c * 2 if backward else 0)


def group_norm(backward=False, **kw):
    v = dict(x=A, dy=B if backward else 0, y=0 if backward else B, dx=D if backward else 0, weight=0, bias=0, stats=D + (1 << 34), work=D + (1 << 35),
             dweight=0, dbias=0, images=2, pixels=9, ldx=64, lddy=64, ldy=64, lddx=64, c=64, groups=8, act=1, x_fp32=0, y_fp32=0, eps=1e-5)
    v.update(kw)
    fn = L.lib().geeps_group_norm_backward if backward else L.lib().geeps_group_norm_forward
    return fn(L.GROUP_NORM.pack(*v.values()), None)


def test_packed_arguments_have_the_structures_size():
    class Group(C.Structure):
        _fields_ = [(f"p{i}", C.c_void_p) for i in range(10)] + [(f"n{i}", C.c_longlong) for i in range(6)] + [(f"i{i}", C.c_int) for i in range(5)] + [("eps", C.c_float)]
    assert C.sizeof(Group) == L.GROUP_NORM.size


REFUSED = (-10, -12, -14, -16)
NO_GPU = not torch.cuda.is_available()          # what is not refused is launched, and those addresses are nobody's


@pytest.mark.parametrize("backward", [False, True])
def test_group_norm_refusals(backward):
    call = lambda **kw: group_norm(backward, **kw)
    out = "dx" if backward else "y"
    assert call(groups=7) == -16 and call(groups=0) == -16 and call(groups=65) == -16
    assert call(c=16385, groups=1, ldx=1 << 15, ldy=1 << 15, lddx=1 << 15, lddy=1 << 15) == -10 and call(c=0) == -10
    assert call(x=A + 1) == -14 and call(x=A + 2, x_fp32=1) == -14 and call(stats=D + (1 << 34) + 4) == -14 and call(weight=B - 2) == -14
    assert call(work=D + (1 << 35) + 4) == -14
    assert call(**{out: A + 64}) == -12 and call(**{out: A + 2 * 64 * 17}) == -12          # a shifted overlap
    assert call(**{out: A + 64 * 2 * 5, "ldx": 200}) == -12
    assert call(weight=(D if backward else B) + 4) == -12
    assert call(ldx=63) == 1 and call(eps=-1.0) == 1 and call(act=3) == 1 and call(y_fp32=1) == 1 and call(x=0) == 1 and call(images=-1) == 1
    assert call(images=1 << 20, pixels=1 << 11) == 1 and call(images=1 << 32, pixels=1 << 32) == 1 and work(1 << 32, 1 << 32, 64, 8, backward) == 0
    if backward:
        assert call(dweight=D + (1 << 34)) == -12 and call(dbias=A) == -12 and call(stats=0) == 1
    else:
        assert group_norm(ldx=200, ldy=200, y=A + 2 * 63) == -12
    if NO_GPU:                                                                                  # the launch fails
        assert call(**{out: A}) not in REFUSED
        if backward:
            assert call(dx=B) not in REFUSED
        else:
            assert group_norm(ldx=200, ldy=200, y=A + 2 * 64) not in REFUSED                    # other channels of the same rows


def tensors(ranges, fp32):
    n = len(ranges)
    order = sorted(range(n), key=lambda i: ranges[i])
    arrays = ((C.c_void_p * n)(*[r[0] for r in ranges]), (C.c_longlong * n)(*[r[1] for r in ranges]), (C.c_ubyte * n)(*fp32), (C.c_longlong * n)(*order))
    return L.Tensors(n, *(C.addressof(a) for a in arrays)), arrays


def adamw(params, p32, grads, g32, out=None, o32=None, **kw):
    p, hold = tensors(params, p32)
    g, hold2 = tensors(grads, g32)
    o, hold3 = (None, None) if out is None else tensors(out, o32)
    decay = (C.c_ubyte * len(params))(*[1] * len(params))
    k = L.AdamW()
    k.params, k.grads, k.out, k.decay = C.addressof(p), C.addressof(g), None if o is None else C.addressof(o), C.addressof(decay)
    k.m, k.v, k.exponents, k.steps = D, D + (1 << 34), D + (1 << 35), D + (1 << 36)
    k.beta1, k.beta2, k.eps, k.lr, k.bits, k.blocks = 0.9, 0.999, 1e-8, 0.1, 8, 1 << 30
    for name, v in kw.items():
        setattr(k, name, v)
    return L.lib().geeps_adamw(C.byref(k), None)


def test_adamw_refusals():
    one = dict(params=[(A, 1000)], p32=[1], grads=[(B, 1000)], g32=[1])
    assert adamw([(A + 2, 10)], [1], [(B, 10)], [1]) == -15 and adamw([(A, 10)], [0], [(B + 1, 10)], [0]) == -15
    assert adamw(**one, out=[(B + (1 << 20) + 2, 1000)], o32=[1]) == -15
    assert adamw(**one, m=D + 2) == -15 and adamw(**one, bits=32, v=D + (1 << 34) + 8) == -15 and adamw(**one, steps=D + (1 << 36) + 4) == -15
    assert adamw(**one, lr_ref=D - 2) == -15 and adamw(**one, norm=D - 1) == -15
    assert adamw([(A, 1000)], [1], [(A + 3996, 1000)], [1]) == -13 and adamw([(A, 1000)], [1], [(A, 1000)], [1]) == -13
    assert adamw([(A, 10), (A + 36, 10)], [1, 1], [(B, 10), (B + 40, 10)], [1, 1]) == -13
    assert adamw(**one, out=[(B + 4, 1000)], o32=[1]) == -13 and adamw(**one, out=[(A, 1000)], o32=[1]) == -13
    assert adamw(**one, out=[(B, 1000)], o32=[0]) == -13                                      # the gradients' place, but another type
    assert adamw(**one, m=A) == -13 and adamw(**one, v=B) == -13 and adamw(**one, norm=A + 400) == -13 and adamw(**one, v=D + 512) == -13
    assert adamw(**one, exponents=D + 4) == -13 and adamw(**one, steps=D + 8) == -13 and adamw(**one, lr_ref=D + (1 << 36)) == -13
    assert adamw(**one, blocks=7) == 1 and adamw(**one, bits=16) == 1 and adamw(**one, beta1=1.0) == 1 and adamw(**one, beta2=-0.1) == 1 and adamw(**one, eps=-1.0) == 1
    assert adamw([(A, 10)], [1], [(B, 11)], [1]) == 1 and adamw([(0, 10)], [1], [(B, 10)], [1]) == 1
    # out may be the gradients themselves, and empty tensors may lie anywhere
    if NO_GPU:
        assert adamw(**one, out=[(B, 1000)], o32=[1]) not in (-13, -15)
        assert adamw([(A, 10), (A + 1, 0)], [1, 1], [(B, 10), (A + 3, 0)], [1, 0]) not in (-13, -15)


def test_fp8_refusals():
    def quantize(**kw):
        p = L.QuantizeFp8()
        p.x, p.q, p.scale, p.rows, p.cols, p.ldx, p.ldq = A, B, D, 10, 20, 20, 32
        for k, v in kw.items():
            setattr(p, k, v)
        return L.lib().geeps_quantize_fp8(C.byref(p), None)
    for kw in (dict(x=A + 1), dict(x=A + 2, fp32=1), dict(ldx=19), dict(q=B + 8), dict(ldq=24), dict(ldq=16), dict(scale=0), dict(rows=-1), dict(cols=1 << 30),
               dict(qt=B + 16, scale_t=0, ldqt=16), dict(qt=B + 4, scale_t=D, ldqt=16), dict(qt=B, scale_t=D, ldqt=8)):
        assert quantize(**kw) == 1, kw
    assert quantize(rows=0) == 0 and quantize(q=0) == 0 and quantize(x=0) == 1
    both = dict(qt=B + 4096, scale_t=D + 4096, ldqt=16)
    for kw in (dict(q=A), dict(q=A + 384), dict(scale=A + 399), dict(scale=B + 304), dict(both, qt=B), dict(both, qt=B + 304), dict(both, scale_t=D), dict(both, scale_t=D + 511),
               dict(both, scale_t=A), dict(both, qt=D + 496)):
        assert quantize(**kw) == -12, kw

    def gemm(**kw):
        p = L.GemmFp8()
        p.A, p.B, p.scale_a, p.scale_b, p.C, p.M, p.N, p.K, p.lda, p.ldb, p.ldc = A, B, D, D + 512, D + 4096, 100, 200, 300, 304, 304, 200
        for k, v in kw.items():
            setattr(p, k, v)
        return L.lib().geeps_gemm_fp8(C.byref(p), None)
    for kw in (dict(A=A + 8), dict(scale_b=D + 8), dict(lda=303), dict(lda=288), dict(ldb=310), dict(ldc=199), dict(K=0), dict(M=-1), dict(N=1 << 30),
               dict(bn=96, cluster=1), dict(bn=32, cluster=1), dict(bn=256, cluster=1), dict(bn=64, cluster=3), dict(bn=64, cluster=2), dict(bn=64, cluster=16),
               dict(bn=64, cluster=-2, C=D + 4098), dict(bn=64, cluster=-2, ldc=201), dict(bn=96, cluster=-2), dict(bn=64, cluster=-2, swap=1)):
        assert gemm(**kw) == 1, kw
    assert gemm(M=0) == 0 and gemm(N=0) == 0
    for kw in (dict(A=0), dict(B=0), dict(scale_a=0), dict(scale_b=0), dict(C=0), dict(C=D + 4097), dict(C=D + 4098, out_fp32=1), dict(bias=D + 2), dict(status=D + 3)):
        assert gemm(**kw) == 1, kw
    for kw in (dict(C=A), dict(C=A + 304 * 99 + 298), dict(C=B - 2), dict(C=D - 39998), dict(C=D + 512 + 1022), dict(bias=D + 4096), dict(status=D + 4096 + 39996)):
        assert gemm(**kw) == -12, kw


def test_a_copied_matrix_has_its_own_memory():
    a = F.Fp8Matrix(5, 20, "cpu")
    a.q.copy_(torch.arange(100.0).view(5, 20))
    a.scale.fill_(127)
    for b in (copy.deepcopy(a), pickle.loads(pickle.dumps(a))):
        assert b._at == (b.q.data_ptr(), b.scale.data_ptr()) and b._at[0] != a._at[0] and b._at[1] != a._at[1] and b.q.stride() == (32, 1)
        assert torch.equal(b.dequantize(), a.dequantize()) and (b.rows, b.cols, b.pitch, b.device) == (5, 20, 32, -1)
    with pytest.raises(AttributeError):
        a.q = a.q.clone()
    with pytest.raises(AttributeError):
        a.scale = a.scale.clone()


@pytest.mark.parametrize("options", [["--model", "inception_bn_small", "--fp8-linear"], ["--model", "alexnet", "--norm", "group"], ["--adam-bits", "8"]])
def test_the_trainer_refuses_options_without_effect(options, capsys):
    with pytest.raises(SystemExit):
        train.main(options)
    assert "is for" in capsys.readouterr().err


def test_the_inception_models_with_group_norms():
    for make in (inception_bn_small, inception_bn_22k):
        batch, group = make(), make(norm="group")
        b, g = list(batch.all_layers()), list(group.all_layers())
        assert [type(l) for l in b] == [BatchNorm if isinstance(l, GroupNorm) else type(l) for l in g]
        assert [l.name for l in b if hasattr(l, "cout")] == [l.name for l in g if hasattr(l, "cout")]
        convs = {l.name: l.cout for l in g if hasattr(l, "cout")}
        norms = [l for l in g if isinstance(l, GroupNorm)]
        assert len(norms) == sum(isinstance(l, BatchNorm) for l in b) == len(convs)
        assert all(l.act == "relu" and l.groups == norm_groups(convs[l.name[:-3]]) and convs[l.name[:-3]] % l.groups == 0 for l in norms)
    assert [norm_groups(c) for c in (1, 3, 24, 80, 96, 160, 576)] == [1, 1, 8, 16, 32, 32, 32]
    with pytest.raises(ValueError, match="norm"):
        inception_bn_small(norm="layer")


def fp8_shape(m, n, k, fp32, plan=(0, 0, 0), odd=False):
    """Tile width, CTAs that share K, operands swapped, CTAs, tiles, k tiles, stages, sets of scales, columns of TMEM."""
    p, out = L.GemmFp8(), (C.c_int * 9)()
    p.C, p.M, p.N, p.K, p.out_fp32 = D, m, n, k, int(fp32)
    p.ldc = n + 1 if odd else (n + 7) // 8 * 8
    p.bn, p.cluster, p.swap = plan
    assert L.lib().geeps_gemm_fp8_shape(C.byref(p), out) == 0, (m, n, k, plan)
    return list(out)


def read_while_overwritten(m, n, k, fp32, plan=(0, 0, 0), odd=False):
    """Follows the products of a CTA in the order in which they are issued.  The k tile at place i of that order is issued when its stage
    has arrived, so the one at i - stages has been waited for; a tile's first when the tile before the last has left its accumulator.
    Places at which a set of scales is written that a k tile not yet waited for reads."""
    bn, cluster, swap, ctas, tiles, kt, stages, sets, columns = fp8_shape(m, n, k, fp32, plan, odd)
    assert 2 * bn + 16 * sets <= columns <= 512 and 2 <= stages
    if cluster > 1:                      # a slice of one tile, whole quads in all but the last one
        kt, count = min(kt, -(-((kt + 3) // 4) // cluster) * 4), 1
    else:
        count = -(-tiles // (ctas // 2 if cluster < 0 else ctas))
    reader, ends, bad, i, at = [-1] * sets, [], [], 0, 0
    for t in range(min(count, 12)):      # by then the pattern has come round
        for j in range(kt):
            if j % 4 == 0:
                done = max(i - stages, ends[t - 2] if t >= 2 else -1)
                if reader[at] > done:
                    bad.append((t, j, i - reader[at]))
                now, at = at, (at + 1) % sets
            reader[now] = i
            i += 1
        ends.append(i - 1)
    return bad


@pytest.mark.parametrize("kt", list(range(1, 20)) + [37, 38, 72])
def test_fp8_scales_are_not_overwritten_before_the_products_that_read_them_are_done(kt):
    k = kt * 128 - 5
    assert fp8_shape(128 * 148 * 6, 32, k, False, (32, 1, 0))[4:6] == [888, kt]          # six tiles a CTA
    for fp32 in (False, True):
        for bn in (64, 128, 192):
            for plan, odd in (((bn, 1, 0), False), ((bn, 1, 0), True), ((bn, 1, 1), False), ((bn, -2, 0), False)):
                assert not read_while_overwritten(128 * 120, 64 * 150, k, fp32, plan, odd), (plan, fp32, odd)
        assert not read_while_overwritten(128 * 1500, 32, k, fp32, (32, 1, 0)) and not read_while_overwritten(32, 128 * 1500, k, fp32, (32, 1, 1))
        for m, n in ((16384, 256), (32768, 32), (32768, 64), (4096, 1000), (200, 60000)):      # as the sizes choose
            assert not read_while_overwritten(m, n, k, fp32) and not read_while_overwritten(m, n, k, fp32, odd=True)
    if kt in (16, 37, 38, 72):           # where four slices of whole quads are there
        assert not read_while_overwritten(100, 300, k, False, (64, 4, 0))


def test_group_norms_of_too_many_channels_are_refused_before_a_launch_shape_is_sought():
    """In a process of its own: what went wrong here was a division by zero, which ends the process."""
    code = """
import ctypes as C
from geeps_b200.ops import _lib as L
from geeps_b200.ops import functional as F
out = (C.c_int * 9)()
for c in (16385, 16392, 25600, 32768, 40000, 1 << 30):
    for groups in (1, c):
        for backward in (0, 1):
            assert F.group_norm_work(4, 50, c, groups, bool(backward)) == 0, (c, groups, backward)
            for vec in ((0, 1) if c % 8 == 0 else (0,)):
                assert L.lib().geeps_group_norm_shape(C.c_longlong(4), C.c_longlong(50), c, groups, backward, vec, 0, 0, out) == -10, (c, groups, backward, vec)
assert L.lib().geeps_group_norm_shape(C.c_longlong(4), C.c_longlong(50), 16384, 1, 1, 1, 0, 0, out) == 0 and F.group_norm_work(4, 50, 16384, 1, True) > 0
print("through")
"""
    got = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), timeout=300)
    assert got.returncode == 0 and got.stdout.strip() == "through", (got.returncode, got.stderr[-500:])


@pytest.mark.parametrize("rank", [0, 2])
def test_states_that_were_resumed_are_saved_before_the_first_step_too(rank, tmp_path):
    """A rank that the saved job did not have takes rank 0's."""
    from geeps_b200.parallel.ps_module import _AdamW
    kept = dict(m=torch.arange(256, dtype=torch.uint8), v=torch.arange(256, dtype=torch.uint8).flip(0), exponents=torch.full((2, 2), 40, dtype=torch.uint8),
                steps=torch.tensor([7, 0]))
    for d, clock in (("old", 8), ("new", 9)):
        (tmp_path / d / f"snapshot.{clock}").mkdir(parents=True)
        (tmp_path / d / "LATEST").write_text(str(clock))
    torch.save(kept, tmp_path / "old" / "snapshot.8" / "adamw.0")
    first = _AdamW(torch.device("cpu"), 1, 0.1, 0.0, bits=8)
    first.resume(str(tmp_path / "old"), rank)
    first.save(str(tmp_path / "new" / "snapshot.9"), rank)
    again = _AdamW(torch.device("cpu"), 1, 0.1, 0.0, bits=8)
    again.resume(str(tmp_path / "new"), rank)
    assert again._resumed is not None and all(torch.equal(again._resumed[k], kept[k]) for k in kept)


def test_workers_round_with_bits_of_their_own():
    """A step's random bits are a hash of seed x 0x100000001B3 + step: no worker meets another's in 2^32 steps."""
    from geeps_b200.parallel.ps_module import _AdamW
    for seed in (0, 7, -1, (1 << 64) - 1):
        at = [_AdamW(torch.device("cpu"), 8, 0.1, 0.0, rank=r, seed=seed).seed for r in range(8)]
        assert at[0] == seed
        keys = sorted((s & 0xFFFFFFFFFFFFFFFF) * 0x100000001B3 % (1 << 64) for s in at)
        assert all(b - a > 1 << 32 for a, b in zip(keys, keys[1:])) and keys[0] + (1 << 64) - keys[-1] > 1 << 32
    assert _AdamW(torch.device("cpu"), 8, 0.1, 0.0, rank=3).seed is None


@pytest.mark.parametrize("momentum", ["0.5", "0.9"])
def test_the_trainer_refuses_a_momentum_beside_adamw(momentum, capsys):
    with pytest.raises(SystemExit):
        train.main(["--optimizer", "adamw", "--momentum", momentum, "--max-iter", "0", "--synthetic-images", "0"])
    assert "--momentum is for --optimizer sgd" in capsys.readouterr().err


def test_a_snapshot_without_states_is_not_resumed_in_silence(tmp_path):
    from geeps_b200.parallel.ps_module import _AdamW
    (tmp_path / "snapshot.4").mkdir()
    (tmp_path / "LATEST").write_text("4")
    a = _AdamW(torch.device("cpu"), 1, 0.1, 0.0)
    with pytest.warns(UserWarning, match="snapshot.4 has no AdamW states"):
        a.resume(str(tmp_path), 0)
    assert a._resumed is None
