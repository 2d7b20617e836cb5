"""Host side of the norm and clipping kernels: launch shapes, workspaces and refusals, which need no GPU."""
import ctypes as C

import pytest

from geeps_b200.ops import _lib as L


def shape(rows, c, backward=True, mode=3, gate_rows=0, vec=True, types=(0, 0)):
    out = (C.c_int * 10)()
    assert L.lib().geeps_norm_shape(C.c_longlong(rows), C.c_longlong(gate_rows), c, mode, int(backward), int(vec), *types, out) == 0
    return list(out)


@pytest.mark.parametrize("c", [1, 7, 8, 9, 64, 72, 96, 136, 255, 256, 257, 576, 1000, 1024, 2048, 4095, 4096, 4097, 6144, 6152, 8192, 8193, 12280, 12288, 12296, 16383,
                               16384])
@pytest.mark.parametrize("rows", [1, 5, 300, 50176, 10_000_000])
@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("mode", [1, 2, 3])
def test_shapes_cover_the_rows_within_the_launch_limits(rows, c, backward, mode):
    for types in ((0, 0), (1, 0), (1, 1)):
        for vec in ((True, False) if c % 8 == 0 else (False,)):
            for gate in ((0, rows, max(1, rows // 5 if rows % 5 == 0 else 1)) if mode > 1 else (0,)):
                vectors, slot, slots, blocks, per_sm, depth, smem, large, tiles, width = shape(rows, c, backward, mode, gate, vec, types)
                threads = 512 if large or (not backward and vectors == 4 and c >= (4089 if vec else 4097)) else 256 if not backward else 512 if not vec else 256 if vectors > 2 and mode > 1 else 384
                assert (tiles - 1) * width < c <= tiles * width and (tiles == 1 or (backward and width % 8 == 0))
                assert vectors * slot * 8 >= width and slot * slots <= threads and slots >= 1
                assert slot in (1, 2, 4, 8, 16, 32) or slot % 32 == 0
                assert slot <= 32 or slots <= 15                    # a named barrier for each slot of several warps
                assert 1 <= blocks <= 148 * per_sm and (blocks - 1) * slots < rows
                assert (slot * slots) % 32 == 0                     # whole warps: their lanes meet in shuffles
                assert (0 if large or (threads == 512 and not vec and not backward) else 1) <= depth <= 4
                # dynamic and static shared memory of all blocks of an SM (1 KB of each is the system's)
                fixed = 16 * 64 * 4 + ((4 if tiles > 1 else 2) * 8 * threads if backward else 0) + 1024
                assert per_sm * (smem + fixed) <= 228 * 1024 and smem <= 208 * 1024


def pack(**kw):
    names = ["x", "res", "gate", "out", "y", "dout", "dy", "dx", "dres", "dgate", "scale", "dscale", "work"]
    v = [kw.get(n, 0) for n in names]
    for n in ("post", "pre"):
        v += list(kw.get(n, (0, 0, 0, 0, 0, 0.0, 0)))
    mode = kw.get("mode", (2 if "x" in kw else 0) | (1 if "pre" in kw else 0))
    v += [kw["rows"], kw.get("gate_rows", 0)] + [kw.get("ld", kw["c"])] * 10 + [kw["c"], mode, kw.get("stream_fp32", 0), kw.get("block_fp32", 0), 0]
    return L.RESIDUAL.pack(*v)         # the structure ends on a multiple of eight bytes


def test_packed_arguments_have_the_structures_size():
    class Norm(C.Structure):
        _fields_ = [(n, C.c_void_p) for n in ("weight", "bias", "stats", "dweight", "dbias")] + [("eps", C.c_float), ("kind", C.c_int)]

    class Residual(C.Structure):
        _fields_ = ([(f"p{i}", C.c_void_p) for i in range(13)] + [("post", Norm), ("pre", Norm)]
                    + [(f"n{i}", C.c_longlong) for i in range(12)] + [(f"i{i}", C.c_int) for i in range(5)])
    assert C.sizeof(Residual) == L.RESIDUAL.size
    r = Residual.from_buffer_copy(pack(rows=5, c=8, x=4096, pre=(0, 0, 64, 0, 0, 0.5, 2), gate_rows=3))
    assert (r.p0, r.pre.stats, r.pre.eps, r.pre.kind, r.n0, r.n1, r.n2, r.i0) == (4096, 64, 0.5, 2, 5, 3, 8, 8)


LAYER = (0, 0, 1 << 30, 0, 0, 1e-5, 1)
A, B, D = 1 << 32, 1 << 33, 1 << 34        # addresses that are never touched: every call here is refused


@pytest.mark.parametrize("kw,code", [
    (dict(res=A, y=B, pre=LAYER, rows=4, c=0), -10),
    (dict(res=A, y=B, pre=LAYER, rows=4, c=16385), -10),
    (dict(x=A, res=B, out=D, gate=D + (1 << 20), gate_rows=3, rows=4, c=8), -11),
    (dict(x=A, res=B, out=D, gate=D + (1 << 20), gate_rows=8, rows=4, c=8), -11),
    (dict(x=A, res=B, out=D, gate=D + (1 << 20), gate_rows=0, rows=4, c=8), -11),
    (dict(x=A, res=B, out=A + 16, rows=4, c=8), -12),
    (dict(x=A, res=B, out=D, y=D, pre=LAYER, rows=4, c=8), -12),
    (dict(x=A, res=B, out=A, rows=4, c=8, stream_fp32=1), -12),
    (dict(x=A, res=B, out=B + 8, rows=4, c=8, ld=12), -12),
    (dict(x=A, res=B, rows=4, c=8), 1),
    (dict(res=A, pre=LAYER, rows=4, c=8), 1),
    (dict(res=A, y=B, rows=4, c=8), 1),
    (dict(x=A, res=B, out=D, rows=-1, c=8), 1),
    (dict(x=A, res=B, out=D, rows=4, c=8, mode=3), 1),
    (dict(x=A, res=B, out=D, rows=4, c=8, mode=0), 1),
    (dict(res=B, out=D, rows=4, c=8, mode=2), 1),
    (dict(x=A, res=B, out=D, rows=4, c=8, ld=7), 1),
    (dict(x=A, res=B, out=D, rows=4, c=8, block_fp32=1), 1),
])
def test_refused_forward_calls(kw, code):
    assert L.lib().geeps_residual_forward(pack(**kw), None) == code


@pytest.mark.parametrize("kw,code", [
    (dict(out=A, dy=B, dres=D, pre=(0, 0, 0, 0, 0, 1e-5, 1), rows=4, c=8), 1),
    (dict(x=A, dout=B, dx=D, dres=D, rows=4, c=8), -12),
    (dict(x=A, dout=B, dx=D, rows=4, c=8), 1),
    (dict(x=A, dx=B, dres=D, rows=4, c=8), 1),
    (dict(x=A, dout=B, dx=D, dres=D + (1 << 20), rows=1 << 20, c=8), -12),
    (dict(x=A, dout=B, dx=D, dres=D + (1 << 30), rows=1 << 20, c=8), 1),        # no workspace
])
def test_refused_backward_calls(kw, code):
    assert L.lib().geeps_residual_backward(pack(**kw), None) == code


def test_ranges_of_columns_of_one_matrix_do_not_overlap():
    # refused only for the missing output behind the overlap check
    for x, out in ((A, A + 16), (A + 16, A), (A, A + 16 + 32 * 2)):
        assert L.lib().geeps_residual_forward(pack(x=x, out=out, rows=4, c=8, ld=16), None) == 1
    for x, out in ((A, A + 14), (A + 18, A), (A, A + 16 + 32 * 2 + 2)):
        assert L.lib().geeps_residual_forward(pack(x=x, out=out, rows=4, c=8, ld=16), None) == -12


def test_workspaces():
    def work(rows, gate_rows, c, mode):
        return L.lib().geeps_residual_work(C.c_longlong(rows), C.c_longlong(gate_rows), c, mode)
    assert work(0, 0, 64, 1) == 0 and work(1, 0, 64, 3) == 0
    assert work(1 << 22, 1 << 21, 4096, 2) > 1 << 32
    for rows, gate, c, mode in ((50176, 0, 1024, 1), (50176, 256, 1024, 3), (50176, 50176, 1024, 2), (7, 7, 16, 3), (40, 4, 8192, 3), (999, 3, 77, 2)):
        for types in ((0, 0), (1, 0), (1, 1)):
            for vec in (True, False):
                _, _, slots, blocks, *_ = shape(rows, c, True, mode, gate, vec, types)
                by_image = 0 < gate < rows
                need = (blocks * (4 if mode == 3 else 2) + (3 * blocks * slots + gate if by_image else 0)) * c
                assert work(rows, gate, c, mode) >= (need if blocks > 1 or by_image else 0)


def tensors(ranges, fp32=1):
    n = len(ranges)
    order = sorted(range(n), key=lambda i: ranges[i])
    arrays = ((C.c_void_p * n)(*[r[0] for r in ranges]), (C.c_longlong * n)(*[r[1] for r in ranges]), (C.c_ubyte * n)(*[fp32] * n),
              (C.c_longlong * n)(*order))
    return L.Tensors(n, *(C.addressof(a) for a in arrays)), arrays


@pytest.mark.parametrize("src,dst,code", [
    ([(A, 10), (A + 36, 10)], None, -13),
    ([(A, 10)], [(A + 4, 10)], -13),
    ([(A, 10), (A + 40, 10)], [(A + 40, 10), (A, 10)], -13),
    ([(A, 10), (B, 5)], [(D, 10), (A + 20, 5)], -13),
    ([(A, 10), (B, 5)], [(D, 10), (D + 36, 5)], -13),
    ([(A, 10)], [(A, 9)], 1),
    ([(A, 10)], [(A, 10), (B, 10)], 1),
    ([(0, 10)], None, 1),
    ([(A, -1)], None, 1),
])
def test_refused_clipping_calls(src, dst, code):
    s, hold = tensors(src)
    d, hold2 = tensors(dst) if dst is not None else (None, None)
    assert L.lib().geeps_clip_gradients(C.byref(s), C.byref(d) if d is not None else None, C.c_double(1.0), C.c_void_p(A), C.c_void_p(B), None) == code


@pytest.mark.parametrize("bound", [-1.0, float("nan")])
def test_a_bound_that_is_no_norm_is_refused(bound):
    s, hold = tensors([(A, 10)])
    assert L.lib().geeps_clip_gradients(C.byref(s), None, C.c_double(bound), C.c_void_p(A), C.c_void_p(B), None) == 1


def test_the_trainer_hands_the_bound_to_the_module(monkeypatch):
    import contextlib

    import torch

    import geeps_b200.parallel.ps_module as pm
    import geeps_b200.train as train

    class Stop(Exception):
        pass

    seen = []

    def module(*args, **kw):
        seen.append(kw["clip_gradients"])
        raise Stop
    monkeypatch.setattr(pm, "PSModule", module)
    monkeypatch.setattr(torch.cuda, "set_device", lambda d: None)
    monkeypatch.setattr(torch.cuda, "Stream", lambda **kw: object())
    monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext())
    for args in ([], ["--clip-gradients", "35"]):
        with pytest.raises(Stop):
            train.main(["--model", "inception_bn_small", "--batch", "2", "--synthetic-images", "4", "--source-size", "32"] + args)
    assert seen == [None, 35.0]


def test_a_bound_needs_a_gpu():
    from geeps_b200.models.net import Net
    from geeps_b200.ops.layers import Input, Linear
    from geeps_b200.parallel.ps_module import PSModule
    from geeps_b200.utils.config import GeePsConfig
    for bound in (1.0, -1.0, float("nan")):
        with pytest.raises(ValueError, match="clip_gradients"):
            PSModule(Net("n", Input(), [Linear("f", 8, fp32_out=True)]), (2, 8, 1, 1), GeePsConfig(tcp_base_port=31990), device="cpu", clip_gradients=bound)


def test_tensors_of_the_host_are_refused():
    import torch

    from geeps_b200.ops import functional as F
    x = torch.zeros(4, 8)
    for call in (lambda: F.norm_forward(x, x, F.Norm("rms")), lambda: F.residual_forward(x, x, x), lambda: F.clip_gradients([x], 1.0, torch.zeros(2))):
        with pytest.raises((ValueError, RuntimeError), match="CUDA|cpu"):
            call()
    with pytest.raises(ValueError, match="need x"):
        F.residual_forward(x, None, x)
    with pytest.raises(ValueError, match="need x"):
        F.residual_backward(x, x, None, x)


S = 1 << 30


@pytest.mark.parametrize("kw,code", [
    (dict(res=A, y=B, pre=(0, 0, S + 4, 0, 0, 1e-5, 1)), -14),
    (dict(x=A, res=B, out=D, post=(0, 0, S + 12, 0, 0, 1e-5, 2)), -14),
    (dict(res=A, y=B, pre=(0, 0, B + 56, 0, 0, 1e-5, 1)), -12),                       # statistics in an output
    (dict(res=A, y=B, pre=(0, 0, A + 56, 0, 0, 1e-5, 1)), -12),                       # ... in an input
    (dict(res=A, y=B, pre=(B + 60, 0, S, 0, 0, 1e-5, 1)), -12),                       # a parameter in an output
    (dict(res=A, y=B, pre=(S + 28, 0, S, 0, 0, 1e-5, 1)), -12),                       # ... in statistics
    (dict(x=A, res=B, out=D, mode=3, pre=(0, 0, S, 0, 0, 1e-5, 1), post=(0, 0, S + 24, 0, 0, 1e-5, 1)), -12),
    (dict(res=A, mode=1, pre=(A + 60, 0, S, 0, 0, 1e-5, 1)), 1),                      # two inputs may share; the output is missing
    (dict(res=A, mode=1, pre=(S + 32, S + 32, S, 0, 0, 1e-5, 1)), 1),
])
def test_refused_vectors_forward(kw, code):
    assert L.lib().geeps_residual_forward(pack(**{"rows": 4, "c": 8, **kw}), None) == code


@pytest.mark.parametrize("kw,code", [
    (dict(pre=(0, 0, S + 4, 0, 0, 1e-5, 1)), -14),
    (dict(pre=(0, 0, S, 0, 0, 1e-5, 1), work=S + 4), -14),
    (dict(pre=(0, 0, S, S + 28, 0, 1e-5, 1)), -12),
    (dict(pre=(0, 0, S, S + 32, S + 60, 1e-5, 1)), -12),
    (dict(pre=(S + 64, 0, S, S + 68, 0, 1e-5, 1)), -12),
    (dict(pre=(0, 0, S, B + 60, 0, 1e-5, 1)), -12),
    (dict(pre=(0, 0, S, A - 28, 0, 1e-5, 1)), -12),
    (dict(pre=(0, 0, S, 0, D + 60, 1e-5, 1)), -12),
    (dict(pre=(0, 0, S, S + 32, S + 64, 1e-5, 1), dres=0), 1),                        # side by side; the output is missing
    (dict(pre=(0, 0, S, B + 64, A - 32, 1e-5, 1), dres=0), 1),
])
def test_refused_vectors_backward(kw, code):
    assert L.lib().geeps_residual_backward(pack(**{"rows": 4, "c": 8, "out": A, "dy": B, "dres": D, **kw}), None) == code


@pytest.mark.parametrize("result,work", [(A + 36, B), (D + 4, B), (B, A - 8), (B, D + 32), (A - 4, B), (B, B + 8 - 8), (B + 8, B)])
def test_a_result_or_workspace_in_a_gradient_is_refused(result, work):
    s, hold = tensors([(A, 10)])
    d, hold2 = tensors([(D, 10)])
    assert L.lib().geeps_clip_gradients(C.byref(s), C.byref(d), C.c_double(1.0), C.c_void_p(result), C.c_void_p(work), None) == -13


@pytest.mark.parametrize("rows,gate,c,mode", [(3325, 0, 8972, 3), (7, 1, 16384, 3), (1, 0, 16384, 1), (450, 50, 12288, 2), (5000, 5000, 16383, 3), (40, 8, 9001, 2)])
def test_workspaces_of_rows_in_tiles(rows, gate, c, mode):
    """Four values a row, and the sums of a tile at a time."""
    for types in ((0, 0), (1, 0), (1, 1)):
        for vec in (True, False):
            *_, slots, blocks, _, _, _, _, tiles, width = shape(rows, c, True, mode, gate, vec, types)
            if tiles == 1:
                continue
            by_image = 0 < gate < rows
            need = (blocks * (4 if mode == 3 else 2) if blocks > 1 or by_image else 0) + (3 * blocks * slots + gate if by_image else 0)
            assert L.lib().geeps_residual_work(C.c_longlong(rows), C.c_longlong(gate), c, mode) >= 4 * rows + need * width
