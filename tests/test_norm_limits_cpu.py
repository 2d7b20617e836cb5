"""Limits of the norm and join kernels' launches and of their argument checks, which need no GPU."""
import ctypes as C

import pytest

from geeps_b200.ops import _lib as L

TYPES = ((0, 0), (1, 0), (1, 1))
SIZES = [(70000, 2, 4), (100000, 2, 3), (75776, 2, 1), (75775, 3, 7), (65532, 5, 8), (56832, 2, 8), (400000, 2, 2), (1 << 20, 8, 1), (1, 60000, 8),
         (9000, 40, 40), (40000, 3, 129), (30, 900, 9000), (1 << 22, 2, 16), (7, 1, 8), (3, 5, 16384)]


def sums_shape(rows, images, c, mode, vec, types):
    out = (C.c_int * 4)()
    assert L.lib().geeps_norm_sums_shape(C.c_longlong(rows), C.c_longlong(images), c, mode, int(vec), *types, out) == 0
    return list(out)


@pytest.mark.parametrize("images,pixels,c", SIZES)
@pytest.mark.parametrize("mode", [2, 3])
def test_the_launch_that_joins_the_sums_fits_a_grid(images, pixels, c, mode):
    """A grid has at most 65535 blocks along y, and an image's shares are few where there are many images."""
    for types in TYPES:
        for vec in ((True, False) if c % 8 == 0 else (False,)):
            x, y, parts, merged = sums_shape(images * pixels, images, c, mode, vec, types)
            assert 0 <= x <= 512 and 0 <= y <= 65535, (x, y, parts, merged)
            assert parts in (1, 2, 4, 8, 16, 32) and merged in (1, 2, 4, 8, 16, 32)


A, B, D = 1 << 32, 1 << 33, 1 << 34        # addresses that are never touched: every call here is refused


def pack(**kw):
    v = [kw.get(n, 0) for n in ("x", "res", "gate", "out", "y", "dout", "dy", "dx", "dres", "dgate", "scale", "dscale", "work")]
    for n in ("post", "pre"):
        v += list(kw.get(n, (0, 0, 0, 0, 0, 0.0, 0)))
    mode = kw.get("mode", (2 if "x" in kw else 0) | (1 if "pre" in kw else 0))
    v += [kw["rows"], kw.get("gate_rows", 0)] + [kw.get("ld" + n, kw.get("ld", kw["c"])) for n in
                                                 ("x", "res", "gate", "out", "y", "dout", "dy", "dx", "dres", "dgate")]
    return L.RESIDUAL.pack(*v, kw["c"], mode, kw.get("stream_fp32", 0), kw.get("block_fp32", 0), 0)


@pytest.mark.parametrize("ld", [8, 9, 12, 16, 20, 24, 25, 31, 32, 40, 48, 1000, 1001])
def test_two_outputs_on_the_same_rows_are_refused(ld):
    """Any pitch; without the overlap the missing dout would be what is refused."""
    lib = L.lib()
    assert lib.geeps_residual_backward(pack(x=A, dx=D, dres=D, rows=4, c=8, ld=ld), None) == -12
    assert lib.geeps_residual_backward(pack(x=A, dx=B, dres=D, rows=4, c=8, ld=ld), None) == 1
    assert lib.geeps_residual_forward(pack(x=A, out=D, y=D, pre=(0, 0, 0, 0, 0, 1e-5, 1), rows=4, c=8, ld=ld), None) == -12
    # an output and an input of another type at the same address and pitch in bytes
    assert lib.geeps_residual_forward(pack(x=A, out=A, ldx=2 * ld, ldout=ld, rows=4, c=8, stream_fp32=1), None) == -12
    assert lib.geeps_residual_forward(pack(x=A, out=A + 2, ldx=2 * ld, ldout=ld, rows=4, c=8, stream_fp32=1), None) == -12


@pytest.mark.parametrize("ld", [16, 20, 24, 31, 33])
def test_ranges_of_columns_side_by_side_are_not(ld):
    lib = L.lib()
    for x, out in ((A, A + 16), (A + 2 * (ld - 8), A), (A, A + 2 * ld * 2 + 16), (A + 2 * ld * 2 + 16, A)):
        assert lib.geeps_residual_forward(pack(x=x, out=out, rows=4, c=8, ld=ld), None) == 1       # res is missing
    assert lib.geeps_residual_forward(pack(x=A, out=A + 2 * (ld - 7), rows=4, c=8, ld=ld), None) == -12


@pytest.mark.parametrize("shift,code", [(0, -12), (2, -12), (14, -12), (-14, -12), (16, 1), (-16, 1)])
def test_single_rows_without_a_pitch(shift, code):
    assert L.lib().geeps_residual_backward(pack(x=A, dx=D, dres=D + shift, rows=1, c=8, ld=0), None) == code


@pytest.mark.parametrize("kw,code", [
    (dict(stream_fp32=0, block_fp32=1), 1),
    (dict(mode=1), 1),
    (dict(mode=3), 1),
    (dict(post=(0, 0, 1 << 30 | 4, 0, 0, 1e-5, 1)), -14),
    (dict(gate_rows=-3), -11),
    (dict(gate_rows=(1 << 30) + 1), 1),
    (dict(gate=B, dgate=B + 16, gate_rows=4), -12),
    (dict(gate=B, dgate=D, gate_rows=4, lddgate=7), 1),
    (dict(gate=B, dgate=D, gate_rows=4, dscale=D + 60), -12),
])
def test_calls_without_rows_are_checked_like_others(kw, code):
    """A gate without rows to go with was let through whatever else was wrong."""
    assert L.lib().geeps_residual_backward(pack(**{"x": A, "gate": B, "gate_rows": 4, "rows": 0, "c": 8, **kw}), None) == code


S = 1 << 30
NORM = (0, 0, S, 0, 0, 1e-5, 1)


@pytest.mark.parametrize("kw", [
    dict(x=A + 1), dict(out=D + 1), dict(res=B + 1), dict(y=S + 4097, pre=(0, 0, 0, 0, 0, 1e-5, 1)), dict(gate=S + 4097, gate_rows=4),
    dict(res=B + 2, stream_fp32=1), dict(out=D + 2, stream_fp32=1), dict(x=A + 2, stream_fp32=1, block_fp32=1),
    dict(gate=S + 4098, gate_rows=1, stream_fp32=1, block_fp32=1),
    dict(scale=S + 4098), dict(post=(S + 4098, 0, 0, 0, 0, 1e-5, 1)), dict(post=(0, S + 4097, 0, 0, 0, 1e-5, 1)),
    dict(y=S + 8192, pre=(S + 4098, 0, 0, 0, 0, 1e-5, 1)), dict(y=S + 8192, pre=(0, S + 4098, 0, 0, 0, 1e-5, 1)),
])
def test_addresses_between_values_are_refused_forward(kw):
    """A value is read at a multiple of its size; a kernel that is given another address faults.  (Without the refusal the missing
    output or input of each of these calls would be what is refused.)"""
    kw = {"x": A, "res": B, "out": D, "rows": 4, "c": 8, **kw}
    kw["out" if kw["out"] == D else "res"] = 0
    assert L.lib().geeps_residual_forward(pack(**kw), None) == -14


@pytest.mark.parametrize("kw", [
    dict(x=A + 1), dict(dout=B + 1), dict(dx=D + 1), dict(gate=S + 4096, gate_rows=4, dgate=S + 8193), dict(dy=S + 4097, out=S + 8192, pre=NORM),
    dict(dy=S + 4096, out=S + 8193, pre=NORM), dict(dout=B + 2, stream_fp32=1), dict(dx=D + 2, stream_fp32=1, block_fp32=1), dict(dscale=S + 4098),
    dict(post=(0, 0, S, S + 4098, 0, 1e-5, 1)), dict(post=(0, 0, S, 0, S + 4097, 1e-5, 1)), dict(scale=S + 4098),
    dict(dy=S + 4096, out=S + 8192, pre=(0, 0, S, S + 16386, 0, 1e-5, 1)), dict(dy=S + 4096, out=S + 8192, pre=(0, 0, S, 0, S + 16387, 1e-5, 1)),
    dict(rows=0, dscale=S + 4098),
])
def test_addresses_between_values_are_refused_backward(kw):
    assert L.lib().geeps_residual_backward(pack(**{"x": A, "dout": B, "dx": D, "rows": 4, "c": 8, **kw}), None) == -14       # dres is missing


def test_dres_between_values_is_refused():
    assert L.lib().geeps_residual_backward(pack(x=A, dout=B, dres=D + 1, rows=4, c=8), None) == -14       # dx is missing
    assert L.lib().geeps_residual_backward(pack(x=A, dout=B, dres=D + 2, rows=4, c=8, stream_fp32=1), None) == -14
    assert L.lib().geeps_residual_backward(pack(x=A, dout=B, dres=D + 2, rows=4, c=8), None) == 1
    assert L.lib().geeps_residual_backward(pack(x=A + 2, dout=B + 4, dres=D + 4, rows=4, c=8, stream_fp32=1), None) == 1


@pytest.mark.parametrize("backward", [0, 1])
@pytest.mark.parametrize("mode", [1, 2, 3])
@pytest.mark.parametrize("vec", [1, 0])
def test_there_is_a_kernel_for_every_width(backward, mode, vec):
    """Only the kernels that some width asks for are built."""
    lib, out, rows = L.lib(), (C.c_int * 10)(), 34993
    for gate in ((0,) if mode == 1 else (0, 7, rows)):
        for types in TYPES:
            for c in range(8 if vec else 1, 16385, 8 if vec else 1):
                if lib.geeps_norm_shape(C.c_longlong(rows), C.c_longlong(gate), c, mode, backward, vec, *types, out) != 0:
                    raise AssertionError((gate, types, c, list(out)))
