"""Refusals of the clipping call that need no GPU: addresses that no value lies at."""
import ctypes as C

import pytest

from geeps_b200.ops import _lib as L

A, B, D = 1 << 32, 1 << 33, 1 << 34        # addresses that are never touched: every call here is refused


def tensors(ranges, fp32):
    n = len(ranges)
    order = sorted(range(n), key=lambda i: ranges[i])
    arrays = ((C.c_void_p * n)(*[r[0] for r in ranges]), (C.c_longlong * n)(*[r[1] for r in ranges]), (C.c_ubyte * n)(*fp32), (C.c_longlong * n)(*order))
    return L.Tensors(n, *(C.addressof(a) for a in arrays)), arrays


def clip(src, src32, dst=None, dst32=None, bound=1.0, result=B, work=B + 64):
    s, hold = tensors(src, src32)
    d, hold2 = (None, None) if dst is None else tensors(dst, dst32)
    return L.lib().geeps_clip_gradients(C.byref(s), None if d is None else C.byref(d), C.c_double(bound), C.c_void_p(result), C.c_void_p(work), None)


@pytest.mark.parametrize("src,src32,dst,dst32", [
    ([(A + 1, 10)], [0], None, None), ([(A + 1, 10)], [1], None, None), ([(A + 2, 10)], [1], None, None),
    ([(A, 10), (D + 3, 1)], [1, 0], None, None), ([(A, 100000), (D + 2, 5)], [0, 1], None, None),
    ([(A, 10)], [1], [(D + 1, 10)], [0]), ([(A, 10)], [0], [(D + 2, 10)], [1]),
])
def test_tensors_between_values_are_refused(src, src32, dst, dst32):
    assert clip(src, src32, dst, dst32) == -15


@pytest.mark.parametrize("result,work", [(B + 2, D), (B + 1, D), (B, D + 4), (B, D + 1)])
def test_a_result_and_a_workspace_between_values_are_refused(result, work):
    assert clip([(A, 10)], [1], result=result, work=work) == -15
    assert clip([(A, 100000)], [0], result=result, work=work) == -15


def test_tensors_without_values_may_lie_anywhere():
    """Refused only because the result lies in a tensor."""
    assert clip([(A, 10), (D + 1, 0)], [1, 1], result=A) == -13
    assert clip([(A, 10), (0, 0)], [1, 1], [(D, 10), (3, 0)], [0, 0], result=D) == -13
