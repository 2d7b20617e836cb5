"""Casts to e4m3 with a scale for each block of 128, and products of such matrices, against 64-bit arithmetic."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def rounded(x, tile=False):
    """e4m3 values [rows, cols] and exponents of x by the definition, in 64 bits."""
    rows, cols = x.shape
    h = 128 if tile else 1
    full = torch.zeros(-(-rows // h) * h, -(-cols // 128) * 128, dtype=torch.float64, device=x.device)
    full[:rows, :cols] = x.double()
    b = full.view(full.shape[0] // h, h, full.shape[1] // 128, 128)
    top = b.abs().amax((1, 3), keepdim=True)
    m, e = torch.frexp(top)                                   # top = m 2^e, m in [0.5, 1): 448 = 0.875 x 2^9
    e = torch.where(top > 0, (e - 9 + (m > 0.875).int()).clamp(min=-127), -127)
    v = b * torch.exp2(-e.double())
    step = torch.exp2((torch.frexp(v).exponent - 4).clamp(min=-9).double())
    q = torch.round(v / step) * step
    return q.reshape(full.shape)[:rows, :cols], e.expand(-1, h, -1, 1).reshape(full.shape[0], -1)[:rows]


def values(q, e):
    return q * torch.exp2(e.double()).repeat_interleave(128, 1)[:, :q.shape[1]]


def same(got, x, tile=False):
    q, e = rounded(x, tile)
    assert torch.equal(got.exponents().int() - 127, e.int())
    assert torch.equal(got.q.double(), q)


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (7, 500), (128, 512), (130, 1000), (300, 129), (257, 4096)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tile", [False, True])
def test_casts_are_the_definition_bit_for_bit(rows, cols, dtype, tile):
    from geeps_b200.ops import functional as F
    gen = torch.Generator(device=DEV).manual_seed(rows * 1000 + cols)
    x = (torch.randn(rows, cols, generator=gen, device=DEV) * torch.exp(3 * torch.randn(rows, 1, generator=gen, device=DEV))).to(dtype)
    x[rows // 2, cols // 3:] = 0
    a, t = F.Fp8Matrix(rows, cols, DEV), F.Fp8Matrix(cols, rows, DEV)
    F.quantize_fp8(x, a, transposed=t, tile=tile)
    same(a, x, tile)
    same(t, x.T, tile)
    same(F.quantize_fp8(x, tile=tile), x, tile)
    t2 = F.quantize_fp8(x, transposed=F.Fp8Matrix(cols, rows, DEV), tile=tile)
    assert torch.equal(t2.q.view(torch.uint8), t.q.view(torch.uint8)) and torch.equal(t2.exponents(), t.exponents())


def plain(a, b):
    return values(a.q.double(), a.exponents().int() - 127) @ values(b.q.double(), b.exponents().int() - 127).T


def tolerance(a, b, out, K):
    """Products of two e4m3 values have 8 bits and are exact; the sum of K of them in fp32 is off by at most K steps of 2^-23 of the
    sum of magnitudes (the accumulator may cut instead of round); then the output's own rounding."""
    mags = values(a.q.double().abs(), a.exponents().int() - 127) @ values(b.q.double().abs(), b.exponents().int() - 127).T
    half = 2.0 ** -8 if out.dtype is torch.bfloat16 else 2.0 ** -24
    return K * 2.0 ** -23 * mags, half


@pytest.mark.parametrize("plan", [(0, 0, 0), (64, 1, 0), (64, 1, 1), (128, 1, 0), (192, 1, 0), (192, 2, 1), (32, 4, 1), (128, 2, 0), (64, 8, 0), (64, -2, 0), (128, -2, 0), (192, -2, 0)])
@pytest.mark.parametrize("M,N,K", [(7, 4096, 4096), (200, 333, 3712), (300, 520, 3900)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_products_match_64_bits(M, N, K, dtype, plan):
    from geeps_b200.ops import functional as F
    gen = torch.Generator(device=DEV).manual_seed(M + N + K)
    x = torch.randn(M, K, generator=gen, device=DEV) * torch.exp(torch.randn(M, (K + 127) // 128, generator=gen, device=DEV)).repeat_interleave(128, 1)[:, :K]
    w = torch.randn(N, K, generator=gen, device=DEV) * torch.exp(torch.randn(N, (K + 127) // 128, generator=gen, device=DEV)).repeat_interleave(128, 1)[:, :K]
    bias = torch.randn(N, generator=gen, device=DEV)
    a, b = F.quantize_fp8(x), F.quantize_fp8(w)
    if plan[0] == 32 and M > 32:
        plan = (64, 4, 1)          # 32 columns are for a single tile
    # CTA pairs store rows of whole 16 bytes
    out = torch.full((M, (N + 7) // 8 * 8 if plan[1] < 0 else N), float("nan"), dtype=dtype, device=DEV)[:, :N]
    F.matmul_fp8(a, b, out, bias=bias, plan=plan)
    want = plain(a, b) + bias.double()
    sums, half = tolerance(a, b, out, K)
    off = (out.double() - want).abs()
    print("largest error in units of its bound", (off / (sums + half * want.abs() + 1e-30)).max().item(), "of the sum of magnitudes", (off / sums).max().item())
    assert (off <= sums + half * (want.abs() + sums)).all()
