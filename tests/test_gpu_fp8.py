"""Casts to e4m3 with a scale for each block of 128, and products of such matrices, against 64-bit arithmetic."""
import copy
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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tile", [False, True])
@pytest.mark.parametrize("pitch", [300, 304])
def test_scales_change_where_the_definition_says(dtype, tile, pitch):
    """Largest magnitudes at and around 1.75 x 2^k (448 = 1.75 x 2^8), powers of two, the largest finite number, and rows whose other
    values end in every bit."""
    from geeps_b200.ops import functional as F
    edge = torch.tensor([1.75, 1.0, 2.0, 1.75 * 2.0 ** 100, 1.75 * 2.0 ** -118, 448.0, 2.0 ** -126, 1.5 * 2.0 ** 127], device=DEV)
    tops = torch.cat([edge, torch.nextafter(edge, edge * 2), torch.nextafter(edge, edge * 0), torch.tensor([torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal], device=DEV)])
    for shift in range(tops.numel()):
        n = 256 if not tile else 128
        top = (tops[shift:shift + 1] if tile else tops.roll(shift)[torch.arange(n, device=DEV) % tops.numel()]).view(-1, 1)
        x = (top * (2 * torch.rand(n, pitch, device=DEV) - 1)).to(dtype)[:, :300]
        x[:, 7::128] = top.to(dtype)
        a, t = F.Fp8Matrix(n, 300, DEV), F.Fp8Matrix(300, n, DEV)
        F.quantize_fp8(x, a, transposed=t, tile=tile)
        same(a, x, tile)
        same(t, x.T, tile)
        same(F.quantize_fp8(x, tile=tile), x, tile)
        if not tile:
            y = x.T.contiguous()                # the tops by columns
            F.quantize_fp8(y, t, transposed=a)
            same(a, x)
            same(t, y)
            break


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


def test_blocks_that_are_not_finite_are_nan_and_zeros_are_zeros():
    from geeps_b200.ops import functional as F
    x = torch.randn(5, 300, device=DEV)
    x[1, 130] = float("inf")
    x[2, 299] = float("nan")
    x[3] = 0.0
    for kw in (dict(), dict(transposed=F.Fp8Matrix(300, 5, DEV))):
        q = F.quantize_fp8(x, F.Fp8Matrix(5, 300, DEV), **kw)
        e = q.exponents()
        assert (e == 255).nonzero().tolist() == [[1, 1], [2, 2]]
        d = q.dequantize()
        assert d[1, 128:256].isnan().all() and d[2, 256:].isnan().all() and (d[3] == 0).all() and d[0].isfinite().all() and d[1, :128].isfinite().all()
    t = kw["transposed"].dequantize()
    assert t[130].isnan().all() and t[299].isnan().all() and t[:130].isfinite().all()
    w = F.quantize_fp8(torch.randn(40, 300, device=DEV))
    out = torch.zeros(5, 40, device=DEV)
    F.matmul_fp8(q, w, out, relu=True)
    assert out[1].isnan().all() and out[2].isnan().all() and (out[3] == 0).all() and out[0].isfinite().all() and (out[0] >= 0).all()


def test_extreme_sizes_of_values():
    """Scales at both ends of their range; the smallest fp32 values are below it and become zeros."""
    from geeps_b200.ops import functional as F
    x = torch.tensor([[3.0e38], [1e-30], [2.0 ** -127], [2.0 ** -135], [1e-45], [448.0], [449.0], [448.0 * 2 ** -20]], device=DEV).repeat(1, 128)
    q = F.quantize_fp8(x)
    # 3.0e38 = 1.76 x 2^127, so e = 127 - 7; 1e-30 = 1.27 x 2^-100, so e = -100 - 8
    assert q.exponents().view(-1).tolist() == [127 + 120, 127 - 108, 0, 0, 0, 127, 128, 107]
    d = q.dequantize().double()
    assert ((d - x.double()).abs() <= x.double().abs() * 2.0 ** -4 + 2.0 ** -137).all() and d[5, 0] == 448.0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_of_wider_matrices_at_any_address(dtype):
    """Inputs and outputs whose rows begin anywhere; what lies beside an output stays as it was."""
    from geeps_b200.ops import functional as F
    M, N, K = 70, 90, 260
    big = torch.randn(M, K + 7, device=DEV).to(dtype)
    w = F.quantize_fp8(torch.randn(N, K, device=DEV))
    for shift in (0, 1, 3):
        x = big[:, shift:shift + K]
        a = F.quantize_fp8(x)
        same(a, x)
        t = F.quantize_fp8(x, transposed=F.Fp8Matrix(K, M, DEV))
        same(t, x.T)
        out = torch.full((M, N + 5), 9.0, dtype=dtype, device=DEV)
        F.matmul_fp8(a, w, out[:, shift:shift + N])
        sums, half = tolerance(a, w, out, K)
        exact = plain(a, w)
        assert ((out[:, shift:shift + N].double() - exact).abs() <= sums + half * (exact.abs() + sums)).all()
        assert (out[:, :shift] == 9.0).all() and (out[:, shift + N:] == 9.0).all()


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 33, 127), (2, 64, 128), (33, 32, 129), (129, 1, 640), (31, 200, 50), (128, 128, 512), (257, 65, 513), (8, 3000, 3000)])
def test_small_and_odd_sizes(M, N, K):
    from geeps_b200.ops import functional as F
    a, b = F.quantize_fp8(torch.randn(M, K, device=DEV)), F.quantize_fp8(torch.randn(N, K, device=DEV).bfloat16(), tile=True)
    for dtype in (torch.bfloat16, torch.float32):
        out = torch.full((M, N), float("nan"), dtype=dtype, device=DEV)
        F.matmul_fp8(a, b, out)
        sums, half = tolerance(a, b, out, K)
        exact = plain(a, b)
        assert ((out.double() - exact).abs() <= sums + half * (exact.abs() + sums)).all()
    empty = torch.empty(0, N, device=DEV)
    F.matmul_fp8(F.quantize_fp8(torch.empty(0, K, device=DEV)), b, empty)


def test_offsets_that_pass_32_bits():
    """A matrix of more than 2^31 values, cast both ways, and a product of as many: what lies last is that of the last rows alone."""
    from geeps_b200.ops import functional as F
    rows, cols, last = 65664, 32832, 128
    gen = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(rows, cols, dtype=torch.bfloat16, device=DEV, generator=gen)
    q, t = F.Fp8Matrix(rows, cols, DEV), F.Fp8Matrix(cols, rows, DEV)
    end = x[-last:].clone()
    want, want_t = F.Fp8Matrix(last, cols, DEV), F.Fp8Matrix(cols, last, DEV)
    F.quantize_fp8(end, want, transposed=want_t)
    for both in (False, True):
        q.q.view(torch.uint8).zero_()
        F.quantize_fp8(x, q, transposed=t if both else None)
        assert torch.equal(q.q[-last:].view(torch.uint8), want.q.view(torch.uint8)) and torch.equal(q.exponents()[-last:], want.exponents())
    assert torch.equal(t.q[:, -last:].view(torch.uint8), want_t.q.view(torch.uint8)) and torch.equal(t.exponents()[:, -1:], want_t.exponents())
    del x, q, t, end, want, want_t
    a, b = F.quantize_fp8(torch.randn(rows, 200, device=DEV, generator=gen)), F.quantize_fp8(torch.randn(cols, 200, device=DEV, generator=gen))
    for n in (cols, cols - 1):                  # rows that TMA stores, and rows that it does not
        if n < cols:
            b = F.quantize_fp8(b.dequantize()[:n])
        out = torch.empty(rows, n, dtype=torch.bfloat16, device=DEV)
        F.matmul_fp8(a, b, out)
        e = F.Fp8Matrix(last, 200, DEV)
        F.quantize_fp8(a.dequantize()[-last:], e)
        ref = plain(e, b)
        mags, half = tolerance(e, b, out, 200)
        assert ((out[-last:].double() - ref).abs() <= mags + half * (ref.abs() + mags)).all()
        del out


def test_gradients_of_a_layer():
    """Forward and both gradients as a layer forms them, each operand cast once: against the products of what the casts stand for."""
    from geeps_b200.ops import functional as F
    M, N, K = 150, 260, 390
    x, w, dy = torch.randn(M, K, device=DEV).bfloat16(), torch.randn(N, K, device=DEV).bfloat16(), torch.randn(M, N, device=DEV).bfloat16()
    xq, xt, wq, wt, dq, dt = (F.Fp8Matrix(r, c, DEV) for r, c in ((M, K), (K, M), (N, K), (K, N), (M, N), (N, M)))
    F.quantize_fp8(x, xq, transposed=xt)
    F.quantize_fp8(w, wq, transposed=wt, tile=True)
    F.quantize_fp8(dy, dq, transposed=dt)
    assert torch.equal(wt.dequantize(), wq.dequantize().T)
    for a, b, size in ((xq, wq, (M, N)), (dq, wt, (M, K)), (dt, xt, (N, K))):
        out = torch.empty(size, device=DEV)
        F.matmul_fp8(a, b, out)
        sums, half = tolerance(a, b, out, a.cols)
        exact = plain(a, b)
        assert ((out.double() - exact).abs() <= sums + half * (exact.abs() + sums)).all()
    # and the casts are within half a step of what they stand for: 2^-4 of a value, or of the least of e4m3 (2^-9) of the scale
    for m, t in ((xq, x), (wt, w.T), (dt, dy.T)):
        step = torch.exp2(m.exponents().double() - 127).repeat_interleave(128, 1)[:, :m.cols] * 2.0 ** -10
        assert ((m.dequantize().double() - t.double()).abs() <= t.double().abs() * 2.0 ** -4 + step).all()


def test_products_repeat_on_other_streams_and_in_graphs():
    from geeps_b200.ops import functional as F
    x, w = torch.randn(200, 1500, device=DEV).bfloat16(), F.quantize_fp8(torch.randn(300, 1500, device=DEV), tile=True)
    q = [F.Fp8Matrix(200, 1500, DEV) for _ in range(3)]
    outs = [torch.empty(200, 300, dtype=torch.bfloat16, device=DEV) for _ in range(3)]

    def call(i):
        F.quantize_fp8(x, q[i])
        F.matmul_fp8(q[i], w, outs[i])
    call(0)
    graphs, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for i in (1, 2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(i)
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_a_copied_matrix_multiplies_its_own_values():
    from geeps_b200.ops import functional as F
    a, b = F.quantize_fp8(torch.randn(130, 700, device=DEV)), F.quantize_fp8(torch.randn(40, 700, device=DEV))
    want, got = torch.empty(130, 40, device=DEV), torch.empty(130, 40, device=DEV)
    F.matmul_fp8(a, b, want)
    c = copy.deepcopy(a)
    a.q.zero_()
    F.matmul_fp8(c, b, got)
    assert torch.equal(want, got)


def test_shared_memory_is_refused():
    from geeps_b200.ops import functional as F
    x = torch.zeros(40, 40, device=DEV)
    q = F.quantize_fp8(x)
    with pytest.raises(ValueError, match="overlaps"):
        F.quantize_fp8(x, q, transposed=q)
    out = torch.zeros(1600, dtype=torch.bfloat16, device=DEV)                    # a product into one of its operands, and a cast of itself
    a = F.Fp8Matrix(30, 48, DEV)
    a.__setstate__((30, 48, out.view(torch.uint8)[1600:1600 + 30 * 48].view(30, 48), a.scale))
    with pytest.raises(ValueError, match="overlaps"):
        F.matmul_fp8(a, F.Fp8Matrix(20, 48, DEV), out[600:1200].view(30, 20))
    with pytest.raises(ValueError, match="overlaps"):
        F.quantize_fp8(out[:1440].view(30, 48), a)


def test_refusals():
    from geeps_b200.ops import functional as F
    x = torch.zeros(10, 40, device=DEV)
    a, b = F.quantize_fp8(x), F.quantize_fp8(torch.zeros(20, 40, device=DEV))
    out = torch.zeros(10, 20, device=DEV)
    for match, call in (
            ("columns", lambda: F.quantize_fp8(torch.zeros(3, 0, device=DEV))), ("matrix", lambda: F.quantize_fp8(x.half())),
            ("matrix", lambda: F.quantize_fp8(x.view(-1))), ("contiguous", lambda: F.quantize_fp8(x.t())),
            ("out", lambda: F.quantize_fp8(x, F.Fp8Matrix(10, 41, DEV))), ("transposed", lambda: F.quantize_fp8(x, transposed=F.Fp8Matrix(10, 40, DEV))),
            ("out", lambda: F.quantize_fp8(x, x)), ("Fp8Matrix", lambda: F.Fp8Matrix(10, 0, DEV)),
            ("matmul_fp8: b", lambda: F.matmul_fp8(a, F.quantize_fp8(torch.zeros(20, 41, device=DEV)), out)),
            ("matmul_fp8: a", lambda: F.matmul_fp8(a, b, out[:9])), ("out", lambda: F.matmul_fp8(a, b, out.double())),
            ("out", lambda: F.matmul_fp8(a, b, torch.zeros(20, 10, device=DEV).t())), ("bias", lambda: F.matmul_fp8(a, b, out, bias=torch.zeros(19, device=DEV))),
            ("bias", lambda: F.matmul_fp8(a, b, out, bias=torch.zeros(20, device=DEV).bfloat16()))):
        with pytest.raises(ValueError, match=match):
            call()


@pytest.mark.parametrize("K", [640, 768, 1100])
@pytest.mark.parametrize("plan,M,N", [((64, -2, 0), 16384, 256), ((128, -2, 0), 16384, 512), ((64, 1, 0), 16384, 256), ((64, 1, 1), 250, 16384), ((32, 1, 0), 75776, 32)])
def test_several_tiles_a_cta_with_other_scales_in_every_block(plan, M, N, K):
    """Three tiles of K and more for a CTA, whose k tiles are no whole quads, so that the sets of scales in TMEM come round inside a tile."""
    from geeps_b200.ops import functional as F
    gen = torch.Generator(device=DEV).manual_seed(K + N)
    blocks = (K + 127) // 128

    def spread(rows):          # a block's size is a power of two of its own
        e = torch.randint(-6, 7, (rows, blocks), generator=gen, device=DEV).float()
        return torch.randn(rows, K, generator=gen, device=DEV) * torch.exp2(e).repeat_interleave(128, 1)[:, :K]
    a, b = F.quantize_fp8(spread(M)), F.quantize_fp8(spread(N))
    out = torch.full((M, N), float("nan"), dtype=torch.bfloat16, device=DEV)
    F.matmul_fp8(a, b, out, plan=plan)
    exact = plain(a, b)
    sums, half = tolerance(a, b, out, K)
    assert ((out.double() - exact).abs() <= sums + half * (exact.abs() + sums)).all()


@pytest.mark.parametrize("plan", [(0, 0, 0), (64, 1, 0), (32, 1, 0), (192, 1, 0), (64, -2, 0), (128, -2, 0)])
@pytest.mark.parametrize("N", [1, 5, 8, 33, 90, 100, 250, 257])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_what_lies_behind_the_last_column_stays(N, dtype, plan):
    """Rows on a pitch that TMA stores, whose last column is inside a piece of 16 bytes."""
    from geeps_b200.ops import functional as F
    if plan[0] == 32 and N > 32:
        plan = (128, 1, 0)
    gen = torch.Generator(device=DEV).manual_seed(N)
    for M in (40, 300):
        a, b = F.quantize_fp8(torch.randn(M, 200, generator=gen, device=DEV)), F.quantize_fp8(torch.randn(N, 200, generator=gen, device=DEV))
        bias = torch.randn(N, generator=gen, device=DEV)
        wide = torch.full((M + 2, (N + 47) // 16 * 16), 9.0, dtype=dtype, device=DEV)
        F.matmul_fp8(a, b, wide[:M, :N], bias=bias, relu=True, plan=plan)
        exact = (plain(a, b) + bias.double()).relu()
        sums, half = tolerance(a, b, wide, 200)
        sums = sums + 2.0 ** -23 * bias.double().abs()
        assert ((wide[:M, :N].double() - exact).abs() <= sums + half * (exact.abs() + sums)).all()
        assert (wide[:, N:] == 9.0).all() and (wide[M:] == 9.0).all()
