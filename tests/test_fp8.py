"""The 8-bit linear layer: block-scaled fp8 product, quantisation, residual RMS norm with fp8 output, its backward pass.

Oracles are the formulas in 64 bits.  Products of small integers under power-of-two scales are exact in fp32 in any order, so
those are compared bit for bit; random ones are held to bounds counted from roundings of 2^-24 (fp32, half a step)."""
import ctypes as C
import math

import pytest
import torch

import backup_1_b200 as b
from backup_1_b200 import lib as blib

gpu = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24                       # half a step of fp32, relative
TINY = 2.0 ** -126
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: U}
FLOATS = [torch.bfloat16, torch.float16, torch.float32]
KIND = {b.FP8_E4M3: torch.float8_e4m3fn, b.FP8_E5M2: torch.float8_e5m2}
FMAX = {b.FP8_E4M3: 448.0, b.FP8_E5M2: 57344.0}


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def spread(s, block_rows, rows, cols):
    return s.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :cols]


def cur():
    return torch.cuda.current_stream()


# ---- no GPU needed ------------------------------------------------------------------------------------------------------
def test_calls_without_a_context_are_refused():
    L = b.load_library()
    assert L.decxb_gemm_fp8(None, None, None, None, 0, None, 0, 0, None) == 1
    assert L.decxb_quantize_fp8(None, 0, 1, 1, None, 1, 0, None, None, None) == 1
    assert L.decxb_rmsnorm(None, 0, 1, 1, None, 1, None, 0, None, 0, 0.0, None, 0, None, 0, 0, None, None) == 1
    assert L.decxb_rmsnorm_backward(None, 0, 1, 1, None, 1, None, 1, None, 0, 0.0, None, 0, None, 0, None, None, 0, None) == 1
    n = C.c_size_t(7)
    assert L.decxb_rmsnorm_backward_workspace(None, 1, 1, C.byref(n)) == 1


def test_descriptor_from_tensors():
    code = torch.empty((5, 304), dtype=torch.float8_e4m3fn)[:, :300]
    m = b.Fp8Matrix.of(code, torch.empty((3, 5)).t())
    assert (m.c.rows, m.c.cols, m.c.ld, m.c.scale_row_stride, m.c.scale_block_stride, m.c.type, m.c.block_rows) == (5, 300, 304, 1, 5, 0, 1)
    assert (m.c.data, m.c.scales) == (code.data_ptr(), m.scales.data_ptr())
    w = b.Fp8Matrix.of(torch.empty((200, 256), dtype=torch.float8_e5m2), torch.empty((2, 2)), 128)
    assert (w.c.ld, w.c.scale_row_stride, w.c.scale_block_stride, w.c.type, w.c.block_rows) == (256, 2, 1, 1, 128)
    assert b.Fp8Matrix.empty(3, 130, device="cpu").c.ld == 144
    for data, scales, br in [(code, torch.empty((5, 2)), 1), (code, torch.empty((5, 3)), 64), (code, torch.empty((1, 3)), 1),
                             (code.t(), torch.empty((300, 1)), 1), (code[:1].expand(5, 300), torch.empty((5, 3)), 1)]:
        with pytest.raises(ValueError):
            b.Fp8Matrix.of(data, scales, br)
    for data, scales in [(code.float(), torch.empty((5, 3))), (code, torch.empty((5, 3), dtype=torch.float64))]:
        with pytest.raises(TypeError):
            b.Fp8Matrix.of(data, scales)
    with pytest.raises(TypeError):                      # host memory
        b.Fp8Matrix(torch.zeros(16, 16).numpy(), 4096, 16, 16, 16, 1, 16)


def test_stream_argument():
    class S:
        def __init__(self, h):
            self.cuda_stream = h
    assert blib._stream(None) is None and blib._stream(7) == 7 and blib._stream(S(9)) == 9
    assert blib._stream(S(0)) == 1          # torch's default stream, not the context's own


def test_element_type_argument():
    assert blib._dtype(torch.empty(1, dtype=torch.bfloat16), None) == b.BF16 and blib._dtype(1234, b.F16) == b.F16
    for x, given in [(1234, None), (torch.empty(1, dtype=torch.int32), None), (torch.empty(1), b.F16)]:
        with pytest.raises(TypeError):
            blib._dtype(x, given)


# ---- product ------------------------------------------------------------------------------------------------------------
def int_matrix(g, rows, cols, kind, block_rows, pad=0, offset=0, row_major=False):
    """Small whole numbers as codes, powers of two as scales; `pad` and `offset` in codes, the padding poisoned with NaN."""
    code = torch.randint(-4, 5, (rows, cols), device=DEV, generator=g).float().to(KIND[kind])
    ld = cols + pad
    buf = torch.full((offset + rows * ld + 64,), 0x7F, device=DEV, dtype=torch.uint8)
    data = buf[offset:offset + rows * ld].view(KIND[kind]).view(rows, ld)[:, :cols]
    data.copy_(code)
    r, c = -(-rows // block_rows), -(-cols // 128)
    s = torch.exp2(torch.randint(-2, 3, (r, c), device=DEV, generator=g).float())
    s = s if row_major else s.t().contiguous().t()
    m = b.Fp8Matrix(data, s, rows, cols, ld, s.stride(0), s.stride(1), block_rows, kind)
    return m, code.double() * spread(s, block_rows, rows, cols).double()


def run_gemm(ctx, A, B, dtype, Cin=None, pad=0, offset=0):
    M, N = A.rows, B.rows
    ld = N + pad
    buf = torch.full((offset + M * ld + 32,), float("nan"), device=DEV, dtype=dtype)
    D = buf[offset:offset + M * ld].view(M, ld)
    ctx.gemm_fp8(A, B, D, ld, Cin=Cin, ldc=Cin.stride(0) if Cin is not None else 0, stream=cur())
    ctx.synchronize()
    assert torch.isnan(buf[:offset]).all() and torch.isnan(buf[offset + M * ld:]).all() and torch.isnan(D[:, N:]).all()
    return D[:, :N]


SHAPES = [(1, 1, 1), (1, 128, 128), (1, 300, 515), (2, 16, 16), (7, 130, 129), (16, 256, 1024), (33, 4096, 512), (64, 129, 2000), (65, 384, 640),
          (100, 70, 50), (127, 257, 127), (128, 128, 256), (129, 513, 384), (200, 1000, 130), (256, 256, 2176), (257, 511, 1025),
          (515, 640, 900), (1000, 1111, 300), (2048, 1280, 384), (1100, 4100, 260)]


@gpu
@pytest.mark.parametrize("a_rows,b_rows", [(1, 128), (1, 1), (128, 128), (128, 1)])
@pytest.mark.parametrize("shape", SHAPES)
def test_product_of_whole_numbers_is_exact(ctx, shape, a_rows, b_rows):
    M, N, K = shape
    g = gen(M * 7 + N * 3 + K)
    A, a = int_matrix(g, M, K, b.FP8_E4M3, a_rows, pad=-K % 16)
    B, w = int_matrix(g, N, K, b.FP8_E4M3, b_rows, pad=-K % 16 + 16, row_major=True)
    assert torch.equal(run_gemm(ctx, A, B, torch.float32).double(), a @ w.t())


@gpu
@pytest.mark.parametrize("kinds", [(0, 0), (0, 1), (1, 0), (1, 1)])
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("M,N,K", [(5, 200, 300), (150, 200, 300), (300, 260, 140)])
def test_product_types_addend_and_results_pitch(ctx, M, N, K, dtype, kinds):
    g = gen(5)
    A, a = int_matrix(g, M, K, kinds[0], 1, pad=-K % 16)
    B, w = int_matrix(g, N, K, kinds[1], 128, pad=-K % 16)
    Cin = torch.randint(-50, 50, (M, N + 3), device=DEV, generator=g).to(dtype)
    want = (a @ w.t() + Cin[:, :N].double()).to(dtype)
    assert torch.equal(run_gemm(ctx, A, B, dtype, Cin, pad=5, offset=1), want)
    assert torch.equal(run_gemm(ctx, A, B, dtype, Cin, pad=8, offset=0), want)
    D = Cin.clone()                                    # in place
    ctx.gemm_fp8(A, B, D, N + 3, Cin=D, ldc=N + 3, stream=cur())
    ctx.synchronize()
    assert torch.equal(D[:, :N], want) and torch.equal(D[:, N:], Cin[:, N:])


@gpu
@pytest.mark.parametrize("b_rows", [1, 128])
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("M,N,K,pad", [(2055, 1288, 384, 0), (2055, 1288, 300, 1), (2304, 1283, 130, 5), (40, 20000, 260, 8), (5000, 4200, 640, 0),
                                       (4999, 4101, 390, 3)])
def test_product_of_many_tiles_with_addend(ctx, M, N, K, pad, dtype, b_rows):
    """Addend and result through the copy engine (pitch and N of whole 16-byte pieces) and by the threads, in place too."""
    g = gen(K)
    A, a = int_matrix(g, M, K, b.FP8_E5M2, 1, pad=-K % 16)
    B, w = int_matrix(g, N, K, b.FP8_E4M3, b_rows, pad=-K % 16)
    Cin = torch.randint(-50, 50, (M, N + pad), device=DEV, generator=g).to(dtype)
    want = (a @ w.t() + Cin[:, :N].double()).to(dtype)
    assert torch.equal(run_gemm(ctx, A, B, dtype, Cin, pad=8), want)
    assert torch.equal(run_gemm(ctx, A, B, dtype, None, pad=pad), (a @ w.t()).to(dtype))
    D = Cin.clone()
    for _ in range(2):
        ctx.gemm_fp8(A, B, D, N + pad, Cin=D, ldc=N + pad, stream=cur())
    ctx.synchronize()
    assert torch.equal(D[:, :N], (a @ w.t() + want.double()).to(dtype)) and torch.equal(D[:, N:], Cin[:, N:])


@gpu
@pytest.mark.parametrize("M", [3, 200])
@pytest.mark.parametrize("pad,offset", [(1, 0), (16, 1), (0, 8), (7, 3), (16, 16)])
def test_product_of_operands_at_any_address_and_pitch(ctx, M, pad, offset):
    g = gen(pad * 100 + offset)
    A, a = int_matrix(g, M, 272, b.FP8_E4M3, 1, pad=pad, offset=offset)
    B, w = int_matrix(g, 150, 272, b.FP8_E4M3, 128, pad=offset, offset=pad)
    assert torch.equal(run_gemm(ctx, A, B, torch.float32).double(), a @ w.t())


@gpu
@pytest.mark.parametrize("M,N,K,b_rows", [(1, 512, 4096, 128), (40, 300, 5000, 1), (384, 512, 4096, 128), (700, 300, 2050, 1), (2048, 1024, 512, 128)])
def test_product_of_random_numbers(ctx, M, N, K, b_rows):
    """Bound: the products are exact (8-bit significands); the tensor core adds 128 of them in four steps of at most 33 terms, each
    truncated by less than a step (2 U) of the block's sum of magnitudes; the product of the scales is rounded once
    and the block sums are added with one rounding each: (4 * 33 * 2 + K / 128 + 2) U of the sum of magnitudes."""
    g = gen(M + N)
    a = torch.randn(M, K, device=DEV, generator=g)
    w = torch.randn(N, K, device=DEV, generator=g)
    A, B = b.Fp8Matrix.empty(M, K), b.Fp8Matrix.empty(N, K, b_rows)
    ctx.quantize_fp8(M, K, a, K, A, stream=cur())
    ctx.quantize_fp8(N, K, w, K, B, stream=cur())
    a64 = A.data.double() * spread(A.scales, 1, M, K).double()
    w64 = B.data.double() * spread(B.scales, b_rows, N, K).double()
    want = a64 @ w64.t()
    mag = a64.abs() @ w64.abs().t()
    err = (run_gemm(ctx, A, B, torch.float32).double() - want).abs()
    assert bool((err <= (264 + K / 128 + 2) * U * mag).all())
    # and far inside it on the whole: independent errors of that size would give 1e-6 of the result's norm
    assert float(err.norm() / want.norm()) <= 1e-5
    half = run_gemm(ctx, A, B, torch.bfloat16).double()
    assert bool(((half - want).abs() <= HALF[torch.bfloat16] * want.abs() * 1.01 + (264 + K / 128 + 2) * U * mag).all())


@gpu
def test_product_carries_nan_and_infinity_of_one_row_only(ctx):
    g = gen(3)
    for M in (4, 300):
        A, a = int_matrix(g, M, 512, b.FP8_E4M3, 1)
        B, w = int_matrix(g, 256, 512, b.FP8_E4M3, 128)
        want = a @ w.t()
        A.data[1, 200] = float("nan")
        A.scales[2, 3] = float("inf")
        D = run_gemm(ctx, A, B, torch.float32)
        assert torch.isnan(D[1]).all() and not torch.isfinite(D[2]).any()
        keep = [i for i in range(M) if i not in (1, 2)]
        assert torch.equal(D[keep].double(), want[keep])


@gpu
def test_product_of_zero_rows_and_of_block_of_zeros(ctx):
    A, B = b.Fp8Matrix.empty(0, 256), b.Fp8Matrix.empty(64, 256, 128)
    ctx.gemm_fp8(A, B, torch.empty((0, 64), device=DEV), 64, stream=cur())
    x = torch.zeros((5, 256), device=DEV)
    A = b.Fp8Matrix.empty(5, 256)
    ctx.quantize_fp8(5, 256, x, 256, A, stream=cur())
    ctx.quantize_fp8(64, 256, torch.randn(64, 256, device=DEV), 256, B, stream=cur())
    assert torch.equal(run_gemm(ctx, A, B, torch.bfloat16), torch.zeros((5, 64), device=DEV, dtype=torch.bfloat16))


@gpu
def test_product_refusals(ctx):
    A, B = b.Fp8Matrix.empty(4, 256), b.Fp8Matrix.empty(8, 256, 128)
    D = torch.zeros((4, 8), device=DEV)

    def bad(status, A=A, B=B, D=D, ldd=8, **kw):
        with pytest.raises(b.DecxbError) as e:
            ctx.gemm_fp8(A, B, D, ldd, stream=cur(), **kw)
        assert e.value.status == status, str(e.value)

    bad(3, B=b.Fp8Matrix.empty(8, 255, 128))
    bad(3, ldd=7)
    bad(3, Cin=D, ldc=4)
    bad(13, A=b.Fp8Matrix.empty(4, 0), B=b.Fp8Matrix.empty(8, 0, 128))
    bad(13, D=D.data_ptr() + 2, d_type=b.F32)
    bad(13, D=0, d_type=b.F32)
    bad(13, Cin=D, ldc=9)
    bad(11, D=D.data_ptr(), d_type=7)
    bad(11, A=b.Fp8Matrix(A.data, A.scales, 4, 256, 256, 1, 4, 1, 5))
    bad(13, A=b.Fp8Matrix(A.data, A.scales, 4, 256, 256, 1, 4, 64))
    bad(13, A=b.Fp8Matrix(A.data, A.scales, 4, 256, 256, -1, 4))
    bad(13, A=b.Fp8Matrix(0, A.scales, 4, 256, 256, 1, 4))
    bad(13, A=b.Fp8Matrix(A.data, A.scales.data_ptr() + 2, 4, 256, 256, 1, 4))
    bad(3, A=b.Fp8Matrix(A.data, A.scales, 4, 256, 255, 1, 4))
    bad(104, A=b.Fp8Matrix(A.data, A.scales, 2 ** 31, 256, 256, 1, 4))
    bad(13, D=torch.zeros((4, 8)))                      # not on the context's device
    assert ctx.L.decxb_gemm_fp8(ctx.h, None, B.addr, None, 0, D.data_ptr(), 0, 8, None) == 13
    with pytest.raises(TypeError):
        ctx.gemm_fp8(A, B, D, 8, Cin=D.half(), ldc=8)
    with pytest.raises(b.DecxbError):
        ctx.gemm_fp8(b.Fp8Matrix.empty(4, 256, device="cpu"), B, D, 8)
    with pytest.raises(ValueError):
        b.Fp8Matrix.of(A.data, A.scales.cpu())
    assert bool((D == 0).all())


# ---- quantisation -------------------------------------------------------------------------------------------------------
def blocks_amax(x, block_rows):
    rows, cols = x.shape
    r, c = -(-rows // block_rows), -(-cols // 128)
    p = torch.zeros((r * block_rows, c * 128), device=x.device, dtype=x.dtype)
    p[:rows, :cols] = x.abs()
    return p.view(r, block_rows, c, 128).amax((1, 3))


def want_scales(amax64, kind, rule):
    s = amax64 / FMAX[kind]
    if rule == b.SCALE_POW2:
        m, e = torch.frexp(s)
        s = torch.ldexp(torch.ones_like(s), torch.where(m > 0.5, e, e - 1))
    return s.clamp_min(TINY).float()


def check_codes(code, quotient, kind, delta):
    """Every code is the quotient rounded to nearest, up to a relative error `delta` of the quotient."""
    lo = (quotient * (1 - delta)).float().to(KIND[kind]).double()
    hi = (quotient * (1 + delta)).float().to(KIND[kind]).double()
    c = code.double()
    assert bool(((c >= torch.minimum(lo, hi)) & (c <= torch.maximum(lo, hi))).all())


@gpu
@pytest.mark.parametrize("kind", [b.FP8_E4M3, b.FP8_E5M2])
@pytest.mark.parametrize("rule", [b.SCALE_AMAX, b.SCALE_POW2])
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 130), (128, 128), (127, 300), (260, 129), (600, 1000), (1, 4096), (1500, 8)])
def test_quantise_both_orientations(ctx, rows, cols, dtype, rule, kind):
    """scale: one IEEE division, equal; code: the fp32 quotient (the one in 64 bits, rounded) rounded to the type, equal."""
    g = gen(rows + cols)
    x = (torch.randn(rows, cols, device=DEV, generator=g) * torch.exp2(torch.randint(-8, 9, (rows, 1), device=DEV, generator=g).float())).to(dtype)
    for br, tr in [(1, 1), (128, 128), (1, 128), (128, 1)]:
        Q, T = b.Fp8Matrix.empty(rows, cols, br, kind), b.Fp8Matrix.empty(cols, rows, tr, kind)
        ctx.quantize_fp8(rows, cols, x, cols, Q, T, rule=rule, stream=cur())
        ctx.synchronize()
        for m, y, blk in ((Q, x.double(), br), (T, x.double().t(), tr)):
            s = want_scales(blocks_amax(y, blk), kind, rule)
            assert torch.equal(m.scales, s)
            check_codes(m.data, y / spread(s, blk, *y.shape).double(), kind, 0.0)


@gpu
@pytest.mark.parametrize("pad,offset", [(0, 0), (5, 0), (8, 3), (8, 8)])
def test_quantise_strides_and_one_output(ctx, pad, offset):
    rows, cols = 140, 200
    g = gen(pad + offset)
    buf = torch.full((offset + rows * (cols + pad) + 16,), float("nan"), device=DEV, dtype=torch.bfloat16)
    x = buf[offset:offset + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
    x.copy_(torch.randn(rows, cols, device=DEV, generator=g))
    ref = b.Fp8Matrix.empty(rows, cols)
    ctx.quantize_fp8(rows, cols, x.contiguous(), cols, ref, stream=cur())
    for transposed in (False, True):
        r, c = (cols, rows) if transposed else (rows, cols)
        out = torch.full((offset + r * (c + pad) + 16,), 0x55, device=DEV, dtype=torch.uint8)
        data = out[offset:offset + r * (c + pad)].view(r, c + pad)
        s = torch.full((r, -(-c // 128) + 1), -7.0, device=DEV)          # row by row, one column too many
        m = b.Fp8Matrix(data, s, r, c, c + pad, s.stride(0), s.stride(1))
        ctx.quantize_fp8(rows, cols, x, cols + pad, *((None, m) if transposed else (m, None)), stream=cur())
        ctx.synchronize()
        assert bool((out[:offset] == 0x55).all()) and bool((data[:, c:] == 0x55).all()) and bool((out[offset + r * (c + pad):] == 0x55).all())
        assert bool((s[:, -1] == -7.0).all())
        if not transposed:
            assert torch.equal(data[:, :c], ref.data.view(torch.uint8)) and torch.equal(s[:, :-1], ref.scales)
        else:
            want = b.Fp8Matrix.empty(r, c)
            ctx.quantize_fp8(r, c, x.t().contiguous(), c, want, stream=cur())
            ctx.synchronize()
            assert torch.equal(data[:, :c], want.data.view(torch.uint8)) and torch.equal(s[:, :-1], want.scales)


@gpu
def test_quantise_orientations_of_different_types(ctx):
    x = torch.randn(200, 300, device=DEV)
    Q, T = b.Fp8Matrix.empty(200, 300, 1, b.FP8_E4M3), b.Fp8Matrix.empty(300, 200, 128, b.FP8_E5M2)
    ctx.quantize_fp8(200, 300, x, 300, Q, T, stream=cur())
    ctx.synchronize()
    for m, y, blk, kind in ((Q, x.double(), 1, b.FP8_E4M3), (T, x.double().t(), 128, b.FP8_E5M2)):
        s = want_scales(blocks_amax(y, blk), kind, b.SCALE_AMAX)
        assert torch.equal(m.scales, s)
        check_codes(m.data, y / spread(s, blk, *y.shape).double(), kind, 0.0)


@gpu
@pytest.mark.parametrize("blocks", [(1, 1), (128, 128), (1, 128), (128, 1)])
@pytest.mark.parametrize("dtype", FLOATS)
def test_quantise_special_values_in_every_row_and_column_of_a_tile(ctx, dtype, blocks):
    """Blocks that hold a NaN or an infinity, wherever it lies and whatever its sign, next to blocks that hold none; the
    second row of tiles and the last column of tiles are cut."""
    rows, cols = 200, 600
    g = gen(9)
    x = torch.randn(rows, cols, device=DEV, generator=g).to(dtype)
    x[torch.arange(0, 128, 2), torch.arange(0, 128, 2)] = float("nan")          # tile 0: every other row and column
    x[torch.arange(0, 64), 128 + torch.arange(64, 128)] = -float("inf")         # tile 1: the upper rows, the last columns
    x[torch.arange(128, 200), 256 + torch.arange(0, 72)] = -float("nan")        # a cut tile
    x[:, 384:512] = -x[:, 384:512].abs()                                        # the largest magnitude is negative
    x[199, 599] = float("inf")
    Q, T = b.Fp8Matrix.empty(rows, cols, blocks[0]), b.Fp8Matrix.empty(cols, rows, blocks[1])
    ctx.quantize_fp8(rows, cols, x, cols, Q, T, stream=cur())
    ctx.synchronize()
    for m, y, blk in ((Q, x.double(), blocks[0]), (T, x.double().t(), blocks[1])):
        amax = blocks_amax(y, blk)
        want = torch.where(torch.isfinite(amax), want_scales(amax.nan_to_num(1.0, 1.0), m.type, b.SCALE_AMAX).double(), amax).float()
        assert torch.equal(m.scales.nan_to_num(-1.0, -2.0), want.nan_to_num(-1.0, -2.0))
        scale, code = spread(want, blk, *y.shape).double(), m.data.double()
        none = torch.isnan(scale) | torch.isinf(y)
        assert torch.equal(torch.isnan(code), none)
        assert bool((code[torch.isinf(scale) & ~none] == 0).all())
        ok = torch.isfinite(scale)
        check_codes(m.data[ok], y[ok] / scale[ok], m.type, 0.0)


@gpu
def test_quantise_zeros_nan_infinity_and_tiny(ctx):
    x = torch.randn(6, 256, device=DEV)
    x[0] = 0.0
    x[1, 5] = float("nan")
    x[2, 200] = float("inf")
    x[3] = 1e-42                         # subnormal: under the smallest scale
    x[4, :128] = -0.0
    Q, T = b.Fp8Matrix.empty(6, 256), b.Fp8Matrix.empty(256, 6)
    ctx.quantize_fp8(6, 256, x, 256, Q, T, stream=cur())
    ctx.synchronize()
    s, c = Q.scales, Q.data.float()
    assert bool((s[0] == TINY).all()) and bool((c[0] == 0).all()) and bool((s[3] == TINY).all()) and s[4, 0] == TINY
    assert torch.isnan(s[1, 0]) and torch.isnan(c[1, :128]).all() and torch.isfinite(c[1, 128:]).all() and torch.isfinite(s[1, 1])
    assert s[2, 1] == float("inf") and torch.isnan(c[2, 200]) and bool((c[2, 128:200] == 0).all()) and torch.isfinite(s[2, 0])
    assert torch.isnan(T.scales[5, 0]) and T.scales[200, 0] == float("inf") and torch.isfinite(T.scales[6, 0])


@gpu
def test_quantise_refusals(ctx):
    x = torch.zeros((4, 256), device=DEV)
    Q = b.Fp8Matrix.empty(4, 256)

    def bad(status, rows=4, cols=256, X=x, ldx=256, Q=Q, Qt=None, **kw):
        with pytest.raises(b.DecxbError) as e:
            ctx.quantize_fp8(rows, cols, X, ldx, Q, Qt, stream=cur(), **kw)
        assert e.value.status == status, str(e.value)

    bad(13, Q=None)
    bad(3, rows=5)
    bad(3, Qt=b.Fp8Matrix.empty(4, 256))
    bad(3, ldx=255)
    bad(13, X=0, x_type=b.F32)
    bad(13, X=x.data_ptr() + 1, x_type=b.BF16)
    bad(11, X=x.data_ptr(), x_type=9)
    bad(11, rule=4)
    bad(13, rows=-1)
    bad(13, Q=b.Fp8Matrix(Q.data, Q.scales, 4, 256, 256, 0, 1))      # blocks would share a scale
    bad(13, Q=b.Fp8Matrix(Q.data, Q.scales, 4, 256, 256, 1, 1))
    bad(13, Q=b.Fp8Matrix(Q.data, Q.scales, 4, 256, 256, 1, 4, 2))
    ctx.quantize_fp8(0, 256, torch.empty((0, 256), device=DEV), 256, b.Fp8Matrix.empty(0, 256), stream=cur())
    ctx.quantize_fp8(4, 0, torch.empty((4, 0), device=DEV), 0, None, b.Fp8Matrix.empty(0, 4), stream=cur())
    ctx.synchronize()


# ---- norm ---------------------------------------------------------------------------------------------------------------
NORM_SHAPES = [(1, 1), (1, 8), (3, 7), (5, 128), (2, 130), (9, 1000), (1, 4096), (4, 4100), (3, 8192), (2, 16384), (2, 33000), (1, 40001), (1200, 64),
               (1300, 2056), (1190, 4096)]
# roundings of one value: at most 64 terms in a thread's chain of squares (fewer outside the longest rows), 10 levels of
# shuffles, mean, eps, the reciprocal root's 2 steps, three products: under 96
NORM_U = 96 * U


def norm_ref(x, r, gamma, eps):
    h = x.double() + (r.double() if r is not None else 0.0)
    return h, h / torch.sqrt((h * h).mean(1, keepdim=True) + eps) * gamma.double()


def near(got, want, dtype, rel):
    """One rounding to dtype (half a step of a subnormal at least) on top of a relative error."""
    small = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}[dtype]
    return bool(((got.double() - want).abs() <= (HALF[dtype] * (1 + rel) + rel) * want.abs() + small).all())


@gpu
@pytest.mark.parametrize("dtype,gtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32), (torch.float32, torch.float32),
                                         (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
def test_norm(ctx, rows, cols, dtype, gtype):
    g = gen(rows + cols)
    x = torch.randn(rows, cols, device=DEV, generator=g).to(dtype)
    r = torch.randn(rows, cols, device=DEV, generator=g).to(dtype)
    gamma = (1 + 0.2 * torch.randn(cols, device=DEV, generator=g)).to(gtype)
    long_rows = 1.0 if cols <= 32768 else cols / 32768 * 4
    for res in (None, r):
        h, y = norm_ref(x, res, gamma, 1e-5)
        for kind, rule in ((b.FP8_E4M3, b.SCALE_AMAX), (b.FP8_E5M2, b.SCALE_POW2)):
            H, Y, Q = torch.empty_like(x), torch.empty_like(x), b.Fp8Matrix.empty(rows, cols, 1, kind)
            ctx.rmsnorm(rows, cols, x, cols, gamma, 1e-5, R=res, ldr=cols, H=H, ldh=cols, Y=Y, ldy=cols, Q=Q, rule=rule, stream=cur())
            ctx.synchronize()
            assert near(H, h, dtype, U if dtype == torch.float32 else 2 * U)
            assert near(Y, y, dtype, NORM_U * long_rows)
            s = want_scales(blocks_amax(y, 1), kind, rule).double()
            if rule == b.SCALE_AMAX:
                assert bool(((Q.scales.double() - s).abs() <= (NORM_U * long_rows + 2 * U) * s).all())
            else:
                assert bool(((Q.scales == s) | (Q.scales == 2 * s) | (Q.scales == s / 2)).all())
                assert float((Q.scales != s).float().mean()) <= 0.01
            check_codes(Q.data, y / spread(Q.scales, 1, rows, cols).double(), kind, NORM_U * long_rows + 4 * U)


@gpu
@pytest.mark.parametrize("pad,offset", [(0, 0), (3, 0), (8, 1), (8, 8)])
@pytest.mark.parametrize("cols", [200, 33003])
def test_norm_strides_in_place_and_single_outputs(ctx, cols, pad, offset):
    rows, dtype = 5, torch.bfloat16
    g = gen(pad + offset)

    def view(fill=None):
        buf = torch.full((offset + rows * (cols + pad) + 16,), 7.0, device=DEV, dtype=dtype)
        v = buf[offset:offset + rows * (cols + pad)].view(rows, cols + pad)
        if fill is not None:
            v[:, :cols] = fill
        return buf, v
    x, r = torch.randn(rows, cols, device=DEV, generator=g).to(dtype), torch.randn(rows, cols, device=DEV, generator=g).to(dtype)
    gamma = torch.randn(cols + 3, device=DEV, generator=g).to(dtype)[3:]
    H, Y, Q = torch.empty_like(x), torch.empty_like(x), b.Fp8Matrix.empty(rows, cols)
    ctx.rmsnorm(rows, cols, x, cols, gamma, 0.0, R=r, ldr=cols, H=H, ldh=cols, Y=Y, ldy=cols, Q=Q, stream=cur())
    (bx, vx), (br, vr), (by, vy) = view(x), view(r), view()
    ld = cols + pad
    ctx.rmsnorm(rows, cols, vx, ld, gamma, 0.0, R=vr, ldr=ld, H=vr, ldh=ld, Y=vy, ldy=ld, stream=cur())       # residual updated in place
    ctx.synchronize()
    assert torch.equal(vr[:, :cols], H) and torch.equal(vy[:, :cols], Y) and torch.equal(vx[:, :cols], x)
    for buf, v in ((br, vr), (by, vy)):
        assert bool((buf[:offset] == 7).all()) and bool((v[:, cols:] == 7).all()) and bool((buf[offset + rows * ld:] == 7).all())
    (_, vr2), q2 = view(r), b.Fp8Matrix.empty(rows, cols)
    ctx.rmsnorm(rows, cols, vx, ld, gamma, 0.0, R=vr2, ldr=ld, Y=vx, ldy=ld, stream=cur())                   # normalised in place
    ctx.rmsnorm(rows, cols, x, cols, gamma, 0.0, R=vr2, ldr=ld, Q=q2, stream=cur())                          # codes alone
    ctx.synchronize()
    assert torch.equal(vx[:, :cols], Y) and torch.equal(q2.data.view(torch.uint8), Q.data.view(torch.uint8)) and torch.equal(q2.scales, Q.scales)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_norm_of_many_rows_in_place(ctx, dtype):
    """As many rows as are walked by blocks that fetch ahead: nothing is read after it was overwritten."""
    rows, cols = 3001, 2304
    g = gen(9)
    x, r = (torch.randn(rows, cols, device=DEV, generator=g).to(dtype) for _ in range(2))
    gamma = torch.randn(cols, device=DEV, generator=g)
    H, Y = torch.empty_like(x), torch.empty_like(x)
    ctx.rmsnorm(rows, cols, x, cols, gamma, 1e-5, R=r, ldr=cols, H=H, ldh=cols, Y=Y, ldy=cols, stream=cur())
    h, y = norm_ref(x, r, gamma, 1e-5)
    assert near(H, h, dtype, 2 * U) and near(Y, y, dtype, NORM_U)
    x2, r2 = x.clone(), r.clone()
    ctx.rmsnorm(rows, cols, x2, cols, gamma, 1e-5, R=r2, ldr=cols, H=r2, ldh=cols, Y=x2, ldy=cols, stream=cur())
    ctx.synchronize()
    assert torch.equal(r2, H) and torch.equal(x2, Y)
    one = torch.empty_like(x)
    ctx.rmsnorm(rows, cols, x, cols, gamma, 1e-5, Y=one, ldy=cols, stream=cur())                # without a residual
    assert near(one, norm_ref(x, None, gamma, 1e-5)[1], dtype, NORM_U)


@gpu
def test_norm_of_zero_rows_zeros_nan_and_infinity(ctx):
    x = torch.randn(5, 512, device=DEV)
    x[1] = 0.0
    x[2, 3] = float("nan")
    x[3, 3] = float("inf")
    gamma = torch.ones(512, device=DEV)
    Y, Q = torch.empty_like(x), b.Fp8Matrix.empty(5, 512)
    ctx.rmsnorm(5, 512, x, 512, gamma, 1e-6, Y=Y, ldy=512, Q=Q, stream=cur())
    ctx.rmsnorm(0, 512, torch.empty((0, 512), device=DEV), 512, gamma, 1e-6, Q=b.Fp8Matrix.empty(0, 512), stream=cur())
    ctx.synchronize()
    assert bool((Y[1] == 0).all()) and bool((Q.scales[1] == TINY).all())
    assert torch.isnan(Y[2]).all() and torch.isnan(Q.scales[2]).all() and torch.isnan(Q.data[2].float()).all()
    assert torch.isnan(Y[3, 3]) and bool((Y[3, 4:] == 0).all()) and torch.isnan(Q.scales[3, 0])
    assert torch.isfinite(Y[[0, 4]]).all()


def backward_ref(dy, h, gamma, eps, dr):
    h, dy, gamma = h.double(), dy.double(), gamma.double()
    r = 1.0 / torch.sqrt((h * h).mean(1, keepdim=True) + eps)
    w = dy * gamma
    dx = r * (w - h * r * r * (w * h).mean(1, keepdim=True))
    size = r * (w.abs() + h.abs() * r * r * (w * h).abs().mean(1, keepdim=True))
    if dr is not None:
        dx, size = dx + dr.double(), size + dr.double().abs()
    return dx, (dy * h * r).sum(0), size, (dy * h * r).abs().sum(0)


@gpu
@pytest.mark.parametrize("dtype,gtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32), (torch.float32, torch.float32)])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 4096), (3, 7), (61, 5120), (700, 130), (1200, 64), (5, 9001), (2, 16385), (3, 40001), (900, 1024)])
def test_norm_backward(ctx, rows, cols, dtype, gtype):
    """dx: 96 U (as the norm, whose statistics it has twice: 200 U) of the magnitudes that are added, one rounding;
    dgamma: besides those, one rounding for each addend of the longest chain of its sum."""
    g = gen(rows * 3 + cols)
    h = torch.randn(rows, cols, device=DEV, generator=g).to(dtype)
    dy = torch.randn(rows, cols, device=DEV, generator=g).to(dtype)
    dr = torch.randn(rows, cols, device=DEV, generator=g).to(dtype)
    gamma = (1 + 0.2 * torch.randn(cols, device=DEV, generator=g)).to(gtype)
    n = ctx.rmsnorm_backward_workspace(rows, cols)
    ws = torch.empty(n, device=DEV, dtype=torch.uint8)
    parts = n // (4 * cols)
    longest = -(-rows // parts) + -(-parts // 32) + 6
    wide = 1.0 if cols <= 16384 else cols / 16384 * 4
    for res, work in ((None, ws), (dr, None)):
        dx, dg = torch.empty_like(h), torch.full((cols,), float("nan"), device=DEV)
        args = dict(dR=res, lddr=cols, workspace=work, workspace_bytes=n if work is not None else 0, stream=cur())
        ctx.rmsnorm_backward(rows, cols, dy, cols, h, cols, gamma, 1e-5, dx, cols, dg, **args)
        ctx.synchronize()
        wx, wg, mx, mg = backward_ref(dy, h, gamma, 1e-5, res)
        small = 2.0 ** -25 if dtype == torch.float16 else 0.0
        assert bool(((dx.double() - wx).abs() <= HALF[dtype] * wx.abs() * 1.001 + 200 * wide * U * mx + small).all())
        assert bool(((dg.double() - wg).abs() <= (96 * wide + longest + 4) * U * mg).all())
        again, dg2 = dy.clone(), torch.empty_like(dg)                     # in place of dY; the same bits
        ctx.rmsnorm_backward(rows, cols, again, cols, h, cols, gamma, 1e-5, again, cols, dg2, **args)
        ctx.synchronize()
        assert torch.equal(again, dx) and torch.equal(dg2, dg)


@gpu
def test_norm_backward_against_differences(ctx):
    """Central differences of the forward formula in 64 bits along random directions; step 1e-5: error of the second order, far below."""
    rows, cols, eps = 6, 300, 1e-5
    g = gen(1)
    h = torch.randn(rows, cols, device=DEV, generator=g)
    dy, gamma = torch.randn(rows, cols, device=DEV, generator=g), torch.randn(cols, device=DEV, generator=g)
    dx, dg = torch.empty_like(h), torch.empty_like(gamma)
    ctx.rmsnorm_backward(rows, cols, dy, cols, h, cols, gamma, eps, dx, cols, dg, stream=cur())
    ctx.synchronize()

    def loss(h64, g64):
        return float((dy.double() * h64 / torch.sqrt((h64 * h64).mean(1, keepdim=True) + eps) * g64).sum())
    for k in range(4):
        u = torch.randn(rows, cols, device=DEV, generator=g).double()
        v = torch.randn(cols, device=DEV, generator=g).double()
        t = 1e-5
        slope = (loss(h.double() + t * u, gamma.double() + t * v) - loss(h.double() - t * u, gamma.double() - t * v)) / (2 * t)
        got = float((dx.double() * u).sum() + (dg.double() * v).sum())
        size = float((dx.double() * u).abs().sum() + (dg.double() * v).abs().sum())
        assert abs(got - slope) <= 300 * U * size + 1e-6


@gpu
def test_norm_backward_strides_no_gamma_gradient_and_zero_rows(ctx):
    rows, cols = 7, 130
    h, dy = torch.randn(rows, 140, device=DEV), torch.randn(rows, 133, device=DEV)
    gamma = torch.randn(cols, device=DEV)
    out = torch.full((rows, 137), 3.0, device=DEV)
    ctx.rmsnorm_backward(rows, cols, dy, 133, h, 140, gamma, 1e-5, out, 137, None, stream=cur())
    ctx.synchronize()
    wx, _, mx, _ = backward_ref(dy[:, :cols], h[:, :cols], gamma, 1e-5, None)
    assert bool(((out[:, :cols].double() - wx).abs() <= 201 * U * mx).all()) and bool((out[:, cols:] == 3).all())
    dg = torch.full((cols + 1,), 5.0, device=DEV)
    ctx.rmsnorm_backward(0, cols, 0, cols, 0, cols, gamma, 1e-5, 0, cols, dg, type=b.F32, stream=cur())
    ctx.synchronize()
    assert bool((dg[:cols] == 0).all()) and dg[cols] == 5


@gpu
def test_norm_refusals(ctx):
    x, gamma = torch.zeros((4, 256), device=DEV), torch.ones(256, device=DEV)
    y = torch.zeros_like(x)

    def bad(status, rows=4, cols=256, X=x, ldx=256, G=gamma, eps=1e-6, **kw):
        kw.setdefault("Y", y)
        kw.setdefault("ldy", 256)
        with pytest.raises(b.DecxbError) as e:
            ctx.rmsnorm(rows, cols, X, ldx, G, eps, stream=cur(), **kw)
        assert e.value.status == status, str(e.value)

    bad(13, Y=None)
    bad(13, rows=-1)
    bad(13, cols=0)
    bad(3, ldx=255)
    bad(3, ldy=4)
    bad(13, X=0, type=b.F32)
    bad(13, G=0, gamma_type=b.F32)
    bad(13, eps=-1.0)
    bad(13, eps=float("nan"))
    bad(13, H=y, ldh=256)
    bad(13, Y=x, ldy=300)
    bad(3, Q=b.Fp8Matrix.empty(4, 255))
    bad(13, Q=b.Fp8Matrix.empty(4, 256, 128))
    bad(11, rule=2)
    bad(11, X=x.data_ptr(), type=3, Y=y.data_ptr())
    bad(13, R=torch.zeros((4, 256)), ldr=256)
    with pytest.raises(TypeError):
        ctx.rmsnorm(4, 256, x, 256, gamma, 1e-6, Y=y.half(), ldy=256)
    with pytest.raises(TypeError):
        ctx.rmsnorm(4, 256, x.cpu().numpy(), 256, gamma, 1e-6, Y=y, ldy=256)
    bad(13, X=x.cpu())

    def badb(status, rows=4, dX=y, lddx=256, **kw):
        with pytest.raises(b.DecxbError) as e:
            ctx.rmsnorm_backward(rows, 256, x, 256, x, 256, gamma, 1e-6, dX, lddx, torch.empty(256, device=DEV), stream=cur(), **kw)
        assert e.value.status == status, str(e.value)

    ws = torch.empty(8192, device=DEV, dtype=torch.uint8)
    badb(13, workspace=ws, workspace_bytes=ctx.rmsnorm_backward_workspace(4, 256) - 1)
    badb(13, workspace=ws[4:], workspace_bytes=8000)
    badb(13, dX=x)
    badb(3, lddx=255)
    badb(13, rows=-4)
    ctx.synchronize()


# ---- together -----------------------------------------------------------------------------------------------------------
class Layer:
    """y = rmsnorm(x + r) W^T and the gradients, in 8 bits: what a training step calls."""

    def __init__(self, ctx, tokens, width, out, seed=0):
        g = gen(seed)
        self.ctx, self.dims = ctx, (tokens, width, out)
        bf = torch.bfloat16
        self.x, self.r = (torch.randn(tokens, width, device=DEV, generator=g).to(bf) for _ in range(2))
        self.w = torch.randn(out, width, device=DEV, generator=g) * width ** -0.5
        self.gamma = 1 + 0.1 * torch.randn(width, device=DEV, generator=g)
        self.dout = torch.randn(tokens, out, device=DEV, generator=g).to(bf)
        self.h, self.y = torch.empty_like(self.x), torch.empty_like(self.x)
        e = b.Fp8Matrix.empty
        self.q, self.qt = e(tokens, width), e(width, tokens)
        self.wq, self.wt = e(out, width, 128), e(width, out, 128)
        self.d, self.dt = e(tokens, out, 1, b.FP8_E5M2), e(out, tokens, 1, b.FP8_E5M2)
        self.out, self.dy = torch.empty(tokens, out, device=DEV, dtype=bf), torch.empty_like(self.x)
        self.dx, self.dgamma = torch.empty_like(self.x), torch.empty(width, device=DEV)
        self.dw = torch.ones(out, width, device=DEV)
        self.ws = torch.empty(ctx.rmsnorm_backward_workspace(tokens, width), device=DEV, dtype=torch.uint8)

    def step(self):
        (t, w, o), c, s = self.dims, self.ctx, cur()
        c.quantize_fp8(o, w, self.w, w, self.wq, self.wt, stream=s)
        c.rmsnorm(t, w, self.x, w, self.gamma, 1e-6, R=self.r, ldr=w, H=self.h, ldh=w, Y=self.y, ldy=w, Q=self.q, stream=s)
        c.gemm_fp8(self.q, self.wq, self.out, o, stream=s)
        c.quantize_fp8(t, w, self.y, w, None, self.qt, stream=s)
        c.quantize_fp8(t, o, self.dout, o, self.d, self.dt, stream=s)
        c.gemm_fp8(self.d, self.wt, self.dy, w, stream=s)
        c.gemm_fp8(self.dt, self.qt, self.dw, w, Cin=self.dw, ldc=w, stream=s)
        c.rmsnorm_backward(t, w, self.dy, w, self.h, w, self.gamma, 1e-6, self.dx, w, self.dgamma, dR=self.x, lddr=w,
                           workspace=self.ws, workspace_bytes=self.ws.numel(), stream=s)

    def results(self):
        return [v.clone() for v in (self.h, self.y, self.out, self.dy, self.dw, self.dx, self.dgamma)]

    def check(self, steps=1):
        """Each operator on what it was given; the whole against the layer in 64 bits, off by the codes' roundings."""
        val = lambda m: m.data.double() * spread(m.scales, m.block_rows, m.rows, m.cols).double()  # noqa: E731
        bf = HALF[torch.bfloat16]
        for got, a, w in ((self.out, self.q, self.wq), (self.dy, self.d, self.wt)):
            want, size = val(a) @ val(w).t(), val(a).abs() @ val(w).abs().t()
            assert bool(((got.double() - want).abs() <= bf * want.abs() * 1.01 + 400 * U * size).all())
        want, size = val(self.dt) @ val(self.qt).t(), val(self.dt).abs() @ val(self.qt).abs().t()
        assert bool(((self.dw.double() - 1 - steps * want).abs() <= steps * (500 * U * size + 4 * U * (1 + steps * want.abs()))).all())
        # the layer without rounding: e4m3 codes are off by up to 2^-4, e5m2 by up to 2^-3, independently
        h, y = norm_ref(self.x, self.r, self.gamma, 1e-6)
        exact = y @ self.w.double().t()
        assert float((self.out.double() - exact).norm() / exact.norm()) <= 2.0 ** -4 + 2.0 ** -4 + bf
        exact = self.dout.double() @ self.w.double()
        assert float((self.dy.double() - exact).norm() / exact.norm()) <= 2.0 ** -3 + 2.0 ** -4 + bf


@gpu
@pytest.mark.parametrize("dims", [(1, 512, 384), (40, 1024, 520), (300, 640, 1000), (515, 384, 256)])
def test_layer_forward_and_backward(ctx, dims):
    layer = Layer(ctx, *dims)
    layer.step()
    ctx.synchronize()
    layer.check()


@gpu
def test_layer_captured_and_replayed_twice_side_by_side(ctx):
    """Two layers captured into two graphs that are replayed at the same time on two streams."""
    layers = [Layer(ctx, 200, 640, 384, seed) for seed in (1, 2)]
    for v in layers:
        v.step()                                       # first use loads the kernels
    ctx.synchronize()
    want = [v.results() for v in layers]
    graphs, streams = [], [torch.cuda.Stream() for _ in layers]
    for v, s in zip(layers, streams):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            v.step()
        graphs.append(gr)
    for v in layers:
        v.dw.fill_(1.0)
    torch.cuda.synchronize()
    for _ in range(3):
        for gr, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
    torch.cuda.synchronize()
    ctx.synchronize()
    for v, w in zip(layers, want):
        for a, c in zip(v.results()[:4], w[:4]):
            assert torch.equal(a, c)
        for a, c in zip(v.results()[5:], w[5:]):
            assert torch.equal(a, c)
        v.check(steps=3)


@gpu
def test_capture_refuses_what_needs_scratch(ctx):
    A, _ = int_matrix(gen(1), 4, 256, b.FP8_E4M3, 1, pad=3)
    B, _ = int_matrix(gen(2), 64, 256, b.FP8_E4M3, 128)
    x, gamma = torch.randn(4, 256, device=DEV), torch.ones(256, device=DEV)
    D, dx, dg = torch.empty(4, 64, device=DEV), torch.empty_like(x), torch.empty_like(gamma)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        for call in (lambda: ctx.gemm_fp8(A, B, D, 64, stream=cur()),
                     lambda: ctx.rmsnorm_backward(4, 256, x, 256, x, 256, gamma, 1e-6, dx, 256, dg, stream=cur())):
            with pytest.raises(b.DecxbError) as e:
                call()
            assert e.value.status == 13
        ctx.rmsnorm_backward(4, 256, x, 256, x, 256, gamma, 1e-6, dx, 256, None, stream=cur())
    gr.replay()
    torch.cuda.synchronize()
    assert torch.isfinite(dx).all()


@gpu
def test_pitches_and_offsets_beyond_32_bits(ctx):
    """Three rows 2^31 + 64 elements apart, and results that far apart, in every operator."""
    far, rows, cols = 2 ** 31 + 64, 3, 640
    g = gen(4)
    x = torch.randn(rows, cols, device=DEV, generator=g).to(torch.bfloat16)
    gamma = torch.ones(cols, device=DEV)
    apart = torch.empty(2 * far + cols, device=DEV, dtype=torch.bfloat16)

    def view(t):
        return torch.as_strided(t, (rows, cols), (far, 1))
    view(apart).copy_(x)
    out = torch.empty_like(apart)
    Y, Q, T = torch.empty_like(x), b.Fp8Matrix.empty(rows, cols), b.Fp8Matrix.empty(cols, rows)
    ctx.rmsnorm(rows, cols, x, cols, gamma, 1e-6, Y=Y, ldy=cols, Q=Q, stream=cur())
    ctx.rmsnorm(rows, cols, apart, far, gamma, 1e-6, Y=out, ldy=far, stream=cur())
    assert torch.equal(view(out), Y)
    dx = torch.empty_like(x)
    ctx.rmsnorm_backward(rows, cols, Y, cols, x, cols, gamma, 1e-6, dx, cols, stream=cur())
    ctx.rmsnorm_backward(rows, cols, out, far, apart, far, gamma, 1e-6, out, far, stream=cur())
    assert torch.equal(view(out), dx)
    codes = torch.empty(2 * far + cols, device=DEV, dtype=torch.float8_e4m3fn)
    F = b.Fp8Matrix(codes, torch.empty(rows * 5, device=DEV), rows, cols, far, 5, 1)
    ctx.quantize_fp8(rows, cols, apart, far, F, T, stream=cur())
    ctx.quantize_fp8(rows, cols, x, cols, Q, stream=cur())
    ctx.synchronize()
    assert torch.equal(view(codes).view(torch.uint8), Q.data.view(torch.uint8)) and torch.equal(F.scales.view(rows, 5), Q.scales)
    W, w = int_matrix(g, 256, cols, b.FP8_E4M3, 128)
    near, dist = torch.empty(rows, 256, device=DEV, dtype=torch.bfloat16), apart
    ctx.gemm_fp8(Q, W, near, 256, stream=cur())
    ctx.gemm_fp8(F, W, dist, far, stream=cur())
    ctx.gemm_fp8(F, W, dist, far, Cin=dist, ldc=far, stream=cur())
    ctx.synchronize()
    assert torch.equal(torch.as_strided(dist, (rows, 256), (far, 1)), (near.float() * 2).bfloat16())


@gpu
@pytest.mark.parametrize("short", [16, 0])
def test_quantise_rows_up_to_and_over_16_mib_apart(ctx, short):
    """Whole tiles whose rows lie just under 2^24 bytes apart, and just there, in the input and in both outputs."""
    rows, cols, apart = 128, 256, 2 ** 24 - short
    g = gen(6)
    x = torch.randn(rows, cols, device=DEV, generator=g).to(torch.bfloat16)
    far = torch.empty(rows * apart // 2, device=DEV, dtype=torch.bfloat16)
    torch.as_strided(far, (rows, cols), (apart // 2, 1)).copy_(x)
    q, t = (torch.empty(n * apart, device=DEV, dtype=torch.float8_e4m3fn) for n in (rows, cols))
    Q = b.Fp8Matrix.of(torch.as_strided(q, (rows, cols), (apart, 1)), torch.empty(rows, 2, device=DEV))
    T = b.Fp8Matrix.of(torch.as_strided(t, (cols, rows), (apart, 1)), torch.empty(cols, 1, device=DEV))
    nearQ, nearT = b.Fp8Matrix.empty(rows, cols), b.Fp8Matrix.empty(cols, rows)
    ctx.quantize_fp8(rows, cols, far, apart // 2, Q, T, stream=cur())
    ctx.quantize_fp8(rows, cols, x, cols, nearQ, nearT, stream=cur())
    ctx.synchronize()
    for a, c in ((Q, nearQ), (T, nearT)):
        assert torch.equal(a.data.view(torch.uint8), c.data.view(torch.uint8)) and torch.equal(a.scales, c.scales)


_FIRST_CALL_CAPTURED = r"""
import torch
import backup_1_b200 as b
ctx = b.Context(0)
t, w, o = 130, 512, 384
x, g = torch.randn(t, w, device="cuda").bfloat16(), torch.ones(w, device="cuda")
W = torch.randn(o, w, device="cuda")
q, wq, out = b.Fp8Matrix.empty(t, w), b.Fp8Matrix.empty(o, w, 128), torch.zeros(t, o, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    s = torch.cuda.current_stream()
    ctx.quantize_fp8(o, w, W, w, wq, stream=s)
    ctx.rmsnorm(t, w, x, w, g, 1e-6, Q=q, stream=s)
    ctx.gemm_fp8(q, wq, out, o, stream=s)
graph.replay()
torch.cuda.synchronize()
ctx.synchronize()
first = out.clone()
assert float(first.abs().max()) > 0
ctx.quantize_fp8(o, w, W, w, wq, stream=torch.cuda.current_stream())
ctx.rmsnorm(t, w, x, w, g, 1e-6, Q=q, stream=torch.cuda.current_stream())
ctx.gemm_fp8(q, wq, out, o, stream=torch.cuda.current_stream())
torch.cuda.synchronize()
assert torch.equal(first, out)
print("captured first call ok")
"""


@gpu
def test_the_first_call_of_a_process_may_be_captured():
    import subprocess
    import sys
    from pathlib import Path

    r = subprocess.run([sys.executable, "-c", _FIRST_CALL_CAPTURED], cwd=Path(__file__).resolve().parents[1], capture_output=True,
                       text=True, timeout=300)
    assert r.returncode == 0 and "captured first call ok" in r.stdout, r.stdout[-1000:] + r.stderr[-2000:]


@gpu
def test_two_threads_call_at_once(ctx):
    """Two host threads, each with its own stream, on one context: the results of either alone."""
    import threading

    layers = [Layer(ctx, 300, 384, 512, seed) for seed in (5, 6)]
    want = []
    for v in layers:
        v.step()
        torch.cuda.synchronize()
        want.append(v.results())
    streams = [torch.cuda.Stream() for _ in layers]
    failures = []

    def work(v, s):
        try:
            with torch.cuda.stream(s):
                for _ in range(20):
                    v.dw.fill_(1.0)
                    v.step()
        except Exception as e:       # noqa: BLE001
            failures.append(e)
    threads = [threading.Thread(target=work, args=a) for a in zip(layers, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    ctx.synchronize()
    assert not failures, failures
    for v, w in zip(layers, want):
        for a, c in zip(v.results(), w):
            assert torch.equal(a, c)


@gpu
def test_the_callers_device_is_left_and_errors_have_a_text(ctx):
    L = ctx.L
    before = torch.cuda.current_device()
    A = b.Fp8Matrix.empty(4, 256)
    assert L.decxb_gemm_fp8(ctx.h, A.addr, A.addr, None, 0, None, 0, 4, None) == 13
    assert b"D: null" in L.decxb_last_error(ctx.h)
    assert torch.cuda.current_device() == before


@gpu
def test_calls_on_the_contexts_own_stream_and_on_another(ctx):
    """Without a stream the context's own is used, after torch's current one; with one, the work is ordered on it."""
    layer = Layer(ctx, 64, 256, 128)
    t, w, o = layer.dims
    ctx.quantize_fp8(o, w, layer.w, w, layer.wq)
    ctx.rmsnorm(t, w, layer.x, w, layer.gamma, 1e-6, Q=layer.q)
    ctx.gemm_fp8(layer.q, layer.wq, layer.out, o)
    ctx.synchronize()
    first = layer.out.clone()
    s = torch.cuda.Stream()
    s.wait_stream(cur())
    with torch.cuda.stream(s):
        x2 = layer.x * 1
        ctx.rmsnorm(t, w, x2, w, layer.gamma, 1e-6, Q=layer.q, stream=s)
        ctx.gemm_fp8(layer.q, layer.wq, layer.out, o, stream=s)
        again = layer.out * 1
    s.synchronize()
    assert torch.equal(first, again)
    assert math.isfinite(float(again.float().sum()))


# ---- borders of the scales' rules ---------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("kind", [b.FP8_E4M3, b.FP8_E5M2])
@pytest.mark.parametrize("dtype", FLOATS)
def test_quantise_scales_at_and_next_to_powers_of_two(ctx, dtype, kind):
    """Blocks whose largest magnitude is the type's largest value times a power of two, and the numbers just under and just over:
    amax / FMAX is a power of two itself, where a rule by logarithms is off by a factor of two if the logarithm is a step too large."""
    lo, hi = {torch.bfloat16: (-100, 100), torch.float32: (-100, 100), torch.float16: (-20, 0)}[dtype]
    at = FMAX[kind] * torch.exp2(torch.arange(lo, hi + 1, device=DEV, dtype=torch.float64))
    step = 2 * HALF[dtype]                                   # to the next number up, relative to the power of two below
    amax = torch.cat([at, at * (1 - step / 1.75), at * (1 + step / 1.75)]).to(dtype)      # 448 = 1.75 * 2^8, 57344 = 1.75 * 2^15
    amax = torch.cat([amax[:2 * at.numel()], amax[2 * at.numel():][torch.isfinite(amax[2 * at.numel():])]])
    rows = amax.numel()
    assert torch.unique(amax).numel() == rows
    g = gen(12)
    x = (amax[:, None].double() * (2 * torch.rand(rows, 128, device=DEV, generator=g) - 1).double() * 0.99).to(dtype)
    x[torch.arange(rows), torch.randint(0, 128, (rows,), device=DEV, generator=g)] = amax
    x[::2] = -x[::2]
    for rule in (b.SCALE_AMAX, b.SCALE_POW2):
        Q, T = b.Fp8Matrix.empty(rows, 128, 1, kind), b.Fp8Matrix.empty(128, rows, 1, kind)
        ctx.quantize_fp8(rows, 128, x, 128, Q, T, rule=rule, stream=cur())
        ctx.synchronize()
        for m, y in ((Q, x.double()), (T, x.double().t())):
            s = want_scales(blocks_amax(y, 1), kind, rule)
            assert torch.equal(m.scales, s)
            check_codes(m.data, (y / spread(s, 1, *y.shape).double()).float().double(), kind, 0.0)


# ---- copies that never come ---------------------------------------------------------------------------------------------
class LostCopy:
    """Within it the next launch leaves out the copies of one row or tile; on leaving, the wait for them has run out and was reported."""

    def __init__(self, ctx, which):
        self.ctx, self.which = ctx, which

    def __enter__(self):
        self.ctx.set_wait_limit_ms(30)
        assert self.ctx.L.decxb_inject_lost_copy(self.ctx.h, self.which) == 0

    def __exit__(self, kind, *_):
        self.ctx.L.decxb_inject_lost_copy(self.ctx.h, -1)
        if kind is None:
            with pytest.raises(b.DecxbError) as e:
                self.ctx.synchronize()
            assert e.value.status == 103
        self.ctx.set_wait_limit_ms(1000)


def sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


@gpu
@pytest.mark.parametrize("turn", [0, 2, 3])
@pytest.mark.parametrize("res", [False, True])
def test_norm_leaves_rows_that_did_not_come(ctx, turn, res):
    """A block's row of its first, third or fourth turn does not come: that row and the block's later ones stay as they were, all others are right."""
    cols, grid = 2304, 2 * sms()
    rows = 6 * grid + 11
    g = gen(31)
    x, r = (torch.randn(rows, cols, device=DEV, generator=g).bfloat16() for _ in range(2))
    gamma = torch.randn(cols, device=DEV, generator=g)
    kw = dict(R=r, ldr=cols) if res else {}

    def run():
        Y, Q = torch.full_like(x, 9.0), b.Fp8Matrix.empty(rows, cols)
        Q.data.view(torch.uint8).fill_(0x11)
        Q.scales.fill_(7.0)
        ctx.rmsnorm(rows, cols, x, cols, gamma, 1e-5, Y=Y, ldy=cols, Q=Q, stream=cur(), **kw)
        torch.cuda.synchronize()
        return Y, Q.data.view(torch.uint8).clone(), Q.scales.clone()
    want = run()
    ctx.synchronize()
    with LostCopy(ctx, turn * grid + 5):
        got = run()
    left = torch.zeros(rows, dtype=torch.bool, device=DEV)
    left[torch.arange(turn * grid + 5, rows, grid)] = True
    for v, w, was in zip(got, want, (9.0, 0x11, 7.0)):
        assert torch.equal(v[~left], w[~left]) and bool((v[left] == was).all())
    for v, w in zip(run(), want):
        assert torch.equal(v, w)
    ctx.synchronize()


@gpu
@pytest.mark.parametrize("turn", [0, 3])
@pytest.mark.parametrize("cols,dtype", [(1032, torch.bfloat16), (4096, torch.bfloat16), (5120, torch.float16), (9008, torch.bfloat16), (2048, torch.float32)])
def test_norm_backward_leaves_rows_that_did_not_come(ctx, cols, dtype, turn):
    grid = ctx.rmsnorm_backward_workspace(2 ** 20, cols) // (4 * cols)          # what the device takes at once
    rows = 5 * grid + 3
    g = gen(32)
    h, dy, dr = (torch.randn(rows, cols, device=DEV, generator=g).to(dtype) for _ in range(3))
    gamma = torch.randn(cols, device=DEV, generator=g)
    ws = torch.empty(ctx.rmsnorm_backward_workspace(rows, cols), device=DEV, dtype=torch.uint8)

    def run():
        dx, dg = torch.full_like(h, 9.0), torch.empty(cols, device=DEV)
        ctx.rmsnorm_backward(rows, cols, dy, cols, h, cols, gamma, 1e-5, dx, cols, dg, dR=dr, lddr=cols, workspace=ws, workspace_bytes=ws.numel(), stream=cur())
        torch.cuda.synchronize()
        return dx, dg
    want, dgamma = run()
    ctx.synchronize()
    with LostCopy(ctx, turn * grid + 2):
        got, dgamma_without = run()
    left = torch.zeros(rows, dtype=torch.bool, device=DEV)
    left[torch.arange(turn * grid + 2, rows, grid)] = True
    assert torch.equal(got[~left], want[~left]) and bool((got[left] == 9).all())
    wg, mg = backward_ref(dy[~left], h[~left], gamma, 1e-5, None)[1::2]
    longest = 6 + -(-grid // 32) + 6                       # as in test_norm_backward
    assert bool(((dgamma_without.double() - wg).abs() <= (96 + longest + 4) * U * mg).all())
    again, dg = run()
    assert torch.equal(again, want) and torch.equal(dg, dgamma)
    ctx.synchronize()


@gpu
@pytest.mark.parametrize("M,N,K", [(1, 300, 128), (1, 512, 4096), (20, 700, 2048), (50, 640, 3000), (100, 512, 4096)])
def test_product_of_few_tiles_leaves_a_tile_that_did_not_come(ctx, M, N, K):
    """The last k-block of the first share of tile 1 (128 rows of B) does not come: its columns stay as they were, all others are right."""
    g = gen(33)
    A, a = int_matrix(g, M, K, b.FP8_E4M3, 1, pad=-K % 16)
    B, w = int_matrix(g, N, K, b.FP8_E4M3, 128, pad=-K % 16)
    want = a @ w.t()
    for tile in (0, 1):
        D = torch.full((M, N), 9.0, device=DEV)
        with LostCopy(ctx, tile):
            ctx.gemm_fp8(A, B, D, N, stream=cur())
            torch.cuda.synchronize()
        left = torch.zeros(N, dtype=torch.bool, device=DEV)
        left[tile * 128:tile * 128 + 128] = True
        assert torch.equal(D[:, ~left].double(), want[:, ~left]) and bool((D[:, left] == 9).all())
    assert torch.equal(run_gemm(ctx, A, B, torch.float32).double(), want)


@gpu
@pytest.mark.parametrize("addend", [False, True])
@pytest.mark.parametrize("b_rows", [1, 128])
def test_product_of_many_tiles_leaves_tiles_that_did_not_come(ctx, b_rows, addend):
    """The last k-block of a tile of 256 x 256 does not come: that tile and the later ones of its pair of SMs stay as they were."""
    M, N, K, pairs = 4096, 4096, 512, sms() // 2
    g = gen(34)
    A, a = int_matrix(g, M, K, b.FP8_E4M3, 1)
    B, w = int_matrix(g, N, K, b.FP8_E4M3, b_rows)
    Cin = torch.full((M, N), 3.0, device=DEV) if addend else None
    want = (a @ w.t() + (3.0 if addend else 0.0)).float()
    for tile in (0, pairs + 6):
        D = torch.full((M, N), 9.5, device=DEV)                               
        with LostCopy(ctx, tile):
            ctx.gemm_fp8(A, B, D, N, Cin=Cin, ldc=N if addend else 0, stream=cur())
            torch.cuda.synchronize()
        tiles = lambda v: v.view(16, 256, 16, 256).transpose(1, 2).reshape(256, -1)  # noqa: E731
        left = (tiles(D) == 9.5).all(1)
        assert int(left.sum()) == len(range(tile, 256, pairs))
        assert torch.equal(tiles(D)[~left], tiles(want)[~left])
    assert torch.equal(run_gemm(ctx, A, B, torch.float32, Cin), want)


# ---- two threads ---------------------------------------------------------------------------------------------------------
@gpu
def test_two_threads_are_refused_at_once_and_each_reads_its_own_text(ctx):
    import threading

    A, Q, x = b.Fp8Matrix.empty(4, 256), b.Fp8Matrix.empty(4, 256), torch.zeros((4, 256), device=DEV)
    calls = [(lambda: ctx.gemm_fp8(A, A, x.data_ptr(), 3, d_type=b.F32, stream=cur()), "D: leading dimension smaller than the row length"),
             (lambda: ctx.quantize_fp8(4, 256, x, 256, Q, rule=77, stream=cur()), "scale rule"),
             (lambda: ctx.rmsnorm(4, 256, x, 256, x, -1.0, Y=x, ldy=256, stream=cur()), "eps must be a finite number >= 0")]
    wrong, start = [], threading.Barrier(len(calls))

    def work(call, text):
        torch.cuda.set_device(0)
        start.wait()
        for _ in range(3000):
            try:
                call()
                wrong.append("not refused")
            except b.DecxbError as e:
                if text not in str(e):
                    wrong.append(str(e))
    threads = [threading.Thread(target=work, args=c) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[:5]
    with pytest.raises(b.DecxbError) as e:                  # this thread's own, though others failed later
        ctx.quantize_fp8(4, 256, x, 256, None, stream=cur())
    work_text = []
    t = threading.Thread(target=lambda: work_text.append(ctx.L.decxb_last_error(ctx.h).decode()))
    t.start()
    t.join()
    assert "nothing to write" in str(e.value) and "nothing to write" in work_text[0]       # a thread without a failure reads the last one


# ---- tensors that do not hold what a call reaches -----------------------------------------------------------------------
class Entries:
    """The library, as far as a call that has been let through goes: nothing runs."""

    def __init__(self):
        self.calls = 0

    def __getattr__(self, name):
        def entry(*args):
            self.calls += 1
            return 0
        return entry


def host_context():
    """A context whose device is the host's memory (-1, as its tensors say) and whose entries do nothing."""
    c = b.Context.__new__(b.Context)
    c.L, c.h, c.device = Entries(), None, -1
    return c


def test_tensors_that_are_too_small_or_not_rows_are_refused():
    c, e = host_context(), torch.empty
    bf = dict(dtype=torch.bfloat16)
    A, W, Q, T = (b.Fp8Matrix.empty(r, k, br, device="cpu") for r, k, br in [(4, 256, 1), (8, 256, 128), (4, 256, 1), (256, 4, 1)])
    x, gamma, wide = e(4, 256, **bf), e(256), e(4, 300, **bf)[:, :256]
    ok = [lambda: c.gemm_fp8(A, W, e(4, 8), 8), lambda: c.gemm_fp8(A, W, e(3 * 11 + 8), 11, Cin=e(4, 8), ldc=8),
          lambda: c.gemm_fp8(A, W, e(4, 20)[:, :8], 20), lambda: c.gemm_fp8(A, W, 4096, 8, d_type=b.F16),
          lambda: c.quantize_fp8(4, 256, x, 256, Q, T), lambda: c.quantize_fp8(4, 256, wide, 300, Q), lambda: c.quantize_fp8(4, 256, e(2, 2, 256), 256, Q),
          lambda: c.quantize_fp8(1, 256, e(256), 256, b.Fp8Matrix.empty(1, 256, device="cpu")),
          lambda: c.quantize_fp8(0, 256, e(0, 256), 256, b.Fp8Matrix.empty(0, 256, device="cpu")),
          lambda: c.rmsnorm(4, 256, wide, 300, gamma, 1e-6, R=x, ldr=256, H=x, ldh=256, Y=wide, ldy=300, Q=Q),
          lambda: c.rmsnorm_backward(4, 256, x, 256, wide, 300, gamma, 1e-6, x, 256, gamma, dR=x, lddr=256, workspace=e(300), workspace_bytes=1200),
          lambda: c.rmsnorm_backward(0, 256, x, 256, x, 256, gamma, 1e-6, x, 256, gamma)]
    for call in ok:
        call()
    assert c.L.calls == len(ok)
    g2 = e(512)[::2]
    bad = [lambda: c.gemm_fp8(A, W, e(4, 7), 8), lambda: c.gemm_fp8(A, W, e(3, 8), 8), lambda: c.gemm_fp8(A, W, e(3 * 11 + 7), 11),
           lambda: c.gemm_fp8(A, W, e(8, 4).t(), 8), lambda: c.gemm_fp8(A, W, e(4, 8), 8, Cin=e(8).expand(4, 8), ldc=8),
           lambda: c.gemm_fp8(A, W, e(4, 8), 8, Cin=e(3, 8), ldc=8),
           lambda: c.quantize_fp8(4, 256, e(3, 256), 256, Q), lambda: c.quantize_fp8(4, 256, e(256, 4).t(), 256, Q), lambda: c.quantize_fp8(4, 256, wide, 301, Q),
           lambda: c.quantize_fp8(4, 256, e(1, 256).expand(4, 256), 256, Q), lambda: c.quantize_fp8(4, 256, x[3:], 256, None, T),
           lambda: c.rmsnorm(4, 256, x[1:], 256, gamma, 1e-6, Q=Q), lambda: c.rmsnorm(4, 256, x, 256, gamma[1:], 1e-6, Q=Q),
           lambda: c.rmsnorm(4, 256, x, 256, g2, 1e-6, Q=Q), lambda: c.rmsnorm(4, 256, x, 256, gamma, 1e-6, R=x, ldr=257, Q=Q),
           lambda: c.rmsnorm(4, 256, x, 256, gamma, 1e-6, H=x[:3], ldh=256), lambda: c.rmsnorm(4, 256, x, 256, gamma, 1e-6, Y=x[:3], ldy=256),
           lambda: c.rmsnorm_backward(4, 256, x[1:], 256, x, 256, gamma, 1e-6, x, 256), lambda: c.rmsnorm_backward(4, 256, x, 256, x[1:], 256, gamma, 1e-6, x, 256),
           lambda: c.rmsnorm_backward(4, 256, x, 256, x, 256, gamma[1:], 1e-6, x, 256), lambda: c.rmsnorm_backward(4, 256, x, 256, x, 256, gamma, 1e-6, x[1:], 256),
           lambda: c.rmsnorm_backward(4, 256, x, 256, x, 256, gamma, 1e-6, x, 256, e(255)), lambda: c.rmsnorm_backward(4, 256, x, 256, x, 256, gamma, 1e-6, x, 256, g2),
           lambda: c.rmsnorm_backward(0, 256, x, 256, x, 256, gamma, 1e-6, x, 256, e(255)),
           lambda: c.rmsnorm_backward(4, 256, x, 256, x, 256, gamma, 1e-6, x, 256, dR=x[1:], lddr=256),
           lambda: c.rmsnorm_backward(4, 256, x, 256, x, 256, gamma, 1e-6, x, 256, gamma, workspace=e(299), workspace_bytes=1200)]
    for i, call in enumerate(bad):
        with pytest.raises(b.DecxbError) as err:
            call()
        assert err.value.status == 13, i
    assert c.L.calls == len(ok)


def test_the_default_streams_handle_is_not_the_contexts_own_stream():
    assert blib._stream(0) == 1 and blib._stream(2) == 2


def test_calls_without_a_stream_wait_for_torch_whichever_argument_is_torchs(monkeypatch):
    waits = []

    class OnDevice:
        """As much of a CUDA tensor as a call looks at."""
        is_cuda, device, dtype = True, "cuda:0", torch.float32

        def get_device(self):
            return -1

        def numel(self):
            return 1 << 20

        def is_contiguous(self):
            return True

        def data_ptr(self):
            return 4096

    class Stream:
        def synchronize(self):
            waits.append(1)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream())
    c, t, p = host_context(), OnDevice(), 4096
    raw = b.Fp8Matrix(p, p, 4, 256, 256, 1, 4)
    raw_t, mixed = b.Fp8Matrix(p, p, 256, 4, 16, 1, 256), b.Fp8Matrix(p, p, 4, 256, 256, 1, 4)
    mixed.data = t
    f = dict(x_type=b.F32)
    calls = [lambda **s: c.gemm_fp8(raw, raw, t, 4, **s), lambda **s: c.gemm_fp8(raw, mixed, p, 4, d_type=b.F32, **s),
             lambda **s: c.gemm_fp8(raw, raw, p, 4, Cin=t, ldc=4, d_type=b.F32, **s),
             lambda **s: c.quantize_fp8(4, 256, p, 256, mixed, **f, **s), lambda **s: c.quantize_fp8(4, 256, t, 256, raw, raw_t, **s),
             lambda **s: c.rmsnorm(4, 256, p, 256, p, 1e-6, Y=t, ldy=256, type=b.F32, gamma_type=b.F32, **s),
             lambda **s: c.rmsnorm(4, 256, p, 256, t, 1e-6, Y=p, ldy=256, type=b.F32, **s),
             lambda **s: c.rmsnorm_backward(4, 256, t, 256, p, 256, p, 1e-6, p, 256, type=b.F32, gamma_type=b.F32, **s),
             lambda **s: c.rmsnorm_backward(4, 256, p, 256, p, 256, p, 1e-6, p, 256, t, type=b.F32, gamma_type=b.F32, **s)]
    for i, call in enumerate(calls):
        call()
        assert len(waits) == i + 1, i
    for call in calls:
        call(stream=7)
    c.gemm_fp8(raw, raw, p, 4, d_type=b.F32)               # nothing of torch's
    assert len(waits) == len(calls)


@gpu
def test_a_call_on_the_default_streams_handle_follows_what_is_queued_there(ctx):
    """The input is still being written when the call is made, and torch reads the result without waiting."""
    rows, cols = 4096, 4096
    x = torch.empty(rows, cols, device=DEV)
    gamma, Y = torch.ones(cols, device=DEV), torch.zeros(rows, cols, device=DEV)
    big = torch.randn(8192, 8192, device=DEV)
    with torch.cuda.stream(torch.cuda.default_stream()):
        for _ in range(8):
            big = big @ big * 1e-2                          # some milliseconds
        x.fill_(2.0)
        ctx.rmsnorm(rows, cols, x, cols, gamma, 0.0, Y=Y, ldy=cols, stream=torch.cuda.current_stream().cuda_stream)
        got = Y.clone()
    torch.cuda.synchronize()
    assert bool((got - 1).abs().max() <= 8 * U)


@gpu
def test_products_of_every_form_side_by_side(ctx):
    """Four streams with products of one token to many, cut over clusters, two blocks to an SM and pairs, all at once: exact, and all end."""
    g = gen(35)
    shapes = [(1, 4096, 2048), (1, 6000, 4096), (20, 12000, 1024), (64, 20000, 512), (40, 5000, 4096), (100, 512, 2048), (2048, 1280, 384), (1, 20000, 640)]
    made = []
    for M, N, K in shapes:
        A, a = int_matrix(g, M, K, b.FP8_E4M3, 1)
        B, w = int_matrix(g, N, K, b.FP8_E4M3, 128)
        made.append((A, B, torch.empty((M, N), device=DEV), (a @ w.t()).float()))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    for turn in range(12):
        for i, s in enumerate(streams):
            for j in range(len(made)):
                A, B, D, _ = made[(j + turn + 2 * i) % len(made)]
                if j % 4 == i:
                    ctx.gemm_fp8(A, B, D, D.shape[1], stream=s)
        torch.cuda.synchronize()
    ctx.synchronize()
    for A, B, D, want in made:
        for s in streams:
            D.fill_(-1.0)
            torch.cuda.synchronize()
            ctx.gemm_fp8(A, B, D, D.shape[1], stream=s)
            torch.cuda.synchronize()
            assert torch.equal(D, want)


@gpu
def test_tensor_probes_of_two_contexts_beside_products(ctx):
    """Two threads probe the tensor cores, each on its own context, while products run on two more streams: all end, the products are exact."""
    import threading

    other, g = b.Context(0), gen(36)
    made = []
    for M, N, K in [(1, 6000, 4096), (64, 20000, 512), (2048, 1280, 384)]:
        A, a = int_matrix(g, M, K, b.FP8_E4M3, 1)
        B, w = int_matrix(g, N, K, b.FP8_E4M3, 128)
        made.append((A, B, torch.empty((M, N), device=DEV), (a @ w.t()).float()))
    torch.cuda.synchronize()
    rates = []
    threads = [threading.Thread(target=lambda c=c, p=p: rates.append(c.probe_tensor_peak(p, 20.0)["tensor_tflops"])) for c, p in ((ctx, 1), (other, 3))]
    for t in threads:
        t.start()
    streams = [torch.cuda.Stream() for _ in made]
    for _ in range(100):
        for (A, B, D, _), s in zip(made, streams):
            ctx.gemm_fp8(A, B, D, D.shape[1], stream=s)
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    ctx.synchronize()
    other.synchronize()
    other.close()
    assert len(rates) == 2 and min(rates) > 0
    for _, _, D, want in made:
        assert torch.equal(D, want)


@gpu
@pytest.mark.parametrize("kind", ["norm", "backward", "few tiles", "many tiles"])
def test_a_wait_that_gave_up_does_not_cut_later_calls_short(ctx, kind):
    """Two calls whose copies are lost, nothing asked between: the second waits for its own limit, and a third that loses nothing is whole."""
    import time

    g = gen(37)
    if kind in ("norm", "backward"):
        rows, cols = 8 * 2 * sms(), 2304
        x, gamma, Y = torch.randn(rows, cols, device=DEV, generator=g).bfloat16(), torch.ones(cols, device=DEV), torch.empty(rows, cols, device=DEV, dtype=torch.bfloat16)
        if kind == "norm":
            call = lambda: ctx.rmsnorm(rows, cols, x, cols, gamma, 1e-6, Y=Y, ldy=cols, stream=cur())  # noqa: E731
        else:
            call = lambda: ctx.rmsnorm_backward(rows, cols, x, cols, x, cols, gamma, 1e-6, Y, cols, stream=cur())  # noqa: E731
    else:
        M, N, K = (4, 512, 2048) if kind == "few tiles" else (2048, 1280, 384)
        A, _ = int_matrix(g, M, K, b.FP8_E4M3, 1)
        B, _ = int_matrix(g, N, K, b.FP8_E4M3, 128)
        Y = torch.empty(M, N, device=DEV)
        call = lambda: ctx.gemm_fp8(A, B, Y, N, stream=cur())  # noqa: E731
    call()
    ctx.synchronize()
    want = Y.clone()
    try:
        ctx.set_wait_limit_ms(400)
        took = []
        for _ in range(2):
            ctx.L.decxb_inject_lost_copy(ctx.h, 0)
            t0 = time.perf_counter()
            call()
            torch.cuda.synchronize()
            took.append(time.perf_counter() - t0)
        Y.zero_()
        call()
        torch.cuda.synchronize()
        assert torch.equal(Y, want)
        with pytest.raises(b.DecxbError) as e:
            ctx.synchronize()
        assert e.value.status == 103
        assert min(took) >= 0.4, took
    finally:
        ctx.L.decxb_inject_lost_copy(ctx.h, -1)
        ctx.set_wait_limit_ms(1000)
    ctx.synchronize()


# ---- loops over many rows, and every form of a kernel -------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype,gtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32), (torch.float32, torch.float32)])
@pytest.mark.parametrize("rows,cols", [(10000, 64), (10000, 250), (6001, 1032), (3001, 4096), (1301, 5120), (701, 9008), (1301, 5121), (701, 16400), (2501, 2044)])
def test_norm_backward_of_more_rows_than_blocks(ctx, rows, cols, dtype, gtype):
    """Every block (up to 256 columns: every warp) takes several rows: stages that are filled again, sums that alternate, dgamma over the rows of a block;
    dX apart, in place of dY and in place of dR gives the same bits.  Bounds as in test_norm_backward."""
    blocks = ctx.rmsnorm_backward_workspace(rows, cols) // (4 * cols)
    at_once = blocks * (8 if cols <= 256 else 1)
    assert rows > 2 * at_once or (cols <= 256 and rows > at_once)
    g = gen(rows + 5 * cols)
    h, dy, dr = (torch.randn(rows, cols, device=DEV, generator=g).to(dtype) for _ in range(3))
    gamma = (1 + 0.2 * torch.randn(cols, device=DEV, generator=g)).to(gtype)
    n = ctx.rmsnorm_backward_workspace(rows, cols)
    ws = torch.empty(n, device=DEV, dtype=torch.uint8)
    longest = -(-rows // blocks) + -(-blocks // 32) + 6
    wide = 1.0 if cols <= 16384 else cols / 16384 * 4
    small = 2.0 ** -25 if dtype == torch.float16 else 0.0

    def run(y, res, dx):
        dg = torch.full((cols,), float("nan"), device=DEV)
        ctx.rmsnorm_backward(rows, cols, y, cols, h, cols, gamma, 1e-5, dx, cols, dg, dR=res, lddr=cols, workspace=ws, workspace_bytes=n, stream=cur())
        ctx.synchronize()
        return dx, dg
    for res in (None, dr):
        dx, dg = run(dy, res, torch.empty_like(h))
        wx, wg, mx, mg = backward_ref(dy, h, gamma, 1e-5, res)
        assert bool(((dx.double() - wx).abs() <= HALF[dtype] * wx.abs() * 1.001 + 200 * wide * U * mx + small).all())
        assert bool(((dg.double() - wg).abs() <= (96 * wide + longest + 4) * U * mg).all())
        y = dy.clone()
        again, dg2 = run(y, res, y)
        assert torch.equal(again, dx) and torch.equal(dg2, dg)
    r = dr.clone()
    again, dg2 = run(dy, r, r)
    assert torch.equal(again, dx) and torch.equal(dg2, dg)


@gpu
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,cols", [(3, 9001), (2, 10240), (3, 16400), (2, 20003), (2, 32760), (1300, 1028), (40, 5121), (2400, 4096), (5000, 200)])
def test_norm_of_rows_that_need_several_vectors_a_thread_and_ragged_ones(ctx, rows, cols, dtype):
    g = gen(rows + cols)
    x, r = (torch.randn(rows, cols, device=DEV, generator=g).to(dtype) for _ in range(2))
    gamma = (1 + 0.2 * torch.randn(cols, device=DEV, generator=g)).to(dtype)
    h, y = norm_ref(x, r, gamma, 1e-5)
    H, Y, Q = torch.empty_like(x), torch.empty_like(x), b.Fp8Matrix.empty(rows, cols)
    ctx.rmsnorm(rows, cols, x, cols, gamma, 1e-5, R=r, ldr=cols, H=H, ldh=cols, Y=Y, ldy=cols, Q=Q, stream=cur())
    ctx.synchronize()
    assert near(H, h, dtype, U if dtype == torch.float32 else 2 * U) and near(Y, y, dtype, NORM_U)
    s = want_scales(blocks_amax(y, 1), b.FP8_E4M3, b.SCALE_AMAX).double()
    assert bool(((Q.scales.double() - s).abs() <= (NORM_U + 2 * U) * s).all())
    check_codes(Q.data, y / spread(Q.scales, 1, rows, cols).double(), b.FP8_E4M3, NORM_U + 4 * U)


@gpu
@pytest.mark.parametrize("M", [1, 16, 17, 32, 40, 64, 100])
@pytest.mark.parametrize("N,K", [(1000, 8200), (1024, 1024), (4096, 2048), (4090, 4100), (6000, 4096), (12000, 1000), (20000, 640), (40000, 130)])
def test_product_of_few_tokens_in_every_cut(ctx, M, N, K):
    """Eight, four, two shares of K and one, one block to an SM and two, over one wave and several."""
    g = gen(M + N + K)
    A, a = int_matrix(g, M, K, b.FP8_E4M3, 1, pad=-K % 16)
    B, w = int_matrix(g, N, K, b.FP8_E4M3, 128, pad=-K % 16)
    assert torch.equal(run_gemm(ctx, A, B, torch.float32).double(), a @ w.t())


@gpu
@pytest.mark.parametrize("dims", [(40, 1024, 520), (1500, 2304, 256), (3000, 640, 384)])
def test_layers_norm_and_its_gradients_within_the_layer(ctx, dims):
    """What Layer.check leaves out: the sum, the norm's output, dx and dgamma, each on what it was given."""
    layer = Layer(ctx, *dims)
    layer.step()
    ctx.synchronize()
    bf = torch.bfloat16
    h, y = norm_ref(layer.x, layer.r, layer.gamma, 1e-6)
    assert near(layer.h, h, bf, 2 * U) and near(layer.y, y, bf, NORM_U)
    wx, wg, mx, mg = backward_ref(layer.dy, layer.h, layer.gamma, 1e-6, layer.x)
    parts = layer.ws.numel() // (4 * dims[1])
    longest = -(-dims[0] // parts) + -(-parts // 32) + 6
    assert bool(((layer.dx.double() - wx).abs() <= HALF[bf] * wx.abs() * 1.001 + 200 * U * mx).all())
    assert bool(((layer.dgamma.double() - wg).abs() <= (96 + longest + 4) * U * mg).all())


@gpu
@pytest.mark.parametrize("M", [3, 300])
@pytest.mark.parametrize("rows_apart,blocks_apart", [(0, 0), (1, 0), (0, 1), (7, 3)])
def test_product_of_scales_shared_by_stride(ctx, M, rows_apart, blocks_apart):
    """One scale for a whole operand, for all of a row, for all rows of a block column, and scales with gaps."""
    g = gen(41)
    N, K = 260, 640
    made = []
    for n in (M, N):
        code = torch.randint(-4, 5, (n, K), device=DEV, generator=g).float().to(torch.float8_e4m3fn)
        s = torch.exp2(torch.randint(-2, 3, (n * rows_apart + 5 * blocks_apart + 1,), device=DEV, generator=g).float())
        at = (torch.arange(n, device=DEV)[:, None] * rows_apart + (torch.arange(K, device=DEV) // 128)[None, :] * blocks_apart)
        made.append((b.Fp8Matrix(code, s, n, K, K, rows_apart, blocks_apart), code.double() * s.double()[at]))
    (A, a), (B, w) = made
    assert torch.equal(run_gemm(ctx, A, B, torch.float32).double(), a @ w.t())
