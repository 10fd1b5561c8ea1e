"""The operators of a 4-bit transformer block on the B200 against their plain forms in 64 bits:
microscaled quantisation and product, block norms, attention over packed sequences."""
import ctypes as C
import math
import os
import pathlib
import shutil
import subprocess
import sys

import pytest
import torch

import mx_ref

pytestmark = pytest.mark.gpu

F32, F16, BF16 = 0, 1, 30
DEV = "cuda:0"


def _lib():
    from rfdetr_b200 import lib
    return lib.lib()


def _p(t):
    return None if t is None else t.data_ptr()


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _gen(seed):
    g = torch.Generator(DEV)
    g.manual_seed(seed)
    return g


def _mx_buffers(rows, k, fill=0xAB):
    kb = -(-k // 32)
    codes = torch.full((rows, kb * 16), fill, dtype=torch.uint8, device=DEV)
    scales = torch.full((_lib().rfdetr_b200_mx_scale_bytes(rows, k),), fill, dtype=torch.uint8, device=DEV)
    return codes, scales


def _quantize(x, type, k=None):
    rows, k = x.shape[0], k or x.shape[1]
    codes, scales = _mx_buffers(rows, k)
    assert _lib().rfdetr_b200_op_mx_quantize(_p(x), type, x.stride(0), rows, k, _p(codes), codes.shape[1], _p(scales),
                                             _stream()) == 0
    return codes, scales


def _operand(g, rows, k, spread=2.0):
    """A microscaled operand with block scales a few powers of two apart, and its float64 values."""
    x = torch.randn(rows, k, device=DEV, generator=g, dtype=torch.float64)
    x *= torch.exp2(torch.randint(-3, 4, (rows, -(-k // 32)), device=DEV, generator=g).double() * spread / 2
                    ).repeat_interleave(32, 1)[:, :k]
    codes, e = mx_ref.quantize(x)
    return mx_ref.pack(codes).contiguous(), mx_ref.tile_scales(e), mx_ref.values(codes, e)


# ---- quantisation -------------------------------------------------------------

SHAPES = [(1, 1), (1, 32), (3, 31), (2, 33), (1, 4096), (127, 100), (128, 128), (129, 256), (130, 520), (257, 384),
          (5, 1536), (1000, 264), (33, 8200), (2, 100000)]


@pytest.mark.parametrize("type", [F32, F16, BF16])
@pytest.mark.parametrize("rows,k", SHAPES)
def test_quantize_and_back(rows, k, type):
    """Codes, scales and the values read back are the definition's, bit for bit; the zeros that fill
    up the operand are written."""
    t = mx_ref.TYPES[type]
    g = _gen(rows * 31 + k)
    x = (torch.randn(rows, k, device=DEV, generator=g) * torch.exp(2 * torch.randn(rows, k, device=DEV, generator=g))).to(t)
    codes, scales = _quantize(x, type)
    want_c, want_e = mx_ref.quantize(x.double())
    assert torch.equal(codes, mx_ref.pack(want_c))
    assert torch.equal(scales, mx_ref.tile_scales(want_e))
    for bt in (F32, F16, BF16):
        back = torch.full((rows, k + 3), 7.0, dtype=mx_ref.TYPES[bt], device=DEV)
        assert _lib().rfdetr_b200_op_mx_dequantize(_p(codes), codes.shape[1], _p(scales), rows, k, _p(back), bt, k + 3,
                                                   _stream()) == 0
        assert torch.equal(back[:, :k], mx_ref.values(want_c, want_e)[:, :k].to(mx_ref.TYPES[bt]))
        assert (back[:, k:] == 7.0).all()


@pytest.mark.parametrize("type", [F32, F16, BF16])
@pytest.mark.parametrize("offset,pad", [(0, 8), (1, 0), (1, 3), (0, 1), (8, 16)])
def test_quantize_strides_and_alignment(type, offset, pad):
    """Rows with a pitch, starting anywhere: both the 16-byte and the element-wise reads."""
    rows, k = 37, 320
    t = mx_ref.TYPES[type]
    flat = torch.randn(rows * (k + pad) + offset, device=DEV, generator=_gen(5)).to(t)
    x = flat[offset:].view(rows, k + pad)[:, :k]
    codes, scales = _quantize(x, type)
    want_c, want_e = mx_ref.quantize(x.double())
    assert torch.equal(codes, mx_ref.pack(want_c)) and torch.equal(scales, mx_ref.tile_scales(want_e))


@pytest.mark.parametrize("k", [96, 100, 1536])
def test_quantize_writes_its_operand_only(k):
    """Codes with a pitch of their own: nothing between their rows is written, and it reads back."""
    rows, ld = 130, -(-k // 32) * 16 + 48
    x = torch.randn(rows, k, device=DEV, generator=_gen(k)).half()
    codes = torch.full((rows, ld), 0xAB, dtype=torch.uint8, device=DEV)
    n = _lib().rfdetr_b200_mx_scale_bytes(rows, k)
    scales = torch.full((n + 64,), 0xAB, dtype=torch.uint8, device=DEV)
    assert _lib().rfdetr_b200_op_mx_quantize(_p(x), F16, k, rows, k, _p(codes), ld, _p(scales), _stream()) == 0
    want_c, want_e = mx_ref.quantize(x.double())
    assert torch.equal(codes[:, :ld - 48], mx_ref.pack(want_c)) and (codes[:, ld - 48:] == 0xAB).all()
    assert torch.equal(scales[:n], mx_ref.tile_scales(want_e)) and (scales[n:] == 0xAB).all()
    back = torch.zeros(rows, k, dtype=torch.float16, device=DEV)
    assert _lib().rfdetr_b200_op_mx_dequantize(_p(codes), ld, _p(scales), rows, k, _p(back), F16, k, _stream()) == 0
    assert torch.equal(back, mx_ref.values(want_c, want_e)[:, :k].half())


def test_quantize_ties_and_extremes():
    """Every tie of the rounding in both signs, blocks at the ends of f32's range (subnormal and
    largest values), zero blocks, and blocks with infinities and NaN."""
    x = torch.zeros(24, 64)
    x[:, 0] = 4.0
    x[0, 1:9] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.99])
    x[1, 1:9] = -x[0, 1:9]
    x[2] = 0
    x[3] = -0.0
    x[4] = torch.finfo(torch.float32).max
    x[5] = 2.0 ** -126 * torch.linspace(0, 1, 64)       # subnormal
    x[6] = 2.0 ** -149
    x[7, 5] = math.inf
    x[8, 5] = -math.inf
    x[9, 40] = math.nan                                 # its row's other block stays
    x[10] = torch.linspace(-6, 6, 64)
    x[11] = 2.0 ** -128 * torch.linspace(-3, 3, 64)
    x[12:] = torch.exp2(torch.linspace(-140, 127, 12 * 64)).view(12, 64)
    x = x.to(DEV)
    codes, scales = _quantize(x, F32)
    want_c, want_e = mx_ref.quantize(x.double())
    assert torch.equal(scales, mx_ref.tile_scales(want_e))
    assert torch.equal(codes, mx_ref.pack(want_c))
    back = torch.zeros(24, 64, device=DEV)
    assert _lib().rfdetr_b200_op_mx_dequantize(_p(codes), 32, _p(scales), 24, 64, _p(back), F32, 64, _stream()) == 0
    assert torch.isnan(back[7, :32]).all() and torch.isnan(back[9, 32:]).all() and torch.isfinite(back[9, :32]).all()
    want = mx_ref.values(want_c, want_e).float()
    assert torch.equal(torch.nan_to_num(back, nan=1.5), torch.nan_to_num(want, nan=1.5))


@pytest.mark.parametrize("type", [F16, BF16])
def test_quantize_16_bit_extremes(type):
    """Every 16-bit pattern but the NaNs' payloads: subnormals, the largest values, infinities and NaN."""
    t = mx_ref.TYPES[type]
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(t).view(2048, 32).to(DEV)
    mixed = bits.view(-1)[torch.randperm(65536, generator=torch.Generator().manual_seed(0)).to(DEV)].view(2048, 32)
    for x in (bits, mixed):
        codes, scales = _quantize(x, type)
        want_c, want_e = mx_ref.quantize(x.double())
        assert torch.equal(scales, mx_ref.tile_scales(want_e)) and torch.equal(codes, mx_ref.pack(want_c))


@pytest.mark.parametrize("type", [F32, F16, BF16])
@pytest.mark.parametrize("k", [32, 31])
def test_dequantize_every_scale(type, k):
    """All 256 scale bytes with all sixteen codes, to every type: subnormals, overflow and NaN with them."""
    t = mx_ref.TYPES[type]
    codes = torch.arange(16, dtype=torch.uint8, device=DEV).repeat(2).expand(256, 32).contiguous()
    e = torch.arange(256, device=DEV).to(torch.uint8)[:, None]
    out = torch.zeros(256, k, dtype=t, device=DEV)
    assert _lib().rfdetr_b200_op_mx_dequantize(_p(mx_ref.pack(codes).contiguous()), 16, _p(mx_ref.tile_scales(e)), 256, k,
                                               _p(out), type, k, _stream()) == 0
    want = mx_ref.values(codes, e)[:, :k].float().to(t)  # exact in f32, or infinite there and in t
    assert torch.equal(torch.nan_to_num(out, nan=123.0), torch.nan_to_num(want, nan=123.0))
    assert torch.isnan(out[255]).all() and not torch.isnan(out[:255]).any()


@pytest.mark.parametrize("cut", [0, 3])
@pytest.mark.parametrize("units", [65537, 65536, 65541])
def test_quantize_rows_of_many_millions(units, cut):
    """Two rows of 512 `units` - cut columns against the same values in rows of 512, there and back."""
    rows, k, full = 2, 512 * units - cut, 512 * units
    x = torch.zeros(rows, full, dtype=torch.float16, device=DEV)
    x[:, :k] = torch.randn(rows, k, dtype=torch.float16, device=DEV, generator=_gen(units))
    x[1, ::4096] *= 64
    codes, scales = _quantize(x, F16, k)
    want_codes, want_scales = _quantize(x.view(-1, 512), F16)
    assert torch.equal(codes.view(-1, 256), want_codes)

    def untiled(s, rows, blocks):
        r, b = torch.arange(rows, device=DEV)[:, None], torch.arange(blocks, device=DEV)[None]
        return s[((r // 128) * -(-blocks // 4) + b // 4) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + b % 4]

    assert torch.equal(untiled(scales, rows, full // 32).view(-1, 16), untiled(want_scales, rows * units, 16))
    back = torch.full((rows, full), 7.0, dtype=torch.float16, device=DEV)
    assert _lib().rfdetr_b200_op_mx_dequantize(_p(codes), full // 2, _p(scales), rows, k, _p(back), F16, full,
                                               _stream()) == 0
    want = torch.zeros(rows * units, 512, dtype=torch.float16, device=DEV)
    assert _lib().rfdetr_b200_op_mx_dequantize(_p(want_codes), 256, _p(want_scales), rows * units, 512, _p(want), F16,
                                               512, _stream()) == 0
    assert torch.equal(back[:, :k], want.view(rows, full)[:, :k]) and (back[:, k:] == 7.0).all()


def test_quantize_far_rows():
    """Rows whose offset passes 32 bits, on both sides."""
    rows, ld, k = 66000, 33000, 40
    x = torch.empty(rows, ld, dtype=torch.float16, device=DEV)
    x[:, :k] = torch.randn(rows, k, device=DEV, generator=_gen(1)).half()
    codes, scales = _quantize(x, F16, k)
    want_c, want_e = mx_ref.quantize(x[:, :k].double())
    assert torch.equal(codes, mx_ref.pack(want_c)) and torch.equal(scales, mx_ref.tile_scales(want_e))
    x[:, :k] = 0
    assert _lib().rfdetr_b200_op_mx_dequantize(_p(codes), codes.shape[1], _p(scales), rows, k, _p(x), F16, ld,
                                               _stream()) == 0
    assert torch.equal(x[:, :k], mx_ref.values(want_c, want_e)[:, :k].half())


# ---- product --------------------------------------------------------------------


def _gemm_tolerance(A, B, ref, t, act, bias):
    """f32 sums of k exact products: at most k + 2 roundings (or cuts) of 2^-23 of the sum of the
    magnitudes; the activations are within 4e-7 absolute (GELU) or 2^-20 relative (SiLU) and have slopes
    of at most 1.13; then the output's own rounding."""
    mag = A.abs() @ B.abs().T + (bias.double().abs() if bias is not None else 0)
    tol = 1.13 * (A.shape[1] + 2) * 2.0 ** -23 * mag + mx_ref.half_step(t) * ref.abs()
    if t == torch.float16:
        tol = tol + 2.0 ** -25  # half the spacing of its subnormals
    if act == 1:
        tol = tol + 4e-7
    if act == 3:
        tol = tol + 2.0 ** -20 * ref.abs()
    return tol


def _gemm(M, N, K, act, type, with_bias, ldo=None, seed=0):
    g = _gen(seed + M * 7 + N * 3 + K)
    a, sa, A = _operand(g, M, K)
    b, sb, B = _operand(g, N, K)
    B = B / 8
    sb = (sb.int() - 3).clamp_min(0).to(torch.uint8)  # the scales say the same
    bias = torch.randn(N, device=DEV, generator=g) if with_bias else None
    t = mx_ref.TYPES[type]
    ldo = ldo or N
    out = torch.full((M, ldo), 7.0, dtype=t, device=DEV)
    assert _lib().rfdetr_b200_op_mx_gemm(_p(a), a.shape[1], _p(sa), _p(b), b.shape[1], _p(sb), M, N, K, act, _p(bias),
                                         _p(out), type, ldo, _stream()) == 0
    v = A @ B.T
    ref = mx_ref.act(v + bias.double() if with_bias else v, act)
    err = (out[:, :N].double() - ref).abs() - _gemm_tolerance(A, B, ref, t, act, bias)
    assert err.max() <= 0, (err.max().item(), (err > 0).sum().item())
    assert (out[:, N:] == 7.0).all()
    return out


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 128, 64), (1, 4096, 4096), (1, 100, 33), (2, 257, 640), (7, 48, 2048),
                                   (13, 11008, 4096), (16, 384, 96), (17, 4096, 1000), (31, 130, 8192),
                                   (32, 1024, 1024), (33, 520, 512), (64, 2048, 256), (65, 2056, 768), (100, 91, 256),
                                   (127, 129, 128), (128, 128, 128), (129, 257, 257), (300, 1152, 384),
                                   (1000, 1000, 1000), (1616, 1536, 384), (2049, 776, 2000), (4097, 2048, 512),
                                   (24, 200, 5000), (50, 300, 8192), (64, 130, 16384), (70, 64, 16384),
                                   (300, 300, 16384), (257, 129, 10000), (500, 500, 8200), (128, 4096, 8192)])
def test_gemm_shapes(M, N, K):
    _gemm(M, N, K, 0, BF16, False)
    _gemm(M, N, K, 0, F16, True)


@pytest.mark.parametrize("type", [F32, F16, BF16])
@pytest.mark.parametrize("act", [0, 1, 2, 3])
@pytest.mark.parametrize("M,N,K", [(3, 200, 416), (40, 333, 256), (517, 520, 608), (30, 77, 4100), (61, 131, 8192),
                                   (150, 131, 16384)])
def test_gemm_types_and_activations(M, N, K, act, type):
    _gemm(M, N, K, act, type, True)
    _gemm(M, N, K, act, type, False, ldo=N + 5)


@pytest.mark.parametrize("M", [5, 200])
def test_gemm_pitches_and_offsets(M):
    """Operands and output with pitches and starts of their own."""
    N, K = 136, 320
    g = _gen(M)
    a, sa, A = _operand(g, M, K)
    b, sb, B = _operand(g, N, K)
    wide_a = torch.full((M + 1, 192), 0x77, dtype=torch.uint8, device=DEV)
    wide_b = torch.full((N + 1, 176), 0x77, dtype=torch.uint8, device=DEV)
    wide_a[1:, 16:176], wide_b[1:, :160] = a, b
    out = torch.full((M, N + 9), 7.0, dtype=torch.float16, device=DEV)
    view = out.view(-1)[1:]
    assert _lib().rfdetr_b200_op_mx_gemm(wide_a[1:, 16:].data_ptr(), 192, _p(sa), wide_b[1:].data_ptr(), 176, _p(sb), M,
                                         N, K, 0, None, _p(view), F16, N + 9, _stream()) == 0
    ref = A @ B.T
    got = torch.as_strided(out, (M, N), (N + 9, 1), 1).double()
    assert ((got - ref).abs() <= _gemm_tolerance(A, B, ref, torch.float16, 0, None)).all()
    assert (out[:, 0] == 7.0).all() and (out[:, N + 1:] == 7.0).all()


@pytest.mark.parametrize("type", [F32, F16, BF16])
@pytest.mark.parametrize("M,N,K", [(200, 257, 128), (333, 1000, 128), (150, 39, 128), (7, 257, 128), (13, 139, 8192),
                                   (50, 130, 16384), (150, 130, 16384)])
def test_gemm_every_output_alignment(M, N, K, type):
    """Outputs that start at each element of 16 bytes, with pitches that move the rows' boundaries by one,
    two, four or no elements; nothing around them is written."""
    t = mx_ref.TYPES[type]
    g = _gen(M)
    a, sa, A = _operand(g, M, K)
    b, sb, B = _operand(g, N, K)
    ref = A @ B.T
    tol = _gemm_tolerance(A, B, ref, t, 0, None)
    for pad in (0, 1, 2, 3, 4, 7, 8):
        for offset in (0, 1, 2, 5, 8):
            out = torch.full((M * (N + pad) + 32,), 7.0, dtype=t, device=DEV)
            assert _lib().rfdetr_b200_op_mx_gemm(_p(a), K // 2, _p(sa), _p(b), K // 2, _p(sb), M, N, K, 0, None,
                                                 out[offset:].data_ptr(), type, N + pad, _stream()) == 0
            got = torch.as_strided(out, (M, N), (N + pad, 1), offset)
            assert ((got.double() - ref).abs() <= tol).all()
            got.fill_(7.0)
            assert (out == 7.0).all()


@pytest.mark.parametrize("M", [1, 20, 260])
def test_gemm_nan_scale_reaches_its_row_only(M):
    g = _gen(M)
    a, sa, A = _operand(g, M, 512)
    b, sb, B = _operand(g, 300, 512)
    e = torch.full((M, 16), 127, dtype=torch.uint8, device=DEV)
    e[M // 2, 3] = 255
    A = mx_ref.values(mx_ref.unpack(a), e)
    out = torch.zeros(M, 300, device=DEV)
    assert _lib().rfdetr_b200_op_mx_gemm(_p(a), 256, _p(mx_ref.tile_scales(e)), _p(b), 256, _p(sb), M, 300, 512, 0, None,
                                         _p(out), F32, 300, _stream()) == 0
    assert torch.isnan(out[M // 2]).all()
    rest = torch.arange(M, device=DEV) != M // 2
    ref = (A @ B.T)[rest]
    assert ((out[rest].double() - ref).abs() <= _gemm_tolerance(A[rest], B, ref, torch.float32, 0, None)).all()


@pytest.mark.parametrize("act", [1, 2, 3])
@pytest.mark.parametrize("type", [F32, F16, BF16])
@pytest.mark.parametrize("M", [1, 20, 260])
def test_gemm_nan_passes_the_activations(M, type, act):
    """A row with a NaN scale and a column with a NaN bias."""
    g = _gen(M)
    a, sa, A = _operand(g, M, 512)
    b, sb, B = _operand(g, 300, 512)
    e = torch.full((M, 16), 127, dtype=torch.uint8, device=DEV)
    e[M // 2, 3] = 255
    bias = torch.zeros(300, device=DEV)
    bias[77] = math.nan
    out = torch.zeros(M, 300, dtype=mx_ref.TYPES[type], device=DEV)
    assert _lib().rfdetr_b200_op_mx_gemm(_p(a), 256, _p(mx_ref.tile_scales(e)), _p(b), 256, _p(sb), M, 300, 512, act,
                                         _p(bias), _p(out), type, 300, _stream()) == 0
    nan = torch.zeros(M, 300, dtype=torch.bool, device=DEV)
    nan[M // 2] = True
    nan[:, 77] = True
    assert torch.equal(torch.isnan(out), nan)


@pytest.mark.parametrize("M,N", [(3, 200), (257, 520)])
def test_gemm_ignores_what_lies_behind_its_operands(M, N):
    """NaN scales in rows that only fill up the last tile change nothing (nor are they read into a result)."""
    K = 96
    g = _gen(11)
    a, sa, A = _operand(g, M, K)
    b, sb, B = _operand(g, N, K)
    outs = []
    for fill in (0, 255):
        ta, tb = sa.clone(), sb.clone()
        for t, rows in ((ta, M), (tb, N)):
            r = torch.arange(rows, -(-rows // 128) * 128, device=DEV)[:, None]
            c = torch.arange(4, device=DEV)[None]
            t[(r // 128 * 512 + r % 32 * 16 + r // 32 % 4 * 4 + c).reshape(-1)] = fill
        out = torch.zeros(M, N, device=DEV)
        assert _lib().rfdetr_b200_op_mx_gemm(_p(a), a.shape[1], _p(ta), _p(b), b.shape[1], _p(tb), M, N, K, 0, None,
                                             _p(out), F32, N, _stream()) == 0
        outs.append(out)
    assert torch.equal(outs[0], outs[1])


def test_gemm_far_rows():
    """An output whose offsets pass 32 bits."""
    M, N, K, ldo = 66000, 40, 64, 33000
    g = _gen(3)
    a, sa, A = _operand(g, M, K)
    b, sb, B = _operand(g, N, K)
    out = torch.empty(M, ldo, dtype=torch.float16, device=DEV)
    assert _lib().rfdetr_b200_op_mx_gemm(_p(a), 32, _p(sa), _p(b), 32, _p(sb), M, N, K, 0, None, _p(out), F16, ldo,
                                         _stream()) == 0
    ref = A @ B.T
    assert ((out[:, :N].double() - ref).abs() <= _gemm_tolerance(A, B, ref, torch.float16, 0, None)).all()


@pytest.mark.parametrize("M,N,K", [(1, 4096, 4096), (13, 300, 8192), (600, 700, 800), (40, 300, 16384),
                                   (200, 300, 16384)])
def test_gemm_is_deterministic(M, N, K):
    first = _gemm(M, N, K, 0, F32, True)
    for _ in range(3):
        assert torch.equal(first, _gemm(M, N, K, 0, F32, True))


# Shapes that a B200's 148 SMs take with the 256 columns wide tiles: at least 148 tiles of 128 x 256; with pairs of SMs from
# K = 2048 (4096 with GELU or SiLU) where these need no more turns.  Odd numbers of row tiles, rows and columns that end
# inside a tile, K that ends inside a stage.
WIDE = [(2400, 2051, 600), (4097, 2048, 512), (2433, 2304, 1000)]
PAIRS = [(2400, 2051, 2050), (2433, 2304, 4128), (4100, 1300, 4500)]


@pytest.mark.parametrize("type", [F32, F16, BF16])
@pytest.mark.parametrize("act", [0, 1, 2, 3])
@pytest.mark.parametrize("M,N,K", WIDE + PAIRS)
def test_gemm_wide_tiles(M, N, K, act, type):
    _gemm(M, N, K, act, type, True)
    _gemm(M, N, K, act, type, False, ldo=N + 5)


@pytest.mark.parametrize("type", [F32, F16, BF16])
@pytest.mark.parametrize("M,N,K", [WIDE[0], PAIRS[0]])
def test_gemm_wide_tiles_every_output_alignment(M, N, K, type):
    """As test_gemm_every_output_alignment."""
    t = mx_ref.TYPES[type]
    g = _gen(M)
    a, sa, A = _operand(g, M, K)
    b, sb, B = _operand(g, N, K)
    ref = A @ B.T
    tol = _gemm_tolerance(A, B, ref, t, 0, None)
    for pad, offset in ((0, 0), (5, 0), (5, 1), (1, 0), (3, 2), (13, 8), (0, 1)):
        out = torch.full((M * (N + pad) + 32,), 7.0, dtype=t, device=DEV)
        assert _lib().rfdetr_b200_op_mx_gemm(_p(a), a.shape[1], _p(sa), _p(b), b.shape[1], _p(sb), M, N, K, 0, None,
                                             out[offset:].data_ptr(), type, N + pad, _stream()) == 0
        got = torch.as_strided(out, (M, N), (N + pad, 1), offset)
        assert ((got.double() - ref).abs() <= tol).all()
        got.fill_(7.0)
        assert (out == 7.0).all()


@pytest.mark.parametrize("act", [0, 1, 2, 3])
@pytest.mark.parametrize("M,N,K", [WIDE[0], PAIRS[0], PAIRS[1]])
def test_gemm_wide_tiles_nan(M, N, K, act):
    """Rows with a NaN scale and a column with a NaN bias, in every column chunk's epilogue; none but these."""
    g = _gen(M)
    a, sa, A = _operand(g, M, K)
    b, sb, B = _operand(g, N, K)
    rows = [0, 127, 128, 1000, M - 1]
    e = torch.full((M, -(-K // 32)), 127, dtype=torch.uint8, device=DEV)
    e[rows, 3] = 255
    bias = torch.zeros(N, device=DEV)
    bias[[5, 255, 256, 1023, N - 1]] = math.nan
    out = torch.zeros(M, N, dtype=torch.bfloat16, device=DEV)
    assert _lib().rfdetr_b200_op_mx_gemm(_p(a), a.shape[1], _p(mx_ref.tile_scales(e)), _p(b), b.shape[1], _p(sb), M, N, K, act,
                                         _p(bias), _p(out), BF16, N, _stream()) == 0
    nan = torch.isnan(bias)[None].repeat(M, 1)
    nan[rows] = True
    assert torch.equal(torch.isnan(out), nan)


def _exact_operand(g, rows, k):
    """Any codes, scales 1/2, 1 and 2: multiples of 1/4 up to 12, whose products' sums are exact in f32 while the
    sum of their magnitudes is below 2^24 / 16."""
    codes = torch.randint(0, 16, (rows, k), device=DEV, generator=g).to(torch.uint8)
    codes = torch.nn.functional.pad(codes, (0, -k % 32))
    e = torch.randint(126, 129, (rows, -(-k // 32)), device=DEV, generator=g).to(torch.uint8)
    return mx_ref.pack(codes).contiguous(), mx_ref.tile_scales(e), mx_ref.values(codes, e)


EXACT = [(1, 4096, 4096), (1, 130, 16384), (13, 11008, 4096), (16, 500, 8192), (30, 300, 8192), (61, 131, 16384),
         (64, 256, 16384), (150, 131, 16384), (300, 300, 16384), (500, 500, 8200), (200, 700, 1000), (1616, 1152, 384),
         (2400, 2051, 600), (2400, 2051, 2050), (2433, 2304, 8192)]


@pytest.mark.parametrize("M,N,K", EXACT)
def test_gemm_exact_sums(M, N, K):
    """Products whose sums f32 holds exactly in any order: the results are those of 64 bits, rounded once, so a
    block with another's scale, a stage twice or not at all, or a part of K that is missing shows."""
    g = _gen(M + K)
    a, sa, A = _exact_operand(g, M, K)
    b, sb, B = _exact_operand(g, N, K)
    bias = torch.randint(-40, 40, (N,), device=DEV, generator=g).float()
    ref = A @ B.T
    assert (A.abs() @ B.abs().T).max() + 40 < 2 ** 20
    for type, bi in ((F32, None), (F32, bias), (BF16, bias), (F16, None)):
        t = mx_ref.TYPES[type]
        out = torch.full((M, N), 7.0, dtype=t, device=DEV)
        assert _lib().rfdetr_b200_op_mx_gemm(_p(a), a.shape[1], _p(sa), _p(b), b.shape[1], _p(sb), M, N, K, 0, _p(bi), _p(out),
                                             type, N, _stream()) == 0
        assert torch.equal(out, (ref + bi.double() if bi is not None else ref).to(t))


@pytest.mark.parametrize("M,N,K", EXACT)
def test_gemm_one_block_of_each_row(M, N, K):
    """Rows of A with one block that is not zero, another for each row: every block of K counts once, with its own
    scales."""
    g = _gen(M + K + 1)
    kb = -(-K // 32)
    codes = torch.randint(0, 16, (M, kb, 32), device=DEV, generator=g).to(torch.uint8)
    b, sb, B = _exact_operand(g, N, K)
    for first in range(0, kb, max(M, kb // 32)):  # one row at a time: 32 of the blocks
        at = (first + torch.arange(M, device=DEV)) % kb
        here = torch.zeros(M, kb, dtype=torch.bool, device=DEV)
        here[torch.arange(M, device=DEV), at] = True
        c = torch.where(here[..., None], codes, torch.zeros_like(codes)).view(M, -1)
        c = torch.where(torch.arange(c.shape[1], device=DEV) < K, c, torch.zeros_like(c))
        e = torch.randint(126, 129, (M, kb), device=DEV, generator=g).to(torch.uint8)
        A = mx_ref.values(c, e)
        out = torch.full((M, N), 7.0, device=DEV)
        a, sa = mx_ref.pack(c).contiguous(), mx_ref.tile_scales(e)
        assert _lib().rfdetr_b200_op_mx_gemm(_p(a), a.shape[1], _p(sa), _p(b), b.shape[1], _p(sb), M, N, K, 0, None, _p(out),
                                             F32, N, _stream()) == 0
        assert torch.equal(out.double(), A @ B.T)


@pytest.mark.parametrize("M", [1, 20, 260])
@pytest.mark.parametrize("act", [0, 1, 2, 3])
def test_gemm_activations_over_their_range(act, M):
    """act(bias) alone, operands of zeros: GELU is within 3.2e-7 and f32's rounding; SiLU within 2^-17 of itself, the
    fast exponential's 2 + 1.173 |v| steps and the quotient's 2, down to -87, and 0 below; the others are exact."""
    K, N = 64, 4096
    v = torch.cat([torch.linspace(-100, 100, N - 1000), torch.linspace(-8, 8, 990),
                   torch.tensor([0.0, -0.0, 1e-30, -1e-30, 3e38, -3e38, math.inf, 88.0, -86.9, -120.0])]).to(DEV)
    a, b = (torch.zeros(r, K // 2, dtype=torch.uint8, device=DEV) for r in (M, N))
    sa, sb = (torch.zeros(_lib().rfdetr_b200_mx_scale_bytes(r, K), dtype=torch.uint8, device=DEV) for r in (M, N))
    out = torch.full((M, N), 7.0, device=DEV)
    assert _lib().rfdetr_b200_op_mx_gemm(_p(a), K // 2, _p(sa), _p(b), K // 2, _p(sb), M, N, K, act, _p(v), _p(out), F32, N,
                                         _stream()) == 0
    x = v.double()
    if act in (0, 2):
        want = v if act == 0 else v.clamp_min(0)
        assert (out == want).all()
        return
    want = mx_ref.act(x, act)
    want[torch.isposinf(v)] = math.inf
    tol = 3.2e-7 + 2.0 ** -24 * x.abs() if act == 1 else torch.where(x > -87, 2.0 ** -17 * want.abs(), 1e-36)
    fine = torch.isfinite(want)
    assert ((out.double() - want).abs() <= tol)[:, fine].all()
    assert (out[:, ~fine].double() == want[~fine]).all()


@pytest.mark.parametrize("M,N,K", [(1, 40, 2 ** 21), (40, 64, 2 ** 18), (100, 64, 2 ** 18), (1200, 4096, 2 ** 14)])
def test_gemm_long_sums_of_one_sign(M, N, K):
    """Sums that only grow, of terms far apart: the tensor core cuts them with every 64 columns, by less than 2^-23."""
    g = _gen(K)
    ops = []
    for rows in (M, N):
        codes = torch.randint(0, 256, (rows, K // 2), device=DEV, generator=g).to(torch.uint8) & 0x77
        ops.append((codes, torch.randint(122, 132, (rows, K // 32), device=DEV, generator=g).to(torch.uint8)))
    (a, ea), (b, eb) = ops
    out = torch.zeros(M, N, device=DEV)
    assert _lib().rfdetr_b200_op_mx_gemm(_p(a), K // 2, _p(mx_ref.tile_scales(ea)), _p(b), K // 2, _p(mx_ref.tile_scales(eb)),
                                         M, N, K, 0, None, _p(out), F32, N, _stream()) == 0
    ref = torch.zeros(M, N, dtype=torch.float64, device=DEV)
    for c in range(0, K, 2 ** 15):
        A, B = (mx_ref.values(mx_ref.unpack(x[:, c // 2:c // 2 + 2 ** 14]), e[:, c // 32:c // 32 + 1024])[:, :K - c] for x, e in ops)
        ref += A @ B.T
    # then up to eight parts are added, and the result is an f32
    assert ((out.double() - ref).abs() <= (K * 2.0 ** -29 + 9 * 2.0 ** -24) * ref).all()


@pytest.mark.parametrize("M,N,K", [(2400, 2051, 600), (2400, 2051, 2050)])
def test_gemm_wide_tiles_are_deterministic(M, N, K):
    first = _gemm(M, N, K, 1, F32, True)
    for _ in range(3):
        assert torch.equal(first, _gemm(M, N, K, 1, F32, True))


# ---- norms ------------------------------------------------------------------------


def _norm_case(rows, dim, type=F16, resid_type=F32, post=1, pre=1, gate="channel", period=3, scale=0.75, mx=True,
               resid=True, write_x=True, write_h=True, pad=0, offset=0, alias=False, seed=0):
    from rfdetr_b200 import lib

    g = _gen(seed + rows * 5 + dim)
    t, tx = mx_ref.TYPES[type], mx_ref.TYPES[resid_type]

    def matrix(dtype, fill=None):
        flat = torch.empty(rows * (dim + pad) + offset, dtype=dtype, device=DEV)
        if fill is None:
            flat.copy_(torch.randn(flat.numel(), device=DEV, generator=g) * 2 + 0.5)
        else:
            flat.fill_(fill)
        return flat[offset:].view(rows, dim + pad)

    y, x = matrix(t), matrix(tx) if resid else None
    vec = lambda: torch.randn(dim, device=DEV, generator=g) * 0.3 + 1  # noqa: E731
    pw, pb, qw, qb = vec(), vec(), vec(), vec()
    n_gate = {"none": 0, "channel": 1, "group": -(-rows // period)}[gate]
    gt = torch.randn(n_gate, dim, device=DEV, generator=g) if n_gate else None
    y64, x64 = y[:, :dim].double(), (x[:, :dim].double() if resid else None)
    xo = (x if alias else matrix(tx, 7.0)) if write_x else None
    h = (y if alias else matrix(t, 7.0)) if write_h else None
    codes, scales = _mx_buffers(rows, dim) if mx else (None, None)
    args = lib.BlockNorm(y=_p(y), resid=_p(x), post_w=_p(pw), post_b=_p(pb), gate=_p(gt), pre_w=_p(qw), pre_b=_p(qb),
                         out_resid=_p(xo), out=_p(h), mx_codes=_p(codes), mx_scales=_p(scales), rows=rows, dim=dim,
                         type=type, resid_type=resid_type, post=post, pre=pre, ldy=dim + pad, ld_resid=dim + pad,
                         ld_out_resid=dim + pad, ld_out=dim + pad, ld_mx=codes.shape[1] if mx else 0, ld_gate=dim,
                         gate_period=period if gate == "group" else 0, resid_scale=scale, post_eps=1e-5, pre_eps=1e-6)
    assert _lib().rfdetr_b200_op_block_norm(args, _stream()) == 0

    # f32 sums of a row pass through at most 8 * 8 + 5 + 32 additions, so their relative error (all terms
    # of one sign; for a mean, against the mean magnitude) is under 110 * 2^-24
    u = 110 * 2.0 ** -24
    b64, rstd = mx_ref.norm(y64, post, pw, pb, 1e-5)
    slack = u * (b64.abs() + (y64.abs().amax(1, keepdim=True) * rstd * pw.abs() if post else 0))
    if gt is not None:
        gr = gt.double()[torch.arange(rows, device=DEV) // period if gate == "group" else torch.zeros(rows, dtype=torch.long, device=DEV)]
        b64, slack = b64 * gr, slack * gr.abs()
    x1 = b64 + scale * x64 if resid else b64
    slack = slack + 4 * 2.0 ** -24 * (b64.abs() + (x64.abs() if resid else 0))
    if write_x:
        err = (xo[:, :dim].double() - x1).abs() - slack - mx_ref.half_step(tx) * x1.abs() - (2.0 ** -25 if tx == torch.float16 else 0)
        assert err.max() <= 0, err.max()
        if pad and not alias:
            assert (xo[:, dim:] == 7.0).all()
    h64, rstd = mx_ref.norm(x1, pre, qw, qb, 1e-6)
    w = qw.double().abs() * rstd if pre else 1.0
    # an error of x' enters h directly and through the statistics, each by at most its largest in the row
    hs = 3 * slack.amax(1, keepdim=True) * w + u * (h64.abs() + x1.abs().amax(1, keepdim=True) * w + qb.abs())
    if pre:  # dh = h * d(rstd) / rstd: the statistics' relative error from slack, on values up to |h|
        hs = hs + 2 * slack.amax(1, keepdim=True) * rstd * (h64.abs() + qb.abs())
    if write_h:
        err = (h[:, :dim].double() - h64).abs() - hs - mx_ref.half_step(t) * h64.abs() - (2.0 ** -25 if t == torch.float16 else 0)
        assert err.max() <= 0, err.max()
        if pad and not alias:
            assert (h[:, dim:] == 7.0).all()
    if mx:
        # the operand holds some h within that slack: its scale is that of a block maximum within the
        # slack, and every value lies within half a step of E2M1 (or above 6) of an h within the slack
        kb = -(-dim // 32)
        e = scales.view(-1, -(-dim // 128), 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-1, -(-dim // 128) * 4)
        assert (e[rows:] == 0).all() and (e[:, kb:] == 0).all()
        e = e[:rows, :kb]
        got = mx_ref.values(mx_ref.unpack(codes), e)
        pad64 = lambda v: torch.nn.functional.pad(v.expand(rows, dim), (0, -dim % 32)).view(rows, kb, 32)  # noqa: E731
        hb, sb, gb = pad64(h64), pad64(hs), got.view(rows, kb, 32)
        amax = hb.abs().amax(-1)
        lo = torch.floor(torch.log2((amax - sb.amax(-1)).clamp_min(1e-300))) - 2
        hi = torch.floor(torch.log2((amax + sb.amax(-1)).clamp_min(1e-300))) - 2
        ee = e.double() - 127
        assert ((ee >= lo.clamp_min(-127)) & (ee <= hi.clamp_min(-127))).all()
        s = torch.exp2(ee)[..., None]
        a = gb.abs() / s
        step = torch.where(a < 2, 0.25, torch.where(a < 4, 0.5, 1.0))  # half a step beyond a's binade
        step = torch.where(a >= 6, torch.full_like(a, 2.0), step)      # [4, 8) saturates at 6
        assert ((gb - hb).abs() <= step * s + sb).all()
        assert (got.view(rows, -1)[:, dim:] == 0).all()


DIMS = [1, 2, 7, 8, 31, 32, 40, 100, 128, 136, 256, 264, 384, 500, 512, 520, 768, 776, 1000, 1024, 1032, 1500, 2048,
        2056, 4096, 4100, 5120, 8192, 8200, 11008, 16384, 16392, 20001, 32768]


@pytest.mark.parametrize("M,N,K", [(1, 4096, 4096), (1, 128, 16384), (30, 300, 8192), (64, 256, 16384),
                                   (300, 300, 16384)])
def test_gemm_parts_are_all_there_every_time(M, N, K):
    """K split over a cluster, two operands in turn: no result holds a sum of the call before."""
    g = _gen(M)
    b, sb, _ = _operand(g, N, K)
    ops = [_operand(g, M, K)[:2] for _ in range(2)]
    outs = torch.zeros(400, M, N, device=DEV)
    for i in range(400):
        a, sa = ops[i & 1]
        assert _lib().rfdetr_b200_op_mx_gemm(_p(a), K // 2, _p(sa), _p(b), K // 2, _p(sb), M, N, K, 0, None, _p(outs[i]),
                                             F32, N, _stream()) == 0
    assert (outs[0::2] == outs[0]).all() and (outs[1::2] == outs[1]).all()
    assert not torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("dim", DIMS)
def test_block_norm_dims(dim):
    _norm_case(5, dim, post=2, pre=2)
    _norm_case(131, dim, type=BF16, resid_type=BF16, post=1, pre=1, gate="group")


@pytest.mark.parametrize("type,resid_type", [(F32, F32), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("dim", [96, 384, 1001, 2304])
def test_block_norm_types(type, resid_type, dim):
    _norm_case(17, dim, type, resid_type)
    _norm_case(17, dim, type, resid_type, pad=8, post=0, gate="none")
    _norm_case(17, dim, type, resid_type, pad=3, offset=1, post=2, pre=2, gate="group")


@pytest.mark.parametrize("post", [0, 1, 2])
@pytest.mark.parametrize("pre", [0, 1, 2])
@pytest.mark.parametrize("gate", ["none", "channel", "group"])
def test_block_norm_kinds(post, pre, gate):
    _norm_case(40, 384, post=post, pre=pre, gate=gate, scale=1.0)
    _norm_case(9, 200, post=post, pre=pre, gate=gate, period=1, scale=-0.5)


@pytest.mark.parametrize("drop", [dict(resid=False), dict(write_x=False), dict(write_h=False), dict(mx=False),
                                  dict(write_x=False, write_h=False), dict(mx=False, write_x=False),
                                  dict(mx=False, write_h=False), dict(alias=True)])
@pytest.mark.parametrize("dim", [384, 390, 4096])
def test_block_norm_parts(drop, dim):
    _norm_case(21, dim, **drop)


def test_block_norm_many_rows():
    _norm_case(51713, 384, post=0)
    _norm_case(70001, 8, post=2, pre=2)


def test_block_norm_constant_and_special_rows():
    """Rows of equal values (variance 0), zeros, and rows with an infinity or a NaN, which stay in
    their own row: the others are as without them."""
    from rfdetr_b200 import lib

    rows, dim = 9, 384
    y = torch.randn(rows, dim, device=DEV, generator=_gen(2))
    y[1], y[2], y[3, 5], y[4, 6] = 3.5, 0.0, math.inf, math.nan
    w, b = torch.ones(dim, device=DEV), torch.full((dim,), 0.25, device=DEV)
    out = torch.zeros(rows, dim, device=DEV)
    codes, scales = _mx_buffers(rows, dim)
    a = lib.BlockNorm(y=_p(y), pre_w=_p(w), pre_b=_p(b), out=_p(out), mx_codes=_p(codes), mx_scales=_p(scales), rows=rows,
                      dim=dim, type=F32, pre=1, ldy=dim, ld_out=dim, ld_mx=dim // 2, pre_eps=1e-5)
    assert _lib().rfdetr_b200_op_block_norm(a, _stream()) == 0
    assert (out[1] == 0.25).all() and (out[2] == 0.25).all()
    assert torch.isnan(out[3]).any() and torch.isnan(out[4]).all()
    ref, _ = mx_ref.norm(y.double(), 1, w, b, 1e-5)
    keep = [0, 5, 6, 7, 8]
    assert ((out[keep].double() - ref[keep]).abs() < 1e-5).all()
    back = torch.zeros(rows, dim, device=DEV)
    assert _lib().rfdetr_b200_op_mx_dequantize(_p(codes), dim // 2, _p(scales), rows, dim, _p(back), F32, dim,
                                               _stream()) == 0
    assert torch.isnan(back[4]).all() and torch.isfinite(back[keep]).all()


@pytest.mark.parametrize("kind", [1, 2])
@pytest.mark.parametrize("eps", [0.0, 1e-5])
@pytest.mark.parametrize("dim", [50, 384, 2048, 4096])
def test_block_norm_infinite_variance(kind, eps, dim):
    """A row with an infinity, rows of zeros, of very large and of very small values: what the formula
    gives in f32, NaN and zeros in the same places."""
    from rfdetr_b200 import lib

    y = torch.randn(6, dim, device=DEV, generator=_gen(dim))
    y[1, 3] = math.inf
    y[2] = 0
    y[3] *= 1e18
    y[4] *= 1e-18
    y[5] *= 1e25  # its squares are infinite in f32
    w, b = torch.rand(dim, device=DEV, generator=_gen(1)) + 0.5, torch.zeros(dim, device=DEV)
    out = torch.zeros(6, dim, device=DEV)
    a = lib.BlockNorm(y=_p(y), pre_w=_p(w), pre_b=_p(b), out=_p(out), rows=6, dim=dim, type=F32, pre=kind, ldy=dim,
                      ld_out=dim, pre_eps=eps)
    assert _lib().rfdetr_b200_op_block_norm(a, _stream()) == 0
    v = y - y.mean(1, keepdim=True) if kind == 1 else y
    ref = v / torch.sqrt((v * v).mean(1, keepdim=True) + eps) * w + b
    assert torch.equal(torch.isnan(out), torch.isnan(ref))
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isfinite(out), fine)
    # both sides' sums: 110 roundings of 2^-24 each, the mean's against the row's largest value
    assert ((out - ref).abs()[fine] <= 2 * 110 * 2.0 ** -24 * 8 * (1 + ref.abs()[fine])).all()


# ---- attention ----------------------------------------------------------------------


def _attn(lens, heads, kv, d, causal, type, behind=0, seed=0, layout="qkv", gain=1.0, poison=True):
    t = mx_ref.TYPES[type]
    total = sum(lens)
    g = _gen(seed + total + heads * 3 + d)
    ld = (heads + 2 * kv) * d
    if layout == "qkv":
        buf = (torch.randn(total + behind, ld, device=DEV, generator=g) * gain).to(t)
        q, k, v = buf[:, :heads * d], buf[:, heads * d:(heads + kv) * d], buf[:, (heads + kv) * d:]
    else:  # apart, with pitches of their own
        q = (torch.randn(total + behind, heads * d + 8, device=DEV, generator=g) * gain).to(t)[:, :heads * d]
        k = (torch.randn(total + behind, kv * d + 24, device=DEV, generator=g) * gain).to(t)[:, :kv * d]
        v = torch.randn(total + behind, kv * d, device=DEV, generator=g).to(t)
    if behind and poison:
        for x in (q, k, v):
            x[total:] = math.nan
    o = torch.full((total + behind, heads * d + 16), 7.0, dtype=t, device=DEV)
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=DEV)
    scale = d ** -0.5
    assert _lib().rfdetr_b200_op_attention_packed(
        _p(q), _p(k), _p(v), q.stride(0), k.stride(0), v.stride(0), _p(o), o.stride(0), type, _p(cu), len(lens),
        total + behind, max(lens), heads, kv, d, int(causal), scale, _stream()) == 0
    ref, mag = mx_ref.attention(q, k, v, lens, heads, kv, d, causal, scale)
    # p is rounded to the inputs' type for the product with v, the exponential is within 4e-6 (and the
    # scores' f32 sums within d 2^-23 of |q||k|, here under 4e-5 in all); f16 holds a p below 2^-14 in
    # steps of 2^-24; then the output's rounding
    qk = d * 2.0 ** -23 * scale * q[:total].double().abs().amax() * k[:total].double().abs().amax() * d ** 0.5
    u = mx_ref.half_step(t)
    tol = (1.01 * u + 1e-5 + 2 * qk) * mag + u * ref.abs() + 1e-30
    if t == torch.float16:
        tol = tol + max(lens) * 2.0 ** -25 * v[:total].double().abs().amax() + 2.0 ** -25
    err = (o[:total, :heads * d].double() - ref).abs() - tol
    assert err.max() <= 0, (err.max().item(), (err > 0).sum().item())
    assert (o[total:] == 7.0).all() and (o[:, heads * d:] == 7.0).all()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [1, 2, 31, 63, 64, 65, 127, 128, 129, 200, 255, 256, 257, 383, 500, 1025])
def test_attention_lengths(n, d, causal):
    _attn([n], 2, 1, d, causal, BF16)
    _attn([n], 3, 3, d, causal, F16, behind=5)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("type,d", [(F16, 64), (BF16, 64), (F16, 128), (BF16, 128)])
@pytest.mark.parametrize("heads,kv", [(1, 1), (6, 6), (8, 2), (7, 1), (6, 2), (12, 4), (128, 1), (33, 3), (100, 1)])
def test_attention_heads(heads, kv, type, d, causal):
    _attn([5, 0, 140, 1, 33], heads, kv, d, causal, type, behind=3)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_many_sequences(d, causal):
    """Hundreds of sequences, many empty, the last ones too; pitches of their own."""
    g = torch.Generator().manual_seed(4)
    lens = torch.randint(0, 40, (300,), generator=g).tolist()
    lens[7] = 700
    lens[0] = lens[-1] = lens[-2] = 0
    _attn(lens, 4, 2, d, causal, F16, behind=64, layout="apart")
    _attn([1] * 1000, 4, 2, d, causal, BF16)
    _attn([0, 0, 9], 4, 4, d, causal, BF16, behind=200)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("type,d", [(F16, 64), (BF16, 128)])
def test_attention_long(type, d, causal):
    _attn([4000, 37, 2049], 4, 2, d, causal, type)


@pytest.mark.parametrize("type", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_sharp_and_growing_scores(type, d):
    """Scores far apart, with a row maximum that keeps growing along the keys."""
    t = mx_ref.TYPES[type]
    n, heads = 900, 2
    g = _gen(d)
    q = torch.randn(n, heads * d, device=DEV, generator=g)
    k = torch.randn(n, heads * d, device=DEV, generator=g) * torch.linspace(0.1, 4, n, device=DEV)[:, None]
    v = torch.randn(n, heads * d, device=DEV, generator=g)
    q, k, v = q.to(t), k.to(t), v.to(t)
    o = torch.zeros(n, heads * d, dtype=t, device=DEV)
    cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    for causal in (0, 1):
        assert _lib().rfdetr_b200_op_attention_packed(_p(q), _p(k), _p(v), heads * d, heads * d, heads * d, _p(o),
                                                      heads * d, type, _p(cu), 1, n, n, heads, heads, d, causal,
                                                      d ** -0.5, _stream()) == 0
        ref, mag = mx_ref.attention(q, k, v, [n], heads, heads, d, causal, d ** -0.5)
        u = mx_ref.half_step(t)
        # scores reach 4 * d * 4 * 4 / sqrt(d): their f32 sums are off by at most 1e-4
        tol = (1.01 * u + 4e-4) * mag + u * ref.abs() + (n * 2.0 ** -25 * 5 if t == torch.float16 else 1e-30)
        assert ((o.double() - ref).abs() <= tol).all()


def test_attention_equal_scores_average_the_values():
    """Keys that are all zero: the plain mean of the values before each position."""
    n, d = 300, 64
    q = torch.randn(n, d, device=DEV, generator=_gen(0)).half()
    k = torch.zeros(n, d, dtype=torch.float16, device=DEV)
    v = torch.ones(n, d, dtype=torch.float16, device=DEV) * 3
    o = torch.zeros(n, d, dtype=torch.float16, device=DEV)
    cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    assert _lib().rfdetr_b200_op_attention_packed(_p(q), _p(k), _p(v), d, d, d, _p(o), d, F16, _p(cu), 1, n, n, 1, 1, d,
                                                  1, 0.125, _stream()) == 0
    assert (o == 3).all()


@pytest.mark.parametrize("d", [64, 128])
def test_attention_infinities_of_other_sequences(d):
    """A sequence full of NaN and infinities between two others does not reach them."""
    lens, heads = [70, 130, 90], 2
    t = torch.bfloat16
    g = _gen(d)
    x = torch.randn(290, 3 * heads * d, device=DEV, generator=g).to(t)
    clean = x.clone()
    x[70:200] = math.nan
    x[70:200:2] = math.inf
    cu = torch.tensor([0, 70, 200, 290], dtype=torch.int32, device=DEV)
    outs = []
    for z in (x, clean):
        o = torch.zeros(290, heads * d, dtype=t, device=DEV)
        for causal in (0, 1):
            assert _lib().rfdetr_b200_op_attention_packed(
                _p(z), _p(z[:, heads * d:]), _p(z[:, 2 * heads * d:]), 3 * heads * d, 3 * heads * d, 3 * heads * d,
                _p(o), heads * d, BF16, _p(cu), 3, 290, 130, heads, heads, d, causal, d ** -0.5, _stream()) == 0
            outs.append(o.clone())
    for a, b in ((outs[0], outs[2]), (outs[1], outs[3])):
        keep = torch.cat([torch.arange(70), torch.arange(200, 290)]).to(DEV)
        assert torch.equal(a[keep], b[keep]) and torch.isfinite(a[keep]).all()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens,heads,kv", [
    ([129], 1, 1), ([256], 2, 1), ([257], 1, 1), ([385, 0, 128], 2, 2), ([1, 640, 127], 3, 1), ([900, 3, 130], 6, 2),
    ([1500], 8, 2), ([2049, 64], 2, 2), ([700, 700], 28, 7), ([90, 250, 40, 300, 1, 129], 20, 4)])
def test_attention_few_tiles(lens, heads, kv, d, causal):
    """So few tiles that each one's keys are shared out: one block, odd and even numbers of blocks, short last
    blocks, and tiles whose first or second share holds no key that a row sees."""
    _attn(lens, heads, kv, d, causal, BF16, behind=5)
    _attn(lens, heads, kv, d, causal, F16, seed=1, gain=3.0)


@pytest.mark.parametrize("type", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("at", ["first", "last"])
@pytest.mark.parametrize("n,weak", [(65536, -17.46875), (65536, -20.0), (131072, -23.0)])
def test_attention_many_weak_keys(n, weak, at, d, type):
    """One key of weight 1 and many of e^weak, too small for f16 beside it: together they are part of the row."""
    t = mx_ref.TYPES[type]
    q, k = torch.zeros(n, d, dtype=t, device=DEV), torch.zeros(n, d, dtype=t, device=DEV)
    q[:, 0] = 1.0
    k[:, 0] = weak
    one = 0 if at == "first" else n - 1
    k[one, 0] = 0.0
    v = (1 + torch.rand(n, d, device=DEV, generator=_gen(n + d))).to(t)
    v[one] = 0.0
    o = _attention_once(q, k, v, d, type, 0, 1.0)
    w = torch.exp(k[:, 0].double())
    ref = (w @ v.double()) / w.sum()
    # the roundings that _attn counts, with f16's weights within 2^-36 of the largest
    u = mx_ref.half_step(t)
    tol = (1.01 * u + 1e-5) * ref + u * ref + (n * 2.0 ** -36 * 2 + 2.0 ** -25 if t == torch.float16 else 0)
    assert ref.min() > 2 * tol.max()
    assert ((o.double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("type", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("n", [100, 700])
def test_attention_equal_scores_of_great_size(n, sign, d, type):
    """Scores of 2^25, some 3 apart where f32 holds them: the mean of the values."""
    t = mx_ref.TYPES[type]
    q = torch.full((n, d), 1024.0, dtype=t, device=DEV)
    k = torch.full((n, d), sign * 32768.0 / d, dtype=t, device=DEV)
    v = torch.randn(n, d, device=DEV, generator=_gen(d)).to(t)
    o = _attention_once(q, k, v, d, type, 0, 1.0)
    u = mx_ref.half_step(t)
    mean, mag = v.double().mean(0), v.double().abs().mean(0)
    assert ((o.double() - mean).abs() <= (1.01 * u + 1e-5) * mag + u * mean.abs() + 2.0 ** -25).all()


def _attention_once(q, k, v, d, type, causal, scale):
    n = q.shape[0]
    o = torch.full((n, d), 7.0, dtype=q.dtype, device=DEV)
    cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    assert _lib().rfdetr_b200_op_attention_packed(_p(q), _p(k), _p(v), d, d, d, _p(o), d, type, _p(cu), 1, n, n, 1, 1, d,
                                                  causal, scale, _stream()) == 0
    return o


@pytest.mark.parametrize("type", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("at", [0, 1, 12, 13, 14, 31, 63, 77, 127, 130, 159, 190])
def test_attention_nan_keys_reach_the_rows_that_see_them(at, d, type):
    """A key of NaN: all rows without `causal`, with it those from its position on."""
    n, t = 200, mx_ref.TYPES[type]
    q, k, v = (torch.randn(n, d, device=DEV, generator=_gen(at + i)).to(t) for i in range(3))
    k[at] = math.nan
    assert torch.isnan(_attention_once(q, k, v, d, type, 0, d ** -0.5)).all()
    o = _attention_once(q, k, v, d, type, 1, d ** -0.5)
    assert torch.isnan(o[at:]).all() and torch.isfinite(o[:at]).all()


@pytest.mark.parametrize("type", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n,gone", [(100, 30), (300, 128), (300, 200), (520, 384), (140, 140)])
def test_attention_scores_of_minus_infinity(n, gone, d, type):
    """The first keys' scores are all -infinity: weight 0, and NaN for rows that see no others."""
    t = mx_ref.TYPES[type]
    q, k, v = (torch.randn(n, d, device=DEV, generator=_gen(n + i)).to(t) for i in range(3))
    q[:, 0] = 1.0
    k[:gone, 0] = -math.inf
    k[gone:, 0] = 0.0
    for causal in (0, 1):
        o = _attention_once(q, k, v, d, type, causal, d ** -0.5)
        first = gone if causal or gone == n else 0  # rows before it see nothing else
        assert torch.isnan(o[:first]).all()
        if first < n:
            ref, mag = mx_ref.attention(q, k, v, [n], 1, 1, d, causal, d ** -0.5)
            # the roundings that _attn counts
            qk = d * 2.0 ** -23 * q.double().abs().amax() * k[gone:].double().abs().amax()
            u = mx_ref.half_step(t)
            tol = (1.01 * u + 1e-5 + 2 * qk) * mag + u * ref.abs()
            if t == torch.float16:
                tol = tol + n * 2.0 ** -25 * v.double().abs().amax() + 2.0 ** -25
            assert ((o[first:].double() - ref[first:]).abs() <= tol[first:]).all()


@pytest.mark.parametrize("d", [64, 128])
def test_attention_weight_of_unseen_keys_is_zero(d):
    """Values of 2^127 behind a row's own position, which any other weight would show."""
    n = 150
    q, k = (torch.randn(n, d, device=DEV, generator=_gen(i)).bfloat16() for i in range(2))
    v = torch.full((n, d), 2.0 ** 127, device=DEV).bfloat16()
    v[0] = 0.0
    o = _attention_once(q, k, v, d, BF16, 1, d ** -0.5)
    assert (o[0] == 0).all()


@pytest.mark.parametrize("type", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [2 ** 16, 2 ** 18 + 1, 2 ** 19])
def test_attention_long_sums_of_one_sign(n, d, type):
    """Equal weights and values of one sign: the tensor core cuts its sums with every 16 keys, by less than 2^-23."""
    t = mx_ref.TYPES[type]
    q, k = torch.zeros(n, d, dtype=t, device=DEV), torch.zeros(n, d, dtype=t, device=DEV)
    v = (1 + torch.rand(n, d, device=DEV, generator=_gen(n))).to(t)
    o = _attention_once(q, k, v, d, type, 0, 1.0)
    ref = v.double().mean(0)
    # the sum of the weights is one of n / 128 terms a row, of 32 each
    u = mx_ref.half_step(t)
    assert ((o.double() - ref).abs() <= (n * 2.0 ** -27 + (n / 128 + 40) * 2.0 ** -24 + 1e-6 + u) * ref).all()


# Heads of one sequence that a B200's 148 SMs take as single tiles whose keys are shared out, and so many that a CTA has
# two tiles.
FEW_OR_MANY = [1, 160]


def _attention_same_heads(q, k, v, heads, type, causal, scale, lens=None):
    """The same q, k and v [tokens][d] for every head, each with keys of its own; every head's result is the same."""
    n, d = q.shape
    lens = lens or [n]
    q, k, v = (x.repeat(1, heads) for x in (q, k, v))
    o = torch.full((n, heads * d), 7.0, dtype=q.dtype, device=DEV)
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=DEV)
    assert _lib().rfdetr_b200_op_attention_packed(_p(q), _p(k), _p(v), heads * d, heads * d, heads * d, _p(o), heads * d, type,
                                                  _p(cu), len(lens), n, max(lens), heads, heads, d, int(causal), scale,
                                                  _stream()) == 0
    bits = o.view(n, heads, d)
    assert torch.equal(bits.isnan(), bits[:, :1].isnan().expand_as(bits))
    assert torch.equal(bits.nan_to_num(), bits[:, :1].nan_to_num().expand_as(bits))
    return o[:, :d]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens,heads,kv", [([520], 160, 160), ([700, 130, 1, 0, 257], 80, 80), ([1100, 900], 128, 32),
                                           ([300, 385], 224, 32), ([129] * 40, 40, 10)])
def test_attention_two_tiles(lens, heads, kv, d, causal):
    """So many tiles that a CTA takes two of a sequence: both full, the second short or not there, one item or more
    after another."""
    _attn(lens, heads, kv, d, causal, BF16, behind=5)
    _attn(lens, heads, kv, d, causal, F16, seed=1, gain=3.0)


@pytest.mark.parametrize("heads", FEW_OR_MANY)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("type", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [100, 300, 700])
def test_attention_equal_scores_running_mean(n, d, type, causal, heads):
    """Keys that are all zero: the mean of the values up to each position, or of all, which differ from row to row."""
    t = mx_ref.TYPES[type]
    q, k = torch.randn(n, d, device=DEV, generator=_gen(0)).to(t), torch.zeros(n, d, dtype=t, device=DEV)
    v = (torch.linspace(-1, 2, n, device=DEV)[:, None] + torch.randn(n, d, device=DEV, generator=_gen(1)) * 0.1).to(t)
    o = _attention_same_heads(q, k, v, heads, type, causal, 0.125)
    count = torch.arange(1, n + 1, device=DEV, dtype=torch.float64)[:, None]
    mean = v.double().cumsum(0) / count if causal else v.double().mean(0).expand(n, d)
    mag = v.double().abs().cumsum(0) / count if causal else v.double().abs().mean(0).expand(n, d)
    # the weights are all 1, exact in either type: what is left are f32 sums of n terms, and the result's rounding
    u = mx_ref.half_step(t)
    assert ((o.double() - mean).abs() <= (n + 2) * 2.0 ** -23 * mag + u * mean.abs() + 2.0 ** -25).all()


@pytest.mark.parametrize("type", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("at", [0, 13, 63, 127, 128, 200, 255, 256, 300, 383, 400, 519])
def test_attention_two_tiles_nan_keys(at, d, type):
    """As test_attention_nan_keys_reach_the_rows_that_see_them, in CTAs of two tiles."""
    n, t = 520, mx_ref.TYPES[type]
    q, k, v = (torch.randn(n, d, device=DEV, generator=_gen(at + i)).to(t) for i in range(3))
    k[at] = math.nan
    assert torch.isnan(_attention_same_heads(q, k, v, 160, type, 0, d ** -0.5)).all()
    o = _attention_same_heads(q, k, v, 160, type, 1, d ** -0.5)
    assert torch.isnan(o[at:]).all() and torch.isfinite(o[:at]).all()


@pytest.mark.parametrize("type", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n,gone", [(300, 30), (300, 128), (300, 200), (520, 384), (520, 130), (520, 520)])
def test_attention_two_tiles_scores_of_minus_infinity(n, gone, d, type):
    """As test_attention_scores_of_minus_infinity, in CTAs of two tiles."""
    t = mx_ref.TYPES[type]
    q, k, v = (torch.randn(n, d, device=DEV, generator=_gen(n + i)).to(t) for i in range(3))
    q[:, 0] = 1.0
    k[:gone, 0] = -math.inf
    k[gone:, 0] = 0.0
    for causal in (0, 1):
        o = _attention_same_heads(q, k, v, 160, type, causal, d ** -0.5)
        first = gone if causal or gone == n else 0
        assert torch.isnan(o[:first]).all()
        if first < n:
            ref, mag = mx_ref.attention(q, k, v, [n], 1, 1, d, causal, d ** -0.5)
            qk = d * 2.0 ** -23 * q.double().abs().amax() * k[gone:].double().abs().amax()
            u = mx_ref.half_step(t)
            tol = (1.01 * u + 1e-5 + 2 * qk) * mag + u * ref.abs()
            if t == torch.float16:
                tol = tol + n * 2.0 ** -36 * v.double().abs().amax() + 2.0 ** -25
            assert ((o[first:].double() - ref[first:]).abs() <= tol[first:]).all()


@pytest.mark.parametrize("heads", FEW_OR_MANY)
@pytest.mark.parametrize("type", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_infinities_of_long_other_sequences(d, type, heads):
    """A sequence full of NaN and infinities between two others, each of several tiles and key blocks."""
    lens, t = [270, 400, 301], mx_ref.TYPES[type]
    n = sum(lens)
    clean = [torch.randn(n, d, device=DEV, generator=_gen(d + i)).to(t) for i in range(3)]
    dirty = [x.clone() for x in clean]
    for x in dirty:
        x[270:670] = math.nan
        x[270:670:2] = math.inf
    keep = torch.cat([torch.arange(270), torch.arange(670, n)]).to(DEV)
    for causal in (0, 1):
        a, b = (_attention_same_heads(*x, heads, type, causal, d ** -0.5, lens) for x in (dirty, clean))
        assert torch.equal(a[keep], b[keep]) and torch.isfinite(a[keep]).all()


@pytest.mark.parametrize("heads", FEW_OR_MANY)
@pytest.mark.parametrize("d", [64, 128])
def test_attention_unseen_keys_of_several_tiles_weigh_nothing(d, heads):
    """As test_attention_weight_of_unseen_keys_is_zero, over several key blocks: rows up to 300 see zeros only."""
    n = 600
    q, k = (torch.randn(n, d, device=DEV, generator=_gen(i)).bfloat16() for i in range(2))
    v = torch.full((n, d), 2.0 ** 127, device=DEV).bfloat16()
    v[:300] = 0.0
    o = _attention_same_heads(q, k, v, heads, BF16, 1, d ** -0.5)
    assert (o[:300] == 0).all()


@pytest.mark.parametrize("heads", FEW_OR_MANY)
@pytest.mark.parametrize("type", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("fall", [False, True])
def test_attention_growing_scores_of_either_form(fall, d, type, heads):
    """As test_attention_sharp_and_growing_scores, with the largest scores last or first, in both forms."""
    t = mx_ref.TYPES[type]
    n = 900
    gain = torch.linspace(4, 0.1, n, device=DEV) if fall else torch.linspace(0.1, 4, n, device=DEV)
    q, k, v = (torch.randn(n, d, device=DEV, generator=_gen(d + i)) for i in range(3))
    q, k, v = q.to(t), (k * gain[:, None]).to(t), v.to(t)
    for causal in (0, 1):
        o = _attention_same_heads(q, k, v, heads, type, causal, d ** -0.5)
        ref, mag = mx_ref.attention(q, k, v, [n], 1, 1, d, causal, d ** -0.5)
        u = mx_ref.half_step(t)
        tol = (1.01 * u + 4e-4) * mag + u * ref.abs() + (n * 2.0 ** -36 * 5 + 2.0 ** -25 if t == torch.float16 else 1e-30)
        assert ((o.double() - ref).abs() <= tol).all()


def test_attention_far_rows():
    """Token offsets that pass 32 bits."""
    n, ld, d = 66000, 33000 // 8 * 8, 64
    x = torch.empty(n, ld, dtype=torch.bfloat16, device=DEV)
    x[:, :3 * d] = torch.randn(n, 3 * d, device=DEV, generator=_gen(0)).bfloat16()
    lens = [100] * 659 + [50, 50]
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=DEV)
    assert cu[-1] == n
    o = x[:, 4 * d:]
    assert _lib().rfdetr_b200_op_attention_packed(_p(x), _p(x[:, d:]), _p(x[:, 2 * d:]), ld, ld, ld, _p(o), ld, BF16,
                                                  _p(cu), len(lens), n, 100, 1, 1, d, 1, 0.125, _stream()) == 0
    for s in (0, 400, 658, 660):
        a, b = int(cu[s]), int(cu[s + 1])
        ref, mag = mx_ref.attention(x[a:b, :d], x[a:b, d:2 * d], x[a:b, 2 * d:3 * d], [b - a], 1, 1, d, True, 0.125)
        u = 2.0 ** -8
        assert ((o[a:b, :d].double() - ref).abs() <= (1.01 * u + 1e-4) * mag + u * ref.abs()).all()


@pytest.mark.parametrize("type", [F16, BF16])
def test_operators_on_two_streams_at_once(type):
    """Calls that run side by side on two streams give what they give one after the other."""
    L = _lib()
    t = mx_ref.TYPES[type]
    g = _gen(9)
    n, heads, d = 3000, 8, 64
    qkv = torch.randn(2, n, 3 * heads * d, device=DEV, generator=g).to(t)
    cu = torch.tensor([0, 1000, 1001, n], dtype=torch.int32, device=DEV)
    ops = [_operand(g, r, 4096)[:2] for r in (3000, 1024, 8, 4096)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]

    def run(i, o, c, few, stream):
        x, ld = _p(qkv[i]), 3 * heads * d
        rc = L.rfdetr_b200_op_attention_packed(x, x + 2 * heads * d, x + 4 * heads * d, ld, ld, ld, _p(o), heads * d, type,
                                               _p(cu), 3, n, 2000, heads, heads, d, i, 0.125, stream)
        (a, sa), (b, sb), (m, sm), (w, sw) = ops
        rc += L.rfdetr_b200_op_mx_gemm(_p(a), 2048, _p(sa), _p(b), 2048, _p(sb), 3000, 1024, 4096, 1, None, _p(c), type,
                                       1024, stream)
        rc += L.rfdetr_b200_op_mx_gemm(_p(m), 2048, _p(sm), _p(w), 2048, _p(sw), 8, 4096, 4096, 0, None, _p(few), type,
                                       4096, stream)
        assert rc == 0

    def outs():
        return [torch.zeros(r, c, dtype=t, device=DEV) for r, c in ((n, heads * d), (3000, 1024), (8, 4096))]

    want = [outs(), outs()]
    for i in (0, 1):
        run(i, *want[i], _stream())
    torch.cuda.synchronize()
    for _ in range(5):
        got = [outs(), outs()]
        torch.cuda.synchronize()
        for _ in range(3):
            for i in (0, 1):
                run(i, *got[i], streams[i].cuda_stream)
        torch.cuda.synchronize()
        for i in (0, 1):
            for x, y in zip(got[i], want[i]):
                assert torch.equal(x, y)


# ---- together -------------------------------------------------------------------------


def _block(type, lens, dim, heads, kv, d, hidden, bufs, L, lib, stream):
    """One pre- and post-normed transformer block with 4-bit products over packed sequences."""
    n = sum(lens)
    qkv_n = (heads + 2 * kv) * d
    common = dict(rows=n, dim=dim, type=type, resid_type=F32, ldy=dim, ld_resid=dim, ld_out_resid=dim, ld_out=dim,
                  ld_mx=dim // 2, ld_gate=dim, resid_scale=1.0, post_eps=1e-6, pre_eps=1e-6, mx_codes=_p(bufs["c"]),
                  mx_scales=_p(bufs["s"]))
    rc = [L.rfdetr_b200_op_block_norm(lib.BlockNorm(y=_p(bufs["x0"]), pre=2, pre_w=_p(bufs["w1"]), **common), stream)]
    rc.append(L.rfdetr_b200_op_mx_gemm(_p(bufs["c"]), dim // 2, _p(bufs["s"]), _p(bufs["qkv_c"]), dim // 2,
                                       _p(bufs["qkv_s"]), n, qkv_n, dim, 0, _p(bufs["qkv_b"]), _p(bufs["qkv"]), type,
                                       qkv_n, stream))
    q = _p(bufs["qkv"])
    rc.append(L.rfdetr_b200_op_attention_packed(q, q + 2 * heads * d, q + 2 * (heads + kv) * d, qkv_n, qkv_n, qkv_n,
                                                _p(bufs["o"]), heads * d, type, _p(bufs["cu"]), len(lens), n, max(lens),
                                                heads, kv, d, 1, d ** -0.5, stream))
    rc.append(L.rfdetr_b200_op_mx_quantize(_p(bufs["o"]), type, heads * d, n, heads * d, _p(bufs["oc"]), heads * d // 2,
                                           _p(bufs["os"]), stream))
    rc.append(L.rfdetr_b200_op_mx_gemm(_p(bufs["oc"]), heads * d // 2, _p(bufs["os"]), _p(bufs["p_c"]), heads * d // 2,
                                       _p(bufs["p_s"]), n, dim, heads * d, 0, None, _p(bufs["y"]), type, dim, stream))
    rc.append(L.rfdetr_b200_op_block_norm(
        lib.BlockNorm(y=_p(bufs["y"]), resid=_p(bufs["x32"]), post=2, post_w=_p(bufs["w2"]), gate=_p(bufs["gate"]),
                      out_resid=_p(bufs["x1"]), pre=2, pre_w=_p(bufs["w3"]), **common), stream))
    rc.append(L.rfdetr_b200_op_mx_gemm(_p(bufs["c"]), dim // 2, _p(bufs["s"]), _p(bufs["f_c"]), dim // 2,
                                       _p(bufs["f_s"]), n, hidden, dim, 3, None, _p(bufs["hid"]), type, hidden, stream))
    assert rc == [0] * 7


def _block_buffers(type, lens, dim, heads, kv, d, hidden, seed):
    g = _gen(seed)
    t = mx_ref.TYPES[type]
    n = sum(lens)
    qkv_n = (heads + 2 * kv) * d
    b = {}
    b["x0"] = torch.randn(n, dim, device=DEV, generator=g).to(t)
    b["x32"] = b["x0"].float()
    for w in ("w1", "w2", "w3", "gate"):
        b[w] = 1 + 0.1 * torch.randn(dim, device=DEV, generator=g)
    b["qkv_b"] = torch.randn(qkv_n, device=DEV, generator=g) * 0.1
    for name, rows, k in (("qkv", qkv_n, dim), ("p", dim, heads * d), ("f", hidden, dim)):
        b[name + "_c"], b[name + "_s"], b[name + "_v"] = _operand(g, rows, k)
        b[name + "_s"] = (b[name + "_s"].int() - 4).clamp_min(0).to(torch.uint8)
        b[name + "_v"] /= 16
    for name, cols in (("qkv", qkv_n), ("o", heads * d), ("y", dim), ("hid", hidden)):
        b[name] = torch.zeros(n, cols, dtype=t, device=DEV)
    b["x1"] = torch.zeros(n, dim, device=DEV)
    b["c"], b["s"] = _mx_buffers(n, dim)
    b["oc"], b["os"] = _mx_buffers(n, heads * d)
    b["cu"] = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=DEV)
    return b


CONFIG = dict(lens=[150, 1, 0, 300, 77], dim=512, heads=8, kv=2, d=64, hidden=1024)


@pytest.mark.parametrize("type", [F16, BF16])
def test_block_together(type):
    """The calls of one block on a stream: each result against the plain form of its own inputs."""
    from rfdetr_b200 import lib

    c = CONFIG
    n, dim, heads, kv, d = sum(c["lens"]), c["dim"], c["heads"], c["kv"], c["d"]
    t = mx_ref.TYPES[type]
    u = mx_ref.half_step(t)
    b = _block_buffers(type, seed=1, **c)
    _block(type, bufs=b, L=_lib(), lib=lib, stream=_stream(), **c)
    # attention from the qkv that the product wrote
    qkv = b["qkv"]
    ref, mag = mx_ref.attention(qkv[:, :heads * d], qkv[:, heads * d:(heads + kv) * d], qkv[:, (heads + kv) * d:],
                                c["lens"], heads, kv, d, True, d ** -0.5)
    tol = (1.01 * u + 1e-3) * mag + u * ref.abs() + 1e-4
    assert ((b["o"].double() - ref).abs() <= tol).all()
    # its quantisation, bit for bit, and the projection
    codes, e = mx_ref.quantize(b["o"].double())
    assert torch.equal(b["oc"], mx_ref.pack(codes)) and torch.equal(b["os"], mx_ref.tile_scales(e))
    A = mx_ref.values(codes, e)
    ref = A @ b["p_v"].T
    assert ((b["y"].double() - ref).abs() <= _gemm_tolerance(A, b["p_v"], ref, t, 0, None)).all()
    # the residual, and the hidden layer from the operand that the norm wrote
    post, _ = mx_ref.norm(b["y"].double(), 2, b["w2"], None, 1e-6)
    x1 = b["x32"].double() + b["gate"].double() * post
    assert ((b["x1"].double() - x1).abs() <= 1e-5 * (1 + x1.abs())).all()
    e = b["s"].view(-1, dim // 128, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-1, dim // 32)[:n]
    A = mx_ref.values(mx_ref.unpack(b["c"]), e)
    h, _ = mx_ref.norm(x1, 2, b["w3"], None, 1e-6)
    assert (A - h).norm() < 0.15 * h.norm()
    ref = mx_ref.act(A @ b["f_v"].T, 3)
    assert ((b["hid"].double() - ref).abs() <= _gemm_tolerance(A, b["f_v"], ref, t, 3, None)).all()


@pytest.mark.parametrize("type", [F16, BF16])
def test_block_to_its_end(type):
    """The block's second half behind the hidden layer: quantisation, the product back to the residual stream's width,
    norm and residual, and the next block's norm with its operand; directly and captured."""
    from rfdetr_b200 import lib

    c = CONFIG
    n, dim, hidden = sum(c["lens"]), c["dim"], c["hidden"]
    t, L = mx_ref.TYPES[type], _lib()
    b = _block_buffers(type, seed=5, **c)
    g = _gen(6)
    w, sw, W = _operand(g, dim, hidden)
    sw, W = (sw.int() - 4).clamp_min(0).to(torch.uint8), W / 16
    w4, w5 = (1 + 0.1 * torch.randn(dim, device=DEV, generator=g) for _ in range(2))

    def run(stream, hc, hs, z, x2, h, nc, ns):
        _block(type, bufs=b, L=L, lib=lib, stream=stream, **c)
        rc = [L.rfdetr_b200_op_mx_quantize(_p(b["hid"]), type, hidden, n, hidden, _p(hc), hidden // 2, _p(hs), stream)]
        rc.append(L.rfdetr_b200_op_mx_gemm(_p(hc), hidden // 2, _p(hs), _p(w), hidden // 2, _p(sw), n, dim, hidden, 0, None,
                                           _p(z), type, dim, stream))
        rc.append(L.rfdetr_b200_op_block_norm(lib.BlockNorm(
            y=_p(z), resid=_p(b["x1"]), post=2, post_w=_p(w4), out_resid=_p(x2), pre=2, pre_w=_p(w5), out=_p(h),
            mx_codes=_p(nc), mx_scales=_p(ns), rows=n, dim=dim, type=type, resid_type=F32, ldy=dim, ld_resid=dim,
            ld_out_resid=dim, ld_out=dim, ld_mx=dim // 2, resid_scale=1.0, post_eps=1e-6, pre_eps=1e-6), stream))
        assert rc == [0] * 3

    def buffers():
        return [*_mx_buffers(n, hidden), torch.zeros(n, dim, dtype=t, device=DEV), torch.zeros(n, dim, device=DEV),
                torch.zeros(n, dim, dtype=t, device=DEV), *_mx_buffers(n, dim)]

    out = buffers()
    run(_stream(), *out)
    hc, hs, z, x2, h, nc, ns = out
    codes, e = mx_ref.quantize(b["hid"].double())
    assert torch.equal(hc, mx_ref.pack(codes)) and torch.equal(hs, mx_ref.tile_scales(e))
    A = mx_ref.values(codes, e)
    ref = A @ W.T
    assert ((z.double() - ref).abs() <= _gemm_tolerance(A, W, ref, t, 0, None)).all()
    post, _ = mx_ref.norm(z.double(), 2, w4, None, 1e-6)
    want = b["x1"].double() + post
    # the sums' roundings are under 110 * 2^-24 (as in _norm_case), of the norms and of what they are added to
    u = 110 * 2.0 ** -24
    slack = u * (post.abs() + want.abs()) + 4 * 2.0 ** -24 * (post.abs() + b["x1"].double().abs())
    assert ((x2.double() - want).abs() <= slack).all()
    nxt, rstd = mx_ref.norm(want, 2, w5, None, 1e-6)
    worst = slack.amax(1, keepdim=True) * rstd
    tol = worst * (3 * w5.double().abs() + 2 * nxt.abs()) + u * nxt.abs() + mx_ref.half_step(t) * nxt.abs() + 2.0 ** -25
    assert ((h.double() - nxt).abs() <= tol).all()
    e = ns.view(-1, dim // 128, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-1, dim // 32)[:n]
    # E2M1's own steps: at most a sixth of a value in [1, 6] scales, a quarter scale below; 6 stands for up to 8
    v, scale = mx_ref.values(mx_ref.unpack(nc), e), mx_ref.pow2(e.long() - 127).repeat_interleave(32, 1)
    assert ((v - nxt).abs() <= torch.maximum(0.25 * scale, nxt.abs() / 4) + tol).all()

    caught = buffers()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        run(torch.cuda.current_stream().cuda_stream, *caught)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for x, y in zip(caught, out):
        assert torch.equal(x, y)


def test_block_captured_and_replayed():
    """The same calls captured into a CUDA graph on a stream of their own and replayed on new inputs
    give what direct calls give, also while direct calls run on another stream."""
    from rfdetr_b200 import lib

    c = CONFIG
    one, two, plain = (_block_buffers(BF16, seed=s, **c) for s in (1, 2, 2))
    L = _lib()
    _block(BF16, bufs=plain, L=L, lib=lib, stream=_stream(), **c)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        _block(BF16, bufs=one, L=L, lib=lib, stream=torch.cuda.current_stream().cuda_stream, **c)
    for name in one:
        if not name.endswith("_v"):
            one[name].copy_(two[name])
    torch.cuda.synchronize()
    other = _block_buffers(BF16, seed=3, **c)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graph.replay()
    _block(BF16, bufs=other, L=L, lib=lib, stream=_stream(), **c)
    torch.cuda.synchronize()
    for name in ("qkv", "o", "y", "x1", "hid", "c", "s", "oc", "os"):
        assert torch.equal(one[name], plain[name]), name


@pytest.mark.parametrize("rows,dim", [(1, 256), (40, 512), (577, 768), (700, 2048)])
def test_calls_in_a_row_wait_for_each_other(rows, dim):
    """Each call reads what the one before wrote, and overwrites what the one before that read; without a pause, and
    captured, the results are those of calls with a wait after each."""
    from rfdetr_b200 import lib

    L = _lib()
    heads = dim // 64
    g = _gen(rows)
    w, sw, _ = _operand(g, dim, dim)
    sw = (sw.int() - 4).clamp_min(0).to(torch.uint8)
    ones = torch.ones(dim, device=DEV)
    start = torch.randn(rows, dim, device=DEV, generator=g).bfloat16()
    cu = torch.tensor([0, rows], dtype=torch.int32, device=DEV)
    n = L.rfdetr_b200_mx_scale_bytes(rows, dim)

    def run(rounds, pause, b, stream):
        def after(rc):
            assert rc == 0
            if pause:
                torch.cuda.synchronize()

        for _ in range(rounds):
            after(L.rfdetr_b200_op_block_norm(lib.BlockNorm(
                y=_p(b["y"]), resid=_p(b["x"]), pre_w=_p(ones), out_resid=_p(b["x"]), mx_codes=_p(b["c"]), mx_scales=_p(b["s"]),
                rows=rows, dim=dim, type=BF16, resid_type=BF16, pre=2, ldy=dim, ld_resid=dim, ld_out_resid=dim,
                ld_mx=dim // 2, resid_scale=0.5, pre_eps=1e-6), stream))
            after(L.rfdetr_b200_op_mx_gemm(_p(b["c"]), dim // 2, _p(b["s"]), _p(w), dim // 2, _p(sw), rows, dim, dim, 0, None,
                                           _p(b["y"]), BF16, dim, stream))
            after(L.rfdetr_b200_op_attention_packed(_p(b["y"]), _p(b["y"]), _p(b["y"]), dim, dim, dim, _p(b["o"]), dim, BF16,
                                                    _p(cu), 1, rows, rows, heads, heads, 64, 1, 0.125, stream))
            after(L.rfdetr_b200_op_mx_quantize(_p(b["o"]), BF16, dim, rows, dim, _p(b["c"]), dim // 2, _p(b["s"]), stream))
            after(L.rfdetr_b200_op_mx_dequantize(_p(b["c"]), dim // 2, _p(b["s"]), rows, dim, _p(b["y"]), BF16, dim, stream))

    def buffers():
        b = {k: start.clone() for k in ("x", "y", "o")}
        b["c"] = torch.zeros(rows, dim // 2, dtype=torch.uint8, device=DEV)
        b["s"] = torch.zeros(n, dtype=torch.uint8, device=DEV)
        return b

    want, got, caught = buffers(), buffers(), buffers()
    run(30, True, want, _stream())
    assert torch.isfinite(want["x"].float()).all() and not torch.equal(want["x"], start)
    run(30, False, got, _stream())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(10, False, caught, torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for name in want:
        assert torch.equal(got[name], want[name]) and torch.equal(caught[name], want[name]), name


def test_captured_with_copies_and_a_second_stream_between():
    """A graph in which the calls stand behind copies and fills, and behind two streams at once."""
    rows, dim = 33, 256
    g = _gen(9)
    w, sw, W = _operand(g, dim, dim)
    x = torch.zeros(rows, dim, dtype=torch.bfloat16, device=DEV)
    new = torch.randn(rows, dim, device=DEV, generator=g).bfloat16()
    n = _lib().rfdetr_b200_mx_scale_bytes(rows, dim)
    bufs = [(torch.zeros(rows, dim // 2, dtype=torch.uint8, device=DEV), torch.zeros(n, dtype=torch.uint8, device=DEV),
             torch.zeros(rows, dim, device=DEV)) for _ in range(2)]
    total = torch.zeros(rows, dim, dtype=torch.bfloat16, device=DEV)
    back = torch.zeros(rows, dim, device=DEV)
    side = torch.cuda.Stream()

    def branch(c, s, y):
        st = torch.cuda.current_stream().cuda_stream
        c.fill_(0x77)
        assert _lib().rfdetr_b200_op_mx_quantize(_p(x), BF16, dim, rows, dim, _p(c), dim // 2, _p(s), st) == 0
        assert _lib().rfdetr_b200_op_mx_gemm(_p(c), dim // 2, _p(s), _p(w), dim // 2, _p(sw), rows, dim, dim, 0, None, _p(y), F32,
                                             dim, st) == 0

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        main = torch.cuda.current_stream()
        x.copy_(new)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            branch(*bufs[0])
        branch(*bufs[1])
        main.wait_stream(side)
        # the first call behind both streams reads the other stream's operand
        assert _lib().rfdetr_b200_op_mx_dequantize(_p(bufs[0][0]), dim // 2, _p(bufs[0][1]), rows, dim, _p(back), F32, dim,
                                                   main.cuda_stream) == 0
        total.copy_(bufs[0][2] + bufs[1][2])
        assert _lib().rfdetr_b200_op_mx_quantize(_p(total), BF16, dim, rows, dim, _p(bufs[0][0]), dim // 2, _p(bufs[0][1]),
                                                 main.cuda_stream) == 0
    for i in range(3):
        new.copy_(torch.randn(rows, dim, device=DEV, generator=g).bfloat16())
        graph.replay()
        torch.cuda.synchronize()
        codes, e = mx_ref.quantize(new.double())
        A = mx_ref.values(codes, e)
        assert torch.equal(back.double(), A)
        ref = A @ W.T
        tol = _gemm_tolerance(A, W, ref, torch.float32, 0, None)
        assert all(((b[2].double() - ref).abs() <= tol).all() for b in bufs)
        codes, e = mx_ref.quantize(total.double())
        assert torch.equal(bufs[0][0], mx_ref.pack(codes)) and torch.equal(bufs[0][1], mx_ref.tile_scales(e))
        assert torch.equal(total, (bufs[0][2] + bufs[1][2]).bfloat16())


# ---- waits that run out -----------------------------------------------------------------

WAIT_PROBE = r"""
#include "sm100.cuh"
// A wait for an arrival that nobody makes, and the word that it leaves.
__global__ void k_wait(int* err) {
    __shared__ uint64_t bar;
    __shared__ int cta_abort;
    if (threadIdx.x == 0) {
        rfb::mbar_init(&bar, 1);
        cta_abort = 0;
        rfb::fence_mbar_init();
        rfb::mbar_wait(&bar, 0, &cta_abort, nullptr);
    }
    __syncthreads();
    rfb::report_abort(&cta_abort, err);
}
extern "C" int wait_for_nothing(int* err, void* stream) {
    k_wait<<<1, 32, 0, static_cast<cudaStream_t>(stream)>>>(err);
    return (int)cudaGetLastError();
}
"""


def _error_word():
    word = C.c_void_p()
    assert _lib().rfdetr_b200_op_error_word(C.byref(word)) == 0 and word.value
    return word.value


class _DeviceInt:
    """Device memory at an address as torch sees it."""

    def __init__(self, at):
        self.__cuda_array_interface__ = {"shape": (1,), "typestr": "<i4", "data": (at, False), "version": 2}


def test_error_word_stays_zero():
    """The calls of this file leave it alone; it is the same address every time."""
    at = _error_word()
    assert at == _error_word()
    word = torch.as_tensor(_DeviceInt(at), device=DEV)
    _gemm(300, 300, 16384, 0, BF16, False)
    _attn([700, 3], 4, 2, 64, True, BF16)
    assert word.item() == 0


def test_a_wait_that_runs_out_sets_the_error_word(tmp_path):
    """The operators' bounded wait, in a kernel of its own, for an arrival that nobody makes: it returns after its
    two seconds, the context lives on, the word tells, and the caller clears it."""
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    (tmp_path / "probe.cu").write_text(WAIT_PROBE)
    csrc = pathlib.Path(__file__).parents[1] / "rf-detr.cpp_b200" / "csrc"
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O2", "-shared", "-Xcompiler", "-fPIC",
                    "-cudart", "shared", "-I", str(csrc), "-o", str(tmp_path / "probe.so"), str(tmp_path / "probe.cu")],
                   check=True)
    probe = C.CDLL(str(tmp_path / "probe.so")).wait_for_nothing
    probe.argtypes = [C.c_void_p, C.c_void_p]
    at = _error_word()
    word = torch.as_tensor(_DeviceInt(at), device=DEV)
    assert word.item() == 0
    assert probe(at, _stream()) == 0
    # calls behind it run, and neither clear the word nor set it anew
    _gemm(70, 64, 512, 0, BF16, False)
    code = word.item()
    assert code & 0xff == 1
    _attn([200], 2, 1, 128, True, BF16)
    assert word.item() == code
    word.zero_()
    _gemm(70, 64, 512, 0, BF16, False)
    assert word.item() == 0


def test_first_call_of_a_process_may_be_captured():
    """Nothing that a first call sets up keeps it from being captured."""
    code = """
import sys, torch
sys.path[:0] = [%r, %r]
import mx_ref, test_gpu_block4 as t
g = t._gen(0)
(a, sa, A), (b, sb, B) = t._operand(g, 70, 512), t._operand(g, 64, 512)
x = torch.randn(200, 192, device=t.DEV, generator=g).bfloat16()
cu = torch.tensor([0, 200], dtype=torch.int32, device=t.DEV)
y, o = torch.zeros(70, 64, device=t.DEV), torch.zeros(200, 64, device=t.DEV).bfloat16()
graph = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(graph):
    st = torch.cuda.current_stream().cuda_stream
    L = t._lib()
    assert L.rfdetr_b200_op_mx_gemm(t._p(a), 256, t._p(sa), t._p(b), 256, t._p(sb), 70, 64, 512, 0, None, t._p(y), 0, 64, st) == 0
    assert L.rfdetr_b200_op_attention_packed(t._p(x), t._p(x[:, 64:]), t._p(x[:, 128:]), 192, 192, 192, t._p(o), 64, 30, t._p(cu),
                                             1, 200, 200, 1, 1, 64, 1, 0.125, st) == 0
graph.replay()
torch.cuda.synchronize()
assert ((y.double() - A @ B.T).abs() <= t._gemm_tolerance(A, B, A @ B.T, torch.float32, 0, None)).all()
assert torch.isfinite(o.float()).all() and (o[0] == x[0, 128:]).all()
""" % (str(pathlib.Path(__file__).parent), str(pathlib.Path(__file__).parents[1] / "rf-detr.cpp_b200"))
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300)
