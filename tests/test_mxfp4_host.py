"""Argument checks of the 4-bit entry points (before any CUDA call), their sizes, and the numpy statement of the
format that the GPU tests compare with."""
import ctypes as C

import numpy as np
import pytest

from cudanative_jl_b200 import _lib
from cudanative_jl_b200.gemm import mxfp4_scale_bytes
from mxfp4_cases import GRID, pack, quantize, tile, up, values


@pytest.fixture()
def fake_handle():
    buf = C.create_string_buffer(4096)
    return C.cast(buf, C.c_void_p), buf


QUANT = dict(stream=None, trans=0, K=64, cols=8, X=4096, ldx=64, t=_lib.F16, Q=4096, ldq=64, S=4096, off=None, groups=0)
DEQUANT = dict(stream=None, K=64, cols=8, Q=4096, ldq=64, S=4096, Y=4096, ldy=64, t=_lib.F16, off=None, groups=0)
GEMM = dict(stream=None, M=16, N=16, K=64, alpha=1.0, A=4096, lda=64, SA=4096, B=4096, ldb=64, SB=4096, beta=0.0, Cm=None, ldc=16, c=_lib.F32,
            D=4096, ldd=16, d=_lib.F32)
GROUPED = dict(stream=None, M=16, N=16, K=64, alpha=1.0, A=4096, lda=64, stride_a=1024, SA=4096, B=4096, ldb=64, SB=4096, beta=0.0, Cm=None, ldc=16,
               c=_lib.F32, D=4096, ldd=16, d=_lib.F32, off=4096, groups=2)


@pytest.mark.parametrize("change,text", [
    (dict(K=-1), b"negative"), (dict(cols=-1), b"negative"), (dict(t=5), b"values must be"), (dict(ldq=32), b"ldq"), (dict(K=33, ldx=64, ldq=33), b"ldq"),
    (dict(ldq=72), b"ldq"), (dict(groups=-1), b"groups"), (dict(groups=2), b"go together"), (dict(off=4096), b"go together"),
    (dict(off=4096, groups=1025), b"groups"), (dict(Q=None), b"null"), (dict(S=None), b"null"), (dict(Q=4104), b"16-byte"), (dict(S=4100), b"16-byte"),
    (dict(off=4098, groups=1), b"not aligned")])
def test_quantize_refuses(lib, fake_handle, change, text):
    for fn, args, extra in ((lib.b200_mxfp4_quantize, QUANT, {}), (lib.b200_mxfp4_dequantize, DEQUANT, {})):
        merged = {**args, **{k: v for k, v in change.items() if k in args}}
        assert fn(fake_handle[0], *merged.values()) == _lib.INVALID_ARG
        assert text in lib.b200_last_error(), lib.b200_last_error()


def test_quantize_refuses_its_own(lib, fake_handle):
    for fn, args, change in ((lib.b200_mxfp4_quantize, QUANT, dict(ldx=63)), (lib.b200_mxfp4_quantize, QUANT, dict(trans=1, ldx=7)),
                             (lib.b200_mxfp4_quantize, QUANT, dict(trans=2)), (lib.b200_mxfp4_quantize, QUANT, dict(X=None)),
                             (lib.b200_mxfp4_quantize, QUANT, dict(X=4097)), (lib.b200_mxfp4_dequantize, DEQUANT, dict(ldy=63)),
                             (lib.b200_mxfp4_dequantize, DEQUANT, dict(Y=None)), (lib.b200_mxfp4_dequantize, DEQUANT, dict(Y=4098, t=_lib.F32))):
        assert fn(fake_handle[0], *{**args, **change}.values()) == _lib.INVALID_ARG
    assert lib.b200_mxfp4_quantize(fake_handle[0], *{**QUANT, **dict(cols=0, X=None)}.values()) == _lib.OK
    assert lib.b200_mxfp4_quantize(None, *QUANT.values()) == _lib.INVALID_ARG
    assert lib.b200_mxfp4_dequantize(None, *DEQUANT.values()) == _lib.INVALID_ARG


@pytest.mark.parametrize("change,text", [
    (dict(M=-1), b"negative"), (dict(K=0), b"K must be positive"), (dict(lda=32), b"lda and ldb"), (dict(ldb=72), b"lda and ldb"), (dict(ldd=15), b"ldd"),
    (dict(beta=1.0), b"C is null"), (dict(beta=1.0, Cm=4096, ldc=3), b"ldc"), (dict(c=9), b"must be"), (dict(d=9), b"must be"), (dict(A=None), b"null"),
    (dict(SB=None), b"null"), (dict(D=None), b"D is null"), (dict(A=4104), b"16-byte"), (dict(SA=4098), b"16-byte"), (dict(D=4098), b"not aligned"),
    (dict(beta=1.0, Cm=4098), b"not aligned")])
def test_gemm_refuses(lib, fake_handle, change, text):
    for fn, args in ((lib.b200_gemm_mxfp4, GEMM), (lib.b200_gemm_mxfp4_grouped, GROUPED)):
        assert fn(fake_handle[0], *{**args, **change}.values()) == _lib.INVALID_ARG
        assert text in lib.b200_last_error(), lib.b200_last_error()


def test_grouped_gemm_refuses_its_own(lib, fake_handle):
    for change in (dict(groups=-1), dict(groups=1025), dict(off=None), dict(off=4097), dict(stride_a=1023), dict(stride_a=992), dict(stride_a=-32)):
        assert lib.b200_gemm_mxfp4_grouped(fake_handle[0], *{**GROUPED, **change}.values()) == _lib.INVALID_ARG, change
    assert lib.b200_gemm_mxfp4_grouped(fake_handle[0], *{**GROUPED, **dict(groups=0, off=None)}.values()) == _lib.OK
    assert lib.b200_gemm_mxfp4(None, *GEMM.values()) == _lib.INVALID_ARG
    assert lib.b200_gemm_mxfp4_grouped(None, *GROUPED.values()) == _lib.INVALID_ARG


def test_scale_bytes(lib):
    assert mxfp4_scale_bytes(128, 128) == 512
    assert mxfp4_scale_bytes(129, 128) == 1024 and mxfp4_scale_bytes(1, 129) == 1024
    assert mxfp4_scale_bytes(0, 5) == 0 and mxfp4_scale_bytes(5, 0) == 0 and mxfp4_scale_bytes(5, 0, 3) == 0
    for sizes in ([1, 1, 1], [128, 0, 129], [200, 56], [1] * 9):
        need = sum(up(n, 128) // 128 for n in sizes) * 2 * 512
        assert mxfp4_scale_bytes(200, sum(sizes), len(sizes)) >= need
    assert mxfp4_scale_bytes(128, 3, 3) == 3 * 512  # reached: three groups of one column


def test_statement_of_the_format():
    every = np.concatenate([GRID, -GRID])
    x = np.zeros((32, 1))
    x[:16, 0] = every * 2.0 ** -5
    codes, scales = quantize(x)
    assert scales[0, 0] == 122 and np.array_equal(values(codes, scales), x)
    # ties go to the even code, what passes 6 saturates
    x = np.zeros((32, 1))
    x[:9, 0] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.9, 7.999]
    assert np.array_equal(values(*quantize(x))[:9, 0], [0, 1, 1, 2, 2, 4, 4, 6, 6])
    assert quantize(np.full((1, 1), np.inf))[1][0, 0] == 255 and np.isnan(values(*quantize(np.full((32, 1), np.nan)))).all()
    assert quantize(np.zeros((32, 1)))[1][0, 0] == 0
    assert quantize(np.full((32, 1), 2.0 ** -149))[1][0, 0] == 0 and quantize(np.full((32, 1), 3e38))[1][0, 0] == 252
    t = tile(np.arange(2 * 130).reshape(2, 130) % 251).reshape(2, 1, 512)
    assert t[0, 0, 33 % 32 * 16 + 4 + 1] == (130 + 33) % 251 and t[1, 0, 16 + 0] == 129 % 251 and t[1, 0, 2 * 16] == 0
    assert np.array_equal(pack(np.array([[1], [2]] * 16, np.uint8), 64)[:17, 0], [0x21] * 16 + [0])
