"""Argument checks of the grouped products (they come before any CUDA call, so no GPU is needed), and of the
64-bit statements the GPU tests compare with."""
import ctypes as C

import numpy as np
import pytest

from cudanative_jl_b200 import _lib
from grouped_cases import grouped_k_ref, grouped_ref, offsets_of


@pytest.fixture()
def fake_handle():
    # the checks read nothing of the handle; a block of zeros stands for one
    buf = C.create_string_buffer(4096)
    return C.cast(buf, C.c_void_p), buf


GROUPED = dict(stream=None, transA=0, M=16, N=16, K=16, alpha=1.0, A=4096, lda=16, stride_a=256, B=4096, ldb=16, ab=_lib.F16, beta=0.0, Cm=None,
               ldc=16, c=_lib.F32, D=4096, ldd=16, d=_lib.F32, off=4096, groups=2)
GROUPED_K = dict(stream=None, M=16, N=16, K=16, alpha=1.0, A=4096, lda=16, B=4096, ldb=16, ab=_lib.F16, beta=0.0, Cm=None, ldc=16, stride_c=256,
                 c=_lib.F32, D=4096, ldd=16, stride_d=256, d=_lib.F32, off=4096, groups=2)

COMMON = [
    (dict(M=-1), b"negative dimension"),
    (dict(N=-1), b"negative dimension"),
    (dict(K=-1), b"negative dimension"),
    (dict(K=1 << 31, lda=1 << 31, ldb=1 << 31), b"exceeds 2^31"),
    (dict(groups=-1), b"groups must be"),
    (dict(groups=1025), b"groups must be"),
    (dict(ab=_lib.F32), b"A and B must be Float16 or bfloat16"),
    (dict(c=7), b"C and D must be"),
    (dict(d=-1), b"C and D must be"),
    (dict(lda=15), b"lda smaller"),
    (dict(ldb=15), b"ldb smaller"),
    (dict(ldd=15), b"ldd smaller"),
    (dict(beta=1.0, Cm=4096, ldc=15), b"ldc smaller"),
    (dict(beta=1.0), b"C is null"),
    (dict(A=None), b"A or B is null"),
    (dict(B=None), b"A or B is null"),
    (dict(D=None), b"D is null"),
    (dict(off=None), b"offsets is null"),
    (dict(off=4098), b"not aligned"),
    (dict(A=4097), b"not aligned"),
    (dict(D=4098), b"not aligned"),
    (dict(beta=1.0, Cm=4097), b"not aligned"),
]


@pytest.mark.parametrize("change,text", COMMON + [(dict(transA=2), b"transA"), (dict(stride_a=-1), b"negative stride")])
def test_grouped_refuses(lib, fake_handle, change, text):
    args = {**GROUPED, **change}
    assert lib.b200_gemm_grouped(fake_handle[0], *args.values()) == _lib.INVALID_ARG
    assert text in lib.b200_last_error(), lib.b200_last_error()


@pytest.mark.parametrize("change,text", COMMON + [(dict(stride_d=255), b"overlap"), (dict(beta=1.0, Cm=4096, stride_c=-1), b"negative stride")])
def test_grouped_k_refuses(lib, fake_handle, change, text):
    args = {**GROUPED_K, **change}
    assert lib.b200_gemm_grouped_k(fake_handle[0], *args.values()) == _lib.INVALID_ARG
    assert text in lib.b200_last_error(), lib.b200_last_error()


@pytest.mark.parametrize("change", [dict(M=0), dict(N=0, off=None), dict(groups=0, off=None, D=None)])
def test_nothing_to_do_is_no_error(lib, fake_handle, change):
    assert lib.b200_gemm_grouped(fake_handle[0], *{**GROUPED, **change}.values()) == _lib.OK
    assert lib.b200_gemm_grouped_k(fake_handle[0], *{**GROUPED_K, **change}.values()) == _lib.OK


def test_null_handle(lib):
    assert lib.b200_gemm_grouped(None, *GROUPED.values()) == _lib.INVALID_ARG
    assert lib.b200_gemm_grouped_k(None, *GROUPED_K.values()) == _lib.INVALID_ARG


def test_gradients_of_the_statement():
    """The two statements are each other's gradients: central differences of sum(G * D) in float64."""
    r = np.random.default_rng(0)
    off = offsets_of([3, 0, 4])
    W, X, G = r.standard_normal((3, 5, 6)), r.standard_normal((5, 7)), r.standard_normal((6, 7))  # W_e stored K x M

    def loss(W, X):
        return np.sum(G * grouped_ref(list(W), X, None, off, 1.0, 0.0, True, np.zeros((6, 7)))[0])

    dX = grouped_ref(list(W), G, None, off, 1.0, 0.0, False, np.zeros((5, 7)))[0]
    dW = np.stack(grouped_k_ref(X, G, None, off, 1.0, 0.0)[0])
    h = 1e-6
    for x, g, f in ((X, dX, lambda v: loss(W, v)), (W, dW, lambda v: loss(v, X))):
        for i in list(np.ndindex(x.shape))[::7]:
            up, down = x.copy(), x.copy()
            up[i] += h
            down[i] -= h
            assert abs((f(up) - f(down)) / (2 * h) - g[i]) < 1e-6


def test_every_new_entry_point_has_a_julia_wrapper():
    from test_binding_signatures import julia_ccalls

    seen = {name for name, *_ in julia_ccalls()}
    for name in ("b200_gemm_grouped", "b200_gemm_grouped_k", "b200_mxfp4_scale_bytes", "b200_mxfp4_quantize", "b200_mxfp4_dequantize",
                 "b200_gemm_mxfp4", "b200_gemm_mxfp4_grouped"):
        assert name in seen
