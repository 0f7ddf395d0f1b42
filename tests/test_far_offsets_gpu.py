"""Matrices whose elements lie more than 2^31 apart: leading dimensions, matrices per group and columns far from the first one.
The buffers are large and, but for the elements of the product, never touched."""
import numpy as np
import pytest

from cudanative_jl_b200 import _lib
from cudanative_jl_b200.array import CuArray, CuHostArray
from cudanative_jl_b200.bfloat16 import BFloat16
from grouped_cases import close, grouped_k_ref, grouped_ref, memory_type, offsets_of, store, value
from mxfp4_cases import pack, random_operand, tile, values

pytestmark = pytest.mark.gpu

F16, F32 = np.float16, np.float32


class Far:
    """Columns `ld` elements apart, matrices `stride`; only the columns are moved."""

    def __init__(self, elem, rows, cols, ld, stride=0, count=1):
        self.elem, self.rows, self.cols, self.ld, self.stride, self.count = elem, rows, cols, ld, stride, count
        self.buf = CuHostArray(memory_type(elem), shape=((count - 1) * stride + (cols - 1) * ld + rows + 64,))
        assert (count - 1) * stride + (cols - 1) * ld > 2 ** 31

    def _columns(self, host, move):
        size = np.dtype(memory_type(self.elem)).itemsize
        for e in range(self.count):
            for j in range(self.cols):
                move(self.buf.ptr + size * (e * self.stride + j * self.ld), host[e][:, j])
        _lib.check(_lib.lib().b200_stream_sync(None), "sync")

    def put(self, mats):
        mats = [np.asfortranarray(m) for m in mats]
        self._columns(mats, lambda at, col: _lib.check(_lib.lib().b200_memcpy_h2d(at, col.ctypes.data, col.nbytes, None), "h2d"))
        return self

    def get(self):
        out = [np.zeros((self.rows, self.cols), memory_type(self.elem), order="F") for _ in range(self.count)]
        self._columns(out, lambda at, col: _lib.check(_lib.lib().b200_memcpy_d2h(col.ctypes.data, at, col.nbytes, None), "d2h"))
        return [value(m, self.elem) for m in out]


def sync(handle):
    _lib.check(_lib.lib().b200_stream_sync(None), "sync")
    assert handle.device_status()[0] == 0


def normal(r, shape):
    return r.standard_normal(shape).astype(np.float32)


@pytest.mark.parametrize("d_type,c_type", [(F32, F32), (BFloat16, F16)])
@pytest.mark.parametrize("K", [64, 2048])  # the longer one is shared by four CTAs
@pytest.mark.parametrize("kernel", [_lib.KERNEL_TCGEN05, _lib.KERNEL_SIMPLE])
def test_ragged_n(handle, d_type, c_type, K, kernel):
    r = np.random.default_rng(0)
    M, ld, sizes = 72, 2 ** 26, [20, 0, 21]
    N, off = sum(sizes), offsets_of(sizes)
    handle.set_option(_lib.OPT_FORCE_KERNEL, kernel)
    A, B, Cm = [store(normal(r, (K, M)), F16) for _ in sizes], store(normal(r, (K, N)), F16), store(normal(r, (M, N)), c_type)
    a = Far(F16, K, M, K, stride=2 ** 30 + 8, count=3).put(A)
    c, d = Far(c_type, M, N, ld).put([Cm]), Far(d_type, M, N, ld)
    handle.gemm_grouped(True, M, N, K, 1.0, a.buf.ptr, K, a.stride, CuArray(B), K, F16, 0.5, c.buf.ptr, ld, c_type, d.buf.ptr, ld, d_type, CuArray(off), 3)
    sync(handle)
    assert handle.last_launch()["kernel"] == kernel
    exact, S = grouped_ref([value(x, F16) for x in A], value(B, F16), value(Cm, c_type), off, 1.0, 0.5, True, np.zeros((M, N)))
    close(d.get()[0], exact, S, K, d_type)


@pytest.mark.parametrize("d_type", [F32, BFloat16])
@pytest.mark.parametrize("sizes", [[40, 0, 33], [4100, 0, 2100]], ids=str)
@pytest.mark.parametrize("kernel", [_lib.KERNEL_TCGEN05, _lib.KERNEL_SIMPLE])
def test_ragged_k(handle, d_type, sizes, kernel):
    r = np.random.default_rng(1)
    M, N, off, stride = 72, 40, offsets_of(sizes), 2 ** 30 + 7
    K = sum(sizes)
    handle.set_option(_lib.OPT_FORCE_KERNEL, kernel)
    A, B, Cm = store(normal(r, (M, K)), F16), store(normal(r, (N, K)), F16), [store(normal(r, (M, N)), F32) for _ in sizes]
    c, d = Far(F32, M, N, 80, stride=stride, count=3).put(Cm), Far(d_type, M, N, 80, stride=stride, count=3)
    handle.gemm_grouped_k(M, N, K, 1.0, CuArray(A), M, CuArray(B), N, F16, 1.0, c.buf.ptr, 80, stride, F32, d.buf.ptr, 80, stride, d_type, CuArray(off), 3)
    sync(handle)
    exact, S = grouped_k_ref(value(A, F16), value(B, F16), [value(x, F32) for x in Cm], off, 1.0, 1.0)
    for e, got in enumerate(d.get()):
        close(got, exact[e], S[e], sizes[e], d_type, f"group {e}")


@pytest.mark.parametrize("d_type", [F32, BFloat16])
@pytest.mark.parametrize("N", [33, 136])
def test_4_bits(handle, d_type, N):
    r = np.random.default_rng(2)
    M, K, ld = 136, 96, 2 ** 31 // (N - 1) + 64
    (qa, sa), (qb, sb) = random_operand(r, K, M), random_operand(r, K, N)
    Cm = store(normal(r, (M, N)), F32)
    c, d = Far(F32, M, N, ld).put([Cm]), Far(d_type, M, N, ld)
    handle.gemm_mxfp4(M, N, K, 0.25, CuArray(pack(qa, K)), K, CuArray(tile(sa)), CuArray(pack(qb, K)), K, CuArray(tile(sb)), 1.0, c.buf.ptr, ld, F32, d.buf.ptr, ld,
                      d_type)
    sync(handle)
    exact, S = grouped_ref([values(qa, sa)], values(qb, sb), value(Cm, F32), offsets_of([N]), 0.25, 1.0, True, np.zeros((M, N)))
    close(d.get()[0], exact, S, K, d_type)


@pytest.mark.parametrize("elem", [F16, F32])
@pytest.mark.parametrize("trans", [False, True])
def test_quantise(handle, elem, trans):
    """Values far apart in, and back."""
    r = np.random.default_rng(3)
    K, cols = 72, 40
    X = store(normal(r, (cols, K) if trans else (K, cols)), elem)
    ld = 2 ** 31 // (X.shape[1] - 1) // 8 * 8 + 64
    x, y = Far(elem, X.shape[0], X.shape[1], ld).put([X]), Far(elem, K, cols, 2 ** 31 // 39 + 8)
    q, s = CuArray(np.zeros((48, cols), np.uint8, order="F")), CuArray(np.zeros(512, np.uint8))
    handle.mxfp4_quantize(trans, K, cols, x.buf.ptr, ld, elem, q, 96, s)
    handle.mxfp4_dequantize(K, cols, q, 96, s, y.buf.ptr, y.ld, elem)
    sync(handle)
    from mxfp4_cases import quantize

    exact = values(*quantize(value(X.T if trans else X, elem)))[:K]
    assert np.array_equal(y.get()[0], exact)
