"""Long sums of one sign in the grouped and the 4-bit products.  The tensor core truncates when it adds to its accumulator, so
one accumulator for all of K is off by an amount that grows with K; the kernels begin a new one after a fixed number
of products and add them with rounding to nearest.

Tolerance, relative to the sum (one sign: it is the sum of magnitudes), by arithmetic: an instruction drops less than two units
in the last place, 2 * 2^-23, of what its accumulator holds, `steps` instructions to an accumulator; adding the accumulators
takes K / products roundings of 2^-24 each at most, splitting the sum over CTAs four more, scaling by alpha and adding beta * C two;
the result is rounded by half a step, which below the type's normal numbers is half the smallest one (2^-25 in binary16)."""
import numpy as np
import pytest

from cudanative_jl_b200 import _lib
from cudanative_jl_b200.array import Array, CuArray
from cudanative_jl_b200.bfloat16 import BFloat16
from grouped_cases import HALF_STEP, offsets_of, store, value
from mxfp4_cases import pack, tile, values

pytestmark = pytest.mark.gpu

F16, F32 = np.float16, np.float32


def sync(handle):
    _lib.check(_lib.lib().b200_stream_sync(None), "sync")
    assert handle.device_status()[0] == 0


def near(got, exact, elem, K, products, steps, what):
    rel = 2 * steps * 2.0 ** -23 + (K / products + 6) * 2.0 ** -24
    off = np.abs(got - exact) - (rel * exact + HALF_STEP[elem][0] * (1 + rel) * exact + HALF_STEP[elem][1])
    assert np.all(off <= 0), f"{what}: {np.max(np.abs(got - exact) / exact):.3g} of the result"


# a 16-bit result: accumulators of 16384 products for binary16 and 65536 for bfloat16, 16 to an instruction
def near16(got, exact, d_type, K, what):
    products = 16384 if d_type is F16 else 65536
    near(value(got, d_type), exact, d_type, K, products, products // 16, what)


@pytest.fixture(scope="module")
def positive():
    r = np.random.default_rng(1)
    K = 2 ** 20 + 40
    return store(0.1 + r.random((72, K)), F16), store((0.1 + r.random((40, K))) / 64, F16)


@pytest.mark.parametrize("d_type", [F16, BFloat16])
@pytest.mark.parametrize("tile_n,cta_pair", [(0, 0), (64, 1), (128, 1), (256, 1), (256, 2)])
def test_ragged_k(handle, positive, d_type, tile_n, cta_pair):
    """Groups of one accumulator, of a little more, of many; the last one with a ragged end."""
    A, B = positive
    M, N, alpha = 72, 40, 2.0 ** -10
    sizes = [8192, 0, 16400, 24571, 3, 16384, 65536, 65552]
    sizes.append(A.shape[1] - sum(sizes) - 3)
    off, K = offsets_of(sizes), A.shape[1]
    handle.set_option(_lib.OPT_TILE_N, tile_n)
    handle.set_option(_lib.OPT_CTA_PAIR, cta_pair)
    d = CuArray(np.zeros((M, N * len(sizes)), F16 if d_type is F16 else np.uint16, order="F"))
    handle.gemm_grouped_k(M, N, K, alpha, CuArray(A), M, CuArray(B), N, F16, 0.0, None, M, 0, F32, d, M, M * N, d_type, CuArray(off), len(sizes))
    sync(handle)
    got, a, b = Array(d), value(A, F16), value(B, F16)
    for e, n in enumerate(sizes):
        s = slice(off[e], off[e + 1])
        near16(got[:, e * N:(e + 1) * N], alpha * (a[:, s] @ b[:, s].T), d_type, n, f"group of {n}")


@pytest.mark.parametrize("d_type", [F16, BFloat16])
@pytest.mark.parametrize("tile_n,cta_pair", [(0, 0), (64, 1), (128, 1), (256, 2)])
@pytest.mark.parametrize("N", [8, 40])
def test_ragged_n(handle, positive, d_type, tile_n, cta_pair, N):
    A, B = positive
    M, K, alpha = 72, A.shape[1], 2.0 ** -10
    handle.set_option(_lib.OPT_TILE_N, tile_n)
    handle.set_option(_lib.OPT_CTA_PAIR, cta_pair)
    d = CuArray(np.zeros((M, N), F16 if d_type is F16 else np.uint16, order="F"))
    c = store(np.full((M, N), 2.0), F32)
    handle.gemm_grouped(True, M, N, K, alpha, CuArray(np.asfortranarray(A.T)), K, 0, CuArray(np.asfortranarray(B[:N].T)), K, F16, 1.0, CuArray(c), M, F32,
                        d, M, d_type, CuArray(offsets_of([N // 2, 0, N - N // 2])), 3)
    sync(handle)
    near16(Array(d), alpha * (value(A, F16) @ value(B[:N], F16).T) + 2.0, d_type, K, f"tiles of {tile_n}")


# ---- 4-bit operands: 64 products to an instruction; a binary32 result takes 8192 from one accumulator, a 16-bit one 65536
def operand(r, K, cols, spread=4):
    """Elements of one sign, scales that differ; zeros behind K."""
    codes = r.integers(1, 8, ((K + 31) // 32 * 32, cols)).astype(np.uint8)
    codes[K:] = 0
    return codes, (127 + r.integers(-spread, spread + 1, (codes.shape[0] // 32, cols))).astype(np.uint8)


def run_mx(handle, M, N, K, d_type, beta=0.0, sizes=None, alpha=2.0 ** -12):
    r = np.random.default_rng(K + N)
    (qa, sa), (qb, sb) = operand(r, K, M), operand(r, K, N)
    off = None if sizes is None else offsets_of(sizes)
    ld = qa.shape[0]
    d, c = CuArray(np.zeros((M, N), np.uint16 if d_type is BFloat16 else d_type, order="F")), CuArray(np.full((M, N), 2.0, F32, order="F"))
    args = (CuArray(pack(qa, ld)), ld) + (() if off is None else (0,)) + (CuArray(tile(sa)), CuArray(pack(qb, ld)), ld, CuArray(tile(sb, off)), beta, c, M, F32, d, M, d_type)
    if off is None:
        handle.gemm_mxfp4(M, N, K, alpha, *args)
    else:
        handle.gemm_mxfp4_grouped(M, N, K, alpha, *args, CuArray(off), len(sizes))
    sync(handle)
    exact = alpha * (values(qa, sa)[:K].T @ values(qb, sb)[:K]) + beta * 2.0
    products = 8192 if d_type is F32 else 65536
    near(value(Array(d), d_type), exact, d_type, K, products, products // 64, f"{M} x {N} x {K}")
    return handle.last_launch()["tile_n"]


@pytest.mark.parametrize("N,tile_n,beta,expect", [(8, 0, 0.0, 32), (72, 0, 0.0, 128), (136, 0, 0.0, 256), (136, 0, 1.0, 192), (136, 256, 0.0, 256), (8, 128, 1.0, 128)])
def test_mx_binary32(handle, N, tile_n, beta, expect):
    handle.set_option(_lib.OPT_TILE_N, tile_n)
    assert run_mx(handle, 136, N, 262144 + 40, F32, beta=beta) == expect
    for K in (8192, 8193, 16384, 24576 + 31):  # one accumulator, a second one of one value, whole ones
        assert run_mx(handle, 136, N, K, F32, beta=beta) == expect


def test_mx_binary32_groups(handle):
    for sizes in ([5, 0, 3], [70, 0, 1], [300, 0, 129, 64]):
        run_mx(handle, 264, sum(sizes), 40000, F32, sizes=sizes)
    handle.set_option(_lib.OPT_MAX_CTAS, 2)  # many tiles to a CTA: the accumulators go around
    run_mx(handle, 264, 429, 25000, F32, beta=1.0, sizes=[300, 0, 129])
    run_mx(handle, 520, 300, 25000, F32)


@pytest.mark.parametrize("d_type", [F16, BFloat16])
@pytest.mark.parametrize("tile_n", [0, 128, 256])
def test_mx_16_bits(handle, d_type, tile_n):
    handle.set_option(_lib.OPT_TILE_N, tile_n)
    for K in (65536, 65536 + 40, 2 ** 21):
        run_mx(handle, 136 if tile_n == 256 else 8, 8, K, d_type, alpha=2.0 ** -15)
