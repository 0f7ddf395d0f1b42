"""Microscaled 4-bit values through the C ABI: quantisation bit for bit against the numpy statement, products against
float64 on the values that elements and scales stand for."""
import numpy as np
import pytest

from cudanative_jl_b200 import _lib
from cudanative_jl_b200.array import Array, CuArray
from cudanative_jl_b200.bfloat16 import BFloat16
from cudanative_jl_b200.gemm import mxfp4_scale_bytes
from grouped_cases import close, grouped_ref, offsets_of, store, value
from mxfp4_cases import pack, quantize, random_operand, tile, tile_starts, up, values

pytestmark = pytest.mark.gpu

F16, F32 = np.float16, np.float32


def sync(handle, expect=0):
    _lib.check(_lib.lib().b200_stream_sync(None), "sync")
    code, block, detail = handle.device_status()
    assert code == expect, f"device status {code} (block {block}, detail {detail})"


def spread(r, K, cols):
    """Columns and blocks of very different size, exact ties among the values."""
    x = r.standard_normal((K, cols)) * np.exp2(r.integers(-6, 7, (K, cols)).astype(float))
    ties = r.random((K, cols)) < 0.2
    return np.where(ties, r.choice([0.25, 0.75, -1.25, 1.75, 2.5, -3.5, 5.0, 6.0, 0.0, -0.0], (K, cols)), x)


def run_quantize(handle, X, elem, trans, offsets=None, ldx_pad=0, ldq_pad=0):
    """X float64 values exact in elem.  Checks codes, scales and the way back; returns nothing."""
    K, cols = X.shape
    src = store(X.T if trans else X, elem)
    X = value(src.T if trans else src, elem)
    padded = np.full((src.shape[0] + ldx_pad, src.shape[1]), 0x7fff if elem is BFloat16 else np.nan, src.dtype, order="F")
    padded[: src.shape[0]] = src
    ldq = up(K, 32) + ldq_pad
    q = CuArray(np.full((ldq // 2, cols), 0xA5, np.uint8, order="F"))
    groups = 0 if offsets is None else len(offsets) - 1
    s = CuArray(np.full(mxfp4_scale_bytes(K, cols, groups) + 64, 0xA5, np.uint8))
    off = None if offsets is None else CuArray(np.asarray(offsets, np.int32))
    handle.mxfp4_quantize(trans, K, cols, CuArray(padded), padded.shape[0], elem, q, ldq, s, offsets=off, groups=groups)
    sync(handle)
    codes, scales = quantize(X)
    rows = tile_starts(cols, offsets)
    inside = np.zeros(cols, bool)
    for c, n in rows:
        inside[c:c + n] = True
    want = tile(scales, offsets)
    got_s, got_q = Array(s), Array(q)
    assert np.array_equal(got_s[: want.size], want), "scales"
    assert np.all(got_s[want.size:] == 0xA5), "bytes behind the scales were written"
    good = np.repeat(scales != 255, 16, axis=0)
    assert np.array_equal(got_q[: up(K, 32) // 2][:, inside][good[:, inside]], pack(codes, up(K, 32))[:, inside][good[:, inside]]), "elements"
    assert np.all(got_q[up(K, 32) // 2:] == 0xA5) and np.all(got_q[:, ~inside] == 0xA5), "bytes between the columns were written"
    for y_type in (F32, elem):
        y = CuArray(store(np.full((K + 3, cols), -7.25), y_type))
        handle.mxfp4_dequantize(K, cols, q, ldq, s, y, K + 3, y_type, offsets=off, groups=groups)
        sync(handle)
        v = value(Array(y), y_type)
        assert np.all(v[K:] == -7.25) and np.all(v[:, ~inside] == -7.25)
        with np.errstate(over="ignore"):
            exact = value(store(values(codes, scales)[:K], y_type), y_type)
        assert np.array_equal(v[:K][:, inside], exact[:, inside], equal_nan=True), f"values in {y_type}"


@pytest.mark.parametrize("elem", [F16, BFloat16, F32])
@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("K,cols", [(32, 1), (1, 1), (31, 3), (33, 5), (64, 128), (127, 129), (128, 33), (129, 300), (520, 130), (1000, 64)])
def test_quantize(handle, elem, trans, K, cols):
    run_quantize(handle, spread(np.random.default_rng(K * 1000 + cols), K, cols), elem, trans)


@pytest.mark.parametrize("elem", [F16, BFloat16, F32])
@pytest.mark.parametrize("trans", [False, True])
def test_quantize_strides(handle, elem, trans):
    x = spread(np.random.default_rng(3), 200, 140)
    for ldx_pad, ldq_pad in ((1, 0), (8, 32), (3, 64)):
        run_quantize(handle, x, elem, trans, ldx_pad=ldx_pad, ldq_pad=ldq_pad)


@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("sizes,start,tail", [([1], 0, 0), ([5, 0, 130], 0, 0), ([0, 0], 2, 3), ([128, 256, 1, 127], 3, 7), ([1] * 300, 1, 1)])
def test_quantize_groups(handle, trans, sizes, start, tail):
    off = offsets_of(sizes, start)
    run_quantize(handle, spread(np.random.default_rng(4), 160, int(off[-1]) + tail), BFloat16, trans, offsets=off)


@pytest.mark.parametrize("trans", [False, True])
def test_quantize_special_values(handle, trans):
    x = np.zeros((32 * 12, 3))
    x[0, 0] = np.nan
    x[40, 1] = np.inf
    x[41, 2] = -np.inf
    x[64:96] = 2.0 ** -149
    x[96:128] = 2.0 ** -126 * 1.5
    x[128:160] = 3.4e38
    x[160, :] = [1e-45, 1e-40, 1e-38]
    x[192:224] = -0.0
    x[224:256, 0] = np.linspace(-6, 6, 32)
    x[256, 0], x[257, 0] = 3.4e38, 2.0 ** -149
    x[288:320, 1] = 2.0 ** -125
    run_quantize(handle, x.astype(np.float32).astype(np.float64), F32, trans)


def test_quantize_bad_offsets(handle):
    for off in ([0, 5, 3], [-1, 2, 3], [0, 2, 10], [0, 2147483647, 3]):
        q, s = CuArray(np.full((16, 9), 7, np.uint8, order="F")), CuArray(np.full(mxfp4_scale_bytes(32, 9, 2), 7, np.uint8))
        x, o = CuArray(np.ones((32, 9), F32, order="F")), CuArray(np.array(off, np.int32))
        handle.mxfp4_quantize(False, 32, 9, x, 32, F32, q, 32, s, offsets=o, groups=2)
        sync(handle, _lib.STATUS_BAD_OFFSETS)
        assert np.all(Array(q) == 7) and np.all(Array(s) == 7)
        handle.mxfp4_dequantize(32, 9, q, 32, s, x, 32, F32, offsets=o, groups=2)
        sync(handle, _lib.STATUS_BAD_OFFSETS)
        assert np.all(Array(x) == 1)
        handle.gemm_mxfp4_grouped(8, 9, 32, 1.0, q, 32, 256, s, q, 32, s, 0.0, None, 8, F32, x, 32, F32, o, 2)
        sync(handle, _lib.STATUS_BAD_OFFSETS)
        assert np.all(Array(x) == 1)


def run_product(handle, M, K, sizes, *, grouped=True, d_type=BFloat16, c_type=F32, alpha=1.0, beta=0.0, start=0, tail=0, pad=0, one_a=False,
                seed=0, **options):
    r = np.random.default_rng(seed + 7 * M + K)
    off = offsets_of(sizes, start)
    N, E = int(off[-1]) + tail, len(sizes)
    ld = up(K, 32) + 4 * pad // 32 * 32
    A = [random_operand(r, K, M) for _ in range(1 if one_a else E)]
    B = random_operand(r, K, N)
    # bytes behind K and rows of scales of no group: any but a NaN scale may stand there
    a_dev = CuArray(np.concatenate([pack(c, ld, 0x77 if ld > up(K, 32) else 0).ravel("F") for c, _ in A]))
    sa = CuArray(np.concatenate([tile(s) for _, s in A]))
    b_dev = CuArray(pack(B[0], ld, 0x77))
    sb = CuArray(tile(B[1], off if grouped else None))
    Cm = store(r.standard_normal((M, N)), c_type) if beta else None
    D0 = store(np.full((M, N), -7.25), d_type)

    def taller(x):
        out = np.asfortranarray(np.concatenate([x, np.repeat(store(np.full((1, 1), -7.25), d_type if x is D0 else c_type), pad * x.shape[1]).reshape(pad, x.shape[1])]))
        return CuArray(out)

    d_dev = taller(D0)
    c_dev = taller(Cm) if beta else None
    for k in ("TILE_N", "CTA_PAIR"):
        handle.set_option(getattr(_lib, "OPT_" + k), options.get(k.lower(), 0))
    if grouped:
        handle.gemm_mxfp4_grouped(M, N, K, alpha, a_dev, ld, 0 if one_a else ld * M, sa, b_dev, ld, sb, beta, c_dev, M + pad, c_type, d_dev,
                                  M + pad, d_type, CuArray(off), E)
    else:
        handle.gemm_mxfp4(M, N, K, alpha, a_dev, ld, sa, b_dev, ld, sb, beta, c_dev, M + pad, c_type, d_dev, M + pad, d_type)
    sync(handle)
    got = value(Array(d_dev), d_type)
    assert np.all(got[M:] == -7.25), "rows between the columns of D were written"
    a64 = [values(*a)[:K] for a in A]
    exact, S = grouped_ref(a64 * E if one_a else a64, values(*B)[:K], value(Cm, c_type) if beta else None, off, alpha, beta, True, value(D0, d_type))
    outside = np.ones(N, bool)
    outside[int(off[0]):int(off[-1])] = False
    assert np.all(got[:M, outside] == -7.25), "columns of no group were written"
    close(got[:M], exact, S, K, d_type, f"M {M} K {K} sizes {sizes}")


@pytest.mark.parametrize("K", [1, 31, 32, 33, 64, 65, 96, 127, 128, 160, 224, 255, 256, 257, 384, 512, 640, 1000, 2336])
@pytest.mark.parametrize("d_type", [BFloat16, F32])
def test_any_k(handle, K, d_type):
    run_product(handle, 136, K, [72], grouped=False, d_type=d_type)
    run_product(handle, 136, K, [72, 0, 131], d_type=d_type)


@pytest.mark.parametrize("M", [1, 2, 7, 8, 63, 127, 129, 255, 257, 264, 392])
@pytest.mark.parametrize("N", [1, 2, 15, 16, 17, 33, 100, 129, 260])
def test_any_shape(handle, M, N):
    run_product(handle, M, 288, [N], grouped=False)
    run_product(handle, M, 96, [N], grouped=False, d_type=F32)


@pytest.mark.parametrize("sizes", [[1], [0, 1, 0], [5, 0, 17, 33, 0], [31, 32, 33, 1], [64, 65, 127, 3], [128, 129, 200], [256, 300, 1, 255], [0, 0], [700]],
                         ids=str)
@pytest.mark.parametrize("d_type", [BFloat16, F32])
def test_groups(handle, sizes, d_type):
    run_product(handle, 264, 416, sizes, start=3, tail=5, d_type=d_type)


@pytest.mark.parametrize("d_type", [F16, BFloat16, F32])
@pytest.mark.parametrize("c_type", [None, F16, BFloat16, F32])
def test_types(handle, d_type, c_type):
    # scales within 2^+-1: a Float16 result must not overflow
    for sizes in ([40, 3, 90], [260, 0, 41]):
        run_product(handle, 136, 96, sizes, d_type=d_type, c_type=c_type or F32, beta=0.5 if c_type else 0.0, alpha=-0.0625, tail=2)


@pytest.mark.parametrize("tile_n,cta_pair", [(64, 1), (128, 1), (128, 2), (256, 2), (256, 1)])
@pytest.mark.parametrize("d_type", [BFloat16, F32])
def test_tile_options(handle, tile_n, cta_pair, d_type):
    for sizes in ([3, 0, 70, 300, 257, 31], [192, 193, 1, 128, 64, 65]):
        run_product(handle, 392, 544, sizes, tile_n=tile_n, cta_pair=cta_pair, d_type=d_type, tail=9)
    run_product(handle, 520, 1056, [700], grouped=False, tile_n=tile_n, cta_pair=cta_pair, d_type=d_type)


def test_strides_one_matrix_and_many_groups(handle):
    run_product(handle, 136, 100, [40, 0, 93], pad=8, beta=1.0)
    run_product(handle, 136, 100, [40, 0, 93], pad=3, beta=1.0, d_type=F32)
    run_product(handle, 264, 160, [9, 0, 70, 140], one_a=True)
    r = np.random.default_rng(1)
    for groups in (256, 1024):
        run_product(handle, 40, 64, r.integers(0, 4, groups).tolist(), start=1, tail=1)


def test_a_nan_scale_is_its_row_or_column(handle):
    r = np.random.default_rng(2)
    (qa, sa), (qb, sb) = random_operand(r, 96, 40), random_operand(r, 96, 24)
    sa[1, 5], sb[2, 7] = 255, 255
    d = CuArray(np.zeros((40, 24), F32, order="F"))
    handle.gemm_mxfp4(40, 24, 96, 1.0, CuArray(pack(qa, 96)), 96, CuArray(tile(sa)), CuArray(pack(qb, 96)), 96, CuArray(tile(sb)), 0.0, None, 40, F32,
                      d, 40, F32)
    sync(handle)
    want = np.zeros((40, 24), bool)
    want[5, :] = want[:, 7] = True
    assert np.array_equal(np.isnan(Array(d)), want)


def test_a_layer_of_experts_from_16_bit_tokens(handle):
    """Weights of all experts quantised at once, tokens quantised by group, the grouped product: as a serving step
    runs them, on one stream."""
    r = np.random.default_rng(9)
    sizes, K, M = [70, 0, 33, 129, 1], 136, 72
    E, off, T = 5, offsets_of(sizes), sum(sizes)
    W, X = store(r.standard_normal((K, E * M)), BFloat16), store(r.standard_normal((K, T)), BFloat16)
    ld = up(K, 32)
    woff, xoff = CuArray((np.arange(E + 1) * M).astype(np.int32)), CuArray(off)
    qw, sw = CuArray(np.zeros((ld // 2, E * M), np.uint8, order="F")), CuArray(np.zeros(E * mxfp4_scale_bytes(K, M), np.uint8))
    qx, sx = CuArray(np.zeros((ld // 2, T), np.uint8, order="F")), CuArray(np.zeros(mxfp4_scale_bytes(K, T, E), np.uint8))
    d = CuArray(np.zeros((M, T), np.uint16, order="F"))
    handle.mxfp4_quantize(False, K, E * M, CuArray(W), K, BFloat16, qw, ld, sw, offsets=woff, groups=E)
    handle.mxfp4_quantize(False, K, T, CuArray(X), K, BFloat16, qx, ld, sx, offsets=xoff, groups=E)
    handle.gemm_mxfp4_grouped(M, T, K, 1.0, qw, ld, ld * M, sw, qx, ld, sx, 0.0, None, M, BFloat16, d, M, BFloat16, xoff, E)
    sync(handle)
    w, x = values(*quantize(value(W, BFloat16)))[:K], values(*quantize(value(X, BFloat16)))[:K]
    exact, S = grouped_ref([w[:, e * M:(e + 1) * M] for e in range(E)], x, None, off, 1.0, 0.0, True, np.zeros((M, T)))
    close(value(Array(d), BFloat16), exact, S, K, BFloat16)


@pytest.mark.parametrize("max_ctas", [1, 2, 3, 10])
@pytest.mark.parametrize("tile_n", [0, 128, 256])
def test_few_ctas_walk_many_tiles(handle, max_ctas, tile_n):
    """Every barrier goes through many phases, the ring wraps, accumulators change hands; 192-column tiles with a
    short inner dimension or a C, 256 otherwise, 32 and split sums for few columns."""
    handle.set_option(_lib.OPT_MAX_CTAS, max_ctas)
    for K in (96, 544, 1056):
        run_product(handle, 648, K, [3, 0, 70, 300, 1, 700], tile_n=tile_n)
        run_product(handle, 392, K, [700], grouped=False, tile_n=tile_n, d_type=F32, beta=1.0)
    handle.set_option(_lib.OPT_PDL, 0)
    run_product(handle, 264, 1056, [1, 0, 2, 33], tile_n=tile_n)


@pytest.mark.parametrize("d_type", [BFloat16, F32])
def test_few_columns_share_the_inner_dimension(handle, d_type):
    for sizes, M, K in (([1], 130, 8192), ([1, 0, 2], 264, 1312), ([32, 5, 40], 128, 1056), ([1] * 20, 1024, 1024), ([3] * 40, 512, 1056), ([1], 8, 768)):
        run_product(handle, M, K, sizes, d_type=d_type, beta=0.5, c_type=F32)
    for N in (1, 4, 5, 31, 32):
        run_product(handle, 264, 2080, [N], grouped=False, d_type=d_type)


def test_the_exponent_range_of_the_scales(handle):
    """Products of the smallest and the largest scales: 2^-127 * 2^127 and beyond binary32 on either side."""
    K, M, N = 64, 8, 4
    qa, qb = np.full((K, M), 2, np.uint8), np.full((K, N), 2, np.uint8)  # elements 1.0
    sa, sb = np.full((2, M), 127, np.uint8), np.full((2, N), 127, np.uint8)
    sa[:, 0], sa[:, 1], sa[:, 2] = 0, 254, 100
    sb[:, 0], sb[:, 1] = 254, 0
    d = CuArray(np.zeros((M, N), F32, order="F"))
    handle.gemm_mxfp4(M, N, K, 1.0, CuArray(pack(qa, K)), K, CuArray(tile(sa)), CuArray(pack(qb, K)), K, CuArray(tile(sb)), 0.0, None, M, F32, d, M, F32)
    sync(handle)
    got, exact = Array(d).astype(np.float64), K * np.ldexp(1.0, sa[0].astype(int) - 127)[:, None] * np.ldexp(1.0, sb[0].astype(int) - 127)[None]
    normal = (exact >= 2.0 ** -126) & (exact < 2.0 ** 128)
    assert np.array_equal(got[normal], exact[normal])
    assert np.all(np.isinf(got[exact >= 2.0 ** 128]))
    assert np.all(got[exact < 2.0 ** -126] <= 2.0 ** -120)


@pytest.mark.parametrize("band", [1, 2, 3, 5, 64])
@pytest.mark.parametrize("tile_n", [0, 128, 256])
def test_tile_rows_in_bands(handle, band, tile_n):
    """Every tile is placed once, with one band, whole bands and a last band of fewer rows."""
    handle.set_option(_lib.OPT_RASTER_GROUP, band)
    run_product(handle, 1416, 96, [70, 0, 300, 513, 1], tile_n=tile_n, tail=3)
    run_product(handle, 1416, 1056, [520], grouped=False, tile_n=tile_n, d_type=F32, beta=1.0)
