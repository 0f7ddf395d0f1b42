"""Grouped products through the C ABI (b200_gemm_grouped, b200_gemm_grouped_k) against float64."""
import numpy as np
import pytest

from cudanative_jl_b200 import _lib
from cudanative_jl_b200.array import Array, CuArray, pointer
from cudanative_jl_b200.bfloat16 import BFloat16
from grouped_cases import close, grouped_k_ref, grouped_ref, memory_type, offsets_of, store, value

pytestmark = pytest.mark.gpu

F16, F32 = np.float16, np.float32


def sync(handle, expect=0):
    _lib.check(_lib.lib().b200_stream_sync(None), "sync")
    code, block, detail = handle.device_status()
    assert code == expect, f"device status {code} (block {block}, detail {detail})"


def normal(r, shape, scale=1.0):
    return r.standard_normal(shape).astype(np.float32) * np.float32(scale)


def taller(x, ld, fill):
    """Column-major x with leading dimension ld; what is between its columns holds `fill`."""
    out = np.full((ld, x.shape[1]), fill, dtype=x.dtype, order="F")
    out[: x.shape[0]] = x
    return out


def fill_of(elem, v):
    return store(np.array([[v]]), elem)[0, 0]


def run_grouped(handle, sizes, M, K, *, transA=True, ab=BFloat16, d_type=None, c_type=F32, alpha=1.0, beta=0.0, start=0, tail=0, pad=0, one_a=False,
                alias=False, expect=None, seed=0, poison=True, shift=0, **options):
    """One call against the statement; what lies outside a group's columns of B is NaN and of D a sentinel."""
    d_type = ab if d_type is None else d_type
    r = np.random.default_rng(seed)
    off = offsets_of(sizes, start)
    N = int(off[-1]) + tail
    E = len(sizes)
    shape = (K, M) if transA else (M, K)
    A = [store(normal(r, shape, K ** -0.5 if K else 1.0), ab) for _ in range(1 if one_a else E)]
    B = store(normal(r, (K, N)), ab)
    if poison:
        B[:, :start] = fill_of(ab, np.nan)
        B[:, int(off[-1]):] = fill_of(ab, np.inf)
    Cm = store(normal(r, (M, N)), c_type) if beta else None
    sentinel = np.float32(-7.25)
    D0 = Cm.copy(order="F") if alias else store(np.full((M, N), sentinel), d_type)
    lda, ldb, ldd = max(shape[0] + pad, 1), K + pad, M + pad
    nan = fill_of(ab, np.nan)
    a_host = np.concatenate([taller(a, lda, nan).ravel("F") for a in A if a.size]) if K else np.zeros(8, memory_type(ab))
    a_dev = CuArray(np.concatenate([np.full(shift, nan, memory_type(ab)), a_host]))
    b_dev = CuArray(taller(B, max(ldb, 1), nan))
    d_dev = CuArray(taller(D0, ldd, fill_of(d_type, sentinel)))
    c_dev = d_dev if alias else CuArray(taller(Cm, ldd, fill_of(c_type, np.nan))) if beta else None
    for k in ("FORCE_KERNEL", "TILE_N", "CTA_PAIR"):
        handle.set_option(getattr(_lib, "OPT_" + k), options.get(k.lower(), 0))
    handle.gemm_grouped(transA, M, N, K, alpha, pointer(a_dev) + shift, lda, 0 if one_a else lda * shape[1], b_dev, max(ldb, 1), ab, beta, c_dev,
                        ldd, c_type, d_dev, ldd, d_type, CuArray(off), E)
    sync(handle)
    if expect is not None:
        assert handle.last_launch()["kernel"] == expect
    got = Array(d_dev)
    assert np.all(value(got[M:], d_type) == sentinel), "rows between the columns of D were written"
    a64 = [value(a, ab) for a in (A * E if one_a else A)]
    exact, S = grouped_ref(a64, value(B, ab), value(Cm, c_type) if beta else None, off, alpha, beta, transA, value(D0, d_type))
    got = value(got[:M], d_type)
    outside = np.ones(N, bool)
    outside[int(off[0]):int(off[-1])] = False
    assert np.array_equal(got[:, outside], value(D0, d_type)[:, outside]), "columns of no group were written"
    close(got, exact, S, K, d_type, f"sizes {sizes} M {M} K {K}")


SIZES = [[1], [0, 1, 0], [5, 0, 17, 33, 0], [31, 32, 33, 1], [64, 65, 127, 3], [128, 129, 200], [256, 300, 1, 255], [0, 0], [700]]


@pytest.mark.parametrize("sizes", SIZES, ids=str)
@pytest.mark.parametrize("transA", [True, False])
def test_sizes(handle, sizes, transA):
    run_grouped(handle, sizes, 264, 200, transA=transA, expect=_lib.KERNEL_TCGEN05, start=3, tail=5)


@pytest.mark.parametrize("tile_n,cta_pair", [(64, 1), (128, 1), (128, 2), (256, 2)])
@pytest.mark.parametrize("transA", [True, False])
def test_every_tile_shape(handle, tile_n, cta_pair, transA):
    run_grouped(handle, [3, 0, 70, 300, 257, 31], 392, 136, transA=transA, tile_n=tile_n, cta_pair=cta_pair, force_kernel=_lib.KERNEL_TCGEN05, tail=9)


@pytest.mark.parametrize("ab", [F16, BFloat16])
@pytest.mark.parametrize("d_type", [F16, BFloat16, F32])
@pytest.mark.parametrize("c_type", [None, F16, BFloat16, F32])
def test_types(handle, ab, d_type, c_type):
    for sizes in ([40, 3, 90], [260, 0, 41]):
        run_grouped(handle, sizes, 136, 72, ab=ab, d_type=d_type, c_type=c_type or F32, beta=0.5 if c_type else 0.0, alpha=-1.5, tail=2)


@pytest.mark.parametrize("M", [1, 2, 7, 8, 63, 127, 129, 255, 257, 260])
@pytest.mark.parametrize("d_type", [BFloat16, F32])
def test_any_number_of_rows(handle, M, d_type):
    """A stored row by row: M has no alignment rule at all; bulk stores need whole 16-byte chunks, other rows
    are stored one by one."""
    run_grouped(handle, [50, 140, 0, 9], M, 64, d_type=d_type, expect=_lib.KERNEL_TCGEN05)


@pytest.mark.parametrize("K", [0, 1, 8, 15, 16, 24, 63, 64, 65, 128, 513])
@pytest.mark.parametrize("transA", [True, False])
def test_any_k(handle, K, transA):
    run_grouped(handle, [20, 130], 72, K, transA=transA, beta=1.0, c_type=F32)


@pytest.mark.parametrize("transA", [True, False])
def test_unaligned_runs_on_the_simple_kernel(handle, transA):
    run_grouped(handle, [9, 0, 70, 1], 70, 33, transA=transA, pad=1, expect=_lib.KERNEL_SIMPLE, beta=0.25, tail=3, start=2)
    run_grouped(handle, [9, 0, 70, 1], 72, 40, transA=transA, shift=1, expect=_lib.KERNEL_SIMPLE, tail=3, start=2)
    run_grouped(handle, [9, 0, 70, 1], 72, 40, transA=transA, force_kernel=_lib.KERNEL_SIMPLE, expect=_lib.KERNEL_SIMPLE)


def test_one_matrix_for_all_groups_and_in_place(handle):
    run_grouped(handle, [9, 0, 70, 140], 264, 136, one_a=True)
    run_grouped(handle, [9, 0, 70, 140], 264, 136, beta=1.0, c_type=F32, d_type=F32, alias=True, tail=4)
    run_grouped(handle, [9, 0, 70, 140], 264, 136, beta=1.0, c_type=BFloat16, d_type=BFloat16, alias=True, pad=8)


@pytest.mark.parametrize("groups", [255, 256, 257, 1000, 1024])
def test_many_groups(handle, groups):
    r = np.random.default_rng(groups)
    sizes = r.integers(0, 4, groups).tolist()
    run_grouped(handle, sizes, 72, 64, start=1, tail=1)
    run_grouped(handle, [0] * (groups - 1) + [2], 72, 64)
    run_grouped(handle, [2] + [0] * (groups - 1), 72, 64)
    run_grouped(handle, sizes, 70, 33, force_kernel=_lib.KERNEL_SIMPLE)


def test_a_neighbours_nan_stays_its_own(handle):
    """The tile of one group reads columns of the next one: what they hold changes nothing."""
    r = np.random.default_rng(5)
    sizes, M, K = [5, 40, 3], 136, 72
    off = offsets_of(sizes)
    A, X = CuArray(store(normal(r, (K, 3 * M)), F16)), normal(r, (K, 48))
    out = []
    for bad in (None, np.nan, np.inf):
        Y = X.copy()
        if bad is not None:
            Y[:, 5:45] = bad
        d = CuArray(np.zeros((M, 48), np.float32, order="F"))
        handle.gemm_grouped(True, M, 48, K, 1.0, A, K, K * M, CuArray(store(Y, F16)), K, F16, 0.0, None, M, F32, d, M, F32, CuArray(off), 3)
        sync(handle)
        out.append(Array(d))
    for o in out[1:]:
        assert np.array_equal(o[:, :5], out[0][:, :5]) and np.array_equal(o[:, 45:], out[0][:, 45:])
        assert not np.any(np.isfinite(o[:, 5:45]))


BAD = [[0, 5, 3, 9], [-1, 2, 3, 9], [0, 2, 3, 10], [0, 100, 3, 9], [5, 5, 5, 4], [0, 0, -2147483648, 9], [0, 2147483647, 3, 9]]


@pytest.mark.parametrize("off", BAD, ids=str)
@pytest.mark.parametrize("kernel", [_lib.KERNEL_TCGEN05, _lib.KERNEL_SIMPLE])
def test_bad_offsets_write_nothing_and_are_reported(handle, off, kernel):
    """The kernel checks the offsets before it forms an address with one."""
    handle.set_option(_lib.OPT_FORCE_KERNEL, kernel)
    a, b, o = CuArray(np.ones((64, 192), F16, order="F")), CuArray(np.ones((64, 9), F16, order="F")), CuArray(np.array(off, np.int32))
    d = CuArray(np.full((64, 9), 3.5, F32, order="F"))
    handle.gemm_grouped(True, 64, 9, 64, 1.0, a, 64, 4096, b, 64, F16, 0.0, None, 64, F32, d, 64, F32, o, 3)
    sync(handle, _lib.STATUS_BAD_OFFSETS)
    assert np.all(Array(d) == 3.5)
    d = CuArray(np.full((64, 192), 3.5, F32, order="F"))
    handle.gemm_grouped_k(64, 64, 9, 1.0, b, 64, b, 64, F16, 0.0, None, 64, 4096, F32, d, 64, 4096, F32, o, 3)
    sync(handle, _lib.STATUS_BAD_OFFSETS)
    assert np.all(Array(d) == 3.5)


def run_grouped_k(handle, sizes, M, N, *, ab=BFloat16, d_type=F32, c_type=F32, alpha=1.0, beta=0.0, start=0, tail=0, pad=0, gap=0, alias=False,
                  expect=None, seed=0, **options):
    r = np.random.default_rng(seed)
    off = offsets_of(sizes, start)
    K, E = int(off[-1]) + tail, len(sizes)
    A, B = store(normal(r, (M, K)), ab), store(normal(r, (N, K)), ab)
    for x in (A, B):  # infinities times zeros would show as NaN
        x[:, :start] = fill_of(ab, np.nan)
        x[:, int(off[-1]):] = fill_of(ab, np.inf)
    C = [store(normal(r, (M, N)), c_type) for _ in range(E)]
    ldab, ldd = pad, M + pad
    nan, sentinel = fill_of(ab, np.nan), np.float32(-7.25)
    stride = ldd * N + gap

    def pack(mats, elem, fill):
        out = np.full(stride * len(mats), fill_of(elem, fill), memory_type(elem))
        for e, m in enumerate(mats):
            out[e * stride: e * stride + ldd * N].reshape(ldd, N, order="F")[:M] = m
        return out

    d_host = pack(C, c_type, sentinel) if alias else pack([store(np.full((M, N), sentinel), d_type)] * E, d_type, sentinel)
    d_dev = CuArray(d_host)
    c_dev = d_dev if alias else CuArray(pack(C, c_type, np.nan)) if beta else None
    for k in ("FORCE_KERNEL", "TILE_N", "CTA_PAIR"):
        handle.set_option(getattr(_lib, "OPT_" + k), options.get(k.lower(), 0))
    a_dev, b_dev = CuArray(taller(A, M + ldab, nan)), CuArray(taller(B, N + ldab, nan))
    handle.gemm_grouped_k(M, N, K, alpha, a_dev, M + ldab, b_dev, N + ldab, ab, beta, c_dev, ldd, stride, c_type, d_dev, ldd, stride, d_type,
                          CuArray(off), E)
    sync(handle)
    if expect is not None:
        assert handle.last_launch()["kernel"] == expect
    got = Array(d_dev)
    exact, S = grouped_k_ref(value(A, ab), value(B, ab), [value(c, c_type) for c in C], off, alpha, beta)
    for e in range(E):
        mat = got[e * stride: e * stride + ldd * N].reshape(ldd, N, order="F")
        close(value(mat[:M], d_type), exact[e], S[e], sizes[e], d_type, f"group {e} of {sizes}")
        assert np.all(value(mat[M:], d_type) == sentinel), "rows between the columns were written"
        assert np.all(value(got[e * stride + ldd * N:(e + 1) * stride], d_type) == sentinel), "gap between the matrices was written"


SIZES_K = [[1], [0, 1, 0], [15, 16, 17, 0, 31], [63, 64, 65], [48, 80, 112, 128], [1, 2, 3, 4, 5, 6, 7, 8, 9], [200, 0, 333], [0, 0, 0], [1000]]


@pytest.mark.parametrize("sizes", SIZES_K, ids=str)
@pytest.mark.parametrize("beta", [0.0, 1.0])
def test_k_sizes(handle, sizes, beta):
    run_grouped_k(handle, sizes, 264, 200, beta=beta, start=3, tail=5, expect=_lib.KERNEL_TCGEN05)


@pytest.mark.parametrize("tile_n,cta_pair", [(64, 1), (128, 1), (128, 2), (256, 2)])
@pytest.mark.parametrize("beta", [0.0, 0.5])
def test_k_every_tile_shape(handle, tile_n, cta_pair, beta):
    run_grouped_k(handle, [3, 0, 70, 300, 257, 31, 16], 392, 320, tile_n=tile_n, cta_pair=cta_pair, beta=beta, alpha=2.0,
                  force_kernel=_lib.KERNEL_TCGEN05, tail=9)


@pytest.mark.parametrize("ab", [F16, BFloat16])
@pytest.mark.parametrize("d_type", [F16, BFloat16, F32])
@pytest.mark.parametrize("c_type", [None, F16, BFloat16, F32])
def test_k_types(handle, ab, d_type, c_type):
    run_grouped_k(handle, [40, 0, 93], 136, 264, ab=ab, d_type=d_type, c_type=c_type or F32, beta=0.5 if c_type else 0.0, alpha=-1.5)


@pytest.mark.parametrize("M,N", [(1, 1), (7, 9), (8, 264), (250, 40), (136, 1), (257, 300), (128, 96)])
@pytest.mark.parametrize("beta", [0.0, 1.0])
def test_k_any_shape(handle, M, N, beta):
    run_grouped_k(handle, [40, 0, 93], M, N, beta=beta)
    run_grouped_k(handle, [40, 0, 93], M, N, beta=beta, d_type=BFloat16, c_type=F32, gap=8)


def test_k_gaps_and_in_place(handle):
    run_grouped_k(handle, [40, 0, 93], 136, 72, pad=8, gap=24, beta=1.0)
    run_grouped_k(handle, [40, 0, 93], 136, 72, pad=3, gap=1, beta=1.0, expect=_lib.KERNEL_SIMPLE)
    run_grouped_k(handle, [40, 0, 93], 136, 72, gap=1, beta=1.0, expect=_lib.KERNEL_TCGEN05)
    run_grouped_k(handle, [40, 0, 93], 264, 200, beta=1.0, alias=True)
    run_grouped_k(handle, [40, 0, 93], 136, 72, force_kernel=_lib.KERNEL_SIMPLE, beta=0.5, start=2, tail=1)


@pytest.mark.parametrize("groups", [256, 1024])
def test_k_many_groups(handle, groups):
    sizes = np.random.default_rng(groups).integers(0, 20, groups).tolist()
    run_grouped_k(handle, sizes, 40, 24, start=1, tail=1, beta=1.0)
    run_grouped_k(handle, sizes, 264, 136)


def test_k_a_neighbours_nan_stays_its_own(handle):
    r = np.random.default_rng(5)
    off = offsets_of([5, 40, 19])
    X, Y = normal(r, (136, 64)), normal(r, (72, 64))
    out = []
    for bad in (None, np.nan, np.inf):
        x, y = X.copy(), Y.copy()
        if bad is not None:
            x[:, 5:45] = y[:, 5:45] = bad
        d = CuArray(np.zeros((136, 216), np.float32, order="F"))
        handle.gemm_grouped_k(136, 72, 64, 1.0, CuArray(store(x, F16)), 136, CuArray(store(y, F16)), 72, F16, 0.0, None, 136, 136 * 72, F32, d, 136,
                              136 * 72, F32, CuArray(off), 3)
        sync(handle)
        out.append(Array(d))
    for o in out[1:]:
        assert np.array_equal(o[:, :72], out[0][:, :72]) and np.array_equal(o[:, 144:], out[0][:, 144:])
        assert not np.any(np.isfinite(o[:, 72:144]))


def test_a_layer_forward_and_backward(handle):
    """One layer of experts as a training step runs it: forward, input gradient, weight gradient added to what
    is there, all on one stream without a word to the host in between."""
    r = np.random.default_rng(9)
    sizes, K, M = [70, 0, 33, 129], 136, 264
    off, T = offsets_of(sizes), sum(sizes)
    W, X, G = store(normal(r, (K, 4 * M), K ** -0.5), BFloat16), store(normal(r, (K, T)), BFloat16), store(normal(r, (M, T)), BFloat16)
    acc = normal(r, (K, 4 * M))
    Wd, Xd, Gd, od = CuArray(W), CuArray(X), CuArray(G), CuArray(off)
    Y, dX, dW = CuArray(np.zeros((M, T), np.uint16, order="F")), CuArray(np.zeros((K, T), np.uint16, order="F")), CuArray(np.asfortranarray(acc))
    handle.gemm_grouped(True, M, T, K, 1.0, Wd, K, K * M, Xd, K, BFloat16, 0.0, None, M, BFloat16, Y, M, BFloat16, od, 4)
    handle.gemm_grouped(False, K, T, M, 1.0, Wd, K, K * M, Gd, M, BFloat16, 0.0, None, K, BFloat16, dX, K, BFloat16, od, 4)
    handle.gemm_grouped_k(K, M, T, 1.0, Xd, K, Gd, M, BFloat16, 1.0, dW, K, K * M, F32, dW, K, K * M, F32, od, 4)
    sync(handle)
    w = [value(W[:, e * M:(e + 1) * M], BFloat16) for e in range(4)]
    x, g = value(X, BFloat16), value(G, BFloat16)
    close(value(Array(Y), BFloat16), *grouped_ref(w, x, None, off, 1.0, 0.0, True, np.zeros((M, T))), K, BFloat16, "forward")
    close(value(Array(dX), BFloat16), *grouped_ref(w, g, None, off, 1.0, 0.0, False, np.zeros((K, T))), M, BFloat16, "input gradient")
    exact, S = grouped_k_ref(x, g, [acc[:, e * M:(e + 1) * M].astype(np.float64) for e in range(4)], off, 1.0, 1.0)
    close(value(Array(dW), F32), np.hstack(exact), np.hstack(S), max(sizes), F32, "weight gradient")


@pytest.mark.parametrize("max_ctas", [1, 2, 3, 10])
@pytest.mark.parametrize("tile_n,cta_pair", [(0, 0), (64, 1), (128, 1), (128, 2), (256, 2)])
def test_few_ctas_walk_many_tiles(handle, max_ctas, tile_n, cta_pair):
    """Every barrier goes through many phases, the ring wraps, accumulators change hands."""
    handle.set_option(_lib.OPT_MAX_CTAS, max_ctas)
    for d_type in (BFloat16, F32):
        run_grouped(handle, [3, 0, 70, 300, 1, 31], 648, 264, d_type=d_type, tile_n=tile_n, cta_pair=cta_pair)
        run_grouped_k(handle, [3, 0, 70, 300, 1, 31, 129], 392, 328, d_type=d_type, beta=1.0, tile_n=tile_n, cta_pair=cta_pair)
    handle.set_option(_lib.OPT_PDL, 0)
    run_grouped(handle, [1, 0, 2, 7], 648, 1032, tile_n=tile_n, cta_pair=cta_pair)
    run_grouped_k(handle, [5, 77], 264, 72, tile_n=tile_n, cta_pair=cta_pair)


@pytest.mark.parametrize("d_type", [F16, BFloat16, F32])
@pytest.mark.parametrize("transA", [True, False])
def test_few_columns_share_the_inner_dimension(handle, d_type, transA):
    """32-column tiles: two CTAs take half of K each when that evens out the work, one or several tiles a pair."""
    for sizes, M, K in (([1], 130, 2048), ([1, 0, 2], 264, 1304), ([32, 5], 128, 264), ([1] * 20, 1024, 520), ([3] * 40, 512, 1032), ([1], 8, 192)):
        run_grouped(handle, sizes, M, K, transA=transA, d_type=d_type, beta=0.5, c_type=F32)


def test_long_sums_of_one_sign_keep_binary32(handle):
    """A binary32 D sums several accumulators of 512 products, so that the tensor core's truncation does not grow
    with K.  One instruction adds 16 products to the accumulator; what it drops is less than two units in the
    last place of the sum so far: 32 instructions, 2 * 32 * 2^-23 of the sum of magnitudes, and 2^-24 for each of the
    K / 512 additions.  One accumulator for K = 16384 is 1e-4 off on these values."""
    r = np.random.default_rng(3)
    K, M, N = 16384, 136, 136
    A, B = store(np.abs(normal(r, (M, K), 2.0 ** -7)), F16), store(np.abs(normal(r, (N, K))), F16)
    d = CuArray(np.zeros((M, N), F32, order="F"))
    handle.gemm_grouped_k(M, N, K, 1.0, CuArray(A), M, CuArray(B), N, F16, 0.0, None, M, M * N, F32, d, M, M * N, F32, CuArray(offsets_of([K])), 1)
    sync(handle)
    exact = value(A, F16) @ value(B, F16).T
    assert np.all(np.abs(Array(d) - exact) <= (2 * 32 * 2.0 ** -23 + K / 512 * 2.0 ** -24) * exact)
    At, d2 = CuArray(np.asfortranarray(A.T)), CuArray(np.zeros((M, N), F32, order="F"))
    handle.gemm_grouped(True, M, N, K, 1.0, At, K, M * K, CuArray(np.asfortranarray(B.T)), K, F16, 0.0, None, M, F32, d2, M, F32,
                        CuArray(offsets_of([N])), 1)
    sync(handle)
    assert np.all(np.abs(Array(d2) - exact) <= (2 * 32 * 2.0 ** -23 + K / 512 * 2.0 ** -24) * exact)


def test_same_call_twice_is_bitwise_the_same(handle):
    r = np.random.default_rng(4)
    off = CuArray(offsets_of([1, 0, 2, 7, 30]))
    W, X = CuArray(store(normal(r, (1032, 5 * 264)), BFloat16)), CuArray(store(normal(r, (1032, 40)), BFloat16))
    got = []
    for _ in range(4):
        d = CuArray(np.zeros((264, 40), F32, order="F"))
        handle.gemm_grouped(True, 264, 40, 1032, 1.0, W, 1032, 1032 * 264, X, 1032, BFloat16, 0.0, None, 264, F32, d, 264, F32, off, 5)
        sync(handle)
        got.append(Array(d))
    assert all(np.array_equal(g, got[0]) for g in got)


def test_check_on_call_names_the_offsets(handle):
    from cudanative_jl_b200 import B200Error

    handle.set_option(_lib.OPT_CHECK_ON_CALL, 1)
    a, d = CuArray(np.ones((64, 64), F16, order="F")), CuArray(np.zeros((64, 9), F32, order="F"))

    def call(off):
        handle.gemm_grouped(True, 64, 9, 64, 1.0, a, 64, 0, a, 64, F16, 0.0, None, 64, F32, d, 64, F32, CuArray(np.array(off, np.int32)), 2)
        _lib.check(_lib.lib().b200_stream_sync(None), "sync")

    call([0, 7, 3])
    with pytest.raises(B200Error, match="group offsets") as e:
        call([0, 3, 9])
    assert e.value.status == _lib.INVALID_ARG
    call([0, 3, 9])
    assert np.all(Array(d) == 64.0)


def test_streams_and_replayed_graphs():
    """Sizes are read when the kernel runs: a captured layer follows new offsets and inputs.  Two captured layers on
    one handle, replayed at once on two streams, share nothing."""
    torch = pytest.importorskip("torch")
    from cudanative_jl_b200.gemm import Handle, mxfp4_scale_bytes

    torch.cuda.set_device(0)
    E, M, K, T = 4, 264, 256, 300
    with Handle(0) as h:
        gen = torch.Generator(device="cuda").manual_seed(1)
        rand = lambda *s: torch.randn(s, generator=gen, device="cuda").bfloat16()  # noqa: E731

        class Layer:
            def __init__(self):
                self.w, self.x, self.g = rand(E, M, K), rand(T, K), rand(T, M)
                self.off = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
                self.y, self.dx = torch.zeros(T, M, device="cuda"), torch.zeros(T, K, device="cuda")
                self.dw, self.y4 = torch.zeros(E, M, K, device="cuda"), torch.zeros(T, M, device="cuda")
                u8 = lambda n: torch.zeros(n, dtype=torch.uint8, device="cuda")  # noqa: E731
                self.qw, self.sw = u8(E * M * K // 2), u8(E * mxfp4_scale_bytes(K, M))
                self.qx, self.sx = u8(T * K // 2), u8(mxfp4_scale_bytes(K, T, E))
                self.woff = (torch.arange(E + 1, device="cuda") * M).int()

            def run(self):
                s = torch.cuda.current_stream().cuda_stream
                p = lambda t: t.data_ptr()  # noqa: E731
                h.gemm_grouped(True, M, T, K, 1.0, p(self.w), K, M * K, p(self.x), K, BFloat16, 0.0, None, M, F32, p(self.y), M, F32, p(self.off), E, stream=s)
                h.gemm_grouped(False, K, T, M, 1.0, p(self.w), K, M * K, p(self.g), M, BFloat16, 0.0, None, K, F32, p(self.dx), K, F32, p(self.off), E,
                               stream=s)
                h.gemm_grouped_k(K, M, T, 1.0, p(self.x), K, p(self.g), M, BFloat16, 0.0, None, K, K * M, F32, p(self.dw), K, K * M, F32, p(self.off),
                                 E, stream=s)
                h.mxfp4_quantize(False, K, E * M, p(self.w), K, BFloat16, p(self.qw), K, p(self.sw), offsets=p(self.woff), groups=E, stream=s)
                h.mxfp4_quantize(False, K, T, p(self.x), K, BFloat16, p(self.qx), K, p(self.sx), offsets=p(self.off), groups=E, stream=s)
                h.gemm_mxfp4_grouped(M, T, K, 1.0, p(self.qw), K, M * K, p(self.sw), p(self.qx), K, p(self.sx), 0.0, None, M, F32, p(self.y4), M, F32,
                                     p(self.off), E, stream=s)

            def check(self):
                from mxfp4_cases import quantize, values

                o = self.off.tolist()
                w, x, g = (t.double().cpu().numpy() for t in (self.w, self.x, self.g))
                for e in range(E):
                    s = slice(o[e], o[e + 1])
                    for got, a, b, k in ((self.y, x[s], w[e].T, K), (self.dx, g[s], w[e], M)):
                        close(got[s].double().cpu().numpy(), a @ b, np.abs(a) @ np.abs(b), k, F32)
                    close(self.dw[e].double().cpu().numpy(), g[s].T @ x[s], np.abs(g[s]).T @ np.abs(x[s]), max(1, o[e + 1] - o[e]), F32)
                    a, b = values(*quantize(x[s].T)).T if o[e + 1] > o[e] else np.zeros((0, K)), values(*quantize(w[e].T))
                    close(self.y4[s].double().cpu().numpy(), a @ b, np.abs(a) @ np.abs(b), K, F32)

        layers = [Layer(), Layer()]
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        graphs = []
        for layer, stream in zip(layers, streams):
            layer.off.copy_(torch.tensor([0, 10, 10, 200, 300], dtype=torch.int32))
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                layer.run()  # eagerly, on a stream of its own
            torch.cuda.synchronize()
            layer.check()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                layer.run()
            graphs.append(graph)
        for sizes in ([0, 0, 1, 2, 3], [0, 300, 300, 300, 300], [0, 75, 150, 225, 299]):
            for layer, shift in zip(layers, (0, 1)):
                layer.off.copy_(torch.tensor([min(v + shift, T) if v else 0 for v in sizes], dtype=torch.int32))
                layer.x.copy_(rand(T, K))
            torch.cuda.synchronize()
            for _ in range(3):
                for graph, stream in zip(graphs, streams):
                    with torch.cuda.stream(stream):
                        graph.replay()
            torch.cuda.synchronize()
            for layer in layers:
                layer.check()
        assert h.device_status()[0] == 0


@pytest.mark.parametrize("d_type", [F16, BFloat16, F32])
def test_results_on_any_element_border(handle, d_type):
    """D and C begin one element behind a 16-byte border, their leading dimension is odd: still the tcgen05 kernel."""
    r = np.random.default_rng(8)
    M, K, N, ldd = 264, 136, 70, 267
    off = offsets_of([5, 0, 40, 25])
    A, B, Cm = store(normal(r, (K, 4 * M)), BFloat16), store(normal(r, (K, N)), BFloat16), store(normal(r, (M, N)), d_type)
    sentinel = fill_of(d_type, -7.25)

    def behind(x):
        return CuArray(np.concatenate([[sentinel], taller(x, ldd, sentinel).ravel("F")]))

    c, d, da, ba = behind(Cm), behind(np.full((M, N), sentinel)), CuArray(A), CuArray(B)
    handle.gemm_grouped(True, M, N, K, 1.0, da, K, K * M, ba, K, BFloat16, 1.0, pointer(c) + 1, ldd, d_type, pointer(d) + 1, ldd, d_type, CuArray(off), 4)
    sync(handle)
    assert handle.last_launch()["kernel"] == _lib.KERNEL_TCGEN05
    raw = value(Array(d), d_type)
    got = raw[1:].reshape(ldd, N, order="F")
    assert raw[0] == -7.25 and np.all(got[M:] == -7.25)
    a64 = [value(A[:, e * M:(e + 1) * M], BFloat16) for e in range(4)]
    close(got[:M], *grouped_ref(a64, value(B, BFloat16), value(Cm, d_type), off, 1.0, 1.0, True, np.zeros((M, N))), K, d_type)
    # the other ragged dimension: matrices an odd number of elements apart
    X, Y = store(normal(r, (M, 70)), BFloat16), store(normal(r, (40, 70)), BFloat16)
    d2 = CuArray(np.full(1 + 4 * (ldd * 40 + 1), sentinel))
    handle.gemm_grouped_k(M, 40, 70, 1.0, CuArray(X), M, CuArray(Y), 40, BFloat16, 0.0, None, M, 0, F32, pointer(d2) + 1, ldd, ldd * 40 + 1, d_type,
                          CuArray(off), 4)
    sync(handle)
    assert handle.last_launch()["kernel"] == _lib.KERNEL_TCGEN05
    raw = value(Array(d2), d_type)
    exact, S = grouped_k_ref(value(X, BFloat16), value(Y, BFloat16), None, off, 1.0, 0.0)
    for e in range(4):
        at = 1 + e * (ldd * 40 + 1)
        got = raw[at:at + ldd * 40].reshape(ldd, 40, order="F")
        close(got[:M], exact[e], S[e], 40, d_type)
        assert np.all(got[M:] == -7.25) and raw[at - 1] == -7.25


def test_first_call_of_a_process_inside_a_capture():
    """Kernels are loaded and opted in to their shared memory by whichever call comes first, a captured one too."""
    pytest.importorskip("torch")
    import subprocess
    import sys
    from pathlib import Path

    root = Path(__file__).resolve().parent.parent
    code = """
import torch, numpy as np, __graft_entry__ as e
e.load_package()
from cudanative_jl_b200.gemm import Handle, mxfp4_scale_bytes
from cudanative_jl_b200.bfloat16 import BFloat16
h = Handle(0)
x, w = torch.randn(64, 256, device="cuda").bfloat16(), torch.randn(2, 136, 256, device="cuda").bfloat16()
off = torch.tensor([0, 20, 64], dtype=torch.int32, device="cuda")
y, dw = torch.zeros(64, 136, device="cuda"), torch.zeros(2, 136, 256, device="cuda")
q, s = torch.zeros(64, 128, dtype=torch.uint8, device="cuda"), torch.zeros(mxfp4_scale_bytes(256, 64), dtype=torch.uint8, device="cuda")
z, v = torch.zeros(64, 64, device="cuda"), torch.zeros(64, 256, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    st = torch.cuda.current_stream().cuda_stream
    h.gemm_grouped(True, 136, 64, 256, 1.0, w, 256, 136 * 256, x, 256, BFloat16, 0.0, None, 136, np.float32, y, 136, np.float32, off, 2, stream=st)
    h.gemm_grouped_k(256, 136, 64, 1.0, x, 256, y.bfloat16(), 136, BFloat16, 0.0, None, 256, 0, np.float32, dw, 256, 136 * 256, np.float32, off, 2, stream=st)
    h.mxfp4_quantize(False, 256, 64, x, 256, BFloat16, q, 256, s, stream=st)
    h.mxfp4_dequantize(256, 64, q, 256, s, v, 256, np.float32, stream=st)
    h.gemm_mxfp4(64, 64, 256, 1.0, q, 256, s, q, 256, s, 0.0, None, 64, np.float32, z, 64, np.float32, stream=st)
g.replay()
torch.cuda.synchronize()
ref = torch.cat([x[:20].double() @ w[0].double().T, x[20:].double() @ w[1].double().T])
assert (y.double() - ref).norm() < 1e-5 * ref.norm()
yb = y.bfloat16().double()
ref = torch.stack([yb[:20].T @ x[:20].double(), yb[20:].T @ x[20:].double()])
assert (dw.double() - ref).norm() < 1e-5 * ref.norm()
assert torch.equal(z.double(), v.double() @ v.double().T) or (z.double() - v.double() @ v.double().T).norm() < 1e-5 * z.norm()
assert h.device_status()[0] == 0
print("captured first")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured first" in r.stdout, r.stdout + r.stderr


@pytest.mark.parametrize("d_type", [F16, BFloat16, F32])
@pytest.mark.parametrize("beta", [0.0, 1.0])
def test_k_long_groups_share_the_inner_dimension(handle, d_type, beta):
    """Few tiles and long groups: four CTAs take a share of a tile's columns of A and B each; shares that are ragged,
    short or empty, edges in M and N, two rounds of tiles."""
    for sizes, M, N, shared in (([4099], 72, 40, True), ([2048], 136, 72, True), ([9000, 0, 15, 7000], 64, 136, True), ([4096, 4100], 256, 512, True),
                                ([5000, 1, 64, 448], 136, 200, False), ([8000, 1, 64, 448], 136, 200, True), ([3001] * 18, 64, 64, True),
                                ([8200] * 4, 264, 264, True), ([9000, 0, 15, 7000], 64, 130, False), ([5000, 1, 64, 448], 130, 200, False)):
        run_grouped_k(handle, sizes, M, N, d_type=d_type, c_type=d_type if d_type is not F16 else F32, beta=beta, start=2, tail=3)
        assert (handle.last_launch()["split_k"] == 4) == shared
    run_grouped_k(handle, [4099], 71, 33, d_type=d_type, pad=1, beta=beta, expect=_lib.KERNEL_SIMPLE)


@pytest.mark.parametrize("d_type", [F16, BFloat16, F32])
@pytest.mark.parametrize("transA", [True, False])
def test_few_tiles_share_the_inner_dimension(handle, d_type, transA):
    for sizes, M, K in (([70], 72, 2048), ([64, 0, 65, 3, 190], 136, 2056), ([33], 264, 4104), ([400], 520, 8200), ([100, 100], 8, 2311 * 8)):
        run_grouped(handle, sizes, M, K, transA=transA, d_type=d_type, beta=0.5, c_type=F32, start=1, tail=2)
        assert handle.last_launch()["split_k"] == 4
    run_grouped(handle, [70], 71, 2056, d_type=d_type, expect=_lib.KERNEL_TCGEN05)


@pytest.mark.parametrize("band", [1, 2, 3, 5, 64])
@pytest.mark.parametrize("tile_n,cta_pair", [(64, 1), (128, 1), (256, 2)])
def test_tile_rows_in_bands(handle, band, tile_n, cta_pair):
    """Every tile is placed once, with one band, whole bands and a last band of fewer rows."""
    handle.set_option(_lib.OPT_RASTER_GROUP, band)
    run_grouped(handle, [70, 0, 300, 513, 1], 1416, 72, tile_n=tile_n, cta_pair=cta_pair, tail=3)
    run_grouped_k(handle, [70, 0, 33], 1416, 328, tile_n=tile_n, cta_pair=cta_pair)
    handle.set_option(_lib.OPT_MAX_CTAS, 6)
    run_grouped(handle, [70, 0, 300, 513, 1], 1416, 72, tile_n=tile_n, cta_pair=cta_pair, tail=3)


def test_shared_sums_of_poisoned_neighbours_repeat_bitwise(handle):
    """Four CTAs to a tile: a group whose operands are NaN keeps them to itself, and the same call gives the same bits."""
    r = np.random.default_rng(5)
    sizes, M, N = [5003, 64, 0, 4090], 72, 136
    off = offsets_of(sizes, 0)
    K, E = int(off[-1]), len(sizes)
    A, B = store(normal(r, (M, K)), BFloat16), store(normal(r, (N, K)), BFloat16)
    for x in (A, B):
        x[:, off[1]:off[2]] = fill_of(BFloat16, np.nan)
    a_dev, b_dev, o_dev = CuArray(np.asfortranarray(A)), CuArray(np.asfortranarray(B)), CuArray(off)
    got = []
    for _ in range(3):
        d_dev = CuArray(np.full(M * N * E, 7.0, np.float32))
        handle.gemm_grouped_k(M, N, K, 1.0, a_dev, M, b_dev, N, BFloat16, 0.0, None, M, M * N, F32, d_dev, M, M * N, F32, o_dev, E)
        sync(handle)
        assert handle.last_launch()["split_k"] == 4
        got.append(Array(d_dev).reshape(E, N, M).transpose(0, 2, 1))
    assert got[0].tobytes() == got[1].tobytes() == got[2].tobytes()
    assert np.isnan(got[0][1]).all() and not got[0][2].any()
    a, b = value(A, BFloat16), value(B, BFloat16)
    for e in (0, 3):
        s = slice(off[e], off[e + 1])
        close(got[0][e], a[:, s] @ b[:, s].T, np.abs(a[:, s]) @ np.abs(b[:, s]).T, sizes[e], F32, f"group {e}")


def test_shared_sums_stay_within_one_round_of_clusters(handle):
    """A device holds fewer clusters of four than a quarter of its SMs: tiles beyond those would run a round later."""
    run_grouped_k(handle, [2100], 128, 64 * 30)
    assert handle.last_launch()["split_k"] == 4
    for cols in (35, 37, 72):
        run_grouped_k(handle, [2100], 128, 64 * cols)
        launch = handle.last_launch()
        assert launch["split_k"] == 1 or launch["ctas"] >= 4 * cols
    run_grouped_k(handle, [8200], 128, 64 * 60)
    launch = handle.last_launch()
    assert launch["split_k"] == 1 or launch["ctas"] * 2 >= 4 * 60


@pytest.mark.parametrize("d_type", [BFloat16, F32])
def test_shared_sums_in_two_and_three_rounds(handle, d_type):
    """The buffers that the four CTAs send to are used again for the next tile."""
    for K, tiles in ((4100, 50), (8200, 90)):
        run_grouped_k(handle, [K], 128, 64 * tiles, d_type=d_type, beta=1.0)
        launch = handle.last_launch()
        assert launch["split_k"] == 4 or launch["ctas"] * 3 < 4 * tiles
        run_grouped(handle, [64 * tiles - 64], 128, K + 4, d_type=d_type)
        run_grouped_k(handle, [K // 2, K // 2 + K % 2 + 1, K, K - 3], 128, 16 * tiles // 64 * 64, d_type=d_type)


def test_shared_sums_first_called_inside_a_capture():
    """The device is asked for its clusters by the first call that may share K, a captured one too; two captured calls
    replayed at once on two streams share nothing."""
    pytest.importorskip("torch")
    import subprocess
    import sys
    from pathlib import Path

    root = Path(__file__).resolve().parent.parent
    code = """
import torch, numpy as np, __graft_entry__ as e
e.load_package()
from cudanative_jl_b200.gemm import Handle
from cudanative_jl_b200.bfloat16 import BFloat16
h = Handle(0)
T, M, N = 5000, 136, 264
off = torch.tensor([0, 1703, 5000], dtype=torch.int32, device="cuda")
xs, ys = [torch.randn(T, M, device="cuda").bfloat16() for _ in range(2)], [torch.randn(T, N, device="cuda").bfloat16() for _ in range(2)]
ds, gs, streams = [torch.zeros(2, N, M, device="cuda") for _ in range(2)], [], [torch.cuda.Stream() for _ in range(2)]
torch.cuda.synchronize()
for x, y, d, s in zip(xs, ys, ds, streams):
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        for _ in range(3):
            h.gemm_grouped_k(M, N, T, 1.0, x, M, y, N, BFloat16, 0.0, None, M, 0, np.float32, d, M, M * N, np.float32, off, 2,
                             stream=torch.cuda.current_stream().cuda_stream)
    assert h.last_launch()["split_k"] == 4
    gs.append(g)
for _ in range(5):
    for g, s in zip(gs, streams):
        with torch.cuda.stream(s):
            g.replay()
torch.cuda.synchronize()
for x, y, d in zip(xs, ys, ds):
    x, y = x.double(), y.double()
    ref = torch.stack([y[:1703].T @ x[:1703], y[1703:].T @ x[1703:]])
    assert (d.double() - ref).norm() < 1e-5 * ref.norm()
assert h.device_status()[0] == 0
print("captured first")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured first" in r.stdout, r.stdout + r.stderr
