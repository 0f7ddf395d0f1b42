"""Order between the parts of the grouped products, by repetition: what one warp writes to shared memory for another to use."""
import numpy as np
import pytest

from cudanative_jl_b200 import _lib
from cudanative_jl_b200.array import Array, CuArray
from cudanative_jl_b200.bfloat16 import BFloat16
from grouped_cases import close, offsets_of, store, value

pytestmark = pytest.mark.gpu

F32 = np.float32


@pytest.mark.parametrize("tile_n,cta_pair", [(0, 0), (256, 2), (128, 2), (128, 1), (64, 1)])
def test_cleared_rows_behind_a_group(handle, tile_n, cta_pair):
    """Every other group is NaN and every group ends inside a 16-row step: the rows behind it, which are the neighbour's, are
    cleared in both CTAs of a pair before one of them issues the products of both.  A row that came too late is a NaN."""
    r = np.random.default_rng(2)
    sizes = [int(n) for k in range(32) for n in (16 * (k % 9) + 1 + k % 15, 17 + k)]
    off = offsets_of(sizes)
    M, N, K, E = 264, 328, int(off[-1]), len(sizes)
    A, B = store(r.standard_normal((M, K)), BFloat16), store(r.standard_normal((N, K)), BFloat16)
    for e in range(1, E, 2):
        A[:, off[e]:off[e + 1]] = B[:, off[e]:off[e + 1]] = 0x7fc0
    handle.set_option(_lib.OPT_TILE_N, tile_n)
    handle.set_option(_lib.OPT_CTA_PAIR, cta_pair)
    a_dev, b_dev, o_dev = CuArray(A), CuArray(B), CuArray(off)
    first = None
    for _ in range(20):
        d = CuArray(np.zeros((M, N * E), F32, order="F"))
        handle.gemm_grouped_k(M, N, K, 1.0, a_dev, M, b_dev, N, BFloat16, 0.0, None, M, 0, F32, d, M, M * N, F32, o_dev, E)
        _lib.check(_lib.lib().b200_stream_sync(None), "sync")
        assert handle.device_status()[0] == 0
        got = Array(d).tobytes(order="F")
        first = first or got
        assert got == first
    got = np.frombuffer(first, F32).reshape((M, N * E), order="F")
    a, b = value(A, BFloat16), value(B, BFloat16)
    for e in range(E):
        s, mat = slice(off[e], off[e + 1]), got[:, e * N:(e + 1) * N]
        if e % 2:
            assert np.isnan(mat).all()
        else:
            close(mat.astype(np.float64), a[:, s] @ b[:, s].T, np.abs(a[:, s]) @ np.abs(b[:, s]).T, sizes[e], F32, f"group {e}")
