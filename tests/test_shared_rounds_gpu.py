"""Four CTAs to a tile: when the grouped products choose it, and that the buffers they send their sums to are used again, in
two and three rounds of clusters."""
import numpy as np
import pytest

from cudanative_jl_b200 import _lib
from cudanative_jl_b200.array import CuArray, CuHostArray
from cudanative_jl_b200.bfloat16 import BFloat16
from grouped_cases import offsets_of
from test_grouped_gpu import run_grouped, run_grouped_k

pytestmark = pytest.mark.gpu

F16, F32 = np.float16, np.float32
LEAST_K = {1: 1536, 2: 4096, 3: 8192}  # by rounds of clusters


def call(handle, K, tiles):
    """The launch of one group of K columns into `tiles` tiles of 128 x 64; what the operands hold does not matter."""
    M, N = 128, 64 * tiles
    a, b, d = CuHostArray(F16, shape=(M, K)), CuHostArray(F16, shape=(N, K)), CuHostArray(F32, shape=(M, N))
    handle.gemm_grouped_k(M, N, K, 1.0, a, M, b, N, F16, 0.0, None, M, 0, F32, d, M, M * N, F32, CuArray(offsets_of([K])), 1)
    _lib.check(_lib.lib().b200_stream_sync(None), "sync")
    assert handle.device_status()[0] == 0
    return handle.last_launch()


@pytest.fixture()
def clusters(handle):
    launch = call(handle, 8200, 70)
    assert launch["split_k"] == 4 and launch["ctas"] % 4 == 0
    n = launch["ctas"] // 4
    assert 24 <= n <= 37  # three rounds hold 70 tiles; 148 SMs hold no more than 37 clusters of four
    return n


def test_the_rule(handle, clusters):
    for tiles in (1, clusters, clusters + 1, 2 * clusters, 2 * clusters + 1, 3 * clusters, 3 * clusters + 1):
        rounds = -(-tiles // clusters)
        for K in (1528, 1536, 4088, 4096, 8184, 8192):
            launch = call(handle, K, tiles)
            shared = rounds in LEAST_K and K >= LEAST_K[rounds]
            assert (launch["split_k"] == 4) == shared, (K, tiles)
            if shared:
                assert launch["ctas"] == 4 * min(clusters, tiles)


@pytest.mark.parametrize("d_type", [BFloat16, F32])
def test_buffers_are_used_again(handle, clusters, d_type):
    for K, tiles in ((4104, 2 * clusters - 3), (8200, 3 * clusters - 5)):
        run_grouped_k(handle, [K], 128, 64 * tiles, d_type=d_type, beta=1.0)
        assert handle.last_launch()["split_k"] == 4 and handle.last_launch()["ctas"] < 4 * tiles
        run_grouped(handle, [64 * tiles - 64], 128, K, d_type=d_type)
        assert handle.last_launch()["split_k"] == 4 and handle.last_launch()["ctas"] < 4 * tiles
        run_grouped_k(handle, [K - 8, K + 9, K, K - 1], 128, 64 * (tiles // 4), d_type=d_type, beta=1.0)  # a mean of K
        assert handle.last_launch()["split_k"] == 4 and handle.last_launch()["ctas"] < 4 * (tiles // 4 * 4)
