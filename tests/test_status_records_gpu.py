"""What a handle's kernels report: waits that ran out and group offsets that are none are two records.  Neither hides the other,
and a product that looks for its own waits is not failed by an earlier call's offsets."""
import numpy as np
import pytest

from cudanative_jl_b200 import _lib
from cudanative_jl_b200.array import Array, CuArray
from cudanative_jl_b200.gemm import ShardedGemm, mxfp4_scale_bytes

pytestmark = pytest.mark.gpu

F16, F32 = np.float16, np.float32
WAIT = 107  # of the self-test: a barrier that nothing signals


def sync():
    _lib.check(_lib.lib().b200_stream_sync(None), "sync")


def bad_grouped(handle):
    a, d = CuArray(np.ones((64, 192), F16, order="F")), CuArray(np.full((64, 9), 3.5, F32, order="F"))
    handle.gemm_grouped(True, 64, 9, 64, 1.0, a, 64, 4096, a, 64, F16, 0.0, None, 64, F32, d, 64, F32, CuArray(np.array([0, 5, 3, 9], np.int32)), 3)
    sync()
    assert np.all(Array(d) == 3.5)


def bad_grouped_plain(handle):
    handle.set_option(_lib.OPT_FORCE_KERNEL, _lib.KERNEL_SIMPLE)
    bad_grouped(handle)
    handle.set_option(_lib.OPT_FORCE_KERNEL, _lib.KERNEL_AUTO)


def bad_grouped_k(handle):
    for kernel in (_lib.KERNEL_SIMPLE, _lib.KERNEL_AUTO):
        handle.set_option(_lib.OPT_FORCE_KERNEL, kernel)
        a, d = CuArray(np.ones((64, 9), F16, order="F")), CuArray(np.zeros((64, 192), F32, order="F"))
        handle.gemm_grouped_k(64, 64, 9, 1.0, a, 64, a, 64, F16, 0.0, None, 64, 4096, F32, d, 64, 4096, F32, CuArray(np.array([0, 5, 3, 9], np.int32)), 3)
    sync()


def bad_quantize(handle):
    q, s = CuArray(np.zeros((16, 9), np.uint8, order="F")), CuArray(np.zeros(mxfp4_scale_bytes(32, 9, 3), np.uint8))
    handle.mxfp4_quantize(False, 32, 9, CuArray(np.ones((32, 9), F32, order="F")), 32, F32, q, 32, s, offsets=CuArray(np.array([0, 5, 3, 9], np.int32)), groups=3)
    sync()


def bad_mx(handle):
    q, s = CuArray(np.zeros((16, 24), np.uint8, order="F")), CuArray(np.zeros(4 * 512, np.uint8))
    d = CuArray(np.zeros((8, 9), F32, order="F"))
    handle.gemm_mxfp4_grouped(8, 9, 32, 1.0, q, 32, 256, s, q, 32, s, 0.0, None, 8, F32, d, 8, F32, CuArray(np.array([0, 5, 3, 9], np.int32)), 3)
    sync()


BAD = [bad_grouped, bad_grouped_plain, bad_grouped_k, bad_quantize, bad_mx]


@pytest.mark.parametrize("bad", BAD, ids=lambda f: f.__name__)
def test_a_right_product_after_bad_offsets(handle, bad):
    r = np.random.default_rng(0)
    a, b = np.asfortranarray(r.integers(-4, 5, (64, 32)).astype(F16)), np.asfortranarray(r.integers(-4, 5, (32, 48)).astype(F16))
    d = np.zeros((64, 48), F32, order="F")
    bad(handle)
    handle.gemm_host(False, False, 64, 48, 32, 1.0, a, 64, b, 32, 0.0, None, 64, d, 64)
    assert np.array_equal(d, a.astype(F32) @ b.astype(F32))
    code, _, groups = handle.device_status()  # the report is still there
    assert (code, groups) == (_lib.STATUS_BAD_OFFSETS, 3)
    assert handle.device_status()[0] == 0


def test_a_sharded_product_after_bad_offsets(handle):
    sg = ShardedGemm(handle, 256, 128, 128)
    b, d = CuArray(np.zeros((128, 128), F16, order="F")), CuArray(np.zeros((256, 128), F32, order="F"))
    bad_grouped(handle)
    sg.run(1.0, b, 0.0, None, d)
    sg.wait(10000)
    sg.close()
    assert handle.device_status()[0] == _lib.STATUS_BAD_OFFSETS


@pytest.mark.parametrize("bad", BAD, ids=lambda f: f.__name__)
@pytest.mark.parametrize("wait_first", [False, True])
def test_offsets_do_not_hide_a_wait(handle, bad, wait_first):
    def wait():
        _lib.check(_lib.lib().b200_selftest_bounded_wait(handle._h, None, 1_000_000), "selftest")
        sync()

    for f in ((wait, lambda: bad(handle)) if wait_first else (lambda: bad(handle), wait)):
        f()
    assert [handle.device_status()[0] for _ in range(3)] == [WAIT, _lib.STATUS_BAD_OFFSETS, 0]


def test_check_on_call_reports_both(handle):
    from cudanative_jl_b200 import B200Error

    handle.set_option(_lib.OPT_CHECK_ON_CALL, 1)
    a, d = CuArray(np.ones((64, 64), F16, order="F")), CuArray(np.zeros((64, 64), F32, order="F"))
    bad_grouped(handle)
    _lib.check(_lib.lib().b200_selftest_bounded_wait(handle._h, None, 1_000_000), "selftest")
    sync()
    with pytest.raises(B200Error, match="wait id 107") as e:
        handle.gemm(False, False, 64, 64, 64, 1.0, a, 64, a, 64, 0.0, None, 64, d, 64)
    assert e.value.status == _lib.DEVICE_TIMEOUT
    handle.gemm(False, False, 64, 64, 64, 1.0, a, 64, a, 64, 0.0, None, 64, d, 64)  # nothing of its own to report yet
    sync()
    with pytest.raises(B200Error, match="group offsets") as e:
        handle.gemm(False, False, 64, 64, 64, 1.0, a, 64, a, 64, 0.0, None, 64, d, 64)
    assert e.value.status == _lib.INVALID_ARG
    assert handle.device_status()[0] == 0 and np.all(Array(d) == 64)
