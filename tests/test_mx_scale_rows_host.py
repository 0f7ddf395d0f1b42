"""The rows of scale tiles that the grouped 4-bit product copies, from the function that the kernel calls, compiled for the
host: all that a tile's columns need, and none behind the last row that a group uses."""
import ctypes as C
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

CSRC = Path(__file__).resolve().parent.parent / "cudanative.jl_b200" / "csrc"


@pytest.fixture(scope="module")
def scale_rows(tmp_path_factory):
    gxx = shutil.which("g++") or shutil.which("c++")
    if gxx is None:
        pytest.skip("no C++ compiler")
    d = tmp_path_factory.mktemp("scale_rows")
    (d / "f.cpp").write_text('#include "mx_scale_rows.h"\n'
                             'extern "C" void f(int g, int c, int n, int* o) { b200::ScaleRows r = b200::scale_rows(g, c, n); o[0] = r.first; o[1] = r.count; }\n')
    r = subprocess.run([gxx, "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", str(CSRC), str(d / "f.cpp"), "-o", str(d / "f.so")],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    fn, out = C.CDLL(str(d / "f.so")).f, (C.c_int * 2)()

    def call(group_row, col, cols):
        fn(group_row, col, cols, out)
        return out[0], out[1]

    return call


# the GPU tests' sizes among them: with buffers of just the rows in use, a second row for every tile is a row too many
SIZES = [[1], [128, 129, 200], [256, 300, 1, 255], [192, 193, 1, 128, 64, 65], [3, 0, 70, 300, 257, 31], [70, 0, 300, 513, 1], [128], [256], [384, 0, 0], [0, 0, 64]]
R = np.random.default_rng(0)
SIZES += [R.integers(0, 700, int(R.integers(1, 30))).tolist() for _ in range(50)]


@pytest.mark.parametrize("tile_n", [32, 128, 192, 256])
def test_copies_stay_in_the_rows_in_use(scale_rows, tile_n):
    for sizes in SIZES:
        start, used = 0, sum((n + 127) // 128 for n in sizes)
        for n in sizes:
            for col in range(0, n, tile_n):
                cols = min(tile_n, n - col)
                first, count = scale_rows(start, col, cols)
                assert first == start + col // 128 and first + count - 1 == start + (col + cols - 1) // 128
                assert first + count <= used, (sizes, col)
                # the instruction's columns are rounded up: to 32 for pairs of CTAs, to 16 otherwise
                granule = 32 if tile_n >= 192 else 16
                assert col % 128 + -(-cols // granule) * granule <= 128 * count
                assert count <= (tile_n + 127) // 128
            start += (n + 127) // 128
