"""The bounds of the tile products' operands against every address of the
storage they lie in (no GPU: the header is plain C++)."""
import ctypes
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
KERNELS = os.path.join(ROOT, "applegpu-runtime_amd", "csrc", "kernels")
SRC = """
#include "extent.hpp"
extern "C" int64_t columns(int64_t rows, int64_t n, int64_t first, int64_t ld, int planes) {
  return agpu::k::t16::extent_of_columns(rows, n, first, ld, planes);
}
extern "C" int64_t row(int64_t n, int planes) { return agpu::k::t16::row_values(n, planes); }
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("extents")
    src, out = d / "e.cpp", d / "e.so"
    src.write_text(SRC)
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", f"-I{KERNELS}", str(src), "-o", str(out)], check=True)
    lib = ctypes.CDLL(str(out))
    lib.columns.restype = lib.row.restype = ctypes.c_int64
    lib.columns.argtypes = [ctypes.c_int64] * 4 + [ctypes.c_int]
    lib.row.argtypes = [ctypes.c_int64, ctypes.c_int]
    return lib


@pytest.mark.parametrize("block", [32, 64, 128, 256])
@pytest.mark.parametrize("rows,n,ld,off", [
    (5, 64, 64, 0), (8, 64, 128, 0), (8, 64, 128, 64), (8, 64, 512, 448), (3, 72, 136, 64), (16, 264, 1024, 760),
    (2, 520, 1024, 504), (1, 8, 16, 8), (4, 768, 2304, 1536)])
def test_columns_of_a_view_end_with_its_last_row(lib, rows, n, ld, off, block):
    """Rows [off, off + n) of a storage of `rows` x `ld` values that ends behind
    the last: what a block of columns may read reaches its last value and no
    further than the storage."""
    storage = rows * ld
    for first in range(0, n, block):
        for at in range(rows):   # the resource of the stage from row `at` on
            end = off + at * ld + first + lib.columns(rows - at, n, first, ld, 1)
            assert off + (rows - 1) * ld + n <= end <= storage


@pytest.mark.parametrize("n", [1, 31, 32, 33, 64, 515, 1280])
def test_packed_rows_are_read_whole(lib, n):
    """Rows of planes, and 16-bit rows packed to 32 values: all of them, up to
    their zeros, and nothing behind the storage."""
    for planes in (1, 2):
        ld, rows = (n + 31) // 32 * 32 * planes, 7
        assert n <= lib.row(n, planes) <= ld
        for first in range(0, n, 64):
            end = first * planes + lib.columns(rows, n, first, ld, planes)
            assert (rows - 1) * ld + n <= end <= rows * ld
