"""Which kernel takes a product of the quantised linear layer, on the host: the header that the library is built from
(immerdink_b200/csrc/linear/choice.hpp) is compiled with g++ (tests/linear_choice_shim.cpp) and asked."""
import ctypes as C
import os
import subprocess

import pytest

from immerdink_b200 import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A, B = 0x10000000, 0x20000000


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = tmp_path_factory.mktemp("choice") / "linear_choice.so"
    cuda = os.path.join(os.path.dirname(os.path.dirname(build._nvcc())), "include")
    subprocess.run([build._cxx(), "-std=c++17", "-O1", "-shared", "-fPIC", "-I" + build.INCLUDE, "-I" + build.CSRC, "-I" + cuda,
                    os.path.join(ROOT, "tests", "linear_choice_shim.cpp"), "-o", str(so)], check=True)
    lib = C.CDLL(str(so))
    lib.choice_w4.argtypes = [C.c_int64] * 7 + [C.c_int]
    lib.choice_8.argtypes = [C.c_int] + [C.c_int64] * 7
    lib.w4_by_tma.argtypes = [C.c_int64] * 4
    lib.split.argtypes = [C.c_int64, C.c_int64] + [C.c_int] * 5
    return lib


def w4(lib, rows, n, k, x=A, xs=None, w=B, ws=None, group=128):
    pitch = -(-k // 32) * 32
    return chr(lib.choice_w4(rows, n, k, x, pitch if xs is None else xs, w, pitch // 2 if ws is None else ws, group))


def e8(lib, rows, n, k, x=A, xs=None, w=B, ws=None, e4m3=1):
    pitch = -(-k // 16) * 16
    return chr(lib.choice_8(e4m3, rows, n, k, x, pitch if xs is None else xs, w, pitch if ws is None else ws))


def test_depths_that_32_bit_coordinates_hold(lib):
    """A block of k that TMA brings starts at a byte that fits 32 bits with a sign, x of the 4-bit product at 2 k; blocks
    start at multiples of 128 k, up to 255 k before the end of the last one."""
    for k in (1 << 30, (1 << 30) + 64, (1 << 31) - 1):
        assert w4(lib, 33, 1, k) == "a"                  # x by loads, whose offsets are 64-bit
        assert w4(lib, 17, 1, k, w=B + 1) == "a"         # (17 rows whose weights cannot be streamed)
    assert w4(lib, 33, 1, (1 << 30) - 512) == "t"
    assert 2 * ((1 << 30) - 512 + 255) < 1 << 31
    assert lib.w4_by_tma(1, (1 << 31) - 1, B, 1 << 30) == 1    # the weights' bytes are a quarter of that
    # the streamed kernel counts k itself, to the end of the eight warps' pieces of 256 and a step of 128 behind a row's end
    assert w4(lib, 1, 1, (1 << 31) - 4096) == "s"
    assert (1 << 31) - 4096 + 8 * 256 + 128 < 1 << 31
    for k in ((1 << 31) - 4095, (1 << 31) - 1):
        assert w4(lib, 1, 1, k) == "m"
        assert w4(lib, 17, 1, k) == "a"
    # 8 bits: a byte per k
    for rows in (1, 300):
        assert e8(lib, rows, 1, (1 << 31) - 512) == "t"
    assert e8(lib, 1, 1, (1 << 31) - 1) == "m" and e8(lib, 300, 1, (1 << 31) - 1) == "a"


def test_rows_that_tma_brings(lib):
    assert w4(lib, 40, 64, 256) == "t" and w4(lib, 40, 64, 256, x=A + 2) == "m"
    assert w4(lib, 4000, 640, 256, x=A + 2) == "a" and w4(lib, 4000, 640, 256, xs=255) == "a"
    assert w4(lib, 4000, 640, 256, xs=0) == "a"          # a repeated row
    assert w4(lib, 3, 64, 256) == "s" and w4(lib, 3, 64, 256, w=B + 1) == "m" and w4(lib, 3, 64, 256, xs=257) == "m"
    assert w4(lib, 3, 64, 0) == "m" and w4(lib, 300, 64, 0) == "m"
    assert e8(lib, 3, 64, 256) == "t" and e8(lib, 3, 64, 256, w=B + 1) == "m" and e8(lib, 3, 64, 0) == "m"
    assert e8(lib, 3000, 5000, 257, ws=257) == "a" and e8(lib, 300, 50, 257, ws=257) == "m"


def test_clusters_fit_at_once(lib):
    """K is split among as many CTAs as the GPU holds clusters of that size at once, not as many as it has SMs."""
    fits = (148, 74, 33, 15)
    for per_sm in (1, 2):
        for tiles in range(1, 400):
            for steps in (1, 3, 4, 7, 8, 15, 16, 64):
                parts = lib.split(tiles, steps, *fits, per_sm)
                assert parts in (1, 2, 4, 8)
                assert parts == 1 or (tiles <= fits[parts.bit_length() - 1] * per_sm and steps >= 2 * parts)
                assert parts == 8 or tiles > fits[parts.bit_length()] * per_sm or steps < 4 * parts   # no less than that
    assert [lib.split(t, 64, *fits, 1) for t in (15, 16, 33, 34, 74, 75)] == [8, 4, 4, 2, 2, 1]
    assert [lib.split(t, 64, *fits, 2) for t in (30, 32, 37, 74, 148, 149)] == [8, 4, 4, 2, 2, 1]


@pytest.mark.parametrize("rows", [17, 24, 32])
def test_two_streamed_passes_only_where_they_are_quicker(lib, rows):
    for n, k in ((4096, 4096), (3584, 8192), (8192, 4096), (4096, 14336), (8192, 8192), (8192, 28672), (18944, 3584)):
        assert w4(lib, rows, n, k) == "t" and w4(lib, rows, n, k, group=32) == "s"
        assert w4(lib, 16, n, k) == "s" and w4(lib, 33, n, k, group=32) == "t"
    for n, k in ((512, 1024), (1024, 4096), (2048, 2048), (4736, 2816), (14336, 4096), (28672, 8192), (128256, 4096)):
        for group in (32, 64, 128):
            assert w4(lib, rows, n, k, group=group) == "s"


def test_rows_of_x_that_only_loads_bring_stay_streamed(lib):
    """A repeated row of x: the tensor-core kernel would bring it word by word."""
    for rows in (17, 32):
        assert w4(lib, rows, 4096, 4096, xs=0) == "s" and w4(lib, rows, 8192, 8192, xs=4096) == "s"
        assert w4(lib, rows, 4096, 4096, xs=0, x=A + 2) == "a"
