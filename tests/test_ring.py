"""The wait for copies in flight after a bounded wait gave up, on the host: the header that the kernels include
(immerdink_b200/csrc/common/ring.hpp) is compiled with g++ (tests/ring_shim.cpp) and run against a model of a barrier, whose
answer for the parity of the phase before the current one is always yes."""
import ctypes as C
import glob
import os
import subprocess

import pytest

from immerdink_b200 import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = tmp_path_factory.mktemp("ring") / "ring.so"
    subprocess.run([build._cxx(), "-std=c++17", "-O1", "-shared", "-fPIC", "-I" + build.CSRC,
                    os.path.join(ROOT, "tests", "ring_shim.cpp"), "-o", str(so)], check=True)
    lib = C.CDLL(str(so))
    lib.ring_case.argtypes = lib.slots_case.argtypes = [C.c_int] + [C.c_uint32] * 3
    return lib


@pytest.mark.parametrize("slots", [1, 2, 3, 6, 8, 12])
def test_waits_for_every_copy_in_flight_and_no_other(lib, slots):
    for issued in range(4 * slots + 3):
        for open_ in range(min(slots, issued) + 1):
            for at in (0, 1, 2, slots, 20 * slots):
                assert lib.ring_case(slots, issued, open_, at) == 0, (issued, open_, at)


@pytest.mark.parametrize("slots", [1, 2, 5, 8, 32])
def test_waits_for_the_phases_that_are_open(lib, slots):
    for rounds in (0, 1, 2, 7):
        for open_ in range(slots + 1):
            for at in (0, 1, slots, slots + 1, 20 * slots):
                assert lib.slots_case(slots, rounds, open_, at) == 0, (rounds, open_, at)


def test_no_kernel_asks_for_both_parities():
    """A question for both parities of a barrier is always answered yes: it waits for nothing."""
    for f in glob.glob(os.path.join(build.CSRC, "**", "*.cu*"), recursive=True):
        for line in open(f).read().split(";"):
            assert not ("||" in line and line.count("mbar_try_wait") > 1), f
