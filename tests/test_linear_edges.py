"""Calls of the quantised linear layer that have to pass its checks, on the host: each has a misaligned scale or output on
purpose, the check after all others, so that nothing is launched."""
import pytest

from immerdink_b200 import build, linear

OK, INVALID, UNSUPPORTED, ALIASING, MISALIGNED = 0, 1, 2, 3, 5
A, B, D, E, F, G = (0x10000000 * i for i in range(1, 7))   # addresses far apart, never dereferenced


@pytest.fixture(scope="module")
def lib():
    build.build_linear()
    build.build_fastcall()
    return linear.load_library().lib


NORM = dict(rows=1, dim=64, x_type=1, x=A, xs=64, r=F, rs=64, wt=1, w=B, eps=1e-6, h=0, hs=0, qt=3, q=D, qs=64, scale=E + 2, stream=0)
L8 = dict(rows=4, n=8, k=64, type=3, x=A, xs=64, w=B, ws=64, x_scale=D, w_scale=E, ot=1, out=F + 1, os=8, stream=0)
W4 = dict(rows=4, n=8, k=64, group=32, xt=1, x=A, xs=64, w=B, ws=32, st=1, scale=D, ss=2, zeros=E, zs=2, ot=1, out=F + 1, os=8, stream=0)


@pytest.mark.parametrize("change, status", [
    (dict(h=A, hs=256), MISALIGNED), (dict(h=F, rs=256, hs=64), MISALIGNED), (dict(h=A, xs=1 << 50, hs=0), MISALIGNED),
    (dict(qs=1, rs=-5), MISALIGNED),
    (dict(h=A + 2, hs=64), ALIASING), (dict(rows=2, h=A, hs=256), ALIASING),
])
def test_a_single_row_has_no_distance(lib, change, status):
    """A one-row view of a larger array is the same rows whatever its stride: in place it is accepted."""
    assert lib.imd_norm_quantize(*(NORM | change).values()) == status


def test_single_rows_of_products(lib):
    assert lib.imd_scaled_linear(*(L8 | dict(rows=1, xs=-1, os=1)).values()) == MISALIGNED
    assert lib.imd_scaled_linear(*(L8 | dict(n=1, ws=1 << 45)).values()) == MISALIGNED
    assert lib.imd_scaled_linear(*(L8 | dict(ws=1 << 45)).values()) == INVALID
    assert lib.imd_linear_w4(*(W4 | dict(rows=1, xs=-1, os=1)).values()) == MISALIGNED
    assert lib.imd_linear_w4(*(W4 | dict(n=1, ws=-1, ss=-1, zs=-1)).values()) == MISALIGNED
