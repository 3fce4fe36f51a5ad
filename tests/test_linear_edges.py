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


# columns of one buffer whose rows are 4096 bytes apart: x takes bytes 0 to 127 of each
P = 4096


@pytest.mark.parametrize("change, status", [
    (dict(q=A + 128), MISALIGNED), (dict(q=A + 127), ALIASING), (dict(q=A + P - 64), MISALIGNED), (dict(q=A + P - 63), ALIASING),
    (dict(q=A - 64), MISALIGNED), (dict(q=A - 63), ALIASING), (dict(q=A + 200, qs=P + 1), ALIASING), (dict(q=A + 2 * P + 128), MISALIGNED),
    (dict(q=A + 7 * P + 1), ALIASING), (dict(q=A + 8 * P), MISALIGNED), (dict(h=A + 256, hs=P // 2), MISALIGNED),
    (dict(h=F + 128, hs=P // 2), MISALIGNED), (dict(h=A + 64, hs=P // 2), ALIASING), (dict(h=A, hs=P // 2), MISALIGNED),
    (dict(h=A + 128, hs=P // 2, q=A + 256), MISALIGNED), (dict(h=A + 128, hs=P // 2, q=A + 255), ALIASING),
    (dict(w=A + P + 128, q=A + 256), MISALIGNED), (dict(w=A + P + 200, q=A + 256), ALIASING),
    (dict(scale=A + 130), MISALIGNED), (dict(scale=A + 126), ALIASING), (dict(scale=A + P - 30), ALIASING),
    (dict(x=D + 8, xs=0), ALIASING), (dict(x=D + 64, xs=0), MISALIGNED), (dict(x=D - 2 * 64, xs=0), MISALIGNED),
])
def test_columns_of_one_buffer(lib, change, status):
    """What interleaves without sharing a byte does not overlap."""
    call = NORM | dict(rows=8, xs=P // 2, rs=P // 2, qs=P) | change
    assert lib.imd_norm_quantize(*call.values()) == status


def test_columns_of_one_buffer_in_products(lib):
    out = dict(rows=4, out=A + 65, os=P // 2)
    assert lib.imd_scaled_linear(*(L8 | out | dict(xs=P)).values()) == MISALIGNED
    assert lib.imd_scaled_linear(*(L8 | out | dict(xs=P, out=A + 63)).values()) == ALIASING
    assert lib.imd_scaled_linear(*(L8 | out | dict(xs=P + 1)).values()) == ALIASING
    assert lib.imd_scaled_linear(*(L8 | out | dict(xs=P, w=A + 2 * P + 128, ws=P)).values()) == MISALIGNED
    assert lib.imd_scaled_linear(*(L8 | out | dict(xs=P, x_scale=A + 3 * P + 84)).values()) == MISALIGNED   # out: bytes 65 to 80
    assert lib.imd_scaled_linear(*(L8 | out | dict(xs=P, x_scale=A + 3 * P + 72)).values()) == ALIASING
    out = dict(rows=4, out=A + 129, os=P // 2)
    assert lib.imd_linear_w4(*(W4 | out | dict(xs=P // 2)).values()) == MISALIGNED
    assert lib.imd_linear_w4(*(W4 | out | dict(xs=P // 2, out=A + 127)).values()) == ALIASING
    assert lib.imd_linear_w4(*(W4 | out | dict(xs=P // 2, w=A + 256, ws=P, scale=A + 320, ss=P // 2, zeros=A + 400, zs=P)).values()) == MISALIGNED
    assert lib.imd_linear_w4(*(W4 | out | dict(xs=P // 2, zeros=A + 140, zs=P)).values()) == ALIASING


@pytest.mark.parametrize("eps, status", [(0.0, MISALIGNED), (2.0 ** 127, MISALIGNED), (1.8e38, INVALID), (1e39, INVALID), (1e300, INVALID)])
def test_eps_stays_in_the_range_of_32_bits(lib, eps, status):
    """mean + eps is formed in 32 bits: an eps beyond them would turn every row to zeros."""
    assert lib.imd_norm_quantize(*(NORM | dict(eps=eps)).values()) == status
