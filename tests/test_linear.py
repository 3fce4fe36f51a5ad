"""Refusals of the quantised linear layer, on the host: no GPU is needed, nothing is launched."""
import ctypes as C
import os
import re

import pytest

import immerdink_b200 as imd
from immerdink_b200 import build, linear

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OK, INVALID, UNSUPPORTED, ALIASING, MISALIGNED = 0, 1, 2, 3, 5
A, B, D, E, F, G = (0x10000000 * i for i in range(1, 7))   # addresses far apart, never dereferenced


@pytest.fixture(scope="module")
def lib():
    build.build_linear()
    return linear.load_library().lib


def test_exports_are_the_header(lib):
    text = open(os.path.join(ROOT, "include", "immerdink", "immerdink_linear.h")).read()
    names = sorted(set(re.findall(r"IMD_API[^;]*?\b(imd_[a-z0-9_]+)\s*\(", text)))
    assert names == sorted(linear.SIGNATURES)
    import subprocess
    out = subprocess.run(["nm", "-D", "--defined-only", build.LINEAR_LIB], capture_output=True, text=True).stdout
    assert sorted(ln.split()[-1] for ln in out.splitlines() if " T " in ln and "imd_" in ln) == names


def test_device_error_refuses(lib):
    assert lib.imd_linear_device_error(None) == INVALID


def test_missing_library_fails_loudly(monkeypatch):
    monkeypatch.setattr(os.path, "exists", lambda p: False)
    with pytest.raises(OSError, match="no CPU fallback"):
        linear.Library()


NORM = dict(rows=4, dim=64, x_type=1, x=A, xs=64, r=0, rs=0, wt=1, w=B, eps=1e-6, h=0, hs=0, qt=3, q=D, qs=64, scale=E, stream=0)


@pytest.mark.parametrize("change, status", [
    (dict(rows=0), OK), (dict(rows=0, x=0, q=0), OK),
    (dict(rows=-1), INVALID), (dict(dim=0), INVALID), (dict(dim=1 << 31), INVALID), (dict(x_type=3), INVALID),
    (dict(x_type=9), INVALID), (dict(qt=0), INVALID), (dict(wt=4), INVALID), (dict(eps=-1.0), INVALID),
    (dict(eps=float("nan")), INVALID), (dict(eps=float("inf")), INVALID), (dict(wt=2), UNSUPPORTED),
    (dict(x=0), INVALID), (dict(w=0), INVALID), (dict(q=0), INVALID), (dict(scale=0), INVALID),
    (dict(h=F, hs=64), INVALID),                                   # nothing to add
    (dict(xs=-64), INVALID), (dict(qs=63), INVALID), (dict(r=F, rs=64, h=G, hs=63), INVALID),
    (dict(q=A), ALIASING), (dict(scale=D + 8), ALIASING), (dict(r=F, rs=64, h=F + 2, hs=64), ALIASING),
    (dict(r=F, rs=64, h=F, hs=65), ALIASING), (dict(r=F, rs=64, h=B, hs=64), ALIASING),
    (dict(r=F, rs=64, h=D, hs=64), ALIASING), (dict(q=E), ALIASING),
    (dict(x=A + 1), MISALIGNED), (dict(scale=E + 2), MISALIGNED), (dict(w=B + 1), MISALIGNED),
    (dict(x_type=0, wt=0, x=A + 2), MISALIGNED),
])
def test_norm_refusals(lib, change, status):
    assert lib.imd_norm_quantize(*(NORM | change).values()) == status


L8 = dict(rows=4, n=8, k=64, type=3, x=A, xs=64, w=B, ws=64, x_scale=D, w_scale=E, ot=1, out=F, os=8, stream=0)


@pytest.mark.parametrize("change, status", [
    (dict(rows=0), OK), (dict(n=0, out=0), OK),
    (dict(rows=-1), INVALID), (dict(n=1 << 31), INVALID), (dict(k=-1), INVALID), (dict(type=1), INVALID), (dict(ot=3), INVALID),
    (dict(k=131072, xs=131072, ws=131072), UNSUPPORTED),
    (dict(x=0), INVALID), (dict(w=0), INVALID), (dict(x_scale=0), INVALID), (dict(w_scale=0), INVALID), (dict(out=0), INVALID),
    (dict(ws=-1), INVALID), (dict(os=7), INVALID),
    (dict(out=A), ALIASING), (dict(out=B + 8), ALIASING), (dict(out=D), ALIASING), (dict(out=E), ALIASING),
    (dict(out=F + 1), MISALIGNED), (dict(x_scale=D + 2), MISALIGNED), (dict(w_scale=E + 1), MISALIGNED),
])
def test_scaled_linear_refusals(lib, change, status):
    assert lib.imd_scaled_linear(*(L8 | change).values()) == status


W4 = dict(rows=4, n=8, k=64, group=32, xt=1, x=A, xs=64, w=B, ws=32, st=1, scale=D, ss=2, zeros=E, zs=2, ot=1, out=F, os=8, stream=0)


@pytest.mark.parametrize("change, status", [
    (dict(rows=0), OK), (dict(n=0), OK),
    (dict(rows=1 << 31), INVALID), (dict(n=-1), INVALID), (dict(k=-1), INVALID), (dict(group=0), INVALID), (dict(xt=4), INVALID),
    (dict(st=3), INVALID), (dict(ot=3), INVALID),
    (dict(group=16), UNSUPPORTED), (dict(group=48), UNSUPPORTED), (dict(xt=0, ot=0), UNSUPPORTED), (dict(ot=2), UNSUPPORTED),
    (dict(x=0), INVALID), (dict(w=0), INVALID), (dict(scale=0), INVALID), (dict(out=0), INVALID), (dict(xs=-1), INVALID),
    (dict(ss=-1), INVALID), (dict(zs=-1), INVALID), (dict(os=7), INVALID),
    (dict(out=A), ALIASING), (dict(out=B), ALIASING), (dict(out=D), ALIASING), (dict(out=E), ALIASING),
    (dict(x=A + 1), MISALIGNED), (dict(scale=D + 1), MISALIGNED), (dict(out=F + 1), MISALIGNED),
])
def test_linear_w4_refusals(lib, change, status):
    assert lib.imd_linear_w4(*(W4 | change).values()) == status


def arr(shape, dtype, strides=None, ptr=A, readonly=False):
    return imd.DeviceArray(ptr, shape, strides, dtype, readonly)


def test_front_end_refusals(monkeypatch):
    """Types, shapes, strides and read-only outputs are refused before the library is called."""
    x, q, s = arr((4, 64), "f2"), arr((4, 64), "i1", ptr=D), arr((4,), "f4", ptr=E)
    w = arr((64,), "f2", ptr=B)
    for args, kw, exc in [
            ((arr((4, 64), "i1"), w, q, s), {}, TypeError), ((arr((64,), "f2"), w, q, s), {}, ValueError),
            ((arr((4, 64), "f2", (1, 4)), w, q, s), {}, ValueError), ((x, arr((63,), "f2"), q, s), {}, ValueError),
            ((x, arr((64,), "f2", (2,)), q, s), {}, ValueError), ((x, arr((64,), "i1"), q, s), {}, TypeError),
            ((x, w, arr((4, 63), "i1"), s), {}, ValueError), ((x, w, arr((4, 64), "f2"), s), {}, TypeError),
            ((x, w, arr((4, 64), "i1", readonly=True), s), {}, ValueError), ((x, w, q, arr((5,), "f4")), {}, ValueError),
            ((x, w, q, s), dict(residual=arr((3, 64), "f2")), ValueError),
            ((x, w, q, s), dict(residual=arr((4, 64), "f4")), TypeError),
            ((x, w, q, s), dict(residual_out=arr((4, 64), "f2", ptr=F)), ValueError),
            ((object(), w, q, s), {}, TypeError), ((x, w, q, s), dict(eps=-1.0), imd.InvalidValueError)]:
        with pytest.raises(exc):
            imd.norm_quantize(*args, **kw)
    x8, w8, y, xs, ws = arr((4, 64), "i1"), arr((8, 64), "i1", ptr=B), arr((4, 8), "f4", ptr=D), arr((4,), "f4", ptr=E), arr((8,), "f4", ptr=F)
    for args in [(arr((4, 64), "f2"), w8, y, xs, ws), (x8, arr((8, 63), "i1"), y, xs, ws), (x8, w8, arr((8, 4), "f4"), xs, ws),
                 (x8, w8, y, ws, xs), (x8, w8, arr((4, 8), "i1"), xs, ws)]:
        with pytest.raises((TypeError, ValueError)):
            imd.scaled_linear(*args)
    with pytest.raises(imd.AliasingError):
        imd.scaled_linear(x8, w8, arr((4, 8), "f4", ptr=A), xs, ws)
    x4, w4, sc = arr((4, 65), "f2"), arr((8, 33), "u1", ptr=B), arr((8, 3), "f2", ptr=E)
    for args, kw in [((x4, w4, y, sc), dict(group=31)), ((x4, w4, y, sc), dict(group=64)), ((x4, arr((8, 32), "u1"), y, sc), dict(group=32)),
                     ((arr((4, 65), "f4"), w4, y, sc), dict(group=32)), ((x4, w4, y, sc), dict(group=32, zeros=arr((8, 2), "u1"))),
                     ((x4, arr((8, 33), "i1"), y, sc), dict(group=32))]:
        with pytest.raises((TypeError, ValueError)):
            imd.linear_w4(*args, **kw)


def test_host_tensors_are_refused():
    torch = pytest.importorskip("torch")
    x = torch.zeros(2, 8, dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="CUDA memory"):
        imd.norm_quantize(x, x[0], x, x[0])
