"""The short way of calls with PyTorch tensors (csrc/linear/fastcall.c) against the general one of linear.py, on the host: both
are given the same stand-ins for tensors and functions that note what they are called with. Whatever the general way
refuses, the short way does not take; what both take arrives in the C entry the same."""
import ctypes as C
import itertools
import os
import sys
import types

import pytest

import immerdink_b200 as imd
from immerdink_b200 import build, linear

torch = pytest.importorskip("torch")
BF16, F16, F32, I8, E4M3, U8 = torch.bfloat16, torch.float16, torch.float32, torch.int8, torch.float8_e4m3fn, torch.uint8


class Tensor:
    """What both ways read of a PyTorch tensor."""

    def __init__(self, dtype, shape, stride=None, device=0, ptr=0x1000):
        self.dtype, self.shape, self._device, self._ptr = dtype, torch.Size(shape), device, ptr
        if stride is None:
            stride = [1] * len(shape)
            for i in reversed(range(len(shape) - 1)):
                stride[i] = stride[i + 1] * max(shape[i + 1], 1)
        self._stride = tuple(stride)

    def get_device(self):
        return self._device

    def stride(self):
        return self._stride

    def data_ptr(self):
        return self._ptr

    def but(self, **kw):
        new = Tensor(self.dtype, self.shape, self._stride, self._device, self._ptr)
        for k, v in kw.items():
            setattr(new, k, v)
        return new


@pytest.fixture(scope="module")
def ways():
    """(calls noted, short way, general way); a way is called with (name, arguments of the C module's function)."""
    build.build_linear()
    if build.build_fastcall() is None:
        pytest.skip("no Python.h")
    from immerdink_b200 import _fastcall
    noted = []
    device = C.CFUNCTYPE(C.c_int, C.POINTER(C.c_int))(lambda p: p.__setitem__(0, 0) or 0)
    entries, keep = {}, [device]
    for name in ("norm_quantize", "scaled_linear", "linear_w4"):
        args = linear.SIGNATURES["imd_" + name]
        entries[name] = C.CFUNCTYPE(C.c_int, *args)(lambda *a, name=name: noted.append((name, a)) or 0)
    keep.append(entries)
    for dtype, kind in ((BF16, linear.BF16), (F16, linear.F16), (F32, linear.F32), (I8, linear.I8), (E4M3, linear.E4M3), (U8, linear.U8)):
        _fastcall.learn(dtype, kind)
    fake = types.SimpleNamespace(current_device=lambda: 0, lib=types.SimpleNamespace(**{"imd_" + n: f for n, f in entries.items()}))

    def short(name, *args):
        return getattr(_fastcall, name)(C.cast(entries[name], C.c_void_p).value, C.cast(device, C.c_void_p).value, 0, *args)

    def general(name, *args):
        return getattr(linear, "_" + name)(fake, 0, *args)
    yield noted, short, general
    del keep


def norm_args(rows=3, dim=16, t=BF16, wt=None, to=I8, residual=True, out=True):
    return [Tensor(t, (rows, dim), ptr=0x10000), Tensor(wt or t, (dim,), ptr=0x20000), Tensor(to, (rows, dim), ptr=0x30000),
            Tensor(F32, (rows,), ptr=0x40000), 1e-6, Tensor(t, (rows, dim), ptr=0x50000) if residual else None,
            Tensor(t, (rows, dim), ptr=0x60000) if residual and out else None]


def scaled_args(rows=3, n=5, k=16, t=I8, out=BF16):
    return [Tensor(t, (rows, k), ptr=0x10000), Tensor(t, (n, k), ptr=0x20000), Tensor(out, (rows, n), ptr=0x30000),
            Tensor(F32, (rows,), ptr=0x40000), Tensor(F32, (n,), ptr=0x50000)]


def w4_args(rows=3, n=5, k=70, t=BF16, out=None, st=None, zeros=True, group=32):
    groups = -(-k // group)
    return [Tensor(t, (rows, k), ptr=0x10000), Tensor(U8, (n, (k + 1) // 2), ptr=0x20000), Tensor(out or t, (rows, n), ptr=0x30000),
            Tensor(st or t, (n, groups), ptr=0x40000), Tensor(U8, (n, groups), ptr=0x50000) if zeros else None, group]


def strides_of_rows(name, a):
    """The call with the strides of single rows left out, which are not looked at."""
    a = list(a)
    if name == "norm_quantize":
        rows = {4: a[0], 6: a[0], 11: a[0], 14: a[0]}
    elif name == "scaled_linear":
        rows = {5: a[0], 7: a[1], 12: a[0]}
    else:
        rows = {6: a[0], 8: a[1], 11: a[1], 13: a[1], 16: a[0]}
    return [None if i in rows and rows[i] <= 1 else v or 0 for i, v in enumerate(a)]


def both(ways, name, args, taken=None):
    noted, short, general = ways
    noted.clear()
    try:
        general(name, *args)
        want = noted.pop()
    except (TypeError, ValueError, C.ArgumentError):
        want = None
    noted.clear()
    st = short(name, *args)
    assert st in (None, 0) and (st is None) == (not noted)
    if want is None:
        assert st is None, "the short way takes what the general one refuses"
    elif st == 0:
        assert noted[0][0] == want[0] and repr(strides_of_rows(*noted[0])) == repr(strides_of_rows(*want))   # (a NaN is itself)
    if taken is not None:
        assert (st == 0) == taken, (st, want)


def test_what_is_taken(ways):
    for t, to, rows in itertools.product((BF16, F16, F32), (I8, E4M3), (0, 1, 3)):
        for wt in (t, F32):
            both(ways, "norm_quantize", norm_args(rows, 16, t, wt, to), True)
        both(ways, "norm_quantize", norm_args(rows, 16, t, t, to, out=False), True)
        both(ways, "norm_quantize", norm_args(rows, 1, t, t, to, residual=False), True)
    for t, out in itertools.product((I8, E4M3), (BF16, F16, F32)):
        for rows, n, k in ((3, 5, 16), (0, 5, 16), (3, 0, 16), (3, 5, 0), (1, 1, 1)):
            both(ways, "scaled_linear", scaled_args(rows, n, k, t, out), True)
    for t, st, zeros, group in itertools.product((BF16, F16), (BF16, F16, F32), (False, True), (32, 64, 128)):
        for rows, n, k in ((3, 5, 70), (0, 5, 70), (3, 0, 70), (3, 5, 0), (1, 1, 1), (1, 7, 129)):
            for out in (t, F32):
                both(ways, "linear_w4", w4_args(rows, n, k, t, out, st, zeros, group), True)


@pytest.mark.parametrize("name, make", [("norm_quantize", norm_args), ("scaled_linear", scaled_args), ("linear_w4", w4_args)])
def test_every_change_of_one_tensor(ways, name, make):
    """Another type, shape, rank, stride or device of each tensor in turn, and no tensor at all."""
    for i, x in enumerate(make()):
        if not isinstance(x, Tensor):
            continue
        shape, r = tuple(x.shape), len(x.shape)
        changes = [x.but(dtype=d) for d in (BF16, F16, F32, I8, E4M3, U8, torch.float64, torch.int32, torch.float8_e5m2)]
        changes += [x.but(shape=torch.Size(s)) for s in ((shape[0] + 1,) + shape[1:], (0,) + shape[1:], shape[:-1] + (shape[-1] + 1,),
                                                         shape[:-1] + (0,), shape[:-1] + (1,), shape[:-1] + (shape[-1] - 1,))]
        changes += [Tensor(x.dtype, shape + (1,)), Tensor(x.dtype, shape[:1]), Tensor(x.dtype, (1,) + shape), Tensor(x.dtype, ())]
        changes += [x.but(_stride=tuple(s)) for s in ([2] * r, [0] * (r - 1) + [1], [0] * r, [1] * r, [77] * (r - 1) + [1], [1, 4][:r])]
        changes += [x.but(_device=1), x.but(_device=-1), None, 5, "x", object()]
        for c in changes:
            args = make()
            args[i] = c
            both(ways, name, args)


def test_other_arguments(ways):
    for eps in (0, 1, 1e-300, float("nan"), None, "x", [1]):
        args = norm_args()
        args[4] = eps
        both(ways, "norm_quantize", args)
    args = norm_args(residual=False)
    args[6] = Tensor(BF16, (3, 16))
    both(ways, "norm_quantize", args, False)
    for group in (0, 31, 33, 256, -32, None, "32", 32.0, 1 << 70):
        args = w4_args()
        args[5] = group
        both(ways, "linear_w4", args)


def test_one_row_of_a_larger_array(ways):
    args = norm_args(1)
    args[0] = args[0].but(_stride=(64, 1))
    both(ways, "norm_quantize", args, True)
    args = w4_args(1, 1)
    args[1] = args[1].but(_stride=(4096, 1))
    both(ways, "linear_w4", args, True)


def test_built_for_this_interpreter(ways):
    from immerdink_b200 import _fastcall
    import sysconfig
    assert _fastcall.__file__ == build.FASTCALL_LIB and build.FASTCALL_LIB.endswith(sysconfig.get_config_var("EXT_SUFFIX"))


def test_without_the_short_way(monkeypatch, tmp_path):
    """A machine without Python.h builds and runs everything else: calls then go the general way."""
    monkeypatch.setattr(build, "FASTCALL_LIB", str(tmp_path / "_fastcall.so"))
    monkeypatch.setattr(build.sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
    assert build.build_fastcall(force=True) is None and not os.path.exists(build.FASTCALL_LIB)
    build.build_linear()
    monkeypatch.setitem(sys.modules, "immerdink_b200._fastcall", None)
    monkeypatch.delattr(imd, "_fastcall", raising=False)
    lib = linear.Library()
    a = [imd.DeviceArray(0x10000, (3, 16), None, "f2"), imd.DeviceArray(0x20000, (16,), None, "f2"), imd.DeviceArray(0x30000, (3, 16), None, "i1"),
         imd.DeviceArray(0x40000, (3,), None, "f4")]
    with pytest.raises(imd.InvalidValueError):
        imd.norm_quantize(*a, eps=-1.0, lib=lib)
    with pytest.raises(TypeError, match="CUDA memory"):
        imd.norm_quantize(torch.zeros(2, 8, dtype=BF16), *a[1:], lib=lib)
    with pytest.raises(imd.MisalignedError):
        imd.norm_quantize(*a[:3], imd.DeviceArray(0x40002, (3,), None, "f4"), lib=lib)
    with pytest.raises(imd.AliasingError):
        imd.scaled_linear(a[2], a[2], imd.DeviceArray(0x30000, (3, 3), None, "f4"), a[3], a[3], lib=lib)
    with pytest.raises(ValueError):
        imd.linear_w4(a[0], a[2], a[2], a[3], group=31, lib=lib)
