"""The quantised linear layer on caller-owned CUDA arrays, over libimmerdink_linear.so.

    norm_quantize   h = x + residual; y = RMS norm of h; q, scale = y in 8 bits with a scale per row
    scaled_linear   out = x_scale[:, None] * w_scale * (x @ w.T), 8-bit operands
    linear_w4       out = x @ ((w - zeros) * w_scale).T, 4-bit weights, a scale per group of k

Same rules as `contract`: nothing here allocates device memory, copies data or synchronises; a call
checks the arrays on the host and enqueues kernels on the caller's stream (default: the default
stream, also inside `torch.cuda.stream(s)`: pass stream=s there), so it can be captured in a CUDA graph. The caller owns every array. Arrays are PyTorch
tensors, DLPack producers or `__cuda_array_interface__` objects; bfloat16 and float8_e4m3fn need
one of the first two. They must be on the current device, and rows must have unit stride.

Calls with PyTorch tensors take a short way (csrc/linear/fastcall.c) that does the same checks in C; what
it does not take, and everything that is refused, goes through the general path below, and so does every call
where that module was not built (a call then takes longer on the host).

There is no CPU fallback: when the library is missing, the first call raises OSError."""
import ctypes as C
import os
import threading

from . import _arrays
from .device import _error

F32, BF16, F16, I8, E4M3, U8 = 0, 1, 2, 3, 4, 5
_NAMES = {F32: "float32", BF16: "bfloat16", F16: "float16", I8: "int8", E4M3: "float8_e4m3fn", U8: "uint8"}
_SIZES = {F32: 4, BF16: 2, F16: 2, I8: 1, E4M3: 1, U8: 1}
_CAI_TYPES = {"<f4": F32, "<f2": F16, "|i1": I8, "|u1": U8}
_DL_TYPES = {(2, 32, 1): F32, (2, 16, 1): F16, (4, 16, 1): BF16, (0, 8, 1): I8, (1, 8, 1): U8, (10, 8, 1): E4M3}
_TORCH_TYPES = {"torch." + name: code for code, name in _NAMES.items()}

_P, _I, _L = C.c_void_p, C.c_int32, C.c_int64
SIGNATURES = {
    "imd_norm_quantize": [_L, _L, _I, _P, _L, _P, _L, _I, _P, C.c_double, _P, _L, _I, _P, _L, _P, _P],
    "imd_scaled_linear": [_L, _L, _L, _I, _P, _L, _P, _L, _P, _P, _I, _P, _L, _P],
    "imd_linear_w4": [_L, _L, _L, _I, _I, _P, _L, _P, _L, _I, _P, _L, _P, _L, _I, _P, _L, _P],
    "imd_linear_device_error": [C.POINTER(C.c_uint)],
}


class _GeneralOnly:
    """In the place of _fastcall where it was not built: takes no call."""
    norm_quantize = scaled_linear = linear_w4 = learn = staticmethod(lambda *args: None)


def _short_way():
    try:
        from . import _fastcall
    except ImportError:
        return _GeneralOnly
    return _fastcall


class Library:
    """libimmerdink_linear.so. Search order: `path`, $IMMERDINK_LINEAR_LIB,
    $IMMERDINK_LIB_DIR/libimmerdink_linear.so, the package directory."""

    def __init__(self, path=None):
        if path is None:
            tries = [os.environ.get("IMMERDINK_LINEAR_LIB")]
            if os.environ.get("IMMERDINK_LIB_DIR"):
                tries.append(os.path.join(os.environ["IMMERDINK_LIB_DIR"], "libimmerdink_linear.so"))
            tries.append(os.path.join(os.path.dirname(os.path.abspath(__file__)), "libimmerdink_linear.so"))
            path = next((p for p in tries if p and os.path.exists(p)), None)
        if path is None:
            raise OSError("libimmerdink_linear.so not found (build it with `python -m immerdink_b200.build`, "
                          "or set IMMERDINK_LINEAR_LIB); there is no CPU fallback")
        self.path, self.lib = path, C.CDLL(path)
        for name, args in SIGNATURES.items():
            f = getattr(self.lib, name)
            f.restype, f.argtypes = C.c_int, args
        self.fast = _short_way()
        self._address = {name: C.cast(getattr(self.lib, name), C.c_void_p).value for name in SIGNATURES}
        self._local, self._get_device = threading.local(), None
        for name in ("libcudart.so.12", "libcudart.so.13", "libcudart.so"):
            try:
                self._get_device = C.CDLL(name).cudaGetDevice
                break
            except OSError:
                continue
        get_device = 0 if self._get_device is None else C.cast(self._get_device, C.c_void_p).value
        self.norm, self.scaled, self.w4 = ((self._address[name], get_device) for name in
                                           ("imd_norm_quantize", "imd_scaled_linear", "imd_linear_w4"))

    def device_error(self):
        """imd_linear_device_error: the sticky error word, read and cleared (synchronises)."""
        v = C.c_uint(0)
        st = self.lib.imd_linear_device_error(C.byref(v))
        if st:
            raise _error(st, "imd_linear_device_error")
        return int(v.value)

    def current_device(self):
        """The current device's number; None where the runtime cannot be asked."""
        try:
            number, ref = self._local.device
        except AttributeError:   # this thread's first question
            number = C.c_int(0)
            ref = C.byref(number)
            self._local.device = number, ref
        if self._get_device is None or self._get_device(ref) != 0:
            return None
        return number.value


_loaded, _lock = {}, threading.Lock()


def load_library(path=None):
    if isinstance(path, Library):
        return path
    lib = _loaded.get(path)
    if lib is None:
        with _lock:
            lib = _loaded.get(path)
            if lib is None:
                lib = _loaded[path] = Library(path)
    return lib


_torch_types = {}   # dtype object of PyTorch -> type (None: not one of ours)


def _view(x, what, stream, device):
    """(pointer, shape, element strides or None, type, readonly) of a CUDA array."""
    dtype = getattr(x, "dtype", None)
    if dtype is not None and hasattr(x, "data_ptr"):   # a PyTorch tensor: no capsule is made
        if dtype not in _torch_types:
            _torch_types[dtype] = _TORCH_TYPES.get(str(dtype))
            if _torch_types[dtype] is not None:
                _short_way().learn(dtype, _torch_types[dtype])
        on = x.get_device()
        if on < 0:
            raise TypeError(f"{what} is not in CUDA memory")
        if device is not None and on != device:
            raise ValueError(f"{what} is on CUDA device {on}, the current device is {device}")
        return x.data_ptr(), tuple(x.shape), x.stride(), _torch_types[dtype], False
    cai = getattr(x, "__cuda_array_interface__", None)
    if cai is not None:
        ptr, shape, strides, _, readonly, item = _arrays.view(x, stream, device)
        kind = _CAI_TYPES.get(cai["typestr"])
    else:
        ptr, shape, strides, kind, readonly, item = _arrays.dlpack_view(x, stream, device)
        kind = _DL_TYPES.get(kind)
    if strides is not None:
        if any(s % item for s in strides):
            raise ValueError(f"{what}: byte strides must be multiples of the element size")
        strides = tuple(s // item for s in strides)
    return ptr, tuple(shape), strides, kind, readonly


def _matrix(x, what, types, stream, device, out=False):
    """(pointer, rows, columns, row stride, type) of a matrix whose rows have unit stride."""
    ptr, shape, strides, kind, readonly = _view(x, what, stream, device)
    if kind not in types:
        raise TypeError(f"{what}: dtype must be {' or '.join(_NAMES[t] for t in types)}")
    if len(shape) != 2:
        raise ValueError(f"{what}: a matrix is wanted, got shape {shape}")
    if out and readonly:
        raise ValueError(f"{what} is read-only")
    rows, cols = shape
    if strides is None:
        return ptr, rows, cols, cols, kind
    if cols > 1 and strides[1] != 1:
        raise ValueError(f"{what}: rows must have unit stride, got strides {strides}")
    return ptr, rows, cols, strides[0] if rows > 1 else cols, kind


def _vector(x, what, n, types, stream, device, out=False):
    """(pointer, type) of a contiguous vector of n elements."""
    ptr, shape, strides, kind, readonly = _view(x, what, stream, device)
    if kind not in types:
        raise TypeError(f"{what}: dtype must be {' or '.join(_NAMES[t] for t in types)}")
    if shape != (n,):
        raise ValueError(f"{what}: shape must be ({n},), got {shape}")
    if out and readonly:
        raise ValueError(f"{what} is read-only")
    if strides is not None and n > 1 and strides[0] != 1:
        raise ValueError(f"{what} must be contiguous")
    return ptr, kind


def _same(what, got, want):
    if got != want:
        raise ValueError(f"{what}: shape must be {want}, got {got}")


def norm_quantize(x, weight, q, scale, *, eps=1e-6, residual=None, residual_out=None, stream=None, lib=None):
    """RMS norm of the rows of x (+ residual) into 8-bit codes and a scale per row (imd_norm_quantize).

        h = x + residual;  y = h / sqrt(mean(h^2) + eps) * weight;  y ~ scale[:, None] * q

    x, residual: [rows, dim] float32, bfloat16 or float16; weight: [dim] of x's dtype or float32;
    q: [rows, dim] int8 (codes -127..127) or float8_e4m3fn; scale: [rows] float32. residual_out
    ([rows, dim], x's dtype; may be x or residual itself) receives h. A row of zeros gives scale 0;
    a row with a NaN or an infinity gives scale NaN. Returns (q, scale)."""
    lib = load_library(lib)
    s = 0 if stream is None else _arrays.stream_handle(stream)
    st = lib.fast.norm_quantize(*lib.norm, s, x, weight, q, scale, eps, residual, residual_out)
    if st is None:
        st = _norm_quantize(lib, s, x, weight, q, scale, eps, residual, residual_out)
    if st:
        raise _error(st, "imd_norm_quantize")
    return q, scale


def _norm_quantize(lib, s, x, weight, q, scale, eps, residual, residual_out):
    dev = lib.current_device()
    px, rows, dim, sx, tx = _matrix(x, "x", (F32, BF16, F16), s, dev)
    pw, tw = _vector(weight, "weight", dim, (tx, F32) if tx != F32 else (F32,), s, dev)
    pq, qr, qc, sq, tq = _matrix(q, "q", (I8, E4M3), s, dev, True)
    _same("q", (qr, qc), (rows, dim))
    ps, _ = _vector(scale, "scale", rows, (F32,), s, dev, True)
    pr = sr = ph = sh = 0
    if residual is not None:
        pr, r, c, sr, _ = _matrix(residual, "residual", (tx,), s, dev)
        _same("residual", (r, c), (rows, dim))
    if residual_out is not None:
        if residual is None:
            raise ValueError("residual_out is given without a residual")
        ph, r, c, sh, _ = _matrix(residual_out, "residual_out", (tx,), s, dev, True)
        _same("residual_out", (r, c), (rows, dim))
    return lib.lib.imd_norm_quantize(rows, dim, tx, px, sx, pr, sr, tw, pw, eps, ph, sh, tq, pq, sq, ps, s)


def scaled_linear(x, w, out, x_scale, w_scale, *, stream=None, lib=None):
    """out[t, n] = x_scale[t] * w_scale[n] * sum_k x[t, k] * w[n, k] (imd_scaled_linear).

    x: [rows, k], w: [n, k], both int8 (exact 32-bit sums) or both float8_e4m3fn (32-bit float sums);
    x_scale: [rows], w_scale: [n] float32; out: [rows, n] float32, bfloat16 or float16. Returns out."""
    lib = load_library(lib)
    s = 0 if stream is None else _arrays.stream_handle(stream)
    st = lib.fast.scaled_linear(*lib.scaled, s, x, w, out, x_scale, w_scale)
    if st is None:
        st = _scaled_linear(lib, s, x, w, out, x_scale, w_scale)
    if st:
        raise _error(st, "imd_scaled_linear")
    return out


def _scaled_linear(lib, s, x, w, out, x_scale, w_scale):
    dev = lib.current_device()
    px, rows, k, sx, tx = _matrix(x, "x", (I8, E4M3), s, dev)
    pw, n, wk, sw, _ = _matrix(w, "w", (tx,), s, dev)
    _same("w", (n, wk), (n, k))
    po, r, c, so, to = _matrix(out, "out", (F32, BF16, F16), s, dev, True)
    _same("out", (r, c), (rows, n))
    pxs, _ = _vector(x_scale, "x_scale", rows, (F32,), s, dev)
    pws, _ = _vector(w_scale, "w_scale", n, (F32,), s, dev)
    return lib.lib.imd_scaled_linear(rows, n, k, tx, px, sx, pw, sw, pxs, pws, to, po, so, s)


def linear_w4(x, w, out, w_scale, *, zeros=None, group=128, stream=None, lib=None):
    """out[t, n] = sum_k x[t, k] * w_scale[n, k // group] * (w[n, k] - zeros[n, k // group]) (imd_linear_w4).

    x: [rows, k] bfloat16 or float16; w: [n, ceil(k / 2)] uint8, element k in the low (even k) or high
    (odd k) half of byte k // 2; group: 32, 64 or 128; w_scale: [n, ceil(k / group)] float32, bfloat16
    or float16; zeros: the same shape, uint8 0..15 (None: 8); out: [rows, n] float32 or x's dtype.
    Returns out."""
    lib = load_library(lib)
    s = 0 if stream is None else _arrays.stream_handle(stream)
    st = lib.fast.linear_w4(*lib.w4, s, x, w, out, w_scale, zeros, group)
    if st is None:
        st = _linear_w4(lib, s, x, w, out, w_scale, zeros, group)
    if st:
        raise _error(st, "imd_linear_w4")
    return out


def _linear_w4(lib, s, x, w, out, w_scale, zeros, group):
    dev = lib.current_device()
    if group not in (32, 64, 128):
        raise ValueError("group must be 32, 64 or 128")
    px, rows, k, sx, tx = _matrix(x, "x", (BF16, F16), s, dev)
    pw, n, half, sw, _ = _matrix(w, "w", (U8,), s, dev)
    _same("w", (n, half), (n, (k + 1) // 2))
    groups = -(-k // group)
    pws, r, c, ss, ts = _matrix(w_scale, "w_scale", (F32, BF16, F16), s, dev)
    _same("w_scale", (r, c), (n, groups))
    pz = sz = 0
    if zeros is not None:
        pz, r, c, sz, _ = _matrix(zeros, "zeros", (U8,), s, dev)
        _same("zeros", (r, c), (n, groups))
    po, r, c, so, to = _matrix(out, "out", (F32, tx), s, dev, True)
    _same("out", (r, c), (rows, n))
    return lib.lib.imd_linear_w4(rows, n, k, group, tx, px, sx, pw, sw, ts, pws, ss, pz, sz, to, po, so, s)
