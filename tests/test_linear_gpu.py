"""The quantised linear layer against plain 64-bit arithmetic on a GPU.

Tolerances. A rounding to a type with significand spacing eps is off by at most eps / 2 relative to the value
(`half`). A 32-bit sum of m terms with A = sum |term| is off by at most m 2^-23 A: a tensor instruction may cut each term it
aligns (2^-23 of the partial sum, at most A), an ordinary addition rounds (2^-24). In the 2-norm over many outputs the errors
of the accumulations (one per instruction of at least 16 terms, partial sums no larger than the result's spread) add up to no
more than max(sqrt(m), m / 16) 2^-23 of the result."""
import math
import os
import subprocess
import sys

import pytest
import torch

import immerdink_b200 as imd
from immerdink_b200 import linear

pytestmark = pytest.mark.gpu
BF16, F16, F32, I8, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.int8, torch.float8_e4m3fn
U24 = 2.0 ** -24


@pytest.fixture(autouse=True)
def no_wait_gave_up():
    yield
    assert linear.load_library().device_error() == 0


def half(t):
    return torch.finfo(t).eps / 2


def rnd(seed, *shape, dtype=F32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def ints(seed, lo, hi, *shape, dtype=torch.int8):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=torch.int32).to(dtype)


def guarded(rows, cols, dtype, pad=5, skew=0):
    """A matrix with `pad` elements behind each row and rows around it, all 0x5A bytes: (matrix, check)."""
    size = torch.empty(0, dtype=dtype).element_size()
    raw = torch.full(((rows + 2) * (cols + pad) * size + 64,), 0x5A, dtype=torch.uint8, device="cuda")
    flat = raw[skew * size:skew * size + (rows + 2) * (cols + pad) * size].view(dtype).view(rows + 2, cols + pad)
    m = flat[1:rows + 1, :cols]

    def intact():
        keep = raw.clone()
        keep[skew * size:skew * size + (rows + 2) * (cols + pad) * size].view(dtype).view(rows + 2, cols + pad)[1:rows + 1, :cols] = 0
        keep[keep == 0x5A] = 0
        return int(keep.count_nonzero()) == 0
    return m, intact


# ---- norm_quantize -------------------------------------------------------------------------------------------------

def norm_check(x, r, w, q, scale, h, eps, t):
    """q, scale, h against the definition in 64 bits, row by row."""
    xs = x.double() + (r.double() if r is not None else 0.0)
    y = xs * torch.rsqrt(xs.square().mean(1, keepdim=True) + eps) * w.double()
    top = y.abs().amax(1)
    most = 127.0 if q.dtype == I8 else 448.0
    dim = x.shape[1]
    # the sum: each h is off by U24 (2 of its square), a chain of at most max(64, dim / 1024) + 10 additions; half of that goes
    # into the root; then root, reciprocal, mean, two products, division: 8 roundings
    rel = ((max(64, dim / 1024) + 12) / 2 + 1 + 8) * U24
    assert bool(((scale.double() - top / most).abs() <= rel * top / most + 2.0 ** -149).all())
    v = torch.where(top[:, None] > 0, y / (top / most)[:, None], torch.zeros_like(y))
    step = torch.full_like(v, 1.0) if q.dtype == I8 else torch.ldexp(torch.ones_like(v), (torch.frexp(v)[1] - 4).clamp(min=-9))
    # half a step, of a value that is off by rel once more through the scale
    off = (q.double() - v).abs()
    assert bool((off <= step / 2 + 2 * rel * v.abs() + 1e-12).all()), float((off - step / 2 - 2 * rel * v.abs()).max())
    if h is not None:
        tiny = float(torch.finfo(t).smallest_subnormal) if hasattr(torch.finfo(t), "smallest_subnormal") else 2.0 ** -149
        assert bool(((h.double() - xs).abs() <= xs.abs() * (half(t) * (1 + U24) + (U24 if t != F32 else 0)) + tiny).all())


@pytest.mark.parametrize("to", [I8, E4M3])
@pytest.mark.parametrize("t", [BF16, F16, F32])
@pytest.mark.parametrize("rows, dim", [(1, 1), (3, 2), (2, 8), (5, 31), (1, 64), (9, 100), (7, 128), (3, 257), (130, 512), (2, 1000), (3, 1024),
                                       (2, 1025), (1, 4096), (3, 4097), (2, 8192), (2, 8200), (1, 16384), (2, 16400), (1, 32768), (2, 40000), (1, 40001)])
def test_norm_sizes(rows, dim, t, to):
    x, r, w = rnd(1, rows, dim, dtype=t), rnd(2, rows, dim, dtype=t, scale=3.0), (1 + 0.3 * rnd(3, dim)).to(t)
    q, ok_q = guarded(rows, dim, to, pad=(-dim) % 16 + 16)
    h, ok_h = guarded(rows, dim, t, pad=(-dim) % 8 + 8)
    scale, ok_s = guarded(1, rows, F32)
    imd.norm_quantize(x, w, q, scale[0], eps=1e-5, residual=r, residual_out=h)
    norm_check(x, r, w, q, scale[0], h, 1e-5, t)
    assert ok_q() and ok_h() and ok_s()
    q2, s2 = torch.empty(rows, dim, dtype=to, device="cuda"), torch.empty(rows, device="cuda")
    assert imd.norm_quantize(x, w.float(), q2, s2, eps=1e-5, residual=r) == (q2, s2)   # h not wanted, 32-bit weight
    assert torch.equal(q2.view(torch.uint8), q.contiguous().view(torch.uint8)) and torch.equal(s2, scale[0])
    imd.norm_quantize(x, w, q2, s2, eps=0.0)
    norm_check(x, None, w, q2, s2, None, 0.0, t)


@pytest.mark.parametrize("rows", [2, 600])
@pytest.mark.parametrize("dim", [8196, 12001, 14128, 16384, 16385])
def test_norm_long_rows_of_32_bits(rows, dim):
    x, r, w = rnd(1, rows, dim), rnd(2, rows, dim, scale=3.0), 1 + 0.3 * rnd(3, dim)
    h, intact = guarded(rows, dim, F32, pad=(-dim) % 4 + 4)
    for to in (I8, E4M3):
        q, scale = torch.empty(rows, dim, dtype=to, device="cuda"), torch.empty(rows, device="cuda")
        imd.norm_quantize(x, w, q, scale, eps=1e-5, residual=r, residual_out=h)
        norm_check(x, r, w, q, scale, h, 1e-5, F32)
        assert intact()
        imd.norm_quantize(x, w, q, scale)
        norm_check(x, None, w, q, scale, None, 1e-6, F32)
    q2, s2 = torch.empty_like(q), torch.empty_like(scale)
    imd.norm_quantize(x, w, q, scale, residual=r)
    imd.norm_quantize(x, w, q2, s2, residual=r, residual_out=x)        # in place
    assert torch.equal(x, h) and torch.equal(q2.view(I8), q.view(I8)) and torch.equal(s2, scale)


@pytest.mark.parametrize("t, dim", [(BF16, 640), (F16, 4096), (F32, 2052), (BF16, 33000)])
def test_norm_strides_alignment_and_in_place(t, dim):
    rows = 5
    base = rnd(4, rows, dim + 3, dtype=t)
    w = rnd(5, dim + 1, dtype=t)[1:]
    x = base[:, 1:dim + 1]                                       # odd start, odd row distance
    r = rnd(6, 1, dim, dtype=t).expand(rows, dim)                # one residual row for all
    q, s = torch.empty(rows, dim, dtype=I8, device="cuda"), torch.empty(rows, device="cuda")
    h = torch.empty(rows, dim, dtype=t, device="cuda")
    imd.norm_quantize(x, w, q, s, residual=r, residual_out=h)
    norm_check(x, r, w, q, s, h, 1e-6, t)
    q2, s2 = torch.empty_like(q), torch.empty_like(s)
    for target in ("x", "residual"):
        a, b = x.contiguous(), r.contiguous()
        imd.norm_quantize(a, w, q2, s2, residual=b, residual_out=a if target == "x" else b)
        assert torch.equal(a if target == "x" else b, h) and torch.equal(q2, q) and torch.equal(s2, s)


@pytest.mark.parametrize("dim", [96, 1000, 4096, 33001])
@pytest.mark.parametrize("to", [I8, E4M3])
def test_norm_range(dim, to):
    """Rows of zeros, of values whose squares leave 32 bits, and rows with a NaN or an infinity."""
    x = rnd(7, 9, dim)
    x[0] = 0
    x[1] *= 1e25
    x[2] *= 1e-30
    x[3, dim // 2] = math.nan
    x[4, 0] = math.inf
    x[5, dim - 1] = -math.inf
    x[6] = 0
    x[6, dim - 1] = 1e-38                                        # one small value in a row of zeros
    x[7] *= 1e-40                                                # below the normal range
    x[8] = 3e38
    w = 1 + 0.3 * rnd(8, dim)
    for eps in (0.0, 1e-6):
        q, s = torch.empty(9, dim, dtype=to, device="cuda"), torch.empty(9, device="cuda")
        imd.norm_quantize(x, w, q, s, eps=eps)
        good = [0, 1, 2, 6, 7, 8] if eps == 0 else [0, 1, 2, 8]
        xs = x.double()
        if eps == 0:
            xs[0] = 1                                             # 0 / 0 by the formula; defined as zeros
            assert float(s[0]) == 0 and int(q[0].float().count_nonzero()) == 0
            good = good[1:]
        norm_check(x[good], None, w, q[good], s[good], None, eps, F32)
        assert torch.isnan(s[3:6]).all()
        assert int(q[3:6].count_nonzero()) == 0 if to == I8 else torch.isnan(q[3:6].float()).all()
    w[3] = math.nan
    imd.norm_quantize(x, w, q, s)
    assert torch.isnan(s[1:]).all()


@pytest.mark.parametrize("t, dim", [(BF16, 520), (F16, 1024), (F32, 1028), (BF16, 4096), (F32, 4100), (BF16, 8200), (F16, 16384), (F32, 8192), (BF16, 20480), (BF16, 5001), (F32, 1025), (F16, 579)])
def test_norm_rows_in_a_ring(t, dim):
    """Many rows (those that leave the range among them), with and without a residual, in place, broadcast."""
    rows = 5003
    x, w = rnd(11, rows, dim, dtype=t), rnd(12, dim, dtype=t)
    r = rnd(13, 1, dim, dtype=t).expand(rows, dim)
    if t == F32:
        x[17] *= 1e30
        x[4000] *= 1e-35
    x[99], x[1234, dim - 1] = 0, math.nan
    q, s = torch.empty(rows, dim, dtype=E4M3, device="cuda"), torch.empty(rows, device="cuda")
    good = [i for i in range(rows) if i not in (99, 1234)]
    imd.norm_quantize(x, w, q, s, eps=0.0)
    assert float(s[99]) == 0 and bool(torch.isnan(s[1234]))
    norm_check(x[good], None, w, q[good], s[good], None, 0.0, t)
    h = x.clone()
    imd.norm_quantize(h, w, q, s, eps=0.0, residual=r, residual_out=h)
    good = [i for i in range(rows) if i != 1234]
    norm_check(x[good], r[good], w, q[good], s[good], h[good], 0.0, t)


def test_norm_many_rows():
    rows, dim = 70001, 40
    x, w = rnd(9, rows, dim, dtype=BF16), rnd(10, dim, dtype=BF16)
    q, s = torch.empty(rows, dim, dtype=E4M3, device="cuda"), torch.empty(rows, device="cuda")
    imd.norm_quantize(x, w, q, s)
    norm_check(x, None, w, q, s, None, 1e-6, BF16)
    imd.norm_quantize(x[:0], w, q[:0], s[:0])                     # nothing to do


# ---- scaled_linear -------------------------------------------------------------------------------------------------

def check_product(out, want, size, terms, spread_check=True):
    """out against want (64 bits); size = sum of the terms' magnitudes (None: an exact integer sum)."""
    t = out.dtype
    got = out.double()
    tiny = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -25}[t]
    tol = want.abs() * (half(t) * (1 + 8 * U24) + 4 * U24) + tiny
    if size is not None:
        tol = tol + terms * 2.0 ** -23 * size * (1 + half(t))
    off = (got - want).abs()
    assert bool((off <= tol).all()), (float((off / want.abs().clamp(min=1e-30)).max()), float((off - tol).max()))
    if size is not None and t == F32 and want.numel() >= 64:
        assert float(off.norm() / want.norm()) <= max(math.sqrt(terms), terms / 16) * 2.0 ** -23


def operands8(kind, rows, n, k, seed=0):
    if kind == I8:
        x, w = ints(seed + 1, -128, 128, rows, k), ints(seed + 2, -128, 128, n, k)
    else:
        x, w = (rnd(seed + i, m, k, scale=60.0).clamp(-448, 448).to(E4M3) for i, m in ((1, rows), (2, n)))
    return x, w, 0.01 + rnd(seed + 3, rows).abs(), 0.001 * rnd(seed + 4, n)


def want8(x, w, xs, ws):
    s = xs.double()[:, None] * ws.double()
    want = (x.double() @ w.double().t()) * s
    size = None if x.dtype == I8 else (x.double().abs() @ w.double().abs().t()) * s.abs()
    return want, size


ROWS8 = [1, 2, 7, 8, 9, 16, 17, 31, 33, 64, 65, 127, 128, 129, 200, 256, 257, 300]


@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("n, k", [(1, 1), (5, 16), (16, 64), (128, 128), (257, 144), (300, 1040), (640, 4096), (96, 33), (131, 515)])
def test_scaled_linear_sizes(n, k, kind):
    for i, rows in enumerate(ROWS8):
        x, w, xs, ws = operands8(kind, rows, n, k, seed=10 * i)
        t = (F32, BF16, F16)[i % 3]
        out, intact = guarded(rows, n, t, pad=(0, 3, 8)[i % 3] if n % 8 else 8)
        assert imd.scaled_linear(x, w, out, xs, ws) is out
        want, size = want8(x, w, xs, ws)
        if t == F16:
            want = want.where(want.abs() < 65000, torch.zeros_like(want))
            out = out.where(want != 0, torch.zeros_like(out))
        check_product(out, want, size, k)
        assert intact(), (rows, n, k)


@pytest.mark.parametrize("kind", [I8, E4M3])
def test_scaled_linear_large(kind):
    for rows, n, k in [(2000, 1300, 2064), (515, 4100, 1024), (1, 20000, 2048), (48, 2048, 16384), (4097, 130, 256)]:
        x, w, xs, ws = operands8(kind, rows, n, k, seed=rows)
        out = torch.empty(rows, n, dtype=F32, device="cuda")
        imd.scaled_linear(x, w, out, xs, ws)
        check_product(out, *want8(x, w, xs, ws), k)


@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("rows", [3, 40, 300])
def test_scaled_linear_strides(rows, kind):
    n, k = 150, 272
    x, w, xs, ws = operands8(kind, rows, n, k)
    out = torch.empty(rows, n, dtype=F32, device="cuda")
    imd.scaled_linear(x, w, out, xs, ws)
    check_product(out, *want8(x, w, xs, ws), k)
    for pad, start in [(16, 16), (16, 0), (5, 1), (3, 0)]:        # rows apart, odd starts and odd distances
        bx = torch.zeros(rows, k + pad + start, dtype=torch.uint8, device="cuda").view(kind)
        bw = torch.zeros(n, k + pad + start, dtype=torch.uint8, device="cuda").view(kind)
        bx.view(torch.uint8).fill_(0x7F), bw.view(torch.uint8).fill_(0x7F)   # NaN in e4m3
        bx[:, start:start + k], bw[:, start:start + k] = x, w
        got, intact = guarded(rows, n, F32, pad=start + 1, skew=start)
        imd.scaled_linear(bx[:, start:start + k], bw[:, start:start + k], got, xs, ws)
        if kind == I8:
            assert torch.equal(got, out)
        check_product(got, *want8(x, w, xs, ws), k)
        assert intact()
    one = x[:1].expand(rows, k)                                   # one row repeated
    imd.scaled_linear(one, w, out, xs, ws)
    check_product(out, *want8(one, w, xs, ws), k)


@pytest.mark.parametrize("rows", [2, 40, 200])
def test_scaled_linear_special_values(rows):
    n, k = 200, 512
    x, w, xs, ws = operands8(I8, rows, n, k)
    x.fill_(-128), w.fill_(-128)
    x[1], xs[0], ws[3] = 127, math.nan, math.inf
    out = torch.empty(rows, n, device="cuda")
    imd.scaled_linear(x, w, out, xs, ws)
    assert torch.isnan(out[0]).all() and torch.isinf(out[1:, 3]).all()
    want, _ = want8(x, w, xs, ws)
    keep = torch.arange(n, device="cuda") != 3
    check_product(out[1:, keep], want[1:, keep], None, k)
    x, w, xs, ws = operands8(E4M3, rows, n, k)
    x[1, 5], w[7, 400] = math.nan, math.nan
    imd.scaled_linear(x, w, out, xs, ws)
    bad = torch.zeros(rows, n, dtype=torch.bool, device="cuda")
    bad[1], bad[:, 7] = True, True
    assert torch.equal(torch.isnan(out), bad)                     # a NaN stays in its row and column
    x[1, 5], w[7, 400] = 448, 448
    imd.scaled_linear(x, w, out, xs, ws)
    check_product(out, *want8(x, w, xs, ws), k)


def test_scaled_linear_depth():
    """k = 0 gives zeros; the deepest int8 sum is exact; one more is refused."""
    for kind in (I8, E4M3):
        out = torch.full((3, 5), 7.0, dtype=BF16, device="cuda")
        x, w, xs, ws = operands8(kind, 3, 5, 0)
        imd.scaled_linear(x, w, out, xs, ws)
        assert int(out.count_nonzero()) == 0
    for rows in (1, 40, 130):
        x, w = torch.full((rows, 131071), -128, dtype=I8, device="cuda"), torch.full((4, 131071), -128, dtype=I8, device="cuda")
        out = torch.empty(rows, 4, device="cuda")
        imd.scaled_linear(x, w, out, torch.ones(rows, device="cuda"), torch.ones(4, device="cuda"))
        assert bool((out == float(131071 * 16384)).all())
    x = torch.zeros(1, 131072, dtype=I8, device="cuda")
    with pytest.raises(imd.NotSupportedError):
        imd.scaled_linear(x, x, torch.empty(1, 1, device="cuda"), torch.ones(1, device="cuda"), torch.ones(1, device="cuda"))


# ---- linear_w4 -----------------------------------------------------------------------------------------------------

def operands4(t, rows, n, k, group, zeros, seed=0, st=None):
    groups = -(-k // group)
    x = rnd(seed + 1, rows, k, dtype=t)
    w = ints(seed + 2, 0, 256, n, (k + 1) // 2, dtype=torch.uint8)
    scale = (0.01 + rnd(seed + 3, n, groups, scale=0.05)).to(st or t)
    z = ints(seed + 4, 0, 16, n, groups, dtype=torch.uint8) if zeros else None
    return x, w, scale, z


def want4(x, w, scale, z, group):
    k = x.shape[1]
    q = torch.stack((w & 15, w >> 4), 2).flatten(1)[:, :k].double()
    at = torch.arange(k, device="cuda") // group
    q = (q - (8.0 if z is None else z.double()[:, at])) * scale.double()[:, at]
    return x.double() @ q.t(), x.double().abs() @ q.abs().t()


@pytest.mark.parametrize("t", [BF16, F16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n, k", [(1, 1), (3, 2), (16, 32), (130, 128), (17, 129), (200, 511), (256, 1024), (130, 1056), (520, 4096)])
def test_linear_w4_sizes(n, k, group, t):
    for i, rows in enumerate([1, 2, 5, 8, 9, 16, 17, 33, 64, 65, 130, 257]):
        x, w, scale, z = operands4(t, rows, n, k, group, i % 2 == 0, 10 * i, (None, F32, F16, BF16)[i % 4])
        out, intact = guarded(rows, n, (F32, t)[i % 3 == 2], pad=(0, 3, 8)[i % 3] if n % 8 else 8)
        assert imd.linear_w4(x, w, out, scale, zeros=z, group=group) is out
        check_product(out, *want4(x, w, scale, z, group), k)
        assert intact(), (rows, n, k)


@pytest.mark.parametrize("t, group, zeros", [(BF16, 128, False), (F16, 64, True), (BF16, 32, True)])
def test_linear_w4_large(t, group, zeros):
    for rows, n, k in [(1, 12000, 4096), (700, 1300, 2048), (33, 260, 16384), (2100, 100, 320), (16, 4096, 1000)]:
        x, w, scale, z = operands4(t, rows, n, k, group, zeros, rows)
        out = torch.empty(rows, n, dtype=F32, device="cuda")
        imd.linear_w4(x, w, out, scale, zeros=z, group=group)
        check_product(out, *want4(x, w, scale, z, group), k)


@pytest.mark.parametrize("rows", [2, 20, 150])
def test_linear_w4_strides_and_special_values(rows):
    n, k, group = 100, 384, 64
    x, w, scale, z = operands4(BF16, rows, n, k, group, True)
    want, size = want4(x, w, scale, z, group)
    for pad, start in [(16, 16), (8, 0), (5, 1)]:
        bx = torch.full((rows, k + pad + start), math.nan, dtype=BF16, device="cuda")
        bw = torch.full((n, k // 2 + pad + start), 255, dtype=torch.uint8, device="cuda")
        bs = torch.full((n, 6 + start), math.nan, dtype=BF16, device="cuda")
        bz = torch.full((n, 6 + start), 255, dtype=torch.uint8, device="cuda")
        bx[:, start:start + k], bw[:, start:start + k // 2], bs[:, :6], bz[:, :6] = x, w, scale, z
        got, intact = guarded(rows, n, F32, pad=start + 1, skew=start)
        imd.linear_w4(bx[:, start:start + k], bw[:, start:start + k // 2], got, bs[:, :6], zeros=bz[:, :6], group=group)
        check_product(got, want, size, k)
        assert intact()
    out = torch.empty(rows, n, device="cuda")
    one = scale[:, :1].expand(n, 6)                                # a scale per row: stride 0 would repeat groups, so it is laid out
    with pytest.raises(ValueError):
        imd.linear_w4(x, w, out, one, zeros=z, group=group)
    shared = scale[:1].expand(n, 6)                                # one row of scales for all outputs
    imd.linear_w4(x, w, out, shared, zeros=z, group=group)
    check_product(out, *want4(x, w, shared, z, group), k)
    x[1, 7], scale[9, 2] = math.inf, math.nan
    imd.linear_w4(x, w, out, scale, zeros=z, group=group)
    fine = torch.isfinite(out)
    assert not fine[1].any() and not fine[:, 9].any()              # an infinity and a NaN stay in their row and column
    keep = torch.arange(n, device="cuda") != 9
    others = torch.arange(rows, device="cuda") != 1
    x[1, 7] = 0
    scale[9, 2] = 0
    want, size = want4(x, w, scale, z, group)
    check_product(out[others][:, keep], want[others][:, keep], size[others][:, keep], k)
    empty = torch.full((rows, n), 7.0, dtype=BF16, device="cuda")
    imd.linear_w4(x[:, :0], w[:, :0], empty, scale[:, :0], group=group)
    assert int(empty.count_nonzero()) == 0


@pytest.mark.parametrize("t", [BF16, F16])
@pytest.mark.parametrize("n, k, group", [(130, 2048, 128), (300, 4096, 64), (129, 1792, 32), (700, 1152, 128), (19000, 1024, 128)])
def test_linear_w4_layouts_give_the_same(n, k, group, t):
    """Scales and outputs at other addresses, row distances and types: the values of the call that reads and writes whole units."""
    groups = k // group
    for rows in (3, 17, 40, 128, 200, 300) if n < 10000 else (40,):
        x, w, scale, z = operands4(t, rows, n, k, group, True, rows)
        out = torch.empty(rows, n, device="cuda")
        imd.linear_w4(x, w, out, scale, zeros=z, group=group)
        check_product(out, *want4(x, w, scale, z, group), k)
        for start, pad in [(1, 0), (0, 1), (0, 8), (8, 8), (3, 5)]:
            base = torch.full((n * (groups + pad) + start + 16,), math.nan, dtype=t, device="cuda")
            moved = base[start:start + n * (groups + pad)].view(n, groups + pad)[:, :groups]
            moved.copy_(scale)
            got = torch.empty_like(out)
            imd.linear_w4(x, w, got, moved, zeros=z, group=group)
            assert torch.equal(got, out), (rows, start, pad)
        got = torch.empty_like(out)
        imd.linear_w4(x, w, got, scale.float(), zeros=z, group=group)   # (another order of the sums is allowed)
        check_product(got, *want4(x, w, scale, z, group), k)
        for dtype in (F32, t):
            for skew, pad in [(0, -n % 8 + 8), (1, 3), (2, -n % 4 + 4), (0, -n % 2 + 1)]:
                got, intact = guarded(rows, n, dtype, pad=pad, skew=skew)
                imd.linear_w4(x, w, got, scale, zeros=z, group=group)
                assert torch.equal(got, out.to(dtype)) and intact(), (rows, dtype, skew, pad)


@pytest.mark.parametrize("k", [1, 2, 130, 255, 257, 1000, 2051])
def test_padded_rows_of_odd_length(k):
    """Rows in whole 16-byte units whose last unit is only partly theirs: what lies behind a row's end is a NaN or any
    nibble and is not seen."""
    n, group, pitch = 70, 32, -(-k // 32) * 32
    for rows in (1, 2, 16, 20, 40, 300):
        x, w, scale, z = operands4(BF16, rows, n, k, group, True, rows)
        bx = torch.full((rows, pitch), math.nan, dtype=BF16, device="cuda")
        bw = torch.full((n, pitch // 2), 255, dtype=torch.uint8, device="cuda")
        bx[:, :k], bw[:, :(k + 1) // 2] = x, w
        if k % 2:
            bw[:, k // 2] |= 0xF0
        out, intact = guarded(rows, n, F32, pad=3)
        imd.linear_w4(bx[:, :k], bw[:, :(k + 1) // 2], out, scale, zeros=z, group=group)
        check_product(out, *want4(x, w, scale, z, group), k)
        assert intact()
        for kind in (I8, E4M3):
            x, w, xs, ws = operands8(kind, rows, n, k, rows)
            bx = torch.full((rows, pitch), 0x7F, dtype=torch.uint8, device="cuda").view(kind)
            bw = torch.full((n, pitch), 0x7F, dtype=torch.uint8, device="cuda").view(kind)
            bx[:, :k], bw[:, :k] = x, w
            imd.scaled_linear(bx[:, :k], bw[:, :k], out, xs, ws)
            check_product(out, *want8(x, w, xs, ws), k)
            assert intact()


@pytest.mark.parametrize("rows, n, k", [(130, 1100, 8191), (40, 3001, 9001), (700, 901, 2047)])
def test_unaligned_rows_with_much_work(rows, n, k):
    """Odd row lengths on the tensor-core kernels: no row starts at a unit of anything."""
    for kind in (I8, E4M3):
        x, w, xs, ws = operands8(kind, rows, n, k, 7)
        out, intact = guarded(rows, n, F32, pad=1)
        imd.scaled_linear(x, w, out, xs, ws)
        check_product(out, *want8(x, w, xs, ws), k)
        assert intact()
    for t, group in ((BF16, 128), (F16, 32)):
        x, w, scale, z = operands4(t, rows, n, k, group, True, 8)
        imd.linear_w4(x, w, out, scale, zeros=z, group=group)
        check_product(out, *want4(x, w, scale, z, group), k)
        assert intact()


# ---- together ------------------------------------------------------------------------------------------------------

class Layer:
    """A feed-forward block as a decoder runs it: norm to 8 bits, 8-bit up projection, activation, 4-bit down
    projection, and the next norm, which adds the block's output to the residual stream."""

    def __init__(self, rows, dim, hidden, kind, seed=0):
        self.kind, self.group = kind, 64
        self.x, self.stream = rnd(seed + 1, rows, dim, dtype=BF16), rnd(seed + 2, rows, dim, dtype=BF16, scale=2.0)
        self.norm, self.next = (1 + 0.1 * rnd(seed + 3, dim)).to(BF16), (1 + 0.1 * rnd(seed + 4, dim)).to(BF16)
        up = rnd(seed + 5, hidden, dim, scale=dim ** -0.5)
        most = 127.0 if kind == I8 else 448.0
        self.up_scale = up.abs().amax(1) / most
        up = up / self.up_scale[:, None]
        self.up = up.round().to(I8) if kind == I8 else up.to(E4M3)
        self.down = ints(seed + 6, 0, 256, dim, hidden // 2, dtype=torch.uint8)
        self.down_scale = (0.3 * hidden ** -0.5 * (0.5 + rnd(seed + 7, dim, hidden // self.group).abs())).to(BF16)
        self.h = torch.empty_like(self.x)
        self.q, self.s = torch.empty(rows, dim, dtype=kind, device="cuda"), torch.empty(rows, device="cuda")
        self.mid = torch.empty(rows, hidden, dtype=BF16, device="cuda")
        self.act = torch.empty_like(self.mid)
        self.y = torch.empty_like(self.x)
        self.h2, self.q2, self.s2 = torch.empty_like(self.x), torch.empty_like(self.q), torch.empty_like(self.s)

    def __call__(self, stream=None):
        imd.norm_quantize(self.x, self.norm, self.q, self.s, residual=self.stream, residual_out=self.h, stream=stream)
        imd.scaled_linear(self.q, self.up, self.mid, self.s, self.up_scale, stream=stream)
        torch.mul(torch.sigmoid(self.mid), self.mid, out=self.act)
        imd.linear_w4(self.act, self.down, self.y, self.down_scale, group=self.group, stream=stream)
        imd.norm_quantize(self.y, self.next, self.q2, self.s2, residual=self.h, residual_out=self.h2, stream=stream)
        return [t.clone() for t in (self.h, self.q, self.s, self.mid, self.y, self.h2, self.q2, self.s2)]

    def check(self):
        norm_check(self.x, self.stream, self.norm, self.q, self.s, self.h, 1e-6, BF16)
        check_product(self.mid, *want8(self.q, self.up, self.s, self.up_scale), self.x.shape[1])
        check_product(self.y, *want4(self.act, self.down, self.down_scale, None, self.group), self.act.shape[1])
        norm_check(self.y, self.h, self.next, self.q2, self.s2, self.h2, 1e-6, BF16)


def same(a, b):
    return all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))


@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("rows", [1, 12, 77, 400])
def test_layer(rows, kind):
    layer = Layer(rows, 512, 1536, kind)
    first = layer()
    layer.check()
    assert same(first, layer())                                    # the same bits every time


@pytest.mark.parametrize("rows", [1, 300])
def test_layer_captured(rows):
    """A captured layer replays on new inputs, beside a second graph, and on a stream of its own."""
    a, b = Layer(rows, 512, 1024, I8, 100), Layer(rows, 640, 1280, E4M3, 200)
    eager = [a(), b()]
    graphs = []
    for layer in (a, b):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            layer(s)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = layer(s)
        graphs.append((g, out))
    for g, out in graphs:
        for t in out:
            t.view(torch.uint8).zero_()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        graphs[1][0].replay()
    graphs[0][0].replay()                                          # both in flight
    torch.cuda.synchronize()
    assert same(graphs[0][1], eager[0]) and same(graphs[1][1], eager[1])
    a.x.mul_(0.5)
    graphs[0][0].replay()
    torch.cuda.synchronize()
    a.check()


FIRST_CALL = """
import torch, immerdink_b200 as imd
x = torch.randn(40, 256, device="cuda").bfloat16()
w = torch.randint(0, 256, (300, 128), device="cuda", dtype=torch.uint8)
s = torch.rand(300, 2, device="cuda").bfloat16()
y = torch.zeros(40, 300, device="cuda", dtype=torch.bfloat16)
torch.cuda.synchronize()
g, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
with torch.cuda.graph(g, stream=stream):
    imd.linear_w4(x, w, y, s, stream=stream)
g.replay()
torch.cuda.synchronize()
z = torch.empty_like(y)
imd.linear_w4(x, w, z, s)
torch.cuda.synchronize()
assert torch.equal(y, z) and int(y.count_nonzero()) > 0
"""


def test_first_call_in_a_capture():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALL], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_two_streams_at_once():
    layers = [Layer(64, 1024, 2048, I8, 300), Layer(3, 1024, 2048, E4M3, 400)]
    want = [layer() for layer in layers]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in layers]
    for _ in range(5):
        got = []
        for layer, s in zip(layers, streams):
            with torch.cuda.stream(s):
                got.append(layer(s))
        torch.cuda.synchronize()
        assert all(same(g, w) for g, w in zip(got, want))


def test_arrays_other_than_torch():
    """__cuda_array_interface__ and DLPack producers, and an array of another library's rules."""
    class Dl:
        def __init__(self, t):
            self.t = t

        def __dlpack__(self, **kw):
            return self.t.__dlpack__(**kw)

        def __dlpack_device__(self):
            return self.t.__dlpack_device__()

    x, w, xs, ws = operands8(I8, 20, 40, 64)
    out, out2 = torch.empty(20, 40, device="cuda"), torch.empty(20, 40, device="cuda")
    imd.scaled_linear(x, w, out, xs, ws)
    cai = [imd.DeviceArray(t.data_ptr(), t.shape, None, d) for t, d in ((x, "i1"), (w, "i1"), (out2, "f4"), (xs, "f4"), (ws, "f4"))]
    imd.scaled_linear(*cai)
    assert torch.equal(out, out2)
    t, wt = rnd(3, 4, 96, dtype=BF16), rnd(4, 96, dtype=BF16)
    q, s = (torch.empty(4, 96, dtype=I8, device="cuda") for _ in range(2)), (torch.empty(4, device="cuda") for _ in range(2))
    (q, q2), (s, s2) = q, s
    imd.norm_quantize(t, wt, q, s)
    imd.norm_quantize(Dl(t), Dl(wt), Dl(q2), Dl(s2))
    assert torch.equal(q, q2) and torch.equal(s, s2)
    assert linear.load_library().current_device() == torch.cuda.current_device()


def test_long_offsets():
    """Row offsets beyond 32 bits: rows far apart in one buffer."""
    free, _ = torch.cuda.mem_get_info()
    if free < 14 << 30:
        pytest.skip("not enough free memory")
    far = (1 << 31) + 64
    big = torch.zeros(2 * far + 4096, dtype=torch.uint8, device="cuda")
    rows, k, n = 3, 256, 33
    x, w, xs, ws = operands8(I8, rows, n, k)
    xv = torch.as_strided(big.view(I8), (rows, k), (far, 1))
    xv.copy_(x)
    out = torch.empty(rows, n, device="cuda")
    imd.scaled_linear(xv, w, out, xs, ws)
    check_product(out, *want8(x, w, xs, ws), k)
    t, wt = rnd(3, 2, k, dtype=BF16), rnd(4, k, dtype=BF16)
    tv = torch.as_strided(big.view(BF16), (2, k), (far, 1), 0)
    tv.copy_(t)
    q, s = torch.empty(2, k, dtype=E4M3, device="cuda"), torch.empty(2, device="cuda")
    imd.norm_quantize(tv, wt, q, s)
    norm_check(t, None, wt, q, s, None, 1e-6, BF16)
