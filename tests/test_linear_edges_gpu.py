"""Calls at the edges of what the quantised linear layer accepts, on a GPU, against plain 64-bit arithmetic."""
import pytest
import torch

import immerdink_b200 as imd
from immerdink_b200 import linear

pytestmark = pytest.mark.gpu
BF16, F16, F32, I8, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.int8, torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def no_wait_gave_up():
    yield
    assert linear.load_library().device_error() == 0


@pytest.mark.parametrize("rows, k, skew, gib", [(17, (1 << 30) + 64, 1, 44), (1, (1 << 31) - 1, 0, 8)])
def test_linear_w4_depth_beyond_30_bits(rows, k, skew, gib):
    """Sums whose terms lie at both ends of a row and around 2^29, 2^30 and 2^31: x is zero elsewhere, so a sum has as many
    terms as places; each term and addition rounds once (2^-24), or is cut (2^-23) in a tensor instruction."""
    if torch.cuda.mem_get_info()[0] < gib << 30:
        pytest.skip("not enough free memory")
    places = [p for p in (0, 777, (1 << 29) - 1, 1 << 29, (1 << 30) - 1, 1 << 30, (1 << 31) - 300, k - 130, k - 1) if p < k]
    x = torch.zeros(rows, k, dtype=BF16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(5)
    values = torch.randn(rows, len(places), generator=g, device="cuda").to(BF16)
    x[:, places] = values
    half, groups = (k + 1) // 2, -(-k // 128)
    w = torch.randint(0, 256, (half + skew,), generator=g, device="cuda", dtype=torch.uint8)[skew:].view(1, half)
    scale = (0.5 + torch.rand(1, groups, generator=g, device="cuda")).to(BF16)
    out = torch.empty(rows, 1, device="cuda")
    imd.linear_w4(x, w, out, scale)
    nibble = torch.stack([(w[0, p // 2] >> (4 * (p & 1))) & 15 for p in places]).double() - 8
    terms = values.double() * nibble * torch.stack([scale[0, p // 128] for p in places]).double()
    assert bool(((out[:, 0].double() - terms.sum(1)).abs() <= 2 * len(places) * 2.0 ** -23 * terms.abs().sum(1)).all())
    assert bool((terms[:, len(places) // 2:].abs().sum(1) > 0.01 * terms.abs().sum(1)).all())   # what a short walk would lose


@pytest.mark.parametrize("t", [BF16, F32])
def test_one_row_in_place_whatever_its_stride(t):
    """The last position of a sequence: buf[:, -1] and its view(1, dim) are the same row with different strides."""
    dim = 264
    buf, w = torch.randn(1, 5, dim, device="cuda").to(t), torch.randn(dim, device="cuda").to(t)
    x, same = buf[:, -1], buf[:, -1].view(1, dim)
    assert x.stride(0) != same.stride(0) and x.data_ptr() == same.data_ptr()
    r = torch.randn(1, dim, device="cuda").to(t)
    q, s, h = torch.empty(1, dim, dtype=I8, device="cuda"), torch.empty(1, device="cuda"), torch.empty(1, dim, dtype=t, device="cuda")
    imd.norm_quantize(x.clone(), w, q, s, residual=r, residual_out=h)
    before = buf.clone()
    for out, target in ((same, "x"), (x, "x"), (same, "residual"), (x, "residual")):
        buf.copy_(before)
        q2, s2 = torch.empty_like(q), torch.empty_like(s)
        first = x if out is same else same
        if target == "x":
            imd.norm_quantize(first, w, q2, s2, residual=r, residual_out=out)
        else:
            imd.norm_quantize(r, w, q2, s2, residual=first, residual_out=out)
        assert torch.equal(same, h) and torch.equal(q2, q) and torch.equal(s2, s)
        assert torch.equal(buf[:, :-1], before[:, :-1])


def test_general_way_with_tensors():
    """Without the short way of PyTorch tensors every call does the same."""
    lib = linear.Library()
    lib.fast = linear._GeneralOnly
    for rows in (1, 5):
        x, r, w = (torch.randn(*s, device="cuda").to(BF16) for s in ((rows, 96), (rows, 96), (96,)))
        got = []
        for use in (None, lib):
            q, s, h = torch.empty(rows, 96, dtype=I8, device="cuda"), torch.empty(rows, device="cuda"), torch.empty_like(x)
            y, z = torch.empty(rows, 40, dtype=BF16, device="cuda"), torch.empty(rows, 40, dtype=BF16, device="cuda")
            g = torch.Generator(device="cuda").manual_seed(3)
            w8 = torch.randint(-128, 128, (40, 96), generator=g, device="cuda", dtype=torch.int32).to(I8)
            w4 = torch.randint(0, 256, (40, 48), generator=g, device="cuda", dtype=torch.uint8)
            scale = torch.rand(40, 3, generator=g, device="cuda").to(BF16)
            assert imd.norm_quantize(x, w, q, s, residual=r, residual_out=h, lib=use) == (q, s)
            assert imd.scaled_linear(q, w8, y, s, scale[:, 0].float(), lib=use) is y
            assert imd.linear_w4(x, w4, z, scale, group=32, lib=use) is z
            got.append((q, s, h, y, z))
        assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("rows", [1, 3, 20, 77, 400])
@pytest.mark.parametrize("skew", [0, 1])
def test_columns_of_one_buffer(rows, skew):
    """Inputs and outputs in columns of one buffer, side by side without a byte between them (aligned or not): the same as in
    buffers of their own, and the columns around them stay as they were."""
    dim, n, k = 520, 136, 264
    g = torch.Generator(device="cuda").manual_seed(rows)
    raw = torch.randint(0, 256, (rows, 8192), generator=g, device="cuda", dtype=torch.uint8)
    used = torch.zeros(rows, 8192, dtype=torch.bool, device="cuda")

    def column(dtype, cols, at):
        size = torch.empty(0, dtype=dtype).element_size()
        used[:, at * size:(at + cols) * size] = True
        return raw.view(dtype)[:, at:at + cols]

    x, r, h = (column(BF16, dim, skew + i * dim) for i in range(3))        # bytes 0 to 6 dim
    q = column(I8, dim, 2 * skew + 6 * dim)
    x.normal_(generator=g), r.normal_(generator=g)
    w = torch.randn(dim, generator=g, device="cuda").to(BF16)
    before = raw.clone()
    s, s2, q2, h2 = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"), torch.empty(rows, dim, dtype=I8, device="cuda"), torch.empty(rows, dim, dtype=BF16, device="cuda")
    own_x, own_r = x.contiguous().clone(), r.contiguous().clone()
    imd.norm_quantize(x, w, q, s, residual=r, residual_out=h)
    imd.norm_quantize(own_x, w, q2, s2, residual=own_r, residual_out=h2)
    # (a whole and a shifted row may be summed in another order: the formula within a code, and h, are the same)
    assert torch.equal(h, h2) and bool(((s - s2).abs() <= 1e-6 * s2).all()) and int((q.int() - q2.int()).abs().max()) <= 1
    assert torch.equal(raw[~used], before[~used]) and torch.equal(x, own_x) and torch.equal(r, own_r)
    # 8 bits: x in one column, the output in the next
    q, y = column(I8, k, 0), column(F32, n, (k + 4) // 4 + skew)
    q.copy_(q2[:, :k])
    w8, ws = torch.randint(-128, 128, (n, k), generator=g, device="cuda", dtype=torch.int32).to(I8), torch.rand(n, generator=g, device="cuda")
    y2, used[:] = torch.empty(rows, n, device="cuda"), False
    q, y = column(I8, k, 0), column(F32, n, (k + 4) // 4 + skew)
    before = raw.clone()
    imd.scaled_linear(q, w8, y, s2, ws)
    imd.scaled_linear(q.contiguous(), w8, y2, s2, ws)
    assert torch.equal(y, y2) and torch.equal(raw[~used], before[~used])
    # 4 bits: the same, the output before x
    used[:] = False
    y, x = column(BF16, n, skew), column(BF16, k, n + skew)
    x.copy_(own_x[:, :k])
    w4 = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    scale = torch.rand(n, -(-k // 64), generator=g, device="cuda").to(BF16)
    y2, before = torch.empty(rows, n, dtype=BF16, device="cuda"), raw.clone()
    imd.linear_w4(x, w4, y, scale, group=64)
    imd.linear_w4(x.contiguous(), w4, y2, scale, group=64)
    q4 = torch.stack((w4 & 15, w4 >> 4), 2).flatten(1).double() - 8
    size = x.double().abs() @ (q4.abs() * scale.double().repeat_interleave(64, 1)[:, :k]).t()
    # (other kernels for shifted rows: two sums of k terms, each within k 2^-23 of their size, and two roundings to bf16)
    assert bool(((y.double() - y2.double()).abs() <= 2 * k * 2.0 ** -23 * size + 2 * 2.0 ** -8 * y2.double().abs() + 1e-30).all())
    assert torch.equal(raw[~used], before[~used])


def test_large_eps():
    """Rows and eps at the upper end of 32 bits: the sum of squares leaves the range, mean + eps does not."""
    rows, dim = 4, 300
    x = torch.randn(rows, dim, device="cuda")
    x *= torch.tensor([1.0, 1e17, 1e19, 1e30], device="cuda")[:, None]
    w = 1 + 0.1 * torch.randn(dim, device="cuda")
    for eps in (1e30, 1e37, 2.0 ** 127):
        q, s = torch.empty(rows, dim, dtype=I8, device="cuda"), torch.empty(rows, device="cuda")
        imd.norm_quantize(x, w, q, s, eps=eps)
        y = x.double() * torch.rsqrt(x.double().square().mean(1, keepdim=True) + eps) * w.double()
        top = y.abs().amax(1)
        rel = ((64 + 12) / 2 + 9) * 2.0 ** -24   # a chain of at most 64 additions before the root, 9 roundings after it
        assert bool(((s.double() - top / 127).abs() <= rel * top / 127 + 2.0 ** -149).all())
        v = y / (top / 127)[:, None]
        assert bool(((q.double() - v).abs() <= 0.5 + 2 * rel * v.abs() + 1e-12).all())


@pytest.mark.parametrize("rows, dim", [(1, 4096), (70, 100), (600, 1024), (5003, 640), (5003, 2052), (900, 8192), (300, 5001), (40, 16392), (9, 40001)])
@pytest.mark.parametrize("t, to", [(BF16, E4M3), (BF16, I8), (F16, E4M3), (F16, I8), (F32, E4M3)])
def test_codes_are_the_nearest(rows, dim, t, to):
    """Products g = x w of few bits: Q g / max |g| is either in the middle of two codes, which goes to the even one, or more than
    2^-22 of itself away from it, which 32 bits tell apart (24-bit quotients are off by 2^-24). Codes have to be equal."""
    g = torch.Generator(device="cuda").manual_seed(dim + rows)
    x = torch.randn(rows, dim, generator=g, device="cuda").to(BF16).to(t) if t != F16 else torch.randn(rows, dim, generator=g, device="cuda").to(F16)
    if t == BF16 and to == E4M3:
        w = (1 + 0.2 * torch.randn(dim, generator=g, device="cuda")).to(BF16)   # g: 16 bits, middle of two codes: 5 bits; 2^-21
    else:
        w = torch.exp2(torch.randint(-1, 2, (dim,), generator=g, device="cuda").float()).to(t)   # g: 8 or 11 bits, middle: 5 or 8; 2^-19
    q, s = torch.empty(rows, dim, dtype=to, device="cuda"), torch.empty(rows, device="cuda")
    imd.norm_quantize(x, w, q, s)
    p = x.double() * w.double()
    v = (127.0 if to == I8 else 448.0) * p / p.abs().amax(1, keepdim=True)      # one rounding, to 53 bits
    step = torch.ones_like(v) if to == I8 else torch.ldexp(torch.ones_like(v), (torch.frexp(v)[1] - 4).clamp(min=-9))
    assert torch.equal(torch.round(v / step) * step, q.double())
