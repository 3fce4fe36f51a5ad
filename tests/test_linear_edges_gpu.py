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
