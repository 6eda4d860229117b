"""Rows in 8 bits whose values lie below the normal numbers of 32 bits: codes are still y 127 / max |y| to the nearest."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV, BF = "cuda", torch.bfloat16


def ops():
    from pariskv_b200 import ops as o
    return o


def check(codes, scales, y):
    """y f64 [B,n], whole multiples of 2^-149 of at most 16 bits, so that a quotient is a tie or 2^-17 away from one: 32 bits find its side."""
    assert torch.equal((y * 2.0 ** 149).round(), y * 2.0 ** 149) and y.abs().max() * 2.0 ** 149 < 2 ** 16
    top = y.abs().amax(-1, keepdim=True)
    assert torch.equal(codes.cpu().double(), torch.round(y * 127 / top))
    # the scale is rounded to a multiple of 2^-149
    assert ((scales.cpu().double() - top[:, 0] / 127).abs() <= 2.0 ** -150).all()


@pytest.mark.parametrize("n", [8, 712, 4096, 9000])
@pytest.mark.parametrize("least", [-149, -146])
def test_gated_rows(n, least):
    """silu(g) = g / 2 for g of 2^-60: the products are whole multiples of 2^least, in the second row the largest of them is that itself."""
    g = torch.Generator().manual_seed(n)
    gate, up = torch.randint(1, 16, (3, n), generator=g).double(), torch.randint(-15, 16, (3, n), generator=g).double()
    gate[1], up[1] = 1, torch.randint(0, 2, (n,), generator=g).double()
    up[1, 0] = 1
    gate[2], up[2] = 100, torch.randint(-7, 8, (n,), generator=g).double()
    up[2, 0] = 7   # 700 2^least
    x = torch.cat((gate * 2.0 ** -60, up * 2.0 ** (least + 61)), -1).to(BF).to(DEV)
    codes, scales = ops().quantize_rows_i8(x, gated=True)
    check(codes, scales, gate * up * 2.0 ** least)


@pytest.mark.parametrize("n", [64, 1024])
def test_normed_rows(n):
    """A row whose largest value has a weight of zero, the others one of 2^-133."""
    g = torch.Generator().manual_seed(n)
    h = torch.randint(-127, 128, (4, n), generator=g).float()
    h[:, 0] = 2.0 ** 13 * n ** 0.5
    h[:, 1] = torch.tensor([127.0, 127.0, -90.0, 77.0])
    w = torch.full((n,), 2.0 ** -133)
    w[0] = 0
    x = h.to(BF)
    _, codes, scales = ops().add_rmsnorm_i8(x.to(DEV), None, w.to(BF).to(DEV), eps=0.0)
    rstd = (1 / x.double().square().mean(-1, keepdim=True).sqrt()).float().double()
    y = ((x.double() * rstd).float().double() * 2.0 ** -133 * 2.0 ** 149).round() * 2.0 ** -149   # each product rounded to 32 bits
    y[:, 0] = 0
    assert (y != 0).any(-1).all()
    check(codes, scales, y)
