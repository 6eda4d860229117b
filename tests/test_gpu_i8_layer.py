"""A layer's step in 8 bits, every operator's result against its definition on its own inputs."""
import pytest
import torch

from eight_ref import RefCache, attention, kv_rows
from test_gpu_i8 import BF, DEV, check_codes, ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [1, 5])
def test_a_layer_step_by_step(tokens):
    H, G, width, ff, n, block = 2, 2, 512, 768, 90, 32
    Hq = H * G
    g = torch.Generator().manual_seed(tokens)

    def matrix(rows, cols):
        w = torch.randn(rows, cols, generator=g) / cols ** 0.5
        s = w.abs().amax(-1) / 127
        return torch.round(w / s[:, None]).to(torch.int8).to(DEV), s.to(DEV)

    def product(codes, scales, w):
        """Whole-number sums, as a float times two scales, rounded once."""
        y = ops().matmul_i8(codes, scales, *w)
        want = (codes.double() @ w[0].double().t()) * scales.double()[:, None] * w[1].double()
        assert ((y.double() - want).abs() <= (2.0 ** -8 + 4 * 2.0 ** -24) * want.abs()).all()
        assert want.abs().max() > 0.1
        return y

    def norm(delta, hidden, w):
        h, c, s = ops().add_rmsnorm_i8(delta, hidden, w)
        assert torch.equal(h, (delta.float() + hidden.float()).to(BF))
        # the root, two products, a division, the maximum and 127 / 128 are rounded to 32 bits
        check_codes(c, s, h.double() / torch.sqrt(h.double().square().mean(-1, keepdim=True) + 1e-6) * w.double(), 8 * 2.0 ** -24)
        return h, c, s

    w_qkv, w_o, w_gu, w_d = matrix((Hq + 2 * H) * 128, width), matrix(width, Hq * 128), matrix(2 * ff, width), matrix(width, ff)
    n1, n2 = (1 + 0.1 * torch.randn(2, width, generator=g)).to(BF).to(DEV)
    past = kv_rows(g, H, n)
    cache = ops().Cache8.empty(1, H, 128, block=block, device=DEV)
    ops().cache8_append(cache, past[:, :, 0].transpose(0, 1)[None], past[:, :, 1].transpose(0, 1)[None], torch.tensor([n], dtype=torch.int32, device=DEV))
    hidden, delta = torch.randn(2, tokens, width, generator=g).to(BF).to(DEV)
    length = torch.tensor([n + tokens], dtype=torch.int32, device=DEV)

    h, c, s = norm(delta, hidden, n1)
    qkv = product(c, s, w_qkv).view(1, tokens, Hq + 2 * H, 128)
    ops().cache8_append(cache, qkv[:, :, Hq:Hq + H], qkv[:, :, Hq + H:], length)
    o = ops().cache8_attention(qkv[:, :, :Hq], cache, length)
    rows = torch.cat((past, qkv[0, :, Hq:].unflatten(1, (2, H)).permute(2, 0, 1, 3)), 1)
    want, _, tol = attention(RefCache([rows], block, False), qkv[:, :, :Hq], 128 ** -0.5)
    assert ((o.double() - want).abs() <= tol).all()
    c, s = ops().quantize_rows_i8(o.view(tokens, -1))
    check_codes(c, s, o.view(tokens, -1).double(), 2.0 ** -24)
    y = product(c, s, w_o)
    h2, c, s = norm(y, h, n2)
    gu = product(c, s, w_gu)
    c, s = ops().quantize_rows_i8(gu, gated=True)
    gate, up = gu.double().chunk(2, -1)
    check_codes(c, s, gate / (1 + torch.exp(-gate)) * up, 16 * 2.0 ** -24)
    product(c, s, w_d)


def test_weights_by_rows():
    """A matrix of 16 bits by quantize_rows_i8, as the integration guide has it: a row of zeros gives zeros, no code is beyond 127, and a product is off by half a code of each operand at most."""
    g = torch.Generator().manual_seed(2)
    w = (torch.randn(700, 512, generator=g) * 0.02).to(BF).to(DEV)
    w[3] = 0
    codes, scales = ops().quantize_rows_i8(w)
    assert codes.min() >= -127 and codes.abs().amax(-1).eq(127).sum() == 699 and scales[3] == 0
    x = torch.randn(9, 512, generator=g).to(BF).to(DEV)
    cx, sx = ops().quantize_rows_i8(x)
    y = ops().matmul_i8(cx, sx, codes, scales).double()
    want = x.double() @ w.double().t()
    half_x, half_w = sx.double()[:, None] / 2, scales.double()[:, None] / 2
    bound = half_x * w.double().abs().sum(-1) + (half_w * x.double().abs().sum(-1)).t() + half_x * half_w.t() * 512
    assert ((y - want).abs() <= bound * (1 + 2.0 ** -20) + 2.0 ** -8 * (want.abs() + bound) * 1.001).all() and not y[:, 3].any()
