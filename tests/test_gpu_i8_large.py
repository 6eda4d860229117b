"""Operators of a step in 8 bits where offsets pass 32 bits: a cache of more than 2^32 codes, products and rows of more than 2^31 values."""
import pytest
import torch

from eight_ref import RefCache, kv_rows
from test_gpu_cache8 import DEV, TYPES, i32, ops
from test_gpu_i8 import BF, check_codes, i8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
def test_the_end_of_a_long_cache(dtype):
    """17 million rows, all zeros but the last 67: appended, read back, and seen by the last two tokens beside a score and a value of zero for every other row."""
    block, zeros = 64, 64 * 265625
    rows = kv_rows(torch.Generator().manual_seed(1), 1, 67)
    rows[..., 0, :] *= 4
    n = zeros + 67
    cache = ops().Cache8.empty(1, 1, n + 5, block=block, dtype=dtype, device=DEV)
    assert cache.codes.numel() > 2 ** 32
    new = rows.transpose(0, 1)[None]
    ops().cache8_append(cache, new[:, :, :, 0], new[:, :, :, 1], i32(n))
    ref = RefCache([rows], block, dtype != torch.int8)
    at = torch.arange(zeros - 3, n + 2, device=DEV)[None, None]
    got = ops().cache8_read(cache, i32(n), rows=at)[0, 0]
    assert not got[:3].any() and not got[-2:].any()
    k, v = ref.values(0, 0, 0), ref.values(0, 0, 1)
    for kv, w in ((0, k), (1, v)):
        # one product in 32 bits and one rounding
        assert ((got[3:-2, kv].double() - w).abs() <= 2.0 ** -8 * w.abs() * (1 + 2.0 ** -14)).all()
    q = (2 * torch.randn(1, 2, 3, 128, generator=torch.Generator().manual_seed(2))).to(BF).to(DEV)
    scale = 128 ** -0.5
    out = ops().cache8_attention(q, cache, i32(n)).double()
    for t in range(2):
        s = q[0, t].double() @ k[:66 + t].t() * scale
        e = torch.exp(s)
        total = zeros + e.sum(-1, keepdim=True)
        want, mean = e @ v[:66 + t] / total, e @ v[:66 + t].abs() / total
        move = 2 * 140 * 2.0 ** -24 * (q[0, t].double().abs() @ k[:66 + t].abs().t()).amax(-1, keepdim=True) * scale
        # as in test_gpu_cache8_weights; a thread's sum of weights has a few thousand terms in 32 bits
        assert ((out[0, t] - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -10 + move) * mean).all()
        assert want.abs().max() > 1e-4


def test_products_of_more_values_than_31_bits_count():
    g = torch.Generator().manual_seed(3)
    T, O = 17000, 130000
    x, w, sx, so = i8(g, T, 16), i8(g, O, 16), torch.rand(T, generator=g).to(DEV), torch.rand(O, generator=g).to(DEV)
    y = ops().matmul_i8(x, sx, w, so)
    assert y.numel() > 2 ** 31
    for t in (slice(0, 40), slice(16400, 16700), slice(T - 300, T)):
        assert torch.equal(y[t], ((x[t].double() @ w.double().t()).float() * sx[t, None] * so).to(BF))


def test_a_matrix_of_more_values_than_31_bits_count():
    g = torch.Generator().manual_seed(4)
    O, I = 140000, 16384
    w = torch.randint(-128, 128, (1, I), generator=g).to(torch.int8).to(DEV).repeat(O, 1)
    w[:, 0] = (torch.arange(O, device=DEV) % 251 - 125).to(torch.int8)
    so = torch.rand(O, generator=g).to(DEV)
    assert w.numel() > 2 ** 31
    for T in (1, 2, 20):
        x, sx = i8(g, T, I), torch.rand(T, generator=g).to(DEV)
        y = ops().matmul_i8(x, sx, w, so)
        for o in (slice(0, 200), slice(O - 9000, O)):
            assert torch.equal(y[:, o], ((x.double() @ w[o].double().t()).float() * sx[:, None] * so[o]).to(BF))


def test_rows_of_more_values_than_31_bits_count():
    B, n = 33000, 65536
    x = torch.randn(B, n, device=DEV, dtype=BF, generator=torch.Generator(DEV).manual_seed(5))
    assert x.numel() > 2 ** 31
    w = torch.ones(n, device=DEV, dtype=BF)
    h, c, s = ops().add_rmsnorm_i8(x, None, w)
    assert torch.equal(h[-300:], x[-300:])
    y = x[-300:].double()
    check_codes(c[-300:], s[-300:], y / torch.sqrt(y.square().mean(-1, keepdim=True) + 1e-6), 8 * 2.0 ** -24)
    del h
    c, s = ops().quantize_rows_i8(x)
    check_codes(c[-300:], s[-300:], y, 2.0 ** -24)
    del c
    c, s = ops().quantize_rows_i8(x, gated=True)
    gate, up = y.chunk(2, -1)
    check_codes(c[-300:], s[-300:], gate / (1 + torch.exp(-gate)) * up, 16 * 2.0 ** -24)
