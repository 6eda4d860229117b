"""Attention over the cache in 8 bits where its numbers cover a wide range: weights far below the largest, values and queries of very different sizes, the smallest codes, NaN under weights of next to nothing."""
import pytest
import torch

from eight_ref import RefCache
from test_gpu_cache8 import DEV, TYPES, filled, i32, ops

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def attend_all(ref, queries, scale):
    """(out, lse, tol) in 64 bits, queries bf16 [bs,T,Hq,128], the last T tokens.

    tol: the output's rounding, 2^-8 of it; and of the sum of |p v| the share that moves every weight: a weight as two bf16 numbers (2^-17) of a product in 32 bits; a score's sum of 128 products in 32 bits,
    140 * 2^-24 * |q k| scale, for the weight and for the largest score; the exponent's argument x, up to |x| ln 2, rounded three times, and 2^x to 2^-22; n / 16 sums in 32 bits that round by up to 2^-23."""
    bs, T, Hq, _ = queries.shape
    H = ref.rows[0].shape[0]
    G = Hq // H
    out, lse, tol = torch.zeros(queries.shape, dtype=torch.float64, device=DEV), torch.full((bs, T, Hq), float("-inf"), dtype=torch.float64, device=DEV), torch.zeros(queries.shape, dtype=torch.float64, device=DEV)
    for b in range(bs):
        n = ref.rows[b].shape[1]
        if n == 0:
            continue
        at = torch.arange(n, device=DEV)
        seen = (at <= n - T + torch.arange(T, device=DEV)[:, None])[:, None]   # [T,1,n]
        for h in range(H):
            k, v = ref.values(b, h, 0), ref.values(b, h, 1)
            hq = slice(h * G, (h + 1) * G)
            q = queries[b, :, hq].double()
            s = torch.where(seen, q @ k.t() * scale, float("-inf"))
            p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0) * seen
            o, mean = p @ v, p @ v.abs()
            top = torch.where(seen, s, 0.0).abs().amax(-1, keepdim=True)
            share = 2.0 ** -17 + 2.0 ** -22 + (2 * 140 + 3 * 2) * 2.0 ** -24 * torch.maximum(top, (q.abs() @ k.abs().t()).amax(-1, keepdim=True) * scale) + n / 16 * 2.0 ** -23
            out[b, :, hq], lse[b, :, hq], tol[b, :, hq] = o, torch.logsumexp(s, -1) / torch.log(torch.tensor(2.0, dtype=torch.float64)), 2.0 ** -8 * o.abs() + share * mean
    return out, lse, tol


def check(rows, block, dtype, q, scale=128 ** -0.5):
    cache = filled(rows, block, dtype)
    out = ops().cache8_attention(q, cache, i32(*[r.shape[1] for r in rows]), scale=scale).double()
    want, _, tol = attend_all(RefCache(rows, block, dtype == torch.float8_e4m3fn), q, scale)
    off = (out - want).abs()
    assert (off <= tol + 2.0 ** -126).all(), (float((off / (tol + 2.0 ** -126)).max()), float(out.abs().max()), float(want.abs().max()))


def sink(g, H, n, drop, q_shape):
    """One key that has all but 2^-drop of each weight's share, of value zero, in front of a long tail: the tail is the output.  The tail's scores differ by a fifth of a nat or so."""
    x = torch.zeros(H, n, 2, 128)
    x[:, 0, 0, 0] = drop / (16 * 128 ** -0.5 * 1.4427)
    x[:, 1:, 0, 1] = 2 * torch.randn(H, n - 1, generator=g)
    x[:, 1:, 1] = 1 + 0.25 * torch.randn(H, n - 1, 128, generator=g)
    q = torch.zeros(*q_shape, 128)
    q[..., 0], q[..., 1] = 16.0, 1.0
    return x.to(BF).to(DEV), q.to(BF).to(DEV)


# heads, query heads each, tokens, rows: items of eight, sixteen and 32 query rows (the last two where there are many tiles)
SHAPES = [(1, 4, 1, 9000), (1, 3, 2, 700), (2, 16, 1, 29000), (2, 8, 4, 29000)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,G,T,n", SHAPES)
@pytest.mark.parametrize("drop", [12, 22, 26, 31, 60, 110])
def test_a_long_tail_behind_a_key_of_value_zero(dtype, H, G, T, n, drop):
    g = torch.Generator().manual_seed(drop)
    x, q = sink(g, H, n, drop, (1, T, H * G))
    check([x], 16, dtype, q)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("G", [2, 12])
def test_values_that_begin_with_zeros(dtype, G):
    """Every other tile has values of zero, the others very small ones: what a warp meets first says nothing of what follows."""
    g = torch.Generator().manual_seed(3)
    rows = []
    for _ in range(40):
        x = torch.zeros(4, 700, 2, 128)
        x[:, :, 0] = 0.1 * torch.randn(4, 700, 128, generator=g)
        x[:, :, 1] = 1e-6 * (1 + 0.25 * torch.randn(4, 700, 128, generator=g)) * (torch.arange(700) // 128 % 2)[:, None]
        rows.append(x.to(BF).to(DEV))
    check(rows, 64, dtype, torch.randn(40, 1, 4 * G, 128, generator=g).to(BF).to(DEV))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,G,T,n", SHAPES)
def test_queries_with_a_channel_that_no_key_has(dtype, H, G, T, n):
    """A query's largest value does not cost the others their bits."""
    g = torch.Generator().manual_seed(4)
    x = torch.randn(H, n, 2, 128, generator=g)
    x[:, :, 0, 9] = 0.0
    q = torch.randn(1, T, H * G, 128, generator=g)
    q[..., 9] = 2.0 ** 40
    check([x.to(BF).to(DEV)], 32, dtype, q.to(BF).to(DEV))


@pytest.mark.parametrize("H,G,T,n", SHAPES)
def test_the_smallest_codes(H, G, T, n):
    """e4m3 codes below 2^-6, which are whole multiples of 2^-9, in all channels that count."""
    g = torch.Generator().manual_seed(5)
    x = torch.randint(-7, 8, (H, n, 2, 128), generator=g).float() * 2.0 ** -9
    x[..., 1, :] = x[..., 1, :].abs()
    x[..., 5] = 448.0
    q = 2 * torch.randn(1, T, H * G, 128, generator=g)
    q[..., 5] = 0.0
    check([x.to(BF).to(DEV)], 64, torch.float8_e4m3fn, q.to(BF).to(DEV), scale=3.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,G,T,n", SHAPES)
def test_a_block_that_is_not_a_number_under_weights_of_nothing(dtype, H, G, T, n):
    """A block that holds an infinity reads as NaN: no weight is too small for that, whichever blocks of the grid share the sequence."""
    for row in (40, n // 2, n - 200):
        x, q = sink(torch.Generator().manual_seed(6), H, n, 400, (1, T, H * G))
        x[:, row, 1, 3] = float("inf")
        cache = filled([x], 16, dtype)
        assert ops().cache8_attention(q, cache, i32(n)).isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,G,T,n", SHAPES)
def test_an_infinity_behind_the_blocks_under_weights_of_nothing(dtype, H, G, T, n):
    """A row in 16 bits by itself: the channel is an infinity, or 0 times one, and the others are as they were."""
    x, q = sink(torch.Generator().manual_seed(7), H, n, 400, (1, T, H * G))
    x[:, n - T, 1, 3] = float("inf")   # seen by every token
    assert (n - T) // 16 == n // 16
    out = ops().cache8_attention(q, filled([x], 16, dtype), i32(n))
    assert not out[..., 3].isfinite().any()
    assert out[..., :3].isfinite().all() and out[..., 4:].isfinite().all()
