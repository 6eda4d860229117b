"""What the cache in 8 bits promises, where a mistake would show: what a token does not see, and rows that were taken back."""
import pytest
import torch

from eight_ref import RefCache
from test_gpu_cache8 import DEV, TYPES, append, check_attention, check_cache, filled, i32, ops, queries, samples

pytestmark = pytest.mark.gpu


# heads, query heads each, rows: clusters and ranges, items of eight, sixteen (the last) and 32 query rows; whole blocks only, and rows behind them
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,G,n", [(1, 4, 64), (2, 1, 309), (1, 4, 5000), (2, 2, 29000), (2, 4, 29003), (1, 1, 29003)])
@pytest.mark.parametrize("kind", ["inf", "nan"])
@pytest.mark.parametrize("kv", [0, 1])
def test_a_block_that_some_tokens_do_not_see(dtype, H, G, n, kind, kv):
    """The last whole block holds an infinity or NaN and reads as NaN: the tokens before it get what they got, those that see a row of it get NaN in every channel."""
    block, T = 16, 40
    rows = samples((n,), H=H, seed=n)
    q = queries(torch.Generator().manual_seed(2), 1, T, H * G)
    good = ops().cache8_attention(q, filled(rows, block, dtype), i32(n))
    whole = n // block * block
    first = T - block - (n - whole)   # tokens whose rows end before the block
    assert 0 < first < T
    for at in (whole - block, whole - 5, whole - 1):
        x = rows[0].clone()
        x[:, at, kv, 3] = float(kind)
        out = ops().cache8_attention(q, filled([x], block, dtype), i32(n))
        assert torch.equal(out[:, :first], good[:, :first])
        assert out[:, first:].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("block,recent", [(16, 32), (32, 96), (64, 128), (128, 256)])
@pytest.mark.parametrize("n,more", [(33, 0), (47, 16), (130, 7), (300, 200)])
def test_rows_taken_back(dtype, block, recent, n, more):
    """R - block rows too many, which may complete blocks, are taken back: what is left, and what it becomes with other rows in their place, is as if they had never been there."""
    wrong = recent - block
    kept, bad, good = samples((n,), seed=1)[0], samples((wrong,), seed=2)[0], samples((wrong + more,), seed=3)[0]
    cache = filled([torch.cat((kept, bad), 1)], block, dtype, cap=n + wrong + more, recent=recent, cuts=[[n]])
    # taken back: what is left
    once = filled([kept], block, dtype, cap=n + wrong + more, recent=recent)
    q = queries(torch.Generator().manual_seed(4), 1, 3, 4)
    assert torch.equal(ops().cache8_read(cache, i32(n))[:, :, :n], ops().cache8_read(once, i32(n))[:, :, :n])
    assert torch.equal(ops().cache8_attention(q, cache, i32(n)), ops().cache8_attention(q, once, i32(n)))
    # other rows in their place, a few at first
    rows = torch.cat((kept, good), 1)
    append(cache, [rows[:, :n + 1]], [n + 1], [n])
    append(cache, [rows], [rows.shape[1]], [n + 1])
    check_cache(cache, [rows], block, dtype)
    check_attention([rows], block, dtype, 3, 4, cache=cache)
    got, want = ops().cache8_read(cache, i32(rows.shape[1]))[0, :, :rows.shape[1]].double(), RefCache([rows], block, dtype == torch.float8_e4m3fn)
    for h in range(rows.shape[0]):
        for kv in range(2):
            w = want.values(0, h, kv)
            # one product in 32 bits and one rounding
            assert ((got[h, :, kv] - w).abs() <= 2.0 ** -8 * w.abs() * (1 + 2.0 ** -14)).all()
