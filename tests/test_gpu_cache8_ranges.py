"""Attention over long caches in 8 bits where a thread block has several tiles: items of eight, sixteen and 32 query rows, ranges that end where items do or anywhere, whole items inside a range, two ranges a place, more
samples than a warp has lanes.  One sequence stands for all: its cache is expanded over samples and heads, every sample has a length of its own."""
import pytest
import torch

from eight_ref import code_block, kv_rows
from test_gpu_cache8 import DEV, TYPES, i32, ops, queries

pytestmark = pytest.mark.gpu
TILE = 128


class Shared:
    """A sequence of one head of n rows, its cache with every row in 16 bits too, so that any length is as if there were no more, and what that holds in 64 bits."""

    def __init__(self, n, block, dtype):
        self.n, self.block = n, block
        self.rows = kv_rows(torch.Generator().manual_seed(n), 1, n)
        places = -(-n // block) * block
        self.cache = ops().Cache8.empty(1, 1, n, block=block, dtype=dtype, recent=places, device=DEV)
        x = self.rows.transpose(0, 1)[None]
        ops().cache8_append(self.cache, x[:, :, :, 0], x[:, :, :, 1], i32(n))
        full = n // block * block
        self.values = []
        for kv in range(2):
            parts = [code_block(self.rows[0, j:j + block, kv].double(), dtype == torch.float8_e4m3fn) for j in range(0, full, block)]
            self.values.append(torch.cat([c * s for c, s in parts]))

    def prefix(self, n, kv):
        whole = n // self.block * self.block
        return torch.cat((self.values[kv][:whole], self.rows[0, whole:n, kv].double()))


_shared = {}


def shared(n, block, dtype):
    if (n, block, dtype) not in _shared:
        _shared.clear()
        _shared[n, block, dtype] = Shared(n, block, dtype)
    return _shared[n, block, dtype]


def check(n, block, dtype, lengths, H, T, G, item):
    """item: query rows of an item, and the ranges: (rows, ranges, with what scratch says of both)."""
    from pariskv_b200 import _lib as L
    one, bs, Hq = shared(n, block, dtype), len(lengths), H * G
    rows, ranges = item
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert L.load().pk_cache8_attention_workspace_bytes(bs, T, Hq, H, n) == 2 * ranges * (2 if rows == 32 else 3) * sms * rows * 130 * 4
    tiles = [max(1, -(-(m // block * block) // TILE) + (m % block > 0)) for m in lengths]
    assert sum(tiles) * H * -(-T * G // rows) > ranges * (2 if rows == 32 else 3) * sms   # more tiles than thread blocks
    wide = lambda t: t.expand(bs, H, *t.shape[2:])   # noqa: E731
    cache = ops().Cache8(wide(one.cache.codes), wide(one.cache.scales), wide(one.cache.recent), block)
    q = queries(torch.Generator().manual_seed(bs + T), bs, T, Hq)
    lse = torch.empty(bs, T, Hq, device=DEV)
    scale = 128 ** -0.5
    out = ops().cache8_attention(q, cache, i32(*lengths), lse=lse).double()
    again = ops().cache8_attention(q, cache, i32(*lengths)).double()
    assert torch.equal(out, again)
    for b, m in enumerate(lengths):
        k, v = one.prefix(m, 0), one.prefix(m, 1)
        x = q[b].double()                                                   # [T,Hq,128]
        seen = (torch.arange(m, device=DEV) <= m - T + torch.arange(T, device=DEV)[:, None])[:, None]
        s = torch.where(seen, x @ k.t() * scale, float("-inf"))
        p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0) * seen
        # as in test_gpu_cache8_weights: weights of 17 bits, scores of 128 sums, exponents, sums over the rows
        move = (2 * 140 + 3 * 2) * 2.0 ** -24 * (x.abs() @ k.abs().t()).amax(-1, keepdim=True) * scale if m else 0.0
        tol = 2.0 ** -8 * (p @ v).abs() + (2.0 ** -17 + 2.0 ** -22 + move + m / 16 * 2.0 ** -23) * (p @ v.abs())
        assert ((out[b] - p @ v).abs() <= tol).all(), (b, m, float(((out[b] - p @ v).abs() - tol).max()))
        want = torch.logsumexp(s, -1) / torch.log(torch.tensor(2.0, dtype=torch.float64))
        empty = want == float("-inf")
        assert torch.equal(lse[b] == float("-inf"), empty) and not out[b][empty].any()
        if (~empty).any():
            assert (lse[b][~empty].double() - want[~empty]).abs().max() <= 1.45 * (float(move.max()) if m else 0.0) + m / 16 * 2.0 ** -23 + 2.0 ** -18


UNEVEN = [20000, 17, 12001, 0, 128, 19999, 5000, 1, 129, 8192, 300]
# four and eight query rows are items of eight, 12 of 16, 24 of 32, 40 two of them
CASES = [(1, 4, 8), (1, 8, 8), (3, 4, 16), (6, 4, 32), (5, 8, 32)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,G,rows", CASES)
@pytest.mark.parametrize("block", [16, 128])
def test_ranges_over_the_ends_of_items(dtype, T, G, rows, block):
    """Long and short sequences, one without rows, side by side: a range has the end of an item, whole ones, the begin of another."""
    check(20000, block, dtype, UNEVEN, 2, T, G, (rows, 1))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,G,rows", CASES)
@pytest.mark.parametrize("lengths", [(20000, 19000, 18003, 20000, 17777), (20000, 16001, 14000)])
def test_ranges_that_end_where_the_items_do(dtype, T, G, rows, lengths):
    """Few long items of about the same size: uneven shares of several thread blocks each."""
    check(20000, 64, dtype, list(lengths), 4, T, G, (rows, 1))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,G,rows", CASES)
def test_more_samples_than_lanes(dtype, T, G, rows):
    """40 samples with 20 or so tiles a thread block, the longest in the middle."""
    check(20000, 32, dtype, [(i * 1237 + 300) % 9000 for i in range(20)] + [20000] + [(i * 3001) % 9000 for i in range(19)], 2, T, G, (rows, 1 if T * G <= 32 else 2))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,G,rows", CASES[:3])
@pytest.mark.parametrize("lengths", ["even", "uneven"])
def test_two_ranges_a_place(dtype, T, G, rows, lengths):
    check(20000, 64, dtype, [20000 - 64 * i if lengths == "even" else (20000, 0, 777, 9001)[i % 4] for i in range(36)], 4, T, G, (rows, 2))


def test_tokens_of_a_piece_of_a_prompt():
    """256 tokens: 64 items of 32 query rows a head, the first rows of which end well before the last."""
    check(20000, 64, torch.int8, [20000, 255, 9000], 2, 256, 8, (32, 2))
