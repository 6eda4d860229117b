"""Block bounds, selection of blocks and attention over them against the definitions."""
import pytest
import torch

import many_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rnd(seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return lambda *s: torch.randn(*s, generator=g, device=DEV).to(torch.bfloat16)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("bs,H,cap,lengths", [(1, 1, 1, [1]), (2, 3, 200, [200, 0]), (3, 2, 1000, [999, 64, 65]), (2, 1, 4097, [4097, -3]),
                                              (1, 8, 20000, [30000]), (20, 1, 70, list(range(20)))])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_bounds(bs, H, cap, lengths, block):
    from pariskv_b200 import ops
    keys = rnd(cap + block)(bs, H, cap, 128)
    old = torch.full((bs, H, (cap + block - 1) // block, 2, 128), 9.0, dtype=torch.bfloat16, device=DEV)
    for n_new in (None, 0, 1, 3, block, 2 * block + 1, cap + 5):
        got = old.clone()
        assert ops.block_bounds(keys, i32(lengths), block=block, n_new=n_new, bounds=got) is got
        assert torch.equal(got, R.bounds(keys, lengths, block, old, n_new)), n_new
    want = R.bounds(keys, [cap] * bs, block, old)
    assert torch.equal(ops.block_bounds(keys, block=block), want)


def test_bounds_of_strided_keys_with_nan_and_infinities():
    from pariskv_b200 import ops
    store = rnd(1)(2, 3, 150, 2, 128)
    keys = store[:, :, :, 1]
    keys[0, 0, 5, 7], keys[0, 1, 70, 3], keys[1, 2, 149, 0], keys[1, 0, :, 9] = float("nan"), float("inf"), float("-inf"), -0.0
    big = torch.zeros(2, 3, 5, 2, 128, dtype=torch.bfloat16, device=DEV)
    got = ops.block_bounds(keys, i32([150, 140]), block=32, bounds=big)
    want = R.bounds(keys, [150, 140], 32, torch.zeros_like(big))
    assert torch.equal(got.nan_to_num(77.0, 1e30, -1e30), want.nan_to_num(77.0, 1e30, -1e30))
    assert got[0, 0, 0, :, 7].isnan().all()


SELECT = [(1, 1, 1, 1, 16, [1], 1, 16, 0, 1), (1, 1, 2, 4, 700, [700], 5, 16, 1, 1), (2, 3, 2, 3, 1000, [1000, 2], 6, 32, 1, 2), (1, 2, 1, 8, 5000, [4999], 33, 16, 2, 3),
          (3, 1, 2, 5, 300, [300, 64, 0], 4, 64, 0, 1), (2, 16, 1, 4, 900, [900, 10], 7, 128, 1, 1), (1, 1, 8, 4, 40000, [39990], 32, 64, 1, 2),
          (1, 1, 1, 2, 200000, [199999], 100, 16, 1, 1), (1, 1, 2, 16, 2100, [2100], 40, 64, 3, 4), (2, 40, 1, 1, 260, [260, 39], 3, 16, 0, 2)]


@pytest.mark.parametrize("bs,T,H,G,cap,lengths,n,block,sink,local", SELECT)
def test_selection(bs, T, H, G, cap, lengths, n, block, sink, local):
    from pariskv_b200 import ops
    r = rnd(cap + n)
    keys, q = r(bs, H, cap, 128), r(bs, T, H * G, 128)
    bnd = ops.block_bounds(keys, i32(lengths), block=block, bounds=torch.full((bs, H, (cap + block - 1) // block, 2, 128), float("nan"), dtype=torch.bfloat16, device=DEV))
    got = ops.select_blocks(q, bnd, i32(lengths), n, block=block, sink_blocks=sink, local_blocks=local)
    want = R.select(q.cpu(), bnd.cpu(), lengths, n, block, sink, local)
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("bs,T,H,nb,n", [(4, 1, 16, 3000, 20), (3, 4, 8, 2100, 17), (1, 2, 300, 70, 9), (2, 1, 1, 33, 4)])
@pytest.mark.parametrize("gaps", [False, True])
def test_selection_of_long_rows(bs, T, H, nb, n, gaps):
    """Many steps for every block of the launch; bounds that lie next to each other and bounds with gaps, which hold NaN."""
    from pariskv_b200 import ops
    r = rnd(nb)
    store = torch.full((bs, H, nb + 2, 3, 128), float("nan"), dtype=torch.bfloat16, device=DEV)
    bnd = store[:, :, 1:nb + 1, :2]
    bnd.copy_(r(bs, H, nb, 2, 128).sort(3).values)
    if not gaps:
        bnd = bnd.contiguous()
    lengths = [nb * 32 - 700 * b for b in range(bs)]
    lengths[-1] = nb * 32
    q = r(bs, T, 2 * H, 128)
    got = ops.select_blocks(q, bnd, i32(lengths), n, block=32, sink_blocks=1, local_blocks=2)
    qs, lo, hi = q.double().view(bs, T, H, 2, 128), bnd[..., 0, :].double(), bnd[..., 1, :].double()
    P, N = qs.clamp(min=0).sum(3), qs.clamp(max=0).sum(3)
    score = (torch.einsum("bthd,bhjd->bthj", P, hi) + torch.einsum("bthd,bhjd->bthj", N, lo)).float()
    for b in range(bs):
        for t in range(T):
            seen = (lengths[b] - T + t) // 32 + 1
            s = score[b, t, :, :seen].clone()
            s[:, 0] = s[:, seen - 2:] = float("inf")
            want = s.sort(dim=1, descending=True, stable=True).indices[:, :n].sort(dim=1).values
            assert torch.equal(got[b, t].long(), want), (b, t)


def test_ties_go_to_the_lower_block():
    from pariskv_b200 import ops
    r = rnd(2)
    bnd = r(1, 1, 1, 2, 128).sort(3).values.expand(1, 1, 300, 2, 128).contiguous()
    bnd[:, :, 250] += 8      # one block above the others
    q = r(1, 1, 2, 128).abs()
    got = ops.select_blocks(q, bnd, i32([300 * 16]), 20, block=16, sink_blocks=2, local_blocks=3)
    assert got.flatten().tolist() == list(range(16)) + [250, 297, 298, 299]


@pytest.mark.parametrize("nb,T,n", [(300, 1, 20), (5000, 3, 33), (20000, 1, 7)])
def test_scores_that_32_bit_sums_confuse(nb, T, n):
    """Blocks whose channels are permutations of each other: equal scores, which sums in 32 bits tell apart by their order; and a few that
    are above the others by less than such a sum is off."""
    from pariskv_b200 import ops
    g = torch.Generator().manual_seed(nb)
    base = (torch.randn(128, generator=g) * 1000).to(torch.bfloat16)
    hi = torch.stack([base[torch.randperm(128, generator=g)] for _ in range(nb)])
    better = torch.randperm(nb - 20, generator=g)[:n // 2] + 10
    for i, j in enumerate(better.tolist()):   # the smallest magnitude a little larger: by less than one part in 10^7 of the sum of magnitudes
        at = hi[j].abs().argmin()
        hi[j, at] = hi[j, at].abs() + 2.0 ** -6 * (1 + i % 3)
    bnd = torch.stack((torch.full_like(hi, -3.0), hi), 1).view(1, 1, nb, 2, 128).to(DEV)
    q = torch.ones(1, T, 2, 128, dtype=torch.bfloat16, device=DEV)
    got = ops.select_blocks(q, bnd, i32([nb * 16]), n, block=16, sink_blocks=1, local_blocks=1)
    assert torch.equal(got.cpu(), R.select(q.cpu(), bnd.cpu(), [nb * 16], n, 16, 1, 1))


def test_scores_that_are_not_numbers():
    """NaN above all others, -inf and zeros of both signs below; sink and local blocks all the same."""
    from pariskv_b200 import ops
    bnd = torch.zeros(1, 1, 64, 2, 128, dtype=torch.bfloat16, device=DEV)
    bnd[:, :, :, 1] = 0.0
    bnd[:, :, 5:9] = float("nan")
    bnd[:, :, 20, :] = float("-inf")
    bnd[:, :, 30, :] = float("inf")
    bnd[:, :, 33, :, 0] = -0.0
    q = torch.ones(1, 1, 1, 128, dtype=torch.bfloat16, device=DEV)
    pick = lambda n: ops.select_blocks(q, bnd, i32([64 * 16]), n, block=16, sink_blocks=1, local_blocks=1).flatten().tolist()
    assert pick(2) == [0, 63]
    assert pick(5) == [0, 5, 6, 7, 63]
    assert pick(7) == [0, 5, 6, 7, 8, 30, 63]
    assert pick(9) == [0, 1, 2, 5, 6, 7, 8, 30, 63]
    assert pick(63) == [j for j in range(64) if j != 20]
    assert pick(70) == list(range(64)) + [-1] * 6


@pytest.mark.parametrize("first", [-50.0, 0.001, 10.0, 300.0])
@pytest.mark.parametrize("nb,T", [(60, 1), (3000, 2), (17000, 1)])
def test_more_scores_that_are_not_numbers_than_are_taken(first, nb, T):
    """Twenty NaN among scores of every size: the lowest of them are taken."""
    from pariskv_b200 import ops
    bnd = torch.zeros(1, 1, nb, 2, 128, dtype=torch.bfloat16, device=DEV)
    bnd[0, 0, :, :, 0] = (first + torch.arange(nb, device=DEV) % 40)[:, None].to(torch.bfloat16)
    bnd[:, :, 30:50] = float("nan")
    q = torch.zeros(1, T, 1, 128, dtype=torch.bfloat16, device=DEV)
    q[..., 0] = 1
    got = ops.select_blocks(q, bnd, i32([nb * 16]), 9, block=16, sink_blocks=1, local_blocks=1)
    assert got[0, -1, 0].tolist() == [0, *range(30, 37), nb - 1]
    assert got[0, 0, 0].tolist() == [0, *range(30, 37), nb - 1]


@pytest.mark.parametrize("bs,T,H,G,cap,lengths,n,block,sink,local", SELECT)
def test_attention_over_selected_blocks(bs, T, H, G, cap, lengths, n, block, sink, local):
    from pariskv_b200 import ops
    r = rnd(cap + n + 1)
    keys, values, q = r(bs, H, cap, 128), r(bs, H, cap, 128), r(bs, T, H * G, 128)
    for b, m in enumerate(lengths):
        keys[b, :, m:], values[b, :, m:] = float("nan"), float("nan")
    bnd = ops.block_bounds(keys, i32(lengths), block=block)
    ids = ops.select_blocks(q, bnd, i32(lengths), n, block=block, sink_blocks=sink, local_blocks=local)
    lse = torch.full(q.shape[:3], 7.0, device=DEV)
    out = ops.block_attention(q, keys, values, ids, i32(lengths), block=block, lse=lse)
    want, tol, wl, ltol = R.block_attention(q, keys, values, ids, lengths, block)
    R.close(out, want, tol, "out")
    R.close(lse, wl, ltol, "lse")


@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_lists_in_any_order_with_gaps_and_repeats(block):
    from pariskv_b200 import ops
    r = rnd(block)
    bs, T, H, G, cap, lengths = 2, 3, 2, 4, 900, [900, 333]
    keys, values, q = r(bs, H, cap, 128), r(bs, H, cap, 128), r(bs, T, H * G, 128) * 2
    nb = (cap + block - 1) // block
    ids = torch.randint(-2, nb + 3, (bs, T, H, 9), generator=torch.Generator().manual_seed(block)).to(torch.int32)
    ids[0, 0, 0] = -1
    ids[0, 1, 1, 2:5] = 1
    ids[0, 2, 0, 3] = 2 ** 31 - 1
    ids = ids.to(DEV)
    out = ops.block_attention(q, keys, values, ids, i32(lengths), block=block)
    want, tol, _, _ = R.block_attention(q, keys, values, ids.clamp(max=nb + 3), lengths, block)
    R.close(out, want, tol)
    assert (out[0, 0, :G] == 0).all()


@pytest.mark.parametrize("G,n", [(1, 1), (4, 9), (16, 40), (20, 300)])
def test_a_query_that_is_not_a_number(G, n):
    from pariskv_b200 import ops
    r = rnd(G)
    keys, values, q = r(1, 2, 6000, 128), r(1, 2, 6000, 128), r(1, 2, 2 * G, 128)
    q[0, 1, G] = float("nan")
    ids = torch.arange(n, dtype=torch.int32, device=DEV).expand(1, 2, 2, n).contiguous()
    lse = torch.zeros(1, 2, 2 * G, device=DEV)
    out = ops.block_attention(q, keys, values, ids, i32([6000]), block=16, lse=lse)
    assert out[0, 1, G].isnan().all() and lse[0, 1, G].isnan()
    want, tol, _, _ = R.block_attention(q, keys, values, ids, [6000], 16)
    R.close(out, want, tol)
    assert int(out.isnan().sum()) == 128


def test_strided_cache_and_queries():
    from pariskv_b200 import ops
    r = rnd(4)
    store = r(2, 2, 500, 2, 128)
    keys, values = store[:, :, :, 0], store[:, :, :, 1]
    q = r(2, 5, 12, 128)[:, 1:4, 2:10]
    bnd = ops.block_bounds(keys, i32([500, 77]), block=16)
    ids = ops.select_blocks(q, bnd, i32([500, 77]), 6, block=16)
    assert torch.equal(ids.cpu(), R.select(q.cpu(), bnd.cpu(), [500, 77], 6, 16, 1, 1))
    out = ops.block_attention(q, keys, values, ids, i32([500, 77]), block=16, scale=0.3)
    want, tol, _, _ = R.block_attention(q, keys, values, ids, [500, 77], 16, 0.3)
    R.close(out, want, tol)


def test_one_head_of_keys_for_all():
    """Strides of zero: keys, values and bounds expanded over the KV heads."""
    from pariskv_b200 import ops
    r = rnd(8)
    keys, values, q = r(2, 1, 700, 128).expand(2, 3, 700, 128), r(2, 1, 700, 128).expand(2, 3, 700, 128), r(2, 2, 6, 128)
    bnd = ops.block_bounds(keys[:, :1], i32([700, 65]), block=32).expand(2, 3, 22, 2, 128)
    ids = ops.select_blocks(q, bnd, i32([700, 65]), 5, block=32)
    assert torch.equal(ids.cpu(), R.select(q.cpu(), bnd.cpu(), [700, 65], 5, 32, 1, 1))
    out = ops.block_attention(q, keys, values, ids, i32([700, 65]), block=32)
    want, tol, _, _ = R.block_attention(q, keys, values, ids, [700, 65], 32)
    R.close(out, want, tol)


def test_head_groups_of_every_size():
    from pariskv_b200 import ops
    for G in (1, 2, 7, 9, 16, 17, 32, 128):
        r = rnd(G)
        keys, values, q = r(1, 1, 300, 128), r(1, 1, 300, 128), r(1, 2, G, 128)
        ids = i32([[[[0, 2, 4]], [[1, 2, 4]]]])
        out = ops.block_attention(q, keys, values, ids, i32([290]), block=64)
        want, tol, _, _ = R.block_attention(q, keys, values, ids, [290], 64)
        R.close(out, want, tol, f"G={G}")


def test_captured_step_while_the_sequences_grow():
    """Append a row, update the bounds, select, attend: one captured graph, positions on the device."""
    from pariskv_b200 import ops
    r = rnd(5)
    bs, H, G, cap, block = 2, 2, 4, 600, 32
    keys, values = torch.zeros(bs, H, cap, 128, dtype=torch.bfloat16, device=DEV), torch.zeros(bs, H, cap, 128, dtype=torch.bfloat16, device=DEV)
    start = [500, 95]
    for b in range(bs):
        keys[b, :, :start[b]], values[b, :, :start[b]] = r(H, start[b], 128), r(H, start[b], 128)
    lengths = i32(start)
    bnd = ops.block_bounds(keys, lengths, block=block, bounds=torch.zeros(bs, H, 19, 2, 128, dtype=torch.bfloat16, device=DEV))
    q, k_new, v_new = r(bs, 1, H * G, 128), r(bs, H, 1, 128), r(bs, H, 1, 128)

    def step():
        at = lengths.long()[:, None, None, None].expand(-1, H, 1, 128)
        keys.scatter_(2, at, k_new)
        values.scatter_(2, at, v_new)
        lengths.add_(1)
        ops.block_bounds(keys, lengths, block=block, n_new=1, bounds=bnd)
        ids = ops.select_blocks(q, bnd, lengths, 5, block=block, sink_blocks=1, local_blocks=2)
        return ids, ops.block_attention(q, keys, values, ids, lengths, block=block)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ids, out = step()
    for i in range(70):
        q.copy_(r(bs, 1, H * G, 128)), k_new.copy_(r(bs, H, 1, 128)), v_new.copy_(r(bs, H, 1, 128))
        g.replay()
        if i % 23 == 0 or i == 69:
            n = [s + 2 + i for s in start]
            want = R.bounds(keys, n, block, torch.zeros_like(bnd))
            assert torch.equal(bnd, want)
            assert torch.equal(ids.cpu(), R.select(q.cpu(), want.cpu(), n, 5, block, 1, 2))
            o, tol, _, _ = R.block_attention(q, keys, values, ids, n, block)
            R.close(out, o, tol)


def test_refusals():
    from pariskv_b200 import ops
    r = rnd(6)
    keys, values, q, lengths = r(2, 2, 64, 128), r(2, 2, 64, 128), r(2, 1, 4, 128), i32([64, 3])
    bnd = ops.block_bounds(keys, lengths, block=16)
    ids = ops.select_blocks(q, bnd, lengths, 2, block=16)
    bad = (RuntimeError, TypeError, ValueError)
    for call in (lambda: ops.block_bounds(keys, lengths, block=24), lambda: ops.block_bounds(keys, lengths, block=0), lambda: ops.block_bounds(keys.float(), lengths),
                 lambda: ops.block_bounds(keys, lengths, n_new=1), lambda: ops.block_bounds(keys, lengths, n_new=-1, bounds=bnd),
                 lambda: ops.block_bounds(keys, lengths, block=32, bounds=bnd), lambda: ops.block_bounds(keys, lengths[:1]), lambda: ops.block_bounds(keys[..., :64], lengths),
                 lambda: ops.block_bounds(keys.cpu(), lengths),
                 lambda: ops.select_blocks(q, bnd, lengths, 2, block=16, sink_blocks=2), lambda: ops.select_blocks(q, bnd, lengths, 2, block=16, local_blocks=0),
                 lambda: ops.select_blocks(q, bnd, lengths, 0, block=16), lambda: ops.select_blocks(q[:, :, :3], bnd, lengths, 2, block=16),
                 lambda: ops.select_blocks(q, bnd[:, :, :, :1], lengths, 2, block=16), lambda: ops.select_blocks(q, bnd, lengths.long(), 2, block=16),
                 lambda: ops.block_attention(q, keys, values, ids.long(), lengths, block=16), lambda: ops.block_attention(q, keys, values, ids[:, :, :1], lengths, block=16),
                 lambda: ops.block_attention(q, keys, values, ids, lengths, block=48), lambda: ops.block_attention(q, keys, values[:, :1], ids, lengths, block=16),
                 lambda: ops.block_attention(q, keys, values, ids, None, block=16), lambda: ops.block_attention(q[..., ::2], keys, values, ids, lengths, block=16)):
        with pytest.raises(bad):
            call()
