"""The cache in 8 bits: rows in, rows back, attention over it, against the definitions in 64 bits."""
import pytest
import torch

from eight_ref import RefCache, attention, kv_rows

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.int8, torch.float8_e4m3fn]


def ops():
    from pariskv_b200 import ops as o
    return o


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def append(cache, rows, lengths, before):
    """The rows of each sequence from before[b] on, as one call with counts."""
    T = max(n - m for n, m in zip(lengths, before))
    bs, H = len(rows), rows[0].shape[0]
    new = torch.full((bs, T, H, 2, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    for b, (n, m) in enumerate(zip(lengths, before)):
        new[b, :n - m] = rows[b][:, m:n].transpose(0, 1)
    ops().cache8_append(cache, new[:, :, :, 0], new[:, :, :, 1], i32(*lengths), i32(*[n - m for n, m in zip(lengths, before)]))


def filled(rows, block, dtype, cap=None, recent=None, cuts=None):
    """A cache of these rows, appended in the pieces that `cuts` (lengths per sequence) name."""
    bs, H = len(rows), rows[0].shape[0]
    lengths = [r.shape[1] for r in rows]
    cache = ops().Cache8.empty(bs, H, cap or max(max(lengths), 1), block=block, dtype=dtype, recent=recent, device=DEV)
    before = [0] * bs
    for upto in (cuts or []) + [lengths]:
        append(cache, rows, upto, before)
        before = upto
    return cache


def samples(lengths, H=2, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [kv_rows(g, H, n) for n in lengths]


def check_cache(cache, rows, block, dtype):
    ref = RefCache(rows, block, dtype == torch.float8_e4m3fn)
    R = cache.recent.shape[2]
    for b, x in enumerate(rows):
        n, full = x.shape[1], ref.whole(b)
        for h in range(x.shape[0]):
            for kv in range(2):
                c, s = ref.coded(b, h, kv)
                assert torch.equal(cache.codes[b, h, :full, kv].double(), c)
                # one division in 32 bits
                assert torch.allclose(cache.scales[b, h, :full // block, kv].double(), s, rtol=2.0 ** -24, atol=0)
        kept = torch.arange(max(0, n - R), n, device=DEV)
        assert torch.equal(cache.recent[b][:, kept % R], x[:, kept])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("lengths", [(1, 0), (15, 16), (127, 129), (300, 65)])
def test_append_whole(dtype, block, lengths):
    rows = samples(lengths)
    cache = filled(rows, block, dtype)
    check_cache(cache, rows, block, dtype)
    # nothing behind the whole blocks has been touched
    for b, n in enumerate(lengths):
        assert not cache.codes[b, :, n // block * block:].view(torch.uint8).any() and not cache.scales[b, :, n // block:].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("block,recent", [(16, 16), (16, 32), (32, 32), (64, 192)])
@pytest.mark.parametrize("step", [1, 3, 16, 50, 170])
def test_append_in_pieces_is_append_at_once(dtype, block, recent, step):
    """Also where new rows replace, in the same call, the rows that a block is coded from."""
    lengths = (333, 290)
    rows = samples(lengths, H=1, seed=3)
    cuts = [[min(n, i) for n in lengths] for i in range(7, 333, step)]
    cache = filled(rows, block, dtype, recent=recent, cuts=cuts)
    once = filled(rows, block, dtype, recent=recent)
    check_cache(cache, rows, block, dtype)
    assert torch.equal(cache.codes.view(torch.uint8), once.codes.view(torch.uint8)) and torch.equal(cache.scales, once.scales)


def test_rows_taken_back_leave_no_trace():
    block, n = 16, 40
    rows, other = samples([n], seed=1), samples([n + 30], seed=2)
    mixed = [torch.cat((rows[0][:, :33], other[0][:, 33:]), 1)]
    cache = filled([mixed[0][:, :33]], block, torch.int8, cap=96, recent=32)
    wrong = [torch.cat((rows[0][:, :33], samples([17], seed=5)[0]), 1)]
    append(cache, wrong, [49], [33])        # completes a block, 16 rows = R - block too many
    append(cache, mixed, [33 + 37], [33])   # other rows in their place
    ref = RefCache(mixed, block, False)
    for kv in range(2):
        c, s = ref.coded(0, 0, kv)
        assert torch.equal(cache.codes[0, 0, :64, kv].double(), c)


@pytest.mark.parametrize("dtype", TYPES)
def test_append_layouts(dtype):
    """Separate tensors for K and V, heads innermost, values that are views of a projection's row."""
    block, n, H = 32, 100, 3
    rows = samples([n, n], H=H)
    cap, R = 128, 64
    codes = torch.zeros(2, 2, cap, H, 128, dtype=torch.uint8, device=DEV).view(dtype).permute(1, 3, 2, 0, 4)   # [kv][bs][cap][H]
    scales = torch.zeros(2, 4, 2, H, device=DEV).permute(2, 3, 1, 0)
    recent = torch.zeros(2, 2, H, R, 128, dtype=torch.bfloat16, device=DEV).permute(1, 2, 3, 0, 4)
    cache = ops().Cache8(codes, scales, recent, block)
    qkv = torch.randn(2, n, (2 + 2 * H) * 128, device=DEV).to(torch.bfloat16)
    k, v = (qkv[..., (2 + i * H) * 128:(2 + (i + 1) * H) * 128].unflatten(-1, (H, 128)) for i in (0, 1))
    for b in range(2):
        k[b], v[b] = rows[b][:, :, 0].transpose(0, 1), rows[b][:, :, 1].transpose(0, 1)
    ops().cache8_append(cache, k, v, i32(n, n))
    check_cache(cache, rows, block, dtype)
    got = ops().cache8_read(cache, i32(n, n))
    want = RefCache(rows, block, dtype == torch.float8_e4m3fn)
    for b in range(2):
        for h in range(H):
            for kv in range(2):
                w = want.values(b, h, kv)
                assert ((got[b, h, :n, kv].double() - w).abs() <= 2.0 ** -8 * w.abs() * (1 + 2.0 ** -20)).all()


def test_append_out_of_range():
    """Rows below zero and behind the cache are left out; counts below zero and above T are cut off."""
    block, H = 16, 1
    rows = samples([60], H=H)
    cache = ops().Cache8.empty(4, H, 40, block=block, recent=32, device=DEV)
    new = rows[0].transpose(0, 1)[None].expand(4, -1, -1, -1, -1).contiguous()   # 60 rows
    ops().cache8_append(cache, new[:, :, :, 0], new[:, :, :, 1], i32(50, 20, -5, 33), i32(50, 60, 60, -3))
    part = ops().Cache8(cache.codes[:1], cache.scales[:1], cache.recent[:1], block)
    check_cache(part, [rows[0][:, :40]], block, torch.int8)
    part = ops().Cache8(cache.codes[1:2], cache.scales[1:2], cache.recent[1:2], block)
    check_cache(part, [rows[0][:, 40:60]], block, torch.int8)
    assert not cache.codes[2:].any() and not cache.recent[2:].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_append_values_at_the_borders(dtype):
    """Ties, zeros, the largest and the smallest numbers, infinities and NaN."""
    block = 16
    x = torch.zeros(1, 8 * block, 2, 128)
    x[0, :, :, :64] = torch.arange(-32, 32) / 32.0 * 127          # halves of codes, ties among them
    x[0, :, :, 64] = 127.0
    x[0, block:2 * block] = 0.0
    x[0, 2 * block:3 * block] *= 2.0 ** 120                       # near the top of the range
    x[0, 3 * block:4 * block] *= 2.0 ** -139                      # below the normal numbers
    x[0, 4 * block + 3, 0, 5] = float("inf")
    x[0, 5 * block + 3, 1, 5] = float("nan")
    x[0, 6 * block:7 * block] = torch.randint(-255, 256, (block, 2, 128), generator=torch.Generator().manual_seed(1)).float()   # quotients that are near ties
    x[0, 7 * block:] = torch.randint(1, 256, (block, 2, 128), generator=torch.Generator().manual_seed(2)).float() * 2.0 ** torch.randint(-12, 1, (block, 2, 128)).float()
    rows = [x.to(torch.bfloat16).to(DEV)]
    cache = filled(rows, block, dtype)
    ref = RefCache(rows, block, dtype == torch.float8_e4m3fn)
    for kv in range(2):
        c, s = ref.coded(0, 0, kv)
        assert torch.equal(cache.codes[0, 0, :, kv].double(), c)
        ok = s.isfinite()
        assert torch.equal(cache.scales[0, 0, :, kv].isnan().cpu(), (~ok).cpu())
        assert torch.allclose(cache.scales[0, 0, ok, kv].double(), s[ok], rtol=2.0 ** -24, atol=2.0 ** -150)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("block,lengths", [(16, (0, 1)), (32, (64, 95)), (128, (700, 127)), (64, (64, 63))])
def test_read(dtype, block, lengths):
    rows = samples(lengths)
    cache = filled(rows, block, dtype, cap=max(lengths) + 9)
    ref = RefCache(rows, block, dtype == torch.float8_e4m3fn)
    out = torch.full((2, 2, max(lengths) + 9, 2, 128), 3.0, dtype=torch.bfloat16, device=DEV)
    assert ops().cache8_read(cache, i32(*lengths), out=out) is out
    g = torch.Generator().manual_seed(9)
    at = torch.randint(-3, max(lengths) + 4, (2, 2, 77), generator=g)
    at[..., :4] = torch.tensor([2 ** 40, -2 ** 40, 0, 0])
    listed = ops().cache8_read(cache, i32(*lengths), rows=at.to(DEV))
    short = ops().cache8_read(cache, i32(*lengths), out=torch.full((2, 2, 5, 2, 128), 3.0, dtype=torch.bfloat16, device=DEV))
    assert torch.equal(short, out[:, :, :5])
    for b, n in enumerate(lengths):
        assert (out[b, :, n:] == 3).all()
        for h in range(2):
            for kv in range(2):
                w = ref.values(b, h, kv)
                # one product in 32 bits and one rounding
                assert ((out[b, h, :n, kv].double() - w).abs() <= 2.0 ** -8 * w.abs() * (1 + 2.0 ** -14)).all()
                ok = (at[b, h] >= 0) & (at[b, h] < n)
                assert torch.equal(listed[b, h, ok.to(DEV), kv], out[b, h, at[b, h][ok].to(DEV), kv])
                assert not listed[b, h, (~ok).to(DEV), kv].any()


def queries(g, bs, T, Hq):
    q = torch.randn(bs, T, Hq, 128, generator=g)
    return (q * (4.0 / q.norm(dim=-1, keepdim=True))).to(torch.bfloat16).to(DEV)


def check_attention(rows, block, dtype, T, Hq, scale=128 ** -0.5, cap=None, seed=0, cache=None, q=None):
    cache = cache or filled(rows, block, dtype, cap=cap)
    g = torch.Generator().manual_seed(seed + 77)
    q = queries(g, len(rows), T, Hq) if q is None else q
    lse = torch.empty(len(rows), T, Hq, device=DEV)
    out = ops().cache8_attention(q, cache, i32(*[r.shape[1] for r in rows]), scale=scale, lse=lse)
    want, want_lse, tol = attention(RefCache(rows, block, dtype == torch.float8_e4m3fn), q, scale)
    assert ((out.double() - want).abs() <= tol + 1e-30).all(), ((out.double() - want).abs() - tol).max()
    empty = want_lse == float("-inf")
    assert torch.equal(lse == float("-inf"), empty) and not out[empty].any()
    # the sum's rounding, and that of the scores: 140 * 2^-24 * |q| |k| scale log2 e, with |q| = 4 and keys of a norm up to some 200
    assert (lse[~empty].double() - want_lse[~empty]).abs().max() <= 140 * 2.0 ** -24 * 4 * 200 * scale * 1.45 + 2.0 ** -18 if (~empty).any() else True
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("lengths", [(0, 1), (15, 16), (127, 128), (129, 300), (701, 1000)])
def test_attention_lengths(dtype, block, lengths):
    check_attention(samples(lengths), block, dtype, 1, 8)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,H,G", [(1, 1, 1), (2, 2, 3), (4, 1, 4), (3, 2, 5), (5, 1, 7), (16, 2, 8), (33, 1, 1), (1, 1, 40), (7, 3, 2)])
def test_attention_heads_and_tokens(dtype, T, H, G):
    check_attention(samples((260, T - 1, 77), H=H, seed=T), 32, dtype, T, H * G)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_of_a_long_sequence(dtype):
    """Several blocks of the grid share an item, others have the end of one and the begin of the next."""
    check_attention(samples((30011, 5, 9000), H=1, seed=4), 64, dtype, 2, 4)


@pytest.mark.parametrize("scale", [1e-12, 0.02, 3.0])
def test_attention_scales(scale):
    check_attention(samples((150, 97)), 16, torch.int8, 2, 4, scale=scale)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_values_of_very_different_sizes(dtype):
    """Weights times value scales cover more than fp16 does: the largest scores at the smallest values, and the other way round."""
    rows = samples((500,), H=1)
    size = 2.0 ** torch.linspace(-60, 60, 500)
    for order in (size, size.flip(0)):
        x = rows[0].clone()
        x[0, :, 1] = (x[0, :, 1].float() * order[:, None].to(DEV)).to(torch.bfloat16)
        check_attention([x], 16, dtype, 1, 2)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_queries_of_very_different_sizes(dtype):
    rows = samples((200,), H=1)
    g = torch.Generator().manual_seed(5)
    q = queries(g, 1, 6, 4)
    q[0, 0] *= 0
    q[0, 1] *= 2.0 ** -100
    q[0, 2] *= 2.0 ** -20
    q[0, 3] *= 2.0 ** 3
    q[0, 4, :, 1:] *= 2.0 ** -30
    check_attention(rows, 32, dtype, 6, 4, q=q)


@pytest.mark.parametrize("n", [64, 70, 80])
@pytest.mark.parametrize("dtype", TYPES)
def test_what_a_query_does_not_see_does_not_reach_it(dtype, n):
    """Infinities and NaN in later rows, in whole blocks and behind them, and whatever lies behind the sequence."""
    block, T = 16, 8
    rows = samples((n,), H=1)
    cache = filled(rows, block, dtype, cap=96, recent=32)
    q = queries(torch.Generator().manual_seed(1), 1, T, 4)
    length = i32(n)
    good = ops().cache8_attention(q, cache, length)
    whole = n // block * block
    cache.codes[:, :, whole:] = torch.tensor(127, dtype=torch.int8, device=DEV).view(torch.uint8).view(dtype) if dtype != torch.int8 else 127
    cache.scales[:, :, whole // block:] = float("nan")
    held = torch.arange(whole, n, device=DEV) % 32
    free = torch.ones(32, dtype=torch.bool, device=DEV)
    free[held] = False
    cache.recent[0, :, free] = float("nan")
    assert torch.equal(ops().cache8_attention(q, cache, length), good)
    for kind in (float("inf"), float("nan")):
        for kv in (0, 1):
            x = rows[0].clone()
            x[0, n - 1, kv, 3] = kind
            bad = filled([x], block, dtype, cap=96, recent=32)
            out = ops().cache8_attention(q, bad, length)
            if n > whole:   # the last row is by itself: only the last token sees it
                assert torch.equal(out[:, :-1], good[:, :-1])
                last = out[0, -1]
                if kv == 1:
                    assert (last[:, 3].isnan().all() if kind != kind else (last[:, 3] == kind).all()) and last[:, :3].isfinite().all() and last[:, 4:].isfinite().all()
            else:           # its block reads as NaN: so do the tokens that see a row of it; the block before it they see too
                first = max(0, whole - block - (n - T))
                assert torch.equal(out[:, :first], good[:, :first]) and out[0, -1].isnan().all() if kv == 0 else out[0, -1].isnan().any()


def test_queries_that_are_not_numbers():
    rows = samples((100, 10), H=1)
    q = queries(torch.Generator().manual_seed(1), 2, 2, 4)
    cache = filled(rows, 16, torch.int8)
    good = ops().cache8_attention(q, cache, i32(100, 10))
    q[:, 0, 1, 5], q[:, 1, 2, 0] = float("nan"), float("-inf")
    out = ops().cache8_attention(q, cache, i32(100, 10))
    assert out[:, 0, 1].isnan().all() and out[:, 1, 2].isnan().all()
    keep = torch.ones(2, 2, 4, dtype=torch.bool)
    keep[:, 0, 1] = keep[:, 1, 2] = False
    assert torch.equal(out[keep.to(DEV)], good[keep.to(DEV)])


def test_lengths_outside_the_cache():
    rows = samples((64,), H=1)
    cache = filled(rows, 16, torch.int8)
    q = queries(torch.Generator().manual_seed(1), 1, 2, 4)
    good = ops().cache8_attention(q, cache, i32(64))
    assert torch.equal(ops().cache8_attention(q, cache, i32(1000)), good)
    assert not ops().cache8_attention(q, cache, i32(-7)).any() and not ops().cache8_attention(q, cache, i32(-2 ** 31)).any()


def test_a_graph_of_a_growing_sequence_and_other_streams():
    """One captured step - rows in, attention - serves every length; two graphs and an eager call at once have their own scratch."""
    block, n, T = 16, 50, 60
    rows = samples((n + T,), H=2, seed=8)
    q = queries(torch.Generator().manual_seed(3), 1, T, 8)
    want = []
    cache = filled([rows[0][:, :n]], block, torch.int8, cap=n + T)
    for i in range(T):
        append(cache, [rows[0][:, :n + i + 1]], [n + i + 1], [n + i])
        want.append(ops().cache8_attention(q[:, i:i + 1], cache, i32(n + i + 1)))
    graphs = []
    for _ in range(2):
        c = filled([rows[0][:, :n]], block, torch.int8, cap=n + T)
        k, v, qi, length = torch.empty(1, 1, 2, 128, dtype=torch.bfloat16, device=DEV), torch.empty(1, 1, 2, 128, dtype=torch.bfloat16, device=DEV), torch.empty_like(q[:, :1]), i32(n)
        graph, out = torch.cuda.CUDAGraph(), torch.empty_like(q[:, :1])
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            length.add_(1)
            ops().cache8_append(c, k, v, length)
            ops().cache8_attention(qi, c, length, out=out)
        graphs.append((graph, k, v, qi, length, c, out))   # (the graph does not keep the cache alive)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(T):
        torch.cuda.synchronize()
        for (graph, k, v, qi, length, _, out), s in zip(graphs, streams):
            k.copy_(rows[0][:, n + i, 0][None, None]), v.copy_(rows[0][:, n + i, 1][None, None]), qi.copy_(q[:, i:i + 1])
        torch.cuda.synchronize()
        for (graph, *_), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for g in graphs:
            assert torch.equal(g[-1], want[i])


def test_empty_calls():
    rows = samples((20,), H=1)
    cache = filled(rows, 16, torch.int8)
    before = cache.codes.clone()
    ops().cache8_append(cache, torch.empty(1, 0, 1, 128, dtype=torch.bfloat16, device=DEV), torch.empty(1, 0, 1, 128, dtype=torch.bfloat16, device=DEV), i32(20))
    assert torch.equal(cache.codes, before)
    assert ops().cache8_attention(torch.empty(1, 0, 4, 128, dtype=torch.bfloat16, device=DEV), cache, i32(20)).shape == (1, 0, 4, 128)
    assert ops().cache8_read(cache, i32(20), rows=torch.empty(1, 1, 0, dtype=torch.int64, device=DEV)).shape == (1, 1, 0, 2, 128)
