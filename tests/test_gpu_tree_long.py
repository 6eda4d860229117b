"""Attention for several tokens where a block of the launch has many tiles: rings that are filled again and again, sums that are scaled on the
way, ranges with several whole items.  The tolerance is that of many_ref.py."""
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


def make(seed, bs, T, H, G, cap, lengths, spread=1.0):
    r = rnd(seed)
    d = dict(queries=r(bs, T, H * G, 128) * spread, keys=r(bs, H, cap, 128), values=r(bs, H, cap, 128), draft_keys=r(bs, T, H, 128), draft_values=r(bs, T, H, 128),
             tree_mask=r(bs, T, T) > 0.2, lengths=i32(lengths))
    d["tree_mask"] |= torch.eye(T, dtype=torch.bool, device=DEV)
    d["tree_mask"][:, T // 2] = False
    for b, n in enumerate(lengths):
        d["keys"][b, :, n:] = float("nan")
        d["values"][b, :, n:] = float("nan")
    return d


def check(d, lengths):
    """many_ref.tree, all tokens of a KV head at once."""
    from pariskv_b200 import ops
    q = d["queries"]
    bs, T, Hq, _ = q.shape
    H = d["keys"].shape[1]
    G = Hq // H
    lse = torch.full((bs, T, Hq), 7.0, device=DEV)
    out = ops.tree_attention(**d, lse=lse)
    for b in range(bs):
        n = lengths[b]
        for h in range(H):
            k, v = torch.cat((d["keys"][b, h, :n], d["draft_keys"][b, :, h])).double(), torch.cat((d["values"][b, h, :n], d["draft_values"][b, :, h])).double()
            qs = q[b, :, h * G:h * G + G].reshape(T * G, 128).double()
            hidden = torch.cat((torch.zeros(T, n, dtype=torch.bool, device=DEV), ~d["tree_mask"][b]), 1).repeat_interleave(G, 0)
            s = (qs @ k.t() * 128 ** -0.5).masked_fill(hidden, float("-inf"))
            w = torch.softmax(s, -1).masked_fill(hidden.all(-1, keepdim=True), 0.0)   # (a row that sees nothing: zeros)
            want = w @ v
            ds = (qs.abs() @ k.abs().t()).amax(-1) * 128 ** -0.5 * 128 * 2.0 ** -23
            tol = R.U * want.abs() + (R.U * (1 + R.U) + 2 * ds[:, None] + (n + T) * 2.0 ** -23 + 2.0 ** -20) * (w @ v.abs())
            R.close(out[b, :, h * G:h * G + G].reshape(T * G, 128), want, tol, f"out {b} {h}")
            l = torch.logsumexp(s, -1) / 0.6931471805599453
            R.close(lse[b, :, h * G:h * G + G].reshape(-1), l, (ds + (n + T) * 2.0 ** -23 + 2.0 ** -20) / 0.69 + l.abs() * 2.0 ** -23, f"lse {b} {h}")
    return out


ROWS = [(2, 4), (4, 4), (8, 4), (9, 4), (9, 8), (16, 8), (61, 4), (33, 8), (256, 2)]   # 8, 16, 32 rows per KV head, 36 .. 128, and more


@pytest.mark.parametrize("T,G", ROWS)
def test_many_tiles_of_few_items(T, G):
    check(make(T, 1, T, 8, G, 24100, [24077]), [24077])


@pytest.mark.parametrize("T,G", [(4, 4), (40, 1), (33, 4), (33, 8), (256, 2)])
def test_many_items_of_every_length(T, G):
    """Several whole items in a block's range, and items that begin in one block and end in another."""
    lengths = [(37 * i * i) % 1300 for i in range(40)]
    check(make(T + 1, 40, T, 8, G, 1300, lengths), lengths)


@pytest.mark.parametrize("T,G", ROWS)
@pytest.mark.parametrize("way", ["slow", "fast", "down", "saw"])
def test_scores_that_grow_on_the_way(T, G, way):
    """Scores that grow by about 2 and 20 (log2) from one tile of 128 keys to the next, fall, or rise and fall every few tiles."""
    n = 16000
    d = make(T + 2, 1, T, 4, G, n, [n])
    at = torch.arange(n, device=DEV) / 128
    grow = dict(slow=2 * at, fast=20 * at, down=-5 * at, saw=30 * (at % 7))[way]
    d["queries"][..., 0] = 8
    d["draft_keys"][..., 0] = 0
    d["keys"][..., 0] = (grow * 0.6931 * 128 ** 0.5 / 8).to(torch.bfloat16)
    check(d, [n])


@pytest.mark.parametrize("T,G", [(9, 4), (61, 4)])
@pytest.mark.parametrize("layout", ["pairs", "token_major", "fused_rows"])
def test_strides(T, G, layout):
    bs, H, cap, lengths = 2, 2, 5000, [5000, 3333]
    d = make(T + 3, bs, T, H, G, cap, lengths)
    if layout == "pairs":
        store = torch.stack((d["keys"], d["values"]), 3)
        d["keys"], d["values"] = store[:, :, :, 0], store[:, :, :, 1]
    elif layout == "token_major":
        for name in ("keys", "values"):
            d[name] = d[name].transpose(1, 2).contiguous().transpose(1, 2)
        d["tree_mask"] = d["tree_mask"].transpose(1, 2).contiguous().transpose(1, 2)
    else:
        row = torch.cat((d["queries"], d["draft_keys"], d["draft_values"]), 2)
        d["queries"], d["draft_keys"], d["draft_values"] = row.split((H * G, H, H), 2)
    check(d, lengths)


@pytest.mark.parametrize("T,G", [(9, 8), (61, 4)])
def test_captured_and_replayed_while_the_sequences_grow(T, G):
    from pariskv_b200 import ops
    d = make(T + 4, 2, T, 4, G, 12000, [12000, 12000])
    ops.tree_attention(**d)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.tree_attention(**d)
    for lengths in ([11, 12000], [0, 5000], [11999, 128]):
        d["lengths"].copy_(i32(lengths))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, check(d, lengths))


@pytest.mark.parametrize("G", [1, 4, 8, 16, 20, 32])
def test_many_tiles_of_listed_blocks(G):
    from pariskv_b200 import ops
    r = rnd(G)
    bs, T, H, n, block, lengths = 2, 2, 8, 100, 64, [12000, 6401]
    keys, values, q = r(bs, H, 12000, 128), r(bs, H, 12000, 128), r(bs, T, H * G, 128)
    ids = torch.stack([torch.randperm(190, generator=torch.Generator().manual_seed(i))[:n] for i in range(bs * T * H)]).view(bs, T, H, n).to(torch.int32).to(DEV)
    lse = torch.zeros(bs, T, H * G, device=DEV)
    out = ops.block_attention(q, keys, values, ids, i32(lengths), block=block, lse=lse)
    want, tol, wl, ltol = R.block_attention(q, keys, values, ids, lengths, block)
    R.close(out, want, tol, "out")
    R.close(lse, wl, ltol, "lse")


@pytest.mark.parametrize("T,G", [(4, 4), (9, 4), (40, 4)])
def test_a_chain_of_drafts_is_causal_attention_over_all_blocks(T, G):
    """The tree over a chain's drafts, and attention over every block once the drafts' rows are in the cache."""
    from pariskv_b200 import ops
    n, cap = 3000, 3100
    d = make(T + 5, 1, T, 2, G, cap, [n])
    d["tree_mask"] = torch.ones(1, T, T, dtype=torch.bool, device=DEV).tril()
    tree = check(d, [n])
    keys, values = d["keys"].clone(), d["values"].clone()
    keys[:, :, n:n + T], values[:, :, n:n + T] = d["draft_keys"].transpose(1, 2), d["draft_values"].transpose(1, 2)
    ids = torch.arange(49, dtype=torch.int32, device=DEV).expand(1, T, 2, 49).contiguous()
    out = ops.block_attention(d["queries"], keys, values, ids, i32([n + T]), block=64)
    want, tol, _, _ = R.block_attention(d["queries"], keys, values, ids, [n + T], 64)
    R.close(out, want, tol)
    R.close(tree, want, tol)
