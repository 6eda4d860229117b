"""Attention of drafted tokens over a cache against the definition in 64 bits."""
import math

import pytest
import torch

import many_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(seed, bs, T, H, G, cap, lengths, stale=float("nan"), spread=1.0, shared_mask=False, empty=0.1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).to(torch.bfloat16)
    d = dict(queries=r(bs, T, H * G, 128) * spread, keys=r(bs, H, cap, 128), values=r(bs, H, cap, 128), draft_keys=r(bs, T, H, 128),
             draft_values=r(bs, T, H, 128), lengths=torch.tensor(lengths, dtype=torch.int32, device=DEV))
    mask = torch.rand(1 if shared_mask else bs, T, T, generator=g, device=DEV) < 0.4
    mask |= torch.eye(T, dtype=torch.bool, device=DEV)
    mask &= (torch.rand(mask.shape[0], T, 1, generator=g, device=DEV) >= empty)   # some rows see no draft at all
    d["tree_mask"] = mask.contiguous()
    for b, n in enumerate(lengths):
        d["keys"][b, :, max(0, n):] = stale
        d["values"][b, :, max(0, n):] = stale
    return d


def check(d, scale=128 ** -0.5, **kw):
    from pariskv_b200 import ops
    q = d["queries"]
    lse = torch.full(q.shape[:3], 7.0, device=DEV)
    out = ops.tree_attention(**d, lse=lse, **kw)
    want, tol, wl, ltol = R.tree(q, d["keys"], d["values"], d["draft_keys"], d["draft_values"], d["tree_mask"], d["lengths"].tolist(), scale)
    R.close(out, want, tol, "out")
    R.close(lse, wl, ltol, "lse")
    return out


@pytest.mark.parametrize("bs,T,H,G,cap,lengths", [
    (1, 1, 1, 1, 8, [1]), (1, 1, 1, 1, 1, [0]), (2, 1, 2, 4, 300, [300, 17]), (1, 2, 1, 3, 128, [128]), (1, 5, 2, 4, 129, [129]),
    (3, 7, 2, 5, 260, [0, 255, 257]), (2, 16, 1, 8, 700, [700, 1]), (1, 33, 2, 4, 1000, [999]), (1, 64, 1, 4, 513, [513]),
    (2, 61, 2, 2, 400, [400, 383]), (1, 26, 1, 8, 1500, [1500]), (1, 3, 1, 16, 200, [200]), (1, 2, 1, 128, 150, [149]), (1, 129, 1, 1, 64, [40]),
    (1, 130, 1, 3, 300, [300]), (1, 256, 1, 2, 140, [139]), (17, 2, 1, 4, 300, list(range(0, 289, 18))), (1, 4, 8, 7, 2500, [2477]),
    (4, 13, 2, 4, 1400, [1400, 900, 129, 3]), (2, 9, 3, 6, 100, [-5, 1000])])
def test_against_the_definition(bs, T, H, G, cap, lengths):
    check(make(1000 * T + cap, bs, T, H, G, cap, lengths))


def test_long_context_split_over_many_blocks():
    check(make(3, 1, 3, 2, 4, 40000, [39999]))
    check(make(4, 2, 9, 1, 8, 20000, [20000, 11]))


def test_far_scores_and_one_dominant_row():
    """Scores hundreds apart: a late row that outweighs all before it, and one that came first."""
    d = make(5, 1, 6, 1, 4, 900, [900], spread=30.0)
    check(d)
    d["keys"][0, 0, 3] = d["queries"][0, 0, 0] / 4
    d["keys"][0, 0, 897] = d["queries"][0, 2, 1] / 3
    check(d)


def test_explicit_scale_and_given_output():
    d = make(6, 1, 5, 2, 2, 200, [150])
    out = torch.empty_like(d["queries"])
    from pariskv_b200 import ops
    got = ops.tree_attention(**d, scale=0.5, out=out)
    assert got is out
    want, tol, _, _ = R.tree(*[d[k] for k in ("queries", "keys", "values", "draft_keys", "draft_values", "tree_mask")], d["lengths"].tolist(), 0.5)
    R.close(out, want, tol)


@pytest.mark.parametrize("T,G", [(5, 4), (40, 4)])
def test_what_is_masked_does_not_reach_a_token(T, G):
    """NaN and infinities in the drafts that a token does not see, in the cache behind its end, and in other tokens' queries."""
    d = make(7, 2, T, 2, G, 300, [300, 130])
    m = d["tree_mask"]
    m[:] = torch.eye(T, dtype=torch.bool, device=DEV)
    m[:, :, 0] = True
    m[:, 2, 0] = False
    d["draft_values"][:, 3] = float("nan")
    d["draft_keys"][:, 3] = float("inf")
    d["draft_values"][:, 1, :, 5] = float("inf")
    d["draft_values"][:, 4, :, 9] = float("-inf")
    from pariskv_b200 import ops
    out = ops.tree_attention(**d)
    keep = [t for t in range(T) if t not in (1, 3, 4)]
    want, tol, _, _ = R.tree(d["queries"], d["keys"], d["values"], d["draft_keys"], d["draft_values"], m, [300, 130])
    R.close(out[:, keep], want[:, keep], tol[:, keep])
    assert out[:, 3].isnan().all()                                         # the token that sees the NaN row
    for t, dim, sign in ((1, 5, 1), (4, 9, -1)):                           # an infinite value that is seen
        assert (out[:, t, :, dim] == sign * math.inf).all()
        rest = [i for i in range(128) if i != dim]
        R.close(out[:, t][..., rest], want[:, t][..., rest], tol[:, t][..., rest])


@pytest.mark.parametrize("T,G,n", [(1, 1, 1), (2, 4, 0), (2, 4, 3000), (3, 8, 40), (40, 4, 300), (70, 4, 3000)])
@pytest.mark.parametrize("shared_head", [False, True])
def test_a_query_that_is_not_a_number(T, G, n, shared_head):
    """It comes out as NaN, lse too, where it sees a row; the other queries do not notice."""
    d = make(9, 2, T, 2, G, 3000, [n, 3000], empty=0.0)
    if shared_head:
        for k in ("keys", "values"):
            d[k] = d[k][:, :1].expand(2, 2, 3000, 128)
    d["tree_mask"][:] = torch.eye(T, dtype=torch.bool, device=DEV)
    d["queries"][:, T - 1, G] = float("nan")
    from pariskv_b200 import ops
    lse = torch.zeros(2, T, 2 * G, device=DEV)
    out = ops.tree_attention(**d, lse=lse)
    assert out[:, T - 1, G].isnan().all() and lse[:, T - 1, G].isnan().all()
    want, tol, _, _ = R.tree(*[d[k] for k in ("queries", "keys", "values", "draft_keys", "draft_values", "tree_mask")], [n, 3000])
    R.close(out, want, tol)
    assert int(out.isnan().sum()) == 2 * 128


def test_a_row_of_lowest_scores_is_a_row():
    """Every score at the type's lowest values: the weights are equal, not lost."""
    d = make(8, 1, 2, 1, 1, 64, [64], empty=0.0)
    d["queries"][:] = 0
    d["queries"][..., 0] = 3e19
    d["keys"][..., 0] = -1e19
    d["draft_keys"][..., 0] = -1e19
    from pariskv_b200 import ops
    out = ops.tree_attention(**d)
    for t in range(2):
        see = d["tree_mask"][0, t]
        want = torch.cat((d["values"][0, 0], d["draft_values"][0, see, 0])).double().mean(0)
        assert (out[0, t, 0].double() - want).abs().max() < 2 * R.U


@pytest.mark.parametrize("layout", ["pairs", "window", "fused_rows", "token_major"])
def test_strides(layout):
    bs, T, H, G, cap, lengths = 2, 6, 2, 4, 333, [333, 200]
    d = make(9, bs, T, H, G, cap, lengths)
    if layout == "pairs":          # K and V row of a key next to each other
        store = torch.full((bs, H, cap + 3, 2, 128), float("nan"), dtype=torch.bfloat16, device=DEV)
        store[:, :, :cap, 0], store[:, :, :cap, 1] = d["keys"], d["values"]
        d["keys"], d["values"] = store[:, :, :cap, 0], store[:, :, :cap, 1]
    elif layout == "window":       # a slice of a longer buffer
        for name in ("keys", "values"):
            w = torch.full((bs, H, cap + 60, 128), float("nan"), dtype=torch.bfloat16, device=DEV)
            w[:, :, 8:8 + cap] = d[name]
            d[name] = w[:, :, 8:8 + cap]
    elif layout == "fused_rows":   # q, k and v of a projection's row
        row = torch.full((bs, T, (H * G + 2 * H) * 128 + 16), float("nan"), dtype=torch.bfloat16, device=DEV)
        views = {}
        at = 0
        for name, heads in (("queries", H * G), ("draft_keys", H), ("draft_values", H)):
            v = row.as_strided((bs, T, heads, 128), (row.stride(0), row.stride(1), 128, 1), at)
            v.copy_(d[name])
            views[name] = v
            at += heads * 128
        d.update(views)
    else:                          # [bs, cap, H, 128], as a prompt comes
        for name in ("keys", "values"):
            d[name] = d[name].transpose(1, 2).contiguous().transpose(1, 2)
        d["tree_mask"] = d["tree_mask"].transpose(1, 2).contiguous().transpose(1, 2)
        d["tree_mask"] = d["tree_mask"].to(torch.uint8) * 3
    check(d)


@pytest.mark.parametrize("T", [3, 20])
def test_one_head_of_keys_for_all(T):
    """Strides of zero, which no tensor map takes: a cache, and drafts, expanded over the KV heads."""
    d = make(15, 2, T, 1, 8, 150, [150, 33])
    for names, heads_at in ((("keys", "values"), 1), (("draft_keys", "draft_values"), 2)):
        for name in names:
            d[name] = d[name].expand(*[4 if i == heads_at else n for i, n in enumerate(d[name].shape)])
    check(d)


def test_one_mask_for_the_batch():
    d = make(10, 3, 11, 1, 4, 150, [150, 20, 0], shared_mask=True)
    check(d)


def test_heads_far_apart():
    """Offsets behind 2^31 elements."""
    buf = torch.empty(2 ** 31 + 300 * 128 + 64, dtype=torch.bfloat16, device=DEV)
    d = make(11, 1, 3, 2, 2, 300, [300])
    far = buf.as_strided((1, 2, 300, 128), (2 ** 33, 2 ** 31 + 64, 128, 1))
    for name, other in (("keys", "values"), ("values", "keys")):
        far.copy_(d[name])
        check(dict(d, **{name: far}))
    del buf
    torch.cuda.empty_cache()


def test_captured_and_replayed_while_the_sequences_grow():
    from pariskv_b200 import ops
    d = make(12, 2, 5, 2, 4, 700, [700, 700], stale=0.0)
    d["lengths"][:] = torch.tensor([130, 5], device=DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.tree_attention(**d)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.tree_attention(**d)
    g2 = torch.cuda.CUDAGraph()
    other = dict(d, queries=d["queries"].flip(1).contiguous())
    with torch.cuda.graph(g2):
        out2 = ops.tree_attention(**other)
    for lengths in ([130, 5], [700, 0], [257, 511]):
        d["lengths"].copy_(torch.tensor(lengths, dtype=torch.int32))
        torch.cuda.synchronize()
        with torch.cuda.stream(s):     # two graphs at once
            g.replay()
        g2.replay()
        torch.cuda.synchronize()
        for o, q in ((out, d["queries"]), (out2, other["queries"])):
            want, tol, _, _ = R.tree(q, d["keys"], d["values"], d["draft_keys"], d["draft_values"], d["tree_mask"], lengths)
            R.close(o, want, tol)


def test_two_streams_at_once():
    from pariskv_b200 import ops
    ds = [make(20 + i, 1, 9, 2, 4, 5000, [5000 - i]) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i].append(ops.tree_attention(**ds[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, outs[i][0]) for o in outs[i])
        want, tol, _, _ = R.tree(*[ds[i][k] for k in ("queries", "keys", "values", "draft_keys", "draft_values", "tree_mask")], [5000 - i])
        R.close(outs[i][0], want, tol)


def test_no_tokens():
    from pariskv_b200 import ops
    d = make(13, 2, 1, 1, 2, 16, [16, 3])
    e = {k: (v[:, :0] if k in ("queries", "draft_keys", "draft_values") else v) for k, v in d.items()}
    e["tree_mask"] = d["tree_mask"][:, :0, :0]
    assert ops.tree_attention(**e).shape == (2, 0, 2, 128)


def test_refusals():
    from pariskv_b200 import ops
    d = make(14, 2, 4, 2, 2, 64, [64, 3])
    odd = torch.zeros(2, 2, 64, 132, dtype=torch.bfloat16, device=DEV)[..., :128]
    shifted = torch.zeros(2 * 2 * 64 * 128 + 8, dtype=torch.bfloat16, device=DEV)[4:4 + 2 * 2 * 64 * 128].view(2, 2, 64, 128)
    for change in (dict(keys=d["keys"].float()), dict(keys=odd), dict(values=shifted), dict(lengths=d["lengths"][:1]),
                   dict(lengths=d["lengths"].long()), dict(tree_mask=d["tree_mask"][:, :3]), dict(tree_mask=d["tree_mask"].float()),
                   dict(queries=d["queries"][:, :, :3]), dict(draft_keys=d["draft_keys"][:, :3]), dict(values=d["values"][:, :, :60]),
                   dict(queries=d["queries"][..., :64]), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(keys=d["keys"].cpu()), dict(out=torch.empty(2, 4, 4, 64, dtype=torch.bfloat16, device=DEV)),
                   dict(lse=torch.empty(2, 4, 2, device=DEV))):
        with pytest.raises((RuntimeError, TypeError, ValueError)):
            ops.tree_attention(**{**d, **change})
