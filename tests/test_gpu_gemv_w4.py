"""Products with 4-bit weights against the definition in 64 bits, and the operators of a decode step together."""
import pytest
import torch

import many_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(seed, T, O, I, group, offsets):
    g = torch.Generator(device=DEV).manual_seed(seed)
    codes = torch.randint(0, 16, (O, I), generator=g, device=DEV).to(torch.uint8)
    scales = (torch.rand(O, I // group, generator=g, device=DEV) / I ** 0.5 + 1e-3).to(torch.bfloat16)
    scales[0] = -scales[0]
    off = (torch.randn(O, I // group, generator=g, device=DEV) / I ** 0.5).to(torch.bfloat16) if offsets else None
    x = torch.randn(T, I, generator=g, device=DEV).to(torch.bfloat16)
    return codes, scales, x, off


def check(codes, scales, x, off, gated):
    from pariskv_b200 import ops
    got = ops.gemv_w4(R.pack_w4(codes), scales, x, offsets=off, gated=gated)
    want, tol = R.gemv_w4(codes, scales, x, off, gated)
    assert got.shape == want.shape and got.dtype == torch.bfloat16
    R.close(got, want, tol)
    return got


@pytest.mark.parametrize("O,I", [(2, 128), (64, 128), (66, 1024), (130, 4096), (1030, 640), (302, 12288), (5000, 384), (34, 32768), (6144, 4096), (18, 17408)])
@pytest.mark.parametrize("T", [1, 3, 8, 9, 16])
@pytest.mark.parametrize("group,offsets,gated", [(128, False, False), (64, True, True), (32, True, False), (32, False, True)])
def test_against_the_definition(T, O, I, group, offsets, gated):
    check(*make(T + O + I, T, O, I, group, offsets), gated)


@pytest.mark.parametrize("O", [1, 3, 7, 15, 17, 33, 149, 297])
def test_odd_rows(O):
    for T in (1, 2, 13):
        check(*make(O, T, O, 256, 64, True), False)
        check(*make(O, T, O, 32 * 7, 32, False), False)


@pytest.mark.parametrize("T", list(range(1, 17)))
def test_every_number_of_tokens(T):
    check(*make(T, T, 70, 1120, 32, True), False)


@pytest.mark.parametrize("O,I,group,offsets,gated", [(38000, 4096, 128, False, False), (304200, 512, 64, True, False), (76001, 1568, 32, True, False),
                                                     (75000, 2176, 128, True, True), (19001, 12288, 64, False, False)])
def test_long_products_of_one_and_two_tokens(O, I, group, offsets, gated):
    """What an SM has many stages of takes x in whole numbers: values of very different sizes, zeros, and a group of zeros."""
    for T in (1, 2):
        codes, scales, x, off = make(O + T, T, O, I, group, offsets)
        x[0, ::7] *= 1000
        x[0, 5::11] *= 2.0 ** -20
        x[0, :group] = 0
        x[-1, group:2 * group] *= 2.0 ** -110
        check(codes, scales, x, off, gated)
        if T == 2:
            from pariskv_b200 import ops
            clean = ops.gemv_w4(R.pack_w4(codes), scales, x, offsets=off, gated=gated)
            x[0, 3], x[0, 200] = float("inf"), float("nan")
            got = ops.gemv_w4(R.pack_w4(codes), scales, x, offsets=off, gated=gated)
            assert torch.equal(got[1], clean[1]) and not got[0].isfinite().any()


def test_every_code_and_column():
    """One token per column of a group, each code in turn: no two columns or codes are taken for each other."""
    from pariskv_b200 import ops
    I = 256
    codes = (torch.arange(I, device=DEV)[None, :] * 7 + torch.arange(48, device=DEV)[:, None] * 3).remainder(16).to(torch.uint8)
    scales = torch.ones(48, I // 64, dtype=torch.bfloat16, device=DEV)
    for c in range(0, I, 16):
        x = torch.zeros(16, I, dtype=torch.bfloat16, device=DEV)
        x[torch.arange(16), c + torch.arange(16)] = 1
        got = ops.gemv_w4(R.pack_w4(codes), scales, x)
        assert torch.equal(got, (codes[:, c:c + 16].t().float() - 8).to(torch.bfloat16))


def test_strided_tokens_and_large_values():
    codes, scales, x, off = make(3, 5, 90, 512, 128, True)
    wide = torch.full((5, 640), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide[:, 64:576] = x * 1000
    check(codes, scales, wide[:, 64:576], off, True)
    check(codes, scales, (x * 1e30), off, False)


def test_infinities_stay_in_their_token():
    from pariskv_b200 import ops
    codes, scales, x, off = make(4, 4, 40, 256, 64, False)
    x[1, 17], x[2, 5] = float("inf"), float("nan")
    got = ops.gemv_w4(R.pack_w4(codes), scales, x)
    want, tol = R.gemv_w4(codes, scales, x[[0, 3]])
    R.close(got[[0, 3]], want, tol)
    assert not got[1].isfinite().any() and got[2].isnan().all()


def test_no_tokens_and_refusals():
    from pariskv_b200 import ops
    codes, scales, x, off = make(5, 4, 40, 256, 64, True)
    w = R.pack_w4(codes)
    assert ops.gemv_w4(w, scales, x[:0]).shape == (0, 40)
    bad = (RuntimeError, TypeError, ValueError)
    for call in (lambda: ops.gemv_w4(w, scales[:, :3], x), lambda: ops.gemv_w4(w, scales[:39], x), lambda: ops.gemv_w4(w[:39], scales[:39], x, gated=True),
                 lambda: ops.gemv_w4(w.int(), scales, x), lambda: ops.gemv_w4(w, scales.float(), x), lambda: ops.gemv_w4(w, scales, x.float()),
                 lambda: ops.gemv_w4(w, scales, x[:, :128]), lambda: ops.gemv_w4(w, scales, torch.cat([x] * 5)), lambda: ops.gemv_w4(w, scales, x, offsets=off[:, :2]),
                 lambda: ops.gemv_w4(w.cpu(), scales, x), lambda: ops.gemv_w4(w[:, :16], scales[:, :2], x[:, :32]), lambda: ops.gemv_w4(w, scales, x.t()),
                 lambda: ops.gemv_w4(w, scales[:, :1], x)):
        with pytest.raises(bad):
            call()


@pytest.mark.parametrize("launches", ["dependent", "early loads", "plain"])
def test_a_layer_of_a_step_with_drafts_captured(launches):
    """4-bit projection, tree over the cache, then the accepted rows appended, bounds, selection, attention, 4-bit projection back:
    captured once and replayed, against the same definitions step by step."""
    from pariskv_b200 import _lib, ops
    g = torch.Generator(device=DEV).manual_seed(9)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).to(torch.bfloat16)
    bs, T, H, G, cap, hidden, block = 2, 4, 2, 4, 500, 512, 16
    heads = H * G + 2 * H
    qkv = make(10, bs * T, heads * 128, hidden, 64, False)[:2]
    o = make(11, bs * T, hidden, H * G * 128, 128, True)
    wq, wo = R.pack_w4(qkv[0]), R.pack_w4(o[0])
    keys, values, lengths = r(bs, H, cap, 128), r(bs, H, cap, 128), i32([400, 37])
    mask = torch.tril(torch.ones(1, T, T, dtype=torch.bool, device=DEV))
    bnd = ops.block_bounds(keys, lengths, block=block, bounds=torch.zeros(bs, H, 32, 2, 128, dtype=torch.bfloat16, device=DEV))
    x = r(bs * T, hidden)

    def step():
        rows = ops.gemv_w4(wq, qkv[1], x).view(bs, T, heads, 128)
        q, k, v = rows[:, :, :H * G], rows[:, :, H * G:H * G + H], rows[:, :, H * G + H:]
        tree = ops.tree_attention(q, keys, values, k, v, mask, lengths)
        at = (lengths.long()[:, None] + torch.arange(T, device=DEV))[:, None, :, None].expand(-1, H, -1, 128)
        keys.scatter_(2, at, k.transpose(1, 2))
        values.scatter_(2, at, v.transpose(1, 2))
        n = lengths + T
        ops.block_bounds(keys, n, block=block, n_new=T, bounds=bnd)
        ids = ops.select_blocks(q, bnd, n, 6, block=block, sink_blocks=1, local_blocks=2)
        sparse = ops.block_attention(q, keys, values, ids, n, block=block)
        return rows, tree, ids, sparse, ops.gemv_w4(wo, o[1], sparse.view(bs * T, -1), offsets=o[3])

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    try:
        if launches == "early loads":
            _lib.set_pdl(True)
        elif launches == "plain":
            _lib.set_dependent_launch(False)
        with torch.cuda.graph(graph):
            rows, tree, ids, sparse, y = step()
    finally:
        _lib.set_pdl(False)
    for lens in ([400, 37], [404, 0], [496, 41]):
        x.copy_(r(bs * T, hidden))
        lengths.copy_(i32(lens))
        graph.replay()
        torch.cuda.synchronize()
        want, tol = R.gemv_w4(qkv[0], qkv[1], x)
        R.close(rows.reshape(bs * T, -1), want, tol, "qkv")
        q, k, v = rows[:, :, :H * G], rows[:, :, H * G:H * G + H], rows[:, :, H * G + H:]
        want, tol, _, _ = R.tree(q, keys, values, k, v, mask, lens)
        R.close(tree, want, tol, "tree")
        n = [l + T for l in lens]
        new = R.bounds(keys, n, block, bnd, T)
        assert torch.equal(new, bnd)
        assert torch.equal(ids.cpu(), R.select(q.cpu(), bnd.cpu(), n, 6, block, 1, 2))
        want, tol, _, _ = R.block_attention(q, keys, values, ids, n, block)
        R.close(sparse, want, tol, "sparse")
        # the tree of a chain is causal attention: over all blocks it is the same
        want, tol = R.gemv_w4(o[0], o[1], sparse.reshape(bs * T, -1), o[3])
        R.close(y, want, tol, "out")


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)
