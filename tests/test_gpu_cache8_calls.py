"""Calls of the operators of a step in 8 bits that the documentation allows beside the usual ones: many samples, shared heads, kinds of launch, rows of next to nothing, lengths that change under a graph."""
import pytest
import torch

from eight_ref import RefCache, attention, kv_rows
from test_gpu_cache8 import DEV, TYPES, check_attention, check_cache, filled, i32, ops, queries, samples

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("block,recent", [(128, 128), (128, 384), (16, 16), (32, 96)])
@pytest.mark.parametrize("step", [1, 7, 8, 9, 16, 17, 140])
def test_append_of_steps_of_every_size(dtype, block, recent, step):
    """A warp per row, and rows by blocks; a sequence that ends behind the cache, one that begins before it."""
    n, cap = 420, 400
    rows = samples((n,), H=1, seed=step)
    cache = ops().Cache8.empty(2, 1, cap, block=block, dtype=dtype, recent=recent, device=DEV)
    x = rows[0].transpose(0, 1)[None].expand(2, -1, -1, -1, -1)
    for at in range(0, n, step):
        part = x[:, at:at + step]
        upto = min(n, at + step)
        ops().cache8_append(cache, part[:, :, :, 0], part[:, :, :, 1], i32(upto, upto - 13))
    for b, want in ((0, rows[0][:, :cap]), (1, rows[0][:, 13:413][:, :400])):
        check_cache(ops().Cache8(cache.codes[b:b + 1], cache.scales[b:b + 1], cache.recent[b:b + 1], block), [want], block, dtype)


@pytest.mark.parametrize("lengths", [[(i * 37) % 150 for i in range(70)], [(i * 53) % 700 for i in range(40)]])
def test_attention_of_many_samples(lengths):
    """More samples than a warp has lanes, some of them without rows; short and longer caches."""
    check_attention(samples(lengths, H=1, seed=2), 16, torch.int8, 1, 3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [128, 129, 255, 384, 385, 1024, 1153, 3000, 3200])
@pytest.mark.parametrize("rows", [(1, 4), (3, 4), (4, 8)])
def test_attention_around_the_choices(dtype, n, rows):
    """Tiles, clusters of every size, ranges; eight, sixteen and 32 query rows."""
    check_attention(samples((n,), H=1, seed=n), 128, dtype, rows[0], rows[1])


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_over_shared_heads_and_prompts(dtype):
    """One sequence and head expanded over several: strides of zero."""
    rows = samples((300,), H=1, seed=6)
    cache = filled(rows, 32, dtype)
    wide = ops().Cache8(cache.codes.expand(2, 3, -1, -1, -1), cache.scales.expand(2, 3, -1, -1), cache.recent.expand(2, 3, -1, -1, -1), 32)
    g = torch.Generator().manual_seed(0)
    q = queries(g, 2, 2, 12)
    out = ops().cache8_attention(q, wide, i32(300, 170))
    want, _, tol = attention(RefCache([rows[0].expand(3, -1, -1, -1)], 32, dtype == torch.float8_e4m3fn), q[:1], 128 ** -0.5)
    assert ((out[:1].double() - want).abs() <= tol).all()
    back = ops().cache8_read(wide, i32(300, 300))
    assert torch.equal(back[0, 0, :300], ops().cache8_read(cache, i32(300))[0, 0, :300]) and torch.equal(back[0], back[1])


@pytest.mark.parametrize("order", ["kv first", "heads inside"])
def test_attention_layouts(order):
    rows = samples((333,), H=2, seed=9)
    cache = filled(rows, 64, torch.int8)
    q = queries(torch.Generator().manual_seed(0), 1, 1, 8)
    want = ops().cache8_attention(q, cache, i32(333))
    turn = (3, 0, 1, 2, 4) if order == "kv first" else (0, 2, 3, 1, 4)
    back = [turn.index(i) for i in range(5)]
    other = ops().Cache8(cache.codes.permute(turn).contiguous().permute(back), cache.scales.permute(3, 2, 1, 0).contiguous().permute(3, 2, 1, 0),
                         cache.recent.permute(turn).contiguous().permute(back), 64)
    assert other.codes.stride() != cache.codes.stride()
    assert torch.equal(ops().cache8_attention(q, other, i32(333)), want)


@pytest.mark.parametrize("kind", ["plain", "early"])
def test_steps_under_every_kind_of_launch(kind):
    """Append, attention and norms in a chain, under plain launches and under early loads, give what dependent launches give."""
    from pariskv_b200 import _lib as L
    rows = samples((200,), H=2, seed=12)
    q = queries(torch.Generator().manual_seed(3), 1, 40, 8)
    w = torch.ones(1024, device=DEV, dtype=torch.bfloat16)
    m = torch.randint(-128, 128, (512, 1024), generator=torch.Generator().manual_seed(1)).to(torch.int8).to(DEV)

    def run():
        cache, outs = filled([rows[0][:, :160]], 16, torch.int8, cap=200), []
        length = i32(160)
        for i in range(40):
            length.add_(1)
            ops().cache8_append(cache, rows[0][:, 160 + i, 0][None, None], rows[0][:, 160 + i, 1][None, None], length)
            o = ops().cache8_attention(q[:, i:i + 1], cache, length)
            h, c, s = ops().add_rmsnorm_i8(o.view(1, -1), None, w)
            outs += [o, h, ops().matmul_i8(c, s, m, torch.ones(512, device=DEV))]
        return torch.cat([o.flatten() for o in outs])

    want = run()
    try:
        if kind == "plain":
            L.set_dependent_launch(False)
        else:
            L.set_pdl(True)
        got = run()
    finally:
        L.set_dependent_launch(True)
    assert torch.equal(got, want)


def test_a_graph_over_lengths_that_cross_the_forms():
    """One captured attention over a long cache, whose ranges follow the lengths on the device, from empty to full and back."""
    n = 9000
    rows = samples((n,), H=1, seed=4)
    q = queries(torch.Generator().manual_seed(3), 1, 2, 4)
    cache = filled(rows, 64, torch.int8, recent=9024)   # every row stays in 16 bits too: any length is as if the others had never been
    length, out, lse = i32(n), torch.empty_like(q), torch.empty(1, 2, 4, device=DEV)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops().cache8_attention(q, cache, length, out=out, lse=lse)
    for m in (n, 1, 0, 64, 4097, 130, 8999):
        length.fill_(m)
        graph.replay()
        torch.cuda.synchronize()
        want, _, tol = attention(RefCache([rows[0][:, :m]], 64, False), q, 128 ** -0.5)
        assert ((out.double() - want).abs() <= tol + 1e-30).all()


def test_norm_without_eps_of_next_to_nothing():
    """Rows of 2^-120 and of zeros without an eps: the first as exact arithmetic has it, the second is 0 / 0."""
    x = torch.randn(3, 4096, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    x[1] = 0
    x = (x.float() * torch.tensor([2.0 ** -120, 1.0, 1.0])[:, None]).to(torch.bfloat16).to(DEV)
    w = torch.ones(4096, device=DEV, dtype=torch.bfloat16)
    h, c, s = ops().add_rmsnorm_i8(x, None, w, eps=0.0)
    y = x.double() / x.double().square().mean(-1, keepdim=True).sqrt()
    for i in (0, 2):
        top = y[i].abs().max()
        assert ((c[i].double() - y[i] * 127 / top).abs() <= 0.5 + 127 * 8 * 2.0 ** -24).all() and (s[i] - top / 127).abs() <= 8 * 2.0 ** -24 * top / 127
    assert s[1].isnan() and not c[1].any()


def test_norm_of_the_largest_numbers():
    x = torch.full((2, 512), 3.0e38, device=DEV, dtype=torch.bfloat16)
    x[1, ::2] *= -0.5
    h, c, s = ops().add_rmsnorm_i8(x, None, torch.ones(512, device=DEV, dtype=torch.bfloat16))
    y = x.double() / x.double().square().mean(-1, keepdim=True).sqrt()
    assert ((c.double() * s.double()[:, None] - y).abs() <= s.double()[:, None] * (0.5 + 2.0 ** -10)).all()
    c, s = ops().quantize_rows_i8(x)
    assert (c[0] == 127).all() and s.isfinite().all()


def test_outputs_of_one_call_feed_the_next_without_waiting():
    """Many products of changing shapes back to back: a kernel's blocks may be there while the one before still writes."""
    g = torch.Generator().manual_seed(5)
    ws = [(torch.randint(-8, 9, (o, i), generator=g).to(torch.int8).to(DEV), torch.full((o,), 1.0 / i, device=DEV)) for i, o in ((512, 1024), (1024, 2048), (2048, 512))]
    for T in (1, 3, 7, 40, 130, 300):
        x = torch.randn(T, 512, generator=g).to(torch.bfloat16).to(DEV)
        y, want = x, x
        for _ in range(6):
            for w, s in ws:
                y = ops().matmul_i8(*ops().quantize_rows_i8(y), w, s)
        torch.cuda.synchronize()
        for _ in range(6):
            for w, s in ws:
                c, r = ops().quantize_rows_i8(want)
                torch.cuda.synchronize()
                want = ((c.double() @ w.double().t()).float() * r[:, None] * s).to(torch.bfloat16)
        assert torch.equal(y, want)
