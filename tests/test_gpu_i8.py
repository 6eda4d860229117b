"""Rows as 8-bit whole numbers, products of them, and a whole layer's step in 8 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


def ops():
    from pariskv_b200 import ops as o
    return o


def codes_of(y):
    """y f64 [B,n] -> codes, scales, and where a quotient is so near a tie that 32-bit arithmetic may take the other side."""
    top = y.abs().amax(-1, keepdim=True)
    q = torch.where(top > 0, y * 127 / torch.where(top > 0, top, 1.0), 0.0)
    return torch.round(q), (top / 127)[:, 0], q


def check_codes(codes, scales, y, slack):
    """slack: relative error of y in 32 bits.  A code differs from the rounded quotient only where the quotient is that near to a tie."""
    want, s, q = codes_of(y)
    got = codes.double()
    assert ((got - q).abs() <= 0.5 + 127 * slack).all()
    assert torch.allclose(scales.double(), s, rtol=slack, atol=2.0 ** -149)


@pytest.mark.parametrize("B,n", [(1, 8), (1, 4096), (3, 4096), (2, 4104), (5, 1000), (300, 512), (2, 8192), (2, 20000), (1, 40008), (1, 65536)])
@pytest.mark.parametrize("residual", [True, False])
def test_add_rmsnorm_i8(B, n, residual):
    g = torch.Generator().manual_seed(B + n)
    a, r = (torch.randn(B, n, generator=g) * 3).to(BF).to(DEV), torch.randn(B, n, generator=g).to(BF).to(DEV)
    w = (1 + 0.3 * torch.randn(n, generator=g)).to(BF).to(DEV)
    h, codes, scales = ops().add_rmsnorm_i8(a, r if residual else None, w, eps=1e-5)
    assert torch.equal(h, (a.float() + r.float()).to(BF) if residual else a)
    rstd = 1 / torch.sqrt(h.double().square().mean(-1, keepdim=True) + 1e-5)
    # rstd, two products, the division by amax and amax itself are rounded to 32 bits, and 127 / 128 y
    check_codes(codes, scales, h.double() * rstd * w.double(), 8 * 2.0 ** -24)
    # the same steps in 32 bits give the same codes
    y = h.float() * rstd.float() * w.float()
    top = y.abs().amax(-1, keepdim=True)
    assert torch.equal(codes, torch.round((y * 0.9921875) / (top * 0.0078125)).to(torch.int8))
    assert torch.equal(scales, (top / torch.full_like(top, 127.0))[:, 0])


@pytest.mark.parametrize("B,n", [(1, 8), (2, 4096), (7, 1224), (2, 16392), (130, 256)])
def test_quantize_rows(B, n):
    g = torch.Generator().manual_seed(n)
    x = torch.randint(-255, 256, (B, n), generator=g).float() * 2.0 ** torch.randint(-9, 9, (B, 1), generator=g).float()
    x = x.to(BF).to(DEV)
    codes, scales = ops().quantize_rows_i8(x)
    want, s, _ = codes_of(x.double())
    assert torch.equal(codes.double(), want)   # values of 16 bits: as exact arithmetic has it, ties to the even one
    assert torch.allclose(scales.double(), s, rtol=2.0 ** -24, atol=0)


@pytest.mark.parametrize("B,n", [(1, 8), (3, 4096), (2, 12288), (9, 1000)])
def test_quantize_gated_rows(B, n):
    g = torch.Generator().manual_seed(n + 1)
    x = (torch.randn(B, 2 * n, generator=g) * 4).to(BF).to(DEV)
    x[0, :4] = torch.tensor([300.0, -300.0, 0.0, -87.0])
    codes, scales = ops().quantize_rows_i8(x, gated=True)
    gate, up = x[:, :n].double(), x[:, n:].double()
    # exp to 2 units of its last place, a sum, a quotient, two products: 16 units in all are above it
    check_codes(codes, scales, gate / (1 + torch.exp(-gate)) * up, 16 * 2.0 ** -24)


def test_rows_that_are_not_numbers():
    x = torch.randn(4, 64, device=DEV).to(BF)
    x[1, 3], x[2, 5] = float("inf"), float("nan")
    x[3] = 0
    w = torch.ones(64, device=DEV, dtype=BF)
    for codes, scales in (ops().quantize_rows_i8(x), ops().add_rmsnorm_i8(x, None, w)[1:]):
        assert codes[0].any() and scales[0].isfinite()
        assert not codes[1:].any() and scales[1:3].isnan().all() and scales[3] == 0
        y = ops().matmul_i8(codes, scales, torch.ones(5, 64, dtype=torch.int8, device=DEV), torch.ones(5, device=DEV))
        assert y[0].isfinite().all() and y[1:3].isnan().all() and not y[3].any()


def test_rows_in_place_and_strided():
    from pariskv_b200 import _lib as L
    a, r = torch.randn(3, 72, device=DEV).to(BF)[:, :64], torch.randn(3, 64, device=DEV).to(BF)
    w = torch.ones(64, device=DEV, dtype=BF)
    h, codes, scales = ops().add_rmsnorm_i8(a, r, w)
    c2, s2 = torch.empty_like(codes), torch.empty_like(scales)
    d = [L.desc(t) for t in (a, r, w, r, c2, s2)]
    L.check(L.load().pk_add_rmsnorm_i8(*[L.ref(x) for x in d], 1e-6, L.stream_ptr()))
    assert torch.equal(r, h) and torch.equal(c2, codes) and torch.equal(s2, scales)
    assert torch.equal(ops().quantize_rows_i8(a)[0], ops().quantize_rows_i8(a.contiguous())[0])


def i8(g, *shape):
    return torch.randint(-128, 128, shape, generator=g).to(torch.int8).to(DEV)


def check_matmul(T, O, I, x=None, w=None, out=None):
    g = torch.Generator().manual_seed(T * 31 + O * 7 + I)
    x = i8(g, T, I) if x is None else x
    w = i8(g, O, I) if w is None else w
    sx, so = torch.rand(T, generator=g).to(DEV) * 1e-2, torch.rand(O, generator=g).to(DEV) * 1e-3
    y = ops().matmul_i8(x, sx, w, so, out=out)
    acc = x.double() @ w.double().t()   # whole numbers below 2^53
    want = acc * sx.double()[:, None] * so.double()
    # the sum as a float, two products, and the output's rounding
    assert ((y.double() - want).abs() <= (2.0 ** -8 + 4 * 2.0 ** -24) * want.abs()).all()
    # and the very steps
    assert torch.equal(y, (acc.float() * sx[:, None] * so).to(BF))


@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 33, 64, 65, 129, 257, 700])
@pytest.mark.parametrize("O,I", [(1, 16), (127, 48), (128, 128), (129, 144), (1000, 4096), (6144, 1040)])
def test_matmul_i8(T, O, I):
    check_matmul(T, O, I)


@pytest.mark.parametrize("T,O,I", [(1, 4096, 65536), (3, 30000, 512), (16, 151936, 128), (300, 5000, 12288), (4096, 640, 2048), (5000, 129, 64), (2048, 6144, 4096)])
def test_matmul_i8_long(T, O, I):
    check_matmul(T, O, I)


def test_matmul_i8_extremes():
    """The largest sums that there are."""
    T, O, I = 5, 130, 65536
    check_matmul(T, O, I, x=torch.full((T, I), -128, dtype=torch.int8, device=DEV), w=torch.full((O, I), -128, dtype=torch.int8, device=DEV))
    check_matmul(T, O, I, x=torch.full((T, I), 127, dtype=torch.int8, device=DEV), w=torch.full((O, I), -128, dtype=torch.int8, device=DEV))


def test_matmul_i8_layouts():
    g = torch.Generator().manual_seed(0)
    x, w = i8(g, 9, 256)[:, 32:192], i8(g, 50, 512)[::2, 16:176]
    out = torch.full((9, 30), 5.0, device=DEV, dtype=BF)
    check_matmul(9, 25, 160, x=x, w=w, out=out[:, 2:27])
    assert (out[:, :2] == 5).all() and (out[:, 27:] == 5).all()
    assert ops().matmul_i8(x[:0], torch.empty(0, device=DEV), w, torch.ones(25, device=DEV)).shape == (0, 25)


def test_matmul_i8_twice_and_in_graphs():
    g = torch.Generator().manual_seed(3)
    cases = []
    for T, O, I in ((1, 4096, 4096), (40, 3000, 1024), (600, 1000, 512)):
        x, w, sx, so = i8(g, T, I), i8(g, O, I), torch.rand(T, generator=g).to(DEV), torch.rand(O, generator=g).to(DEV)
        cases.append((x, sx, w, so, ops().matmul_i8(x, sx, w, so)))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        outs = [ops().matmul_i8(*c[:4]) for c in cases for _ in range(2)]
    for _ in range(3):
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for i, o in enumerate(outs):
            assert torch.equal(o, cases[i // 2][4])
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(ops().matmul_i8(*c[:4]))
        torch.cuda.synchronize()
        for c, o in zip(cases, got):
            assert torch.equal(o, c[4])


def test_a_layer_in_8_bits():
    """Norm, q/k/v, rows into the cache, attention, output projection, norm, gate and up, activation, down: as used together, eagerly and as a graph, against the same steps in 64 bits."""
    from eight_ref import RefCache, attention, kv_rows
    H, G, width, ff, n, block = 2, 2, 512, 768, 90, 32
    Hq = H * G
    g = torch.Generator().manual_seed(11)

    def matrix(rows, cols):
        w = torch.randn(rows, cols, generator=g) / cols ** 0.5
        s = w.abs().amax(-1) / 127
        return torch.round(w / s[:, None]).to(torch.int8).to(DEV), s.to(DEV)

    w_qkv, w_o, w_gu, w_d = matrix((Hq + 2 * H) * 128, width), matrix(width, Hq * 128), matrix(2 * ff, width), matrix(width, ff)
    n1, n2 = (1 + 0.1 * torch.randn(2, width, generator=g)).to(BF).to(DEV)
    past = kv_rows(g, H, n)
    cache = ops().Cache8.empty(1, H, 128, block=block, device=DEV)
    ops().cache8_append(cache, past[:, :, 0].transpose(0, 1)[None], past[:, :, 1].transpose(0, 1)[None], torch.tensor([n], dtype=torch.int32, device=DEV))
    hidden, delta = (torch.randn(2, 1, width, generator=g).to(BF).to(DEV))
    length = torch.tensor([n + 1], dtype=torch.int32, device=DEV)

    def step():
        h, c, s = ops().add_rmsnorm_i8(delta, hidden, n1)
        qkv = ops().matmul_i8(c, s, *w_qkv).view(1, 1, Hq + 2 * H, 128)
        ops().cache8_append(cache, qkv[:, :, Hq:Hq + H], qkv[:, :, Hq + H:], length)
        o = ops().cache8_attention(qkv[:, :, :Hq], cache, length)
        y = ops().matmul_i8(*ops().quantize_rows_i8(o.view(1, -1)), *w_o)
        h2, c2, s2 = ops().add_rmsnorm_i8(y, h, n2)
        gu = ops().matmul_i8(c2, s2, *w_gu)
        return h, qkv, o, h2, gu, ops().matmul_i8(*ops().quantize_rows_i8(gu, gated=True), *w_d)

    got = step()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        again = step()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, again):
        assert torch.equal(a, b)
    h, qkv, o, h2, gu, out = got
    value = lambda w: w[0].double() * w[1].double()[:, None]   # noqa: E731
    # each product against 64 bits on its own inputs: an input is off by half a code, scale / 2, at most (and a rounding to 16 bits), whatever its sign

    def near(y, x, w, r=2.0 ** -8):
        unit = x.abs().max() / 127
        bound = (w.abs().sum(-1) * unit * 0.5) + r * (x @ w.t()).abs() + (2.0 ** -8) * 0 + w.abs().sum(-1) * unit * 127 * 2.0 ** -20
        assert ((y.double().view(-1) - (x @ w.t()).view(-1)).abs() <= bound.view(-1) * (1 + 2.0 ** -8)).all()

    norm = lambda x, w: x.double() / torch.sqrt(x.double().square().mean() + 1e-6) * w.double()   # noqa: E731
    assert torch.equal(h, hidden + delta)
    near(qkv, norm(h, n1), value(w_qkv))
    rows = torch.cat((past, qkv[0, 0, Hq:].view(2, H, 128).transpose(0, 1)[:, None]), 1)
    want, _, tol = attention(RefCache([rows], block, False), qkv[:, :, :Hq], 128 ** -0.5)
    assert ((o.double() - want).abs() <= tol).all()
    near(h2.double() - h.double(), o.double().view(1, -1), value(w_o), r=2.0 ** -7 + float(h.abs().max()) / float((o.double().view(1, -1) @ value(w_o).t()).abs().min().clamp(min=1e-3)) * 2.0 ** -7)
    near(gu, norm(h2, n2), value(w_gu))
    gate, up = gu.double().chunk(2, -1)
    near(out, gate / (1 + torch.exp(-gate)) * up, value(w_d))
