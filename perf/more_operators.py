"""The operators of a decode step in 8 bits - the cache and the products: what is measured.

    own                 False: run() computes the plain forms; True: run() calls the framework's kernels
    listed()            the named cases
    draw(rng)           another case of the same ranges
    prepare(case, seed) inputs, on the GPU, as a program holds them
    run(state)          one pass; returns the whole outputs
    work(case)          bytes and operations that a pass cannot do without
    exact(case, seed)   the outputs in 64 bits, from the definitions

Kinds of case
    append   new rows of K and V go into a cache of 8-bit codes: whole blocks are coded, the last rows are kept in 16 bits beside them
    read     rows of that cache back in 16 bits: the whole context, or listed rows
    attend   attention of the last tokens of the sequences over that cache
    norm     residual addition, root-mean-square norm and rounding to 8-bit whole numbers with a scale per token
    linear   the product of such tokens with a matrix of 8-bit whole numbers with a scale per row

The cache: codes [batch, kv_heads, rows, 2 (K and V), 128], whole numbers of 8 bits or e4m3; scales f32 [batch, kv_heads, blocks, 2], so that
a value is code * scale; recent bf16 [batch, kv_heads, R, 2, 128], row r of a sequence at place r % R. The rows of whole blocks are those
of the codes, the rows behind the last whole block those of `recent`.  A block's scale is its largest magnitude / 127 (448 for e4m3).  Codes and
whole numbers come back as they are stored, with their scales beside them: how they are rounded is part of the definition.
"""
import math

import torch

own = False

DEV = "cuda:0"
OUTLIERS = (7, 37, 71, 101)   # channels with large values


def _cache(kind, **kw):
    case = dict(kind=kind, batch=1, kv_heads=8, context_lo=4096, context_hi=4096, block=64, e4m3=False)
    case.update(kw)
    return case


def _append(**kw):
    return _cache("append", **{**dict(new=1), **kw})


def _read(**kw):
    return _cache("read", **{**dict(rows=0), **kw})


def _attend(**kw):
    return _cache("attend", **{**dict(q_heads=32, tokens=1), **kw})


def _norm(**kw):
    case = dict(kind="norm", tokens=1, width=4096, residual=True)
    case.update(kw)
    return case


def _linear(**kw):
    case = dict(kind="linear", tokens=1, out_features=4096, in_features=4096)
    case.update(kw)
    return case


def listed():
    return [
        # a decode step's token of every sequence of a batch: nothing but latency, now and then a block is full
        _append(name="append_1_b16", batch=16, context_lo=1021, context_hi=4096),
        # a long prompt, written once
        _append(name="append_prompt_32k", context_lo=32749, context_hi=32749, new=32749),
        # the rows that a selection names for one layer, brought back for an attention in 16 bits
        _read(name="read_2048_rows", context_lo=131072, context_hi=131072, rows=2048),
        # the context of two sequences of different lengths, as the attention of a further piece of prompt wants it
        _read(name="read_context_b2", batch=2, context_lo=40001, context_hi=65536, block=128, e4m3=True),
        # a chat turn on a short prompt: one token per sequence, nothing but latency
        _attend(name="attend_1_token_701", context_lo=701, context_hi=701),
        # a decode step at the 128K-context configuration
        _attend(name="attend_128k", context_lo=131072, context_hi=131072),
        # the batched configuration: sequences of different lengths, smaller blocks, the other type
        _attend(name="attend_varlen_b16", batch=16, context_lo=16384, context_hi=32768, block=32, e4m3=True),
        # one rank's share of a 64 / 8-head model over 8 GPUs with four drafted tokens per sequence: 32 query rows per KV head
        _attend(name="attend_4_tokens_tp_share_b8", batch=8, kv_heads=1, q_heads=8, tokens=4, context_lo=49999, context_hi=65536),
        # one token
        _norm(name="norm_1"),
        # a prompt's tokens
        _norm(name="norm_prompt_4096", tokens=4096),
        # the q/k/v rows of one token
        _linear(name="linear_qkv_1", out_features=6144),
        # gate and up of a feed-forward layer for a piece of a prompt
        _linear(name="linear_gate_up_2048", tokens=2048, out_features=24576),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("append", "read", "attend", "attend", "attend", "norm", "linear", "linear", "linear"))
    if kind == "norm":
        while True:
            tokens, width = _log(rng, 1, 16384), 8 * _log(rng, 8, 2048)
            if tokens * width <= 4096 * 4096:
                return _norm(tokens=tokens, width=width, residual=rng.random() < 0.7)
    if kind == "linear":
        while True:
            tokens, rows, cols = _log(rng, 1, 4096), _log(rng, 16, 152000), 16 * _log(rng, 4, 1024)
            if rows * cols <= 151936 * 4096 and tokens * rows * cols <= 2048 * 24576 * 4096:
                return _linear(tokens=tokens, out_features=rows, in_features=cols)
    heads = rng.choice((1, 2, 4, 8))
    batch = rng.choice((1, 1, 2, 3, 4, 8, 16))
    common = dict(batch=batch, kv_heads=heads, block=rng.choice((16, 32, 64, 128)), e4m3=rng.random() < 0.5)
    while True:
        hi = _log(rng, 1, 131072)
        lo = max(1, int(hi * rng.uniform(0.3, 1.0)))
        if kind == "append":
            new = rng.choice((1, 1, 5, common["block"] - 1, hi))   # a whole prompt, or a step, which may be run again: no row that it needs is overwritten
            if batch * heads * hi <= 8 * 32749 and (new <= lo or new == hi):
                return _append(context_lo=max(lo, new), context_hi=hi, new=new, **common)
        elif kind == "read":
            rows = rng.choice((0, 0, 1, 100, 2048))
            if batch * heads * hi <= 8 * 131072 and batch * heads * (rows or hi) <= 16 * 65536:
                return _read(context_lo=lo, context_hi=hi, rows=rows, **common)
        else:
            group, tokens = rng.choice((1, 2, 3, 4, 4, 5, 7, 8)), rng.choice((1, 1, 1, 2, 3, 5, 8, 16))
            if batch * heads * hi <= 16 * 8 * 24576 and batch * heads * hi * group * tokens <= 16 * 8 * 24576 * 4:
                return _attend(q_heads=heads * group, tokens=tokens, context_lo=lo, context_hi=hi, **common)


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _lengths(case, seed):
    """Lengths of the samples, the last one the longest; whole numbers that the seed alone decides."""
    g = torch.Generator().manual_seed(seed * 7 + 1)
    ls = torch.randint(case["context_lo"], case["context_hi"] + 1, (case["batch"],), generator=g).tolist()
    ls[-1] = case["context_hi"]
    return ls


def _rows(g, *shape):
    """Rows of K and V [..., 2, 128]: keys with large values in a few channels and norms that vary from token to token."""
    x = torch.randn(*shape, 2, 128, generator=g, device=DEV, dtype=torch.bfloat16)
    x[..., 0, list(OUTLIERS)] *= 8
    x[..., 0, :] *= torch.exp(0.5 * torch.randn(*shape, 1, generator=g, device=DEV)).to(torch.bfloat16)
    return x


def _code_type(case):
    return torch.float8_e4m3fn if case["e4m3"] else torch.int8


def _encode(x, amax, most, kind):
    """Codes of x whose block has the largest magnitude amax (f32, broadcast): x most / amax, rounded.  The power of two on both sides keeps the
    product from overflowing; with inputs of 16 bits the quotient's rounding to 32 bits moves no value to or from the middle of two codes."""
    unit = 128 if most < 128 else 512
    q = (x * (most / unit)) / torch.where(amax > 0, amax * (1 / unit), 1.0)
    q = torch.where(torch.isfinite(amax), q, 0.0)
    return q.to(kind) if kind == torch.float8_e4m3fn else torch.round(q).to(kind)


def _scale(amax, most):
    return torch.where(torch.isfinite(amax), amax / torch.full_like(amax, most), float("nan"))


def _blocks_of(x, case):
    """x f32 [..., blocks, block, 2, 128] -> codes of the same shape, scales [..., blocks, 2]."""
    most = 448.0 if case["e4m3"] else 127.0
    amax = x.abs().amax((-3, -1))
    return _encode(x, amax[..., None, :, None], most, _code_type(case)), _scale(amax, most)


def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def prepare(case, seed):
    g = _generator(seed)
    st = dict(case=case)
    if case["kind"] == "norm":
        tokens, width = case["tokens"], case["width"]
        a = torch.randn(tokens, width, generator=g, device=DEV)
        a[:, ::max(1, width // 8)] *= 10   # a few large channels
        st["a"] = a.to(torch.bfloat16)
        st["residual"] = torch.randn(tokens, width, generator=g, device=DEV).to(torch.bfloat16) * 4 if case["residual"] else None
        st["weight"] = (1 + 0.2 * torch.randn(width, generator=g, device=DEV)).to(torch.bfloat16)
        return st
    if case["kind"] == "linear":
        tokens, rows, cols = case["tokens"], case["out_features"], case["in_features"]
        x = torch.randn(tokens, cols, generator=g, device=DEV)
        x[:, ::max(1, cols // 8)] *= 10
        amax = x.abs().amax(-1)
        st["x"], st["x_scales"] = torch.round(x * (127 / amax)[:, None]).to(torch.int8), amax / 127
        w, s = torch.empty(rows, cols, dtype=torch.int8, device=DEV), torch.empty(rows, device=DEV)
        for r in range(0, rows, 16384):   # weights of a trained layer's spread, rounded row by row
            piece = torch.randn(min(16384, rows - r), cols, generator=g, device=DEV) / cols ** 0.5
            top = piece.abs().amax(-1)
            w[r:r + 16384], s[r:r + 16384] = torch.round(piece * (127 / top)[:, None]).to(torch.int8), top / 127
        st.update(weight=w, weight_scales=s)
        return st
    batch, heads, block = case["batch"], case["kv_heads"], case["block"]
    lengths = _lengths(case, seed)
    st["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    blocks, places = -(-case["context_hi"] // block), 2 * block
    codes = torch.zeros(batch, heads, blocks * block, 2, 128, dtype=torch.uint8, device=DEV)
    scales = torch.zeros(batch, heads, blocks, 2, device=DEV)
    recent = torch.zeros(batch, heads, places, 2, 128, dtype=torch.bfloat16, device=DEV)
    new = case.get("new", 0)
    fresh = torch.empty(batch, new, heads, 2, 128, dtype=torch.bfloat16, device=DEV) if new else None
    queries = []
    for b, n in enumerate(lengths):   # what the cache held before the call
        x = _rows(g, heads, n)
        if new:
            fresh[b] = x[:, n - new:].transpose(0, 1)
        old = n - new
        full = old // block * block
        if full:
            c, scales[b, :, :full // block] = _blocks_of(x[:, :full].float().view(heads, -1, block, 2, 128), case)
            codes[b, :, :full] = c.view(torch.uint8).view(heads, full, 2, 128)
        kept = torch.arange(max(0, old - places), old, device=DEV)
        recent[b][:, kept % places] = x[:, kept]
        if case["kind"] == "attend":   # each token's queries lean towards one of the sequence's keys
            tokens, group = case["tokens"], case["q_heads"] // heads
            pick = (torch.rand(tokens, generator=g, device=DEV) * n).long()
            base = x[:, pick, 0].float().transpose(0, 1)[:, :, None]
            base = base / base.norm(dim=-1, keepdim=True).clamp(min=1e-6)
            q = 0.3 * base + torch.randn(tokens, heads, group, 128, generator=g, device=DEV) / 128 ** 0.5
            queries.append((q * (4.0 / q.norm(dim=-1, keepdim=True))).reshape(tokens, heads * group, 128).to(torch.bfloat16))
        if case["kind"] == "read" and case["rows"]:
            at = torch.rand(heads, case["rows"], generator=g, device=DEV)
            queries.append((at * n).long().clamp(max=n - 1).sort(-1).values)
    st.update(codes=codes.view(_code_type(case)), scales=scales, recent=recent)
    if case["kind"] == "append":
        st.update(keys=fresh[:, :, :, 0].contiguous(), values=fresh[:, :, :, 1].contiguous())
    elif case["kind"] == "attend":
        st["queries"] = torch.stack(queries)
    else:
        st["rows"] = torch.stack(queries) if case["rows"] else None
        st["out"] = torch.zeros(batch, heads, case["rows"] or blocks * block, 2, 128, dtype=torch.bfloat16, device=DEV)
    return st


# ---- the plain forms -------------------------------------------------------------------------------------------------
def _plain_append(st):
    case, lengths, recent, scales = st["case"], st["lengths"].long(), st["recent"], st["scales"]
    block, codes = case["block"], st["codes"].view(torch.uint8)
    batch, heads, cap = codes.shape[:3]
    new = st["keys"].shape[1]
    fresh = torch.stack((st["keys"], st["values"]), 3).transpose(1, 2)   # [batch, heads, new, 2, 128]
    places, blocks = recent.shape[2], scales.shape[2]
    start = (lengths - new)[:, None]
    first = torch.div(start, block, rounding_mode="floor")
    count = min((new + block - 2) // block + 1, blocks)   # blocks that the new rows can touch
    ids = first.clamp(max=blocks - count) + torch.arange(count, device=codes.device)
    rows = (ids[..., None] * block + torch.arange(block, device=codes.device)).view(batch, -1)
    wide = lambda i: i[:, None, :, None, None].expand(-1, heads, -1, 2, 128)   # noqa: E731
    x = torch.where(wide(rows >= start), torch.gather(fresh, 2, wide((rows - start).clamp(0, new - 1))), torch.gather(recent, 2, wide(rows % places)))
    c, s = _blocks_of(x.float().view(batch, heads, count, block, 2, 128), case)
    c = c.view(torch.uint8).view(batch, heads, -1, 2, 128)
    done = (ids >= first) & ((ids + 1) * block <= lengths[:, None])   # blocks that are full now
    at, where = done.repeat_interleave(block, 1), ids[:, None, :, None].expand(-1, heads, -1, 2)
    codes.scatter_(2, wide(rows), torch.where(wide(at), c, torch.gather(codes, 2, wide(rows))))
    scales.scatter_(2, where, torch.where(done[:, None, :, None], s, torch.gather(scales, 2, where)))
    place = torch.arange(places, device=codes.device)
    held = lengths[:, None] - 1 - (lengths[:, None] - 1 - place) % places   # the last row at each place
    held_new = torch.gather(fresh, 2, wide((held - start).clamp(0, new - 1)))
    recent.copy_(torch.where(wide((held >= start) & (held >= 0)), held_new, recent))
    return st["codes"], scales, recent


def _values(st):
    """What the codes stand for, f32 [batch, heads, cap, 2, 128]."""
    return st["codes"].float() * st["scales"].repeat_interleave(st["case"]["block"], 2)[..., None]


def _plain_read(st):
    case, lengths, rows, out, recent = st["case"], st["lengths"].long()[:, None], st["rows"], st["out"], st["recent"]
    full = torch.div(lengths, case["block"], rounding_mode="floor") * case["block"]
    wide = lambda i: i[..., None, None].expand(-1, -1, -1, 2, 128)   # noqa: E731
    if rows is None:
        at = torch.arange(out.shape[2], device=out.device).expand(lengths.shape[0], -1)[:, None].expand(-1, out.shape[1], -1)
        x = _values(st)
    else:
        at = rows
        codes = torch.gather(st["codes"].view(torch.uint8), 2, wide(at)).view(st["codes"].dtype)
        x = codes.float() * torch.gather(st["scales"], 2, torch.div(at, case["block"], rounding_mode="floor")[..., None].expand(-1, -1, -1, 2))[..., None]
    tail = torch.gather(recent, 2, wide(at % recent.shape[2]))
    x = torch.where(wide(at >= full[:, None]), tail, x.to(torch.bfloat16))
    out.copy_(torch.where(wide(at < lengths[:, None]), x, out))
    return out


def _plain_attend(st):
    case, q, lengths, recent = st["case"], st["queries"], st["lengths"].long()[:, None], st["recent"]
    batch, tokens, q_heads, _ = q.shape
    heads, cap = st["codes"].shape[1:3]
    group, places = q_heads // heads, recent.shape[2]
    full = torch.div(lengths, case["block"], rounding_mode="floor") * case["block"]
    at = torch.arange(cap, device=q.device).expand(batch, -1)
    place = torch.arange(places, device=q.device)
    held = lengths - 1 - (lengths - 1 - place) % places
    row = torch.cat((torch.where(at < full, at, -1), torch.where(held >= full, held, -1)), 1)   # -1: not there
    pos = lengths - tokens + torch.arange(tokens, device=q.device)
    seen = (row[:, None] >= 0) & (row[:, None] <= pos[:, :, None])   # [batch, tokens, cap + places]
    kv = torch.cat((_values(st), recent.float()), 2)
    k, v = kv[..., 0, :], torch.where((row >= 0)[:, None, :, None], kv[..., 1, :], 0.0)
    qs = q.view(batch, tokens, heads, group, 128).permute(0, 2, 1, 3, 4).reshape(batch, heads, tokens * group, 128).float()
    s = (qs @ k.transpose(2, 3)) * 128 ** -0.5
    s = torch.where(seen.repeat_interleave(group, 1)[:, None], s, float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(m), 0.0, m))
    total = p.sum(-1, keepdim=True)
    o = (p @ v) / torch.where(total > 0, total, 1.0)
    return o.view(batch, heads, tokens, group, 128).permute(0, 2, 1, 3, 4).reshape(batch, tokens, q_heads, 128).to(torch.bfloat16)


def _plain_norm(st):
    h = st["a"].float()
    h = (h if st["residual"] is None else h + st["residual"].float()).to(torch.bfloat16)
    mean = h.double().square().mean(-1, keepdim=True)   # 64 bits: a code next to a border does not hang on the order of a sum
    rstd = (1 / torch.sqrt(mean + 1e-6)).float()
    y = h.float() * rstd * st["weight"].float()
    amax = y.abs().amax(-1, keepdim=True)
    return h, _encode(y, amax, 127.0, torch.int8), _scale(amax, 127.0).view(-1)


def _plain_linear(st):
    return ((st["x"].float() @ st["weight"].float().t()) * st["x_scales"][:, None] * st["weight_scales"]).to(torch.bfloat16)


# ---- one pass --------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        return {"append": _plain_append, "read": _plain_read, "attend": _plain_attend, "norm": _plain_norm, "linear": _plain_linear}[kind](state)
    from pariskv_b200 import ops
    if kind == "norm":
        return ops.add_rmsnorm_i8(state["a"], state["residual"], state["weight"], eps=1e-6)
    if kind == "linear":
        return ops.matmul_i8(state["x"], state["x_scales"], state["weight"], state["weight_scales"])
    cache = ops.Cache8(state["codes"], state["scales"], state["recent"], case["block"])
    if kind == "append":
        ops.cache8_append(cache, state["keys"], state["values"], state["lengths"])
        return cache.codes, cache.scales, cache.recent
    if kind == "read":
        return ops.cache8_read(cache, state["lengths"], rows=state["rows"], out=state["out"])
    return ops.cache8_attention(state["queries"], cache, state["lengths"])


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "norm":
        values = case["tokens"] * case["width"]
        return {"bytes": values * (7 if case["residual"] else 5) + 4 * case["tokens"] + 2 * case["width"], "flops": 8 * values}
    if case["kind"] == "linear":
        tokens, rows, cols = case["tokens"], case["out_features"], case["in_features"]
        return {"bytes": rows * cols + tokens * cols + 2 * tokens * rows + 4 * (tokens + rows), "flops": 2 * tokens * rows * cols}
    batch, heads, block = case["batch"], case["kv_heads"], case["block"]
    mean = (case["context_lo"] + case["context_hi"]) / 2 * (batch - 1) + case["context_hi"]   # rows of all samples, about
    if case["kind"] == "append":   # the new rows; their codes and scales; the last of them as they are
        new = batch * heads * case["new"]
        kept = batch * heads * min(case["new"], 2 * block)
        return {"bytes": int(512 * new + 256 * new + 8 * new / block + 512 * kept), "flops": int(1024 * new)}
    if case["kind"] == "read":
        rows = heads * (batch * case["rows"] if case["rows"] else mean)
        return {"bytes": int(rows * (256 + 512 + 8 / block) + (8 * rows if case["rows"] else 0)), "flops": int(256 * rows)}
    tokens, q_heads = case["tokens"], case["q_heads"]
    return {"bytes": int(heads * mean * (256 + 8 / block) + 512 * batch * tokens * q_heads), "flops": int(512 * tokens * q_heads * mean)}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------
def _to_e4m3(v):
    """The nearest number of four bits of significand, ties to the even one; steps of 2^-9 below 2^-6."""
    exponent = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(exponent - 3)
    return torch.round(v / step) * step


def _exact_cache(case, seed):
    """The rows of every sample, and what the cache holds of them: the same draws as prepare() makes."""
    g, out = _generator(seed), []
    for n in _lengths(case, seed):
        x = _rows(g, case["kv_heads"], n)
        if case["kind"] == "attend":
            torch.rand(case["tokens"], generator=g, device=DEV)
            torch.randn(case["tokens"], case["kv_heads"], case["q_heads"] // case["kv_heads"], 128, generator=g, device=DEV)
        if case["kind"] == "read" and case["rows"]:
            torch.rand(case["kv_heads"], case["rows"], generator=g, device=DEV)
        out.append(x)
    return out


def _exact_sample(x, case):
    """Codes, scales and values of one sample's whole blocks; x [heads, n, 2, 128] in 64 bits."""
    heads, n = x.shape[:2]
    most, block = (448 if case["e4m3"] else 127), case["block"]
    full = n // block * block
    part = x[:, :full].reshape(heads, full // block, block, 2, 128)
    top = part.abs().permute(0, 1, 3, 2, 4).reshape(heads, full // block, 2, -1).amax(-1) if full else torch.zeros(heads, 0, 2, dtype=x.dtype, device=x.device)
    unit = torch.where(top > 0, top, 1.0)[:, :, None, :, None]
    quotient = part * most / unit
    codes = _to_e4m3(quotient) if case["e4m3"] else torch.round(quotient)
    return codes.reshape(heads, full, 2, 128), top / most, (codes * (top / most)[:, :, None, :, None]).reshape(heads, full, 2, 128)


def exact(case, seed):
    if case["kind"] == "norm":
        st = prepare(case, seed)
        total = st["a"].double() if st["residual"] is None else st["a"].double() + st["residual"].double()
        h = total.float().to(torch.bfloat16)
        hd = h.double()
        y = hd / torch.sqrt(torch.einsum("tw,tw->t", hd, hd) / case["width"] + 1e-6)[:, None] * st["weight"].double()
        top = y.abs().max(-1).values
        return total, torch.round(y / (top / 127)[:, None]).to(torch.int8), top / 127
    if case["kind"] == "linear":
        st = prepare(case, seed)
        w = st["weight"].double() * st["weight_scales"].double()[:, None]
        return torch.einsum("tk,ok->to", st["x"].double() * st["x_scales"].double()[:, None], w)
    block, heads = case["block"], case["kv_heads"]
    samples = _exact_cache(case, seed)
    if case["kind"] == "attend":
        st = prepare(case, seed)
        tokens, group = case["tokens"], case["q_heads"] // heads
        out = torch.zeros(st["queries"].shape, dtype=torch.float64, device=DEV)
        for b, x in enumerate(samples):
            n = x.shape[1]
            for h in range(heads):
                kv = torch.cat((_exact_sample(x[h:h + 1].double(), case)[2][0], x[h, n // block * block:].double()))
                for t in range(tokens):
                    last = n - tokens + t + 1
                    if last > 0:
                        q = st["queries"][b, t, h * group:(h + 1) * group].double()
                        w = torch.softmax(torch.einsum("gd,nd->gn", q, kv[:last, 0]) / math.sqrt(128), -1)
                        out[b, t, h * group:(h + 1) * group] = torch.einsum("gn,nd->gd", w, kv[:last, 1])
        return out
    blocks = -(-case["context_hi"] // block)
    if case["kind"] == "append":
        codes = torch.zeros(case["batch"], heads, blocks * block, 2, 128, dtype=torch.float32 if case["e4m3"] else torch.int8, device=DEV)
        scales = torch.zeros(case["batch"], heads, blocks, 2, dtype=torch.float64, device=DEV)
        recent = torch.zeros(case["batch"], heads, 2 * block, 2, 128, dtype=torch.float64, device=DEV)
        for b, x in enumerate(samples):
            n = x.shape[1]
            full = n // block * block
            for h in range(heads):
                c, s, _ = _exact_sample(x[h:h + 1].double(), case)
                codes[b, h, :full], scales[b, h, :full // block] = c[0].to(codes.dtype), s[0]
            for r in range(max(0, n - 2 * block), n):
                recent[b, :, r % (2 * block)] = x[:, r].double()
        return codes, scales, recent
    out = torch.zeros(case["batch"], heads, case["rows"] or blocks * block, 2, 128, dtype=torch.float64, device=DEV)
    st = prepare(case, seed)
    for b, x in enumerate(samples):
        n = x.shape[1]
        for h in range(heads):
            kv = torch.cat((_exact_sample(x[h:h + 1].double(), case)[2][0], x[h, n // block * block:].double()))
            if case["rows"]:
                out[b, h] = kv[st["rows"][b, h]]
            else:
                out[b, h, :n] = kv
    return out
