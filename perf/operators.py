"""The operators of a decode step with drafted tokens, block selection and 4-bit weights: what is measured.

    own                 False: run() computes the plain forms; True: run() calls the framework's kernels
    listed()            the named cases
    draw(rng)           another case of the same ranges
    prepare(case, seed) inputs, on the GPU, as a program holds them
    run(state)          one pass; returns the whole outputs
    work(case)          bytes and operations that a pass cannot do without
    exact(case, seed)   the outputs in 64 bits, from the definitions

Kinds of case
    tree     attention of T drafted tokens per sequence (a tree, given by a mask) over the cache and the drafts themselves
    bounds   smallest and largest value per channel of every block of keys: of a whole cache, or of the rows just appended
    blocks   selection of blocks by those bounds for every token and KV head, and attention over the selected blocks
    w4       y = x W^T for a few tokens, W of 4-bit codes with a scale (and an offset) per group of columns
"""
import math

import torch

own = False

DEV = "cuda:0"
OUTLIERS = (7, 37, 71, 101)   # key channels with large values


def _tree(**kw):
    case = dict(kind="tree", batch=1, kv_heads=8, q_heads=32, tokens=16, context_lo=4096, context_hi=4096)
    case.update(kw)
    return case


def _bounds(**kw):
    case = dict(kind="bounds", batch=1, kv_heads=8, context_lo=4096, context_hi=4096, block=64, n_new=0)
    case.update(kw)
    return case


def _blocks(**kw):
    case = dict(kind="blocks", batch=1, kv_heads=8, q_heads=32, tokens=1, context_lo=32768, context_hi=32768, block=64,
                n_select=32, sink_blocks=1, local_blocks=2)
    case.update(kw)
    return case


def _w4(**kw):
    case = dict(kind="w4", tokens=1, out_features=4096, in_features=4096, group=128, offsets=False, gated=False)
    case.update(kw)
    return case


def listed():
    return [
        # a chat turn on a short prompt without drafts: one token per sequence, nothing but latency
        _tree(name="tree_1_token_701", tokens=1, context_lo=701, context_hi=701),
        # a batch of requests of different lengths, each with an odd number of drafted tokens
        _tree(name="tree_13_varlen_b4", batch=4, tokens=13, context_lo=2477, context_hi=16384),
        # one rank's share of a 64 / 8-head model over 8 GPUs: one KV head with eight query heads, batch 8
        _tree(name="tree_26_tp_share_b8", batch=8, kv_heads=1, q_heads=8, tokens=26, context_lo=65536, context_hi=65536),
        # a wide tree over the 128K-context configuration
        _tree(name="tree_61_128k", tokens=61, context_lo=131072, context_hi=131072),
        # a decode step's token appended to every sequence of the batched configuration: only the last blocks change
        _bounds(name="bounds_append_b16", batch=16, context_lo=16384, context_hi=32768, n_new=1),
        # the summaries of a long prompt, made once
        _bounds(name="bounds_prompt_128k", context_lo=131072, context_hi=131072),
        # a decode step over 32K keys with a budget of 2048 rows per head
        _blocks(name="blocks_32k", context_lo=32749, context_hi=32749),
        # the batched configuration: sequences of different lengths, smaller blocks
        _blocks(name="blocks_varlen_b16", batch=16, context_lo=16384, context_hi=32768, block=32, n_select=64),
        # the million-token configuration with a chain of four drafted tokens, each choosing for itself
        _blocks(name="blocks_1m_4_tokens", tokens=4, context_lo=1048576, context_hi=1048576, block=128, n_select=24),
        # the q/k/v rows of one token
        _w4(name="w4_qkv_1", out_features=6144, in_features=4096),
        # gate and up of a feed-forward layer for six drafted tokens, small groups with offsets
        _w4(name="w4_gate_up_6", tokens=6, out_features=24576, in_features=4096, group=64, offsets=True, gated=True),
        # the vocabulary of 151936 rows, one token
        _w4(name="w4_vocab_1", out_features=151936, in_features=4096),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("tree", "tree", "bounds", "blocks", "blocks", "w4", "w4"))
    if kind == "w4":
        group = rng.choice((32, 64, 128))
        while True:
            tokens = _log(rng, 1, 16)
            rows, cols = _log(rng, 64, 152000), group * max(1, _log(rng, 256, 16384) // group)
            gated = rng.random() < 0.4
            if rows * cols <= 151936 * 4096 and rows * cols * tokens <= 24576 * 4096 * 6:
                return _w4(tokens=tokens, out_features=2 * ((rows + 1) // 2) if gated else rows, in_features=cols, group=group,
                           offsets=rng.random() < 0.5, gated=gated)
    heads = rng.choice((1, 2, 4, 8))
    batch = rng.choice((1, 1, 2, 3, 4, 8, 16))
    group = rng.choice((1, 2, 3, 4, 4, 5, 7, 8))
    if kind == "tree":
        while True:
            hi, tokens = _log(rng, 1, 131072), _log(rng, 1, 64)
            if batch * heads * hi <= 8 * 131072 and batch * heads * hi * group * tokens <= 8 * 131072 * 4 * 61:
                return _tree(batch=batch, kv_heads=heads, q_heads=heads * group, tokens=tokens,
                             context_lo=max(0, int(hi * rng.uniform(0.3, 1.0)) - 1), context_hi=hi)
    block = rng.choice((16, 32, 64, 128))
    if kind == "bounds":
        while True:
            hi = _log(rng, 1, 131072)
            if batch * heads * hi <= 8 * 131072:
                return _bounds(batch=batch, kv_heads=heads, context_lo=max(1, int(hi * rng.uniform(0.3, 1.0))), context_hi=hi,
                               block=block, n_new=rng.choice((0, 1, 1, 5, 130)))
    while True:
        hi, tokens = _log(rng, 64, 1048576), rng.choice((1, 1, 1, 2, 4, 7, 16))
        n_select = rng.choice((5, 16, 24, 32, 33, 64, 100))
        if (hi + block - 1) // block <= 16384 and batch * heads * hi <= 8 * 1048576 and \
                batch * heads * tokens * n_select * block <= 16 * 8 * 64 * 64:
            return _blocks(batch=batch, kv_heads=heads, q_heads=heads * group, tokens=tokens, block=block, n_select=n_select,
                           context_lo=max(tokens, int(hi * rng.uniform(0.3, 1.0))), context_hi=max(hi, tokens),
                           sink_blocks=rng.choice((0, 1, 2)), local_blocks=rng.choice((1, 2, 3)))


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _lengths(case, seed):
    """Lengths of the samples, the last one the longest; whole numbers that the seed alone decides."""
    lo, hi, n = case["context_lo"], case["context_hi"], case["batch"]
    g = torch.Generator().manual_seed(seed * 7 + 1)
    ls = torch.randint(lo, hi + 1, (n,), generator=g).tolist()
    ls[-1] = hi
    return ls


def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _keys(g, batch, heads, cap):
    """Keys with large values in a few channels and norms that vary from token to token."""
    k = torch.randn(batch, heads, cap, 128, generator=g, device=DEV, dtype=torch.bfloat16)
    k[..., list(OUTLIERS)] *= 8
    k *= torch.exp(0.5 * torch.randn(batch, heads, cap, 1, generator=g, device=DEV)).to(torch.bfloat16)
    return k


def _queries(g, keys, lengths, tokens, q_heads):
    """Each token's queries lean towards one of the sequence's keys."""
    batch, heads = keys.shape[:2]
    group = q_heads // heads
    pick = (torch.rand(batch, heads, tokens, generator=g, device=DEV) * lengths[:, None, None]).long()
    base = torch.gather(keys, 2, pick[..., None].expand(-1, -1, -1, 128)).float()
    base = base / base.norm(dim=-1, keepdim=True).clamp(min=1e-6)
    q = 0.3 * base[:, :, :, None] + torch.randn(batch, heads, tokens, group, 128, generator=g, device=DEV) / 128 ** 0.5
    q = q * (4.0 / q.norm(dim=-1, keepdim=True))
    return q.permute(0, 2, 1, 3, 4).reshape(batch, tokens, q_heads, 128).to(torch.bfloat16).contiguous()


def _tree_mask(batch, tokens, seed):
    """Random trees, one per sequence: a token sees itself and its ancestors."""
    g = torch.Generator().manual_seed(seed * 7 + 2)
    parent = (torch.rand(batch, tokens, generator=g) * torch.arange(tokens)).long() - (torch.rand(batch, tokens, generator=g) < 0.2).long()
    mask = torch.zeros(batch, tokens, tokens, dtype=torch.bool)
    at = torch.arange(batch)
    for t in range(tokens):
        p = parent[:, t] if t else torch.full((batch,), -1)
        mask[:, t] = mask[at, p.clamp(min=0)] & (p >= 0)[:, None]
        mask[:, t, t] = True
    return mask


def _bounds_of(keys, lengths, block):
    """lo / hi per block of the rows below `lengths`; blocks without such rows are zero."""
    batch, heads, cap, _ = keys.shape
    nb = (cap + block - 1) // block
    live = torch.arange(nb * block, device=DEV)[None, :] < lengths[:, None]
    out = torch.empty(batch, heads, nb, 2, 128, dtype=keys.dtype, device=DEV)
    for b in range(batch):
        k = torch.nn.functional.pad(keys[b], (0, 0, 0, nb * block - cap))
        m = live[b][None, :, None]
        out[b, :, :, 0] = torch.where(m, k, float("inf")).view(heads, nb, block, 128).amin(2)
        out[b, :, :, 1] = torch.where(m, k, float("-inf")).view(heads, nb, block, 128).amax(2)
    some = torch.arange(nb, device=DEV)[None, :] * block < lengths[:, None]
    return torch.where(some[:, None, :, None, None], out, 0.0)


def prepare(case, seed):
    g = _generator(seed)
    st = dict(case=case)
    if case["kind"] == "w4":
        rows, cols, group = case["out_features"], case["in_features"], case["group"]
        codes = torch.empty(rows, cols // 2, dtype=torch.uint8, device=DEV)
        scales = torch.empty(rows, cols // group, dtype=torch.bfloat16, device=DEV)
        offsets = torch.empty_like(scales) if case["offsets"] else None
        for r in range(0, rows, 16384):   # weights of a trained layer's spread, rounded to 4 bits group by group
            w = torch.randn(min(16384, rows - r), cols // group, group, generator=g, device=DEV) / cols ** 0.5
            if offsets is not None:
                lo, hi = w.amin(-1), w.amax(-1)
                s, m = ((hi - lo) / 15).to(torch.bfloat16), lo.to(torch.bfloat16)
                offsets[r:r + 16384] = m
                c = torch.round((w - m.float()[..., None]) / s.float()[..., None])
            else:
                s = (w.abs().amax(-1) / 7.5).to(torch.bfloat16)
                c = torch.round(w / s.float()[..., None]) + 8
            scales[r:r + 16384] = s
            c = c.clamp(0, 15).to(torch.uint8).view(-1, cols)
            codes[r:r + 16384] = c[:, 0::2] | (c[:, 1::2] << 4)
        x = torch.randn(case["tokens"], cols, generator=g, device=DEV)
        x[:, :: max(1, cols // 8)] *= 10   # a few large activations
        st.update(codes=codes, scales=scales, offsets=offsets, x=x.to(torch.bfloat16))
        return st
    batch, heads, cap = case["batch"], case["kv_heads"], case["context_hi"]
    st["lengths"] = torch.tensor(_lengths(case, seed), dtype=torch.int32, device=DEV)
    if case["kind"] == "tree":
        cap = max(cap, 1)
        keys = _keys(g, batch, heads, cap)
        tokens = case["tokens"]
        st.update(keys=keys, values=torch.randn(keys.shape, generator=g, device=DEV, dtype=torch.bfloat16),
                  queries=_queries(g, keys, st["lengths"].clamp(min=1), tokens, case["q_heads"]),
                  draft_keys=_keys(g, batch, heads, tokens).transpose(1, 2).contiguous(),
                  draft_values=torch.randn(batch, tokens, heads, 128, generator=g, device=DEV, dtype=torch.bfloat16),
                  mask=_tree_mask(batch, tokens, seed).to(DEV))
        return st
    keys = _keys(g, batch, heads, cap)
    st["keys"] = keys
    if case["kind"] == "bounds":
        # what the cache holds before the call: of the whole cache nothing yet, or the blocks as they were before the new rows
        nb = (cap + case["block"] - 1) // case["block"]
        st["bounds"] = (_bounds_of(keys, (st["lengths"] - case["n_new"]).clamp(min=0), case["block"]) if case["n_new"]
                        else torch.zeros(batch, heads, nb, 2, 128, dtype=torch.bfloat16, device=DEV))
        return st
    st.update(values=torch.randn(keys.shape, generator=g, device=DEV, dtype=torch.bfloat16),
              queries=_queries(g, keys, st["lengths"], case["tokens"], case["q_heads"]),
              bounds=_bounds_of(keys, st["lengths"], case["block"]))
    return st


# ---- the plain forms -------------------------------------------------------------------------------------------------
def _softmax_parts(scores, seen, values):
    """scores [..., n], seen [..., n] -> the weighted mean of values over what is seen, zero where nothing is."""
    s = torch.where(seen, scores, float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(m), 0.0, m))
    total = p.sum(-1, keepdim=True)
    return (p @ values) / torch.where(total > 0, total, 1.0)


def _plain_tree(st):
    q, keys, values, lengths, mask = st["queries"], st["keys"], st["values"], st["lengths"], st["mask"]
    batch, tokens, q_heads, _ = q.shape
    heads, cap = keys.shape[1:3]
    group = q_heads // heads
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    at = torch.arange(cap, device=q.device)
    for b in range(batch):
        live = at < lengths[b]
        qs = q[b].view(tokens, heads, group, 128).permute(1, 0, 2, 3).reshape(heads, tokens * group, 128).float()
        k = torch.cat((keys[b].float(), st["draft_keys"][b].transpose(0, 1).float()), 1)
        v = torch.cat((torch.where(live[None, :, None], values[b].float(), 0.0), st["draft_values"][b].transpose(0, 1).float()), 1)
        seen = torch.cat((live[None].expand(tokens, -1), mask[b]), 1).repeat_interleave(group, 0)
        o = _softmax_parts((qs @ k.transpose(1, 2)) * 128 ** -0.5, seen[None], v)
        out[b] = o.view(heads, tokens, group, 128).permute(1, 0, 2, 3).reshape(tokens, q_heads, 128).to(q.dtype)
    return out


def _plain_bounds(st):
    case, bounds, keys = st["case"], st["bounds"], st["keys"]
    block, n_new = case["block"], case["n_new"]
    at = torch.arange(bounds.shape[2], device=bounds.device)[None, :]
    n = st["lengths"][:, None]
    if not n_new:
        new = _bounds_of(keys, st["lengths"], block)
        bounds.copy_(torch.where((at * block < n)[:, None, :, None, None], new, bounds))
        return bounds
    batch, heads, cap, _ = keys.shape
    count = min((n_new + block - 2) // block + 1, bounds.shape[2])   # blocks that the new rows can touch
    first = torch.div((n - n_new).clamp(min=0), block, rounding_mode="floor").clamp(max=bounds.shape[2] - count)
    ids = first + torch.arange(count, device=keys.device)
    rows = (ids[..., None] * block + torch.arange(block, device=keys.device)).view(batch, -1)
    live = (rows < n)[:, None, :, None]
    k = torch.gather(keys, 2, rows.clamp(max=cap - 1)[:, None, :, None].expand(-1, heads, -1, 128))
    lo = torch.where(live, k, float("inf")).view(batch, heads, count, block, 128).amin(3)
    hi = torch.where(live, k, float("-inf")).view(batch, heads, count, block, 128).amax(3)
    written = (ids * block < n) & (ids >= torch.div((n - n_new).clamp(min=0), block, rounding_mode="floor"))
    where = ids[:, None, :, None, None].expand(-1, heads, -1, 2, 128)
    old = torch.gather(bounds, 2, where)
    bounds.scatter_(2, where, torch.where(written[:, None, :, None, None], torch.stack((lo, hi), 3), old))
    return bounds


def _plain_select(st):
    case, q, bounds = st["case"], st["queries"], st["bounds"]
    batch, tokens, q_heads, _ = q.shape
    heads, nb = bounds.shape[1:3]
    block, n_select = case["block"], case["n_select"]
    qs = q.view(batch, tokens, heads, q_heads // heads, 128).permute(0, 2, 1, 3, 4).double()
    up, down = qs.clamp(min=0).sum(3), qs.clamp(max=0).sum(3)   # [batch, heads, tokens, 128]
    at = torch.arange(nb, device=q.device)
    pos = st["lengths"][:, None] - tokens + torch.arange(tokens, device=q.device)
    last = torch.div(pos, block, rounding_mode="floor")[:, None, :, None]
    seen = (at <= last) & (pos[:, None, :, None] >= 0)
    live = at[None, :] * block < st["lengths"][:, None]
    lo, hi = (torch.where(live[:, None, :, None], bounds[:, :, :, i], 0.0).double().transpose(2, 3) for i in (0, 1))
    score = (up @ hi + down @ lo).float()   # sums in 64 bits: the choice does not hang on their order
    score = torch.where((at < case["sink_blocks"]) | (at > last - case["local_blocks"]), float("inf"), score)
    score = torch.where(seen, score, float("-inf"))
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices
    n = min(n_select, nb)
    ids = order[..., :n]
    ids = torch.where(torch.gather(seen.expand(score.shape), -1, ids), ids, nb).sort(-1).values
    ids = torch.where(ids < nb, ids, -1)
    ids = torch.nn.functional.pad(ids, (0, n_select - n), value=-1)
    return ids.permute(0, 2, 1, 3).to(torch.int32).contiguous()


def _plain_block_attention(st, ids):
    case, q, keys, values, lengths = st["case"], st["queries"], st["keys"], st["values"], st["lengths"]
    batch, tokens, q_heads, _ = q.shape
    heads, cap = keys.shape[1:3]
    group, block = q_heads // heads, case["block"]
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    for b in range(batch):
        for t in range(tokens):
            pos = lengths[b] - tokens + t
            listed_ids = ids[b, t].long()   # [heads, n]
            rows = (listed_ids[..., None] * block + torch.arange(block, device=q.device)).view(heads, -1)
            seen = (rows >= 0) & (rows <= pos) & (listed_ids >= 0).repeat_interleave(block, -1)
            rows = rows.clamp(0, cap - 1)[..., None].expand(-1, -1, 128)
            k = torch.gather(keys[b], 1, rows).float()
            v = torch.where(seen[..., None], torch.gather(values[b], 1, rows).float(), 0.0)
            qs = q[b, t].view(heads, group, 128).float()
            out[b, t] = _softmax_parts((qs @ k.transpose(1, 2)) * 128 ** -0.5, seen[:, None], v).view(q_heads, 128).to(q.dtype)
    return out


def _plain_w4(st):
    case, x = st["case"], st["x"].float()
    outs = []
    for r in range(0, case["out_features"], 16384):
        c = st["codes"][r:r + 16384]
        s = st["scales"][r:r + 16384].float()[..., None]
        codes = torch.stack((c & 15, c >> 4), -1).view(c.shape[0], -1, case["group"]).float()
        w = codes * s + st["offsets"][r:r + 16384].float()[..., None] if case["offsets"] else (codes - 8) * s
        outs.append(x @ w.view(c.shape[0], -1).t())
    y = torch.cat(outs, 1)
    if case["gated"]:
        gate, up = y.chunk(2, 1)
        y = gate / (1 + torch.exp(-gate)) * up
    return y.to(torch.bfloat16)


# ---- one pass --------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        if kind == "tree":
            return _plain_tree(state)
        if kind == "bounds":
            return _plain_bounds(state)
        if kind == "blocks":
            ids = _plain_select(state)
            return ids, _plain_block_attention(state, ids)
        return _plain_w4(state)
    from pariskv_b200 import ops
    if kind == "tree":
        return ops.tree_attention(state["queries"], state["keys"], state["values"], state["draft_keys"], state["draft_values"],
                                  state["mask"], state["lengths"])
    if kind == "bounds":
        return ops.block_bounds(state["keys"], state["lengths"], block=case["block"], n_new=case["n_new"] or None,
                                bounds=state["bounds"])
    if kind == "blocks":
        ids = ops.select_blocks(state["queries"], state["bounds"], state["lengths"], case["n_select"], block=case["block"],
                                sink_blocks=case["sink_blocks"], local_blocks=case["local_blocks"])
        return ids, ops.block_attention(state["queries"], state["keys"], state["values"], ids, state["lengths"], block=case["block"])
    return ops.gemv_w4(state["codes"], state["scales"], state["x"], offsets=state["offsets"], gated=case["gated"])


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "w4":
        rows, cols, tokens = case["out_features"], case["in_features"], case["tokens"]
        per_group = 4 if case["offsets"] else 2
        outs = rows // 2 if case["gated"] else rows
        return {"bytes": rows * cols // 2 + per_group * rows * (cols // case["group"]) + 2 * tokens * (cols + outs),
                "flops": 2 * tokens * rows * cols}
    batch, heads = case["batch"], case["kv_heads"]
    mean = (case["context_lo"] + case["context_hi"]) / 2 * (batch - 1) + case["context_hi"]   # keys of all samples, about
    if case["kind"] == "bounds":
        if case["n_new"]:
            blocks = batch * min((case["n_new"] + case["block"] - 2) // case["block"] + 1, case["context_hi"] // case["block"] + 1)
            # the new rows have to be read, and the bounds they change written
            return {"bytes": heads * (256 * batch * min(case["n_new"], case["context_hi"]) + 512 * blocks),
                    "flops": 256 * heads * batch * case["n_new"]}
        return {"bytes": int(heads * (256 * mean + 512 * mean / case["block"])), "flops": int(256 * heads * mean)}
    tokens, q_heads = case["tokens"], case["q_heads"]
    small = 512 * batch * tokens * q_heads   # queries and outputs
    if case["kind"] == "tree":
        drafts = batch * tokens
        return {"bytes": int(512 * heads * (mean + drafts) + small + batch * tokens * tokens),
                "flops": int(512 * tokens * q_heads * mean)}
    rows = min(case["n_select"] * case["block"] * batch, mean)   # of one token; the others may choose the same
    return {"bytes": int(512 * heads * (mean / case["block"] + rows) + small + 4 * batch * tokens * heads * case["n_select"]),
            "flops": int(512 * tokens * (heads * mean / case["block"] + q_heads * rows))}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------
def _attend_exact(q, k, v):
    """q [g,128], k / v [n,128], all of them seen."""
    if k.shape[0] == 0:
        return torch.zeros_like(q)
    w = torch.softmax(torch.einsum("gd,nd->gn", q, k) / math.sqrt(128), -1)
    return torch.einsum("gn,nd->gd", w, v)


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "w4":
        x, ys = st["x"].double(), []
        for r in range(0, case["out_features"], 8192):
            packed = st["codes"][r:r + 8192].to(torch.int64)
            c = torch.empty(packed.shape[0], case["in_features"], dtype=torch.float64, device=DEV)
            c[:, 0::2], c[:, 1::2] = (packed % 16).double(), torch.div(packed, 16, rounding_mode="floor").double()
            s = st["scales"][r:r + 8192].double().repeat_interleave(case["group"], 1)
            m = st["offsets"][r:r + 8192].double().repeat_interleave(case["group"], 1) if case["offsets"] else -8 * s
            ys.append(torch.einsum("tk,ok->to", x, c * s + m))
        y = torch.cat(ys, 1)
        if case["gated"]:
            half = y.shape[1] // 2
            y = y[:, :half] * torch.sigmoid(y[:, :half]) * y[:, half:]
        return y
    lengths = st["lengths"].tolist()
    keys, heads, block = st["keys"], case["kv_heads"], case.get("block")
    if case["kind"] == "bounds":
        want = st["bounds"].double()
        for b, n in enumerate(lengths):
            first = max(0, n - case["n_new"]) // block if case["n_new"] else 0
            for j in range(first, (n + block - 1) // block) if case["n_new"] else ():
                rows = keys[b, :, j * block:min(n, (j + 1) * block)].double()
                want[b, :, j, 0], want[b, :, j, 1] = rows.min(1).values, rows.max(1).values
            if not case["n_new"]:
                full = n // block
                rows = keys[b, :, :full * block].double().view(heads, full, block, 128)
                if full:
                    want[b, :, :full, 0], want[b, :, :full, 1] = rows.min(2).values, rows.max(2).values
                if n > full * block:
                    rows = keys[b, :, full * block:n].double()
                    want[b, :, full, 0], want[b, :, full, 1] = rows.min(1).values, rows.max(1).values
        return want
    group = case["q_heads"] // heads
    tokens = case["tokens"]
    if case["kind"] == "tree":
        out = torch.empty(st["queries"].shape, dtype=torch.float64, device=DEV)
        for b, n in enumerate(lengths):
            for h in range(heads):
                k = torch.cat((keys[b, h, :n], st["draft_keys"][b, :, h])).double()
                v = torch.cat((st["values"][b, h, :n], st["draft_values"][b, :, h])).double()
                q = st["queries"][b, :, h * group:(h + 1) * group].double()
                hidden = torch.cat((torch.zeros(tokens, n, dtype=torch.bool, device=DEV), ~st["mask"][b]), 1)
                s = torch.einsum("tgd,nd->tgn", q, k) / math.sqrt(128)
                w = torch.softmax(s.masked_fill(hidden[:, None], float("-inf")), -1)
                out[b, :, h * group:(h + 1) * group] = torch.einsum("tgn,nd->tgd", w, v)
        return out
    # blocks: the scores as the definition has them, channel by channel, then the rows of the chosen blocks
    n_select = case["n_select"]
    ids = torch.full((case["batch"], tokens, heads, n_select), -1, dtype=torch.int32)
    out = torch.zeros(st["queries"].shape, dtype=torch.float64, device=DEV)
    for b, n in enumerate(lengths):
        for t in range(tokens):
            pos = n - tokens + t
            if pos < 0:
                continue
            visible = pos // block + 1
            for h in range(heads):
                q = st["queries"][b, t, h * group:(h + 1) * group].double()
                lo, hi = st["bounds"][b, h, :visible, 0].double(), st["bounds"][b, h, :visible, 1].double()
                score = torch.zeros(visible, dtype=torch.float64, device=DEV)
                for row in q:
                    score += torch.maximum(row * lo, row * hi).sum(-1)
                score = score.float()
                score[:case["sink_blocks"]] = float("inf")
                score[max(0, visible - case["local_blocks"]):] = float("inf")
                picks = sorted(range(visible), key=score.tolist().__getitem__, reverse=True)[:n_select]
                picks.sort()
                ids[b, t, h, :len(picks)] = torch.tensor(picks, dtype=torch.int32)
                rows = torch.tensor([r for j in picks for r in range(j * block, min(pos + 1, (j + 1) * block))], device=DEV)
                out[b, t, h * group:(h + 1) * group] = _attend_exact(q, keys[b, h, rows].double(), st["values"][b, h, rows].double())
    return ids.to(DEV), out
