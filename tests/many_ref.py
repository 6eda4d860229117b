"""Plain forms, in 64 bits, of the operators for several tokens a step, and the tolerances that follow from the types.

A bf16 rounding is off by at most half a step, U = 2^-8 of the value.  An attention output is one such rounding of a weighted
mean; the weights may be rounded to bf16 once before they meet the values, which moves the mean by at most U sum p|v|.  A score
is a sum of 128 products in fp32, each addition off by at most a whole step (2^-23) of the sum of absolute values; a weight
moves by that relative to itself, numerator and denominator both."""
import math

import torch

U = 2.0 ** -8


def attend(q, k, v, scale):
    """q [n_q,128], k / v [n,128] (all seen) -> (out, tolerance, lse in log2, its tolerance), in 64 bits."""
    q, k, v = q.double(), k.double(), v.double()
    if k.shape[0] == 0:
        z = torch.zeros_like(q)
        inf = torch.full((q.shape[0],), -math.inf, dtype=torch.float64, device=q.device)
        return z, z, inf, torch.zeros_like(inf)
    s = q @ k.t() * scale
    w = torch.softmax(s, -1)
    out = w @ v
    ds = (q.abs() @ k.abs().t()).amax(-1) * abs(scale) * 128 * 2.0 ** -23
    n = k.shape[0]
    tol = U * out.abs() + (U * (1 + U) + 2 * ds[:, None] + n * 2.0 ** -23 + 2.0 ** -20) * (w @ v.abs())
    lse = torch.logsumexp(s, -1) / math.log(2)
    return out, tol, lse, (ds + n * 2.0 ** -23 + 2.0 ** -20) / math.log(2) + lse.abs() * 2.0 ** -23


def tree(q, keys, values, dk, dv, mask, lengths, scale=128 ** -0.5):
    bs, T, Hq, _ = q.shape
    H = keys.shape[1]
    G = Hq // H
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol, lse, ltol = torch.zeros_like(out), torch.zeros(bs, T, Hq, dtype=torch.float64, device=q.device), torch.zeros(bs, T, Hq, dtype=torch.float64, device=q.device)
    for b in range(bs):
        n = min(max(int(lengths[b]), 0), keys.shape[2])
        for t in range(T):
            see = mask[b if mask.shape[0] > 1 else 0, t].bool()
            for h in range(H):
                k, v = torch.cat((keys[b, h, :n], dk[b, see, h])), torch.cat((values[b, h, :n], dv[b, see, h]))
                g = slice(h * G, h * G + G)
                out[b, t, g], tol[b, t, g], lse[b, t, g], ltol[b, t, g] = attend(q[b, t, g], k, v, scale)
    return out, tol, lse, ltol


def bounds(keys, lengths, block, old, n_new=None):
    out = old.clone()
    for b in range(keys.shape[0]):
        n = min(max(int(lengths[b]), 0), keys.shape[2])
        first = 0 if n_new is None else max(0, n - n_new) // block
        if n_new == 0:
            continue
        for j in range(first, (n + block - 1) // block):
            rows = keys[b, :, j * block:min(n, (j + 1) * block)]
            out[b, :, j, 0], out[b, :, j, 1] = rows.amin(1), rows.amax(1)
    return out


def select(q, bnd, lengths, n_select, block, sink, local):
    bs, T, Hq, _ = q.shape
    H, nb = bnd.shape[1:3]
    G = Hq // H
    ids = torch.full((bs, T, H, n_select), -1, dtype=torch.int32)
    for b in range(bs):
        for t in range(T):
            pos = min(int(lengths[b]), nb * block) - T + t
            seen = pos // block + 1 if pos >= 0 else 0
            if seen == 0:
                continue
            for h in range(H):
                qs = q[b, t, h * G:h * G + G].double()
                lo, hi = bnd[b, h, :seen, 0].double(), bnd[b, h, :seen, 1].double()
                score = torch.maximum(qs[:, None] * lo, qs[:, None] * hi).sum((0, 2)).float()
                order = sorted(range(seen), key=lambda j: (not (j < sink or j >= seen - local), -score[j].item(), j))[:n_select]
                ids[b, t, h, :len(order)] = torch.tensor(sorted(order), dtype=torch.int32)
    return ids


def block_attention(q, keys, values, ids, lengths, block, scale=128 ** -0.5):
    bs, T, Hq, _ = q.shape
    H = keys.shape[1]
    G = Hq // H
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol, lse, ltol = torch.zeros_like(out), torch.zeros(bs, T, Hq, dtype=torch.float64, device=q.device), torch.zeros(bs, T, Hq, dtype=torch.float64, device=q.device)
    for b in range(bs):
        for t in range(T):
            end = min(int(lengths[b]), keys.shape[2]) - T + t + 1
            for h in range(H):
                rows = [r for j in ids[b, t, h].tolist() if j >= 0 for r in range(j * block, min(end, (j + 1) * block))]
                rows = torch.tensor(rows, dtype=torch.long, device=q.device)
                g = slice(h * G, h * G + G)
                out[b, t, g], tol[b, t, g], lse[b, t, g], ltol[b, t, g] = attend(q[b, t, g], keys[b, h, rows], values[b, h, rows], scale)
    return out, tol, lse, ltol


def pack_w4(codes):
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).contiguous()


def gemv_w4(codes, scales, x, offsets=None, gated=False):
    """codes u8 [O,I] unpacked -> (y, tolerance) in 64 bits.  The sums run over at most 32768 products in fp32 and in groups: an
    addition is off by at most a step (2^-23) of the sum of absolute values, of which a path from a product to the result has less than 1024."""
    O, I = codes.shape
    group = I // scales.shape[1]
    s = scales.double().repeat_interleave(group, 1)
    c = codes.double()
    w = c * s + offsets.double().repeat_interleave(group, 1) if offsets is not None else (c - 8) * s
    parts = c.abs() * s.abs() + offsets.double().abs().repeat_interleave(group, 1) if offsets is not None else (c - 8).abs() * s.abs()
    y = x.double() @ w.t()
    d = 1024 * 2.0 ** -23 * (x.double().abs() @ parts.t())
    if not gated:
        return y, U * y.abs() + d * (1 + U)
    g, u = y.chunk(2, 1)
    dg, du = d.chunk(2, 1)
    act = g * torch.sigmoid(g)
    # silu's slope is below 1.1; exp and the division of fp32 are good to 2^-20
    z = act * u
    return z, U * z.abs() + (1 + U) * (1.1 * dg * u.abs() + act.abs() * du + 1.1 * dg * du + 2.0 ** -20 * z.abs())


def close(got, want, tol, what=""):
    got = got.double()
    bad = ~((got - want).abs() <= tol + 1e-30) & ~((got == want) | (got.isnan() & want.isnan()))
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {((got - want).abs() / (tol + 1e-30))[bad].max().item():.2f} tolerances, first at {bad.nonzero()[0].tolist()}"
