"""The operators of a step in 8 bits in 64 bits, from their definitions, one sequence and head at a time."""
import torch

OUTLIERS = (7, 37, 71, 101)


def kv_rows(g, *shape, dev="cuda"):
    """Rows of K and V [..., 2, 128]: keys with large values in a few channels, norms that vary."""
    x = torch.randn(*shape, 2, 128, generator=g)
    x[..., 0, list(OUTLIERS)] *= 8
    x[..., 0, :] *= torch.exp(0.5 * torch.randn(*shape, 1, generator=g))
    return x.to(torch.bfloat16).to(dev)


def to_e4m3(v):
    """The nearest number with four bits of significand, ties to the even one, steps of 2^-9 below 2^-6."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def code_block(x, e4m3):
    """x f64 [block,128] -> codes (as numbers), scale."""
    most = 448 if e4m3 else 127
    top = x.abs().max()
    if not torch.isfinite(top):
        return torch.zeros_like(x), torch.tensor(float("nan"), dtype=torch.float64)
    if top == 0:
        return torch.zeros_like(x), top
    q = x * most / top
    return (to_e4m3(q) if e4m3 else torch.round(q)), top / most


class RefCache:
    """What a cache holds: all rows that were appended, coded from scratch."""

    def __init__(self, rows, block, e4m3):   # rows: list of bf16 [H,n,2,128] per sequence
        self.rows, self.block, self.e4m3 = rows, block, e4m3

    def whole(self, b):
        n = self.rows[b].shape[1]
        return n // self.block * self.block

    def coded(self, b, h, kv):
        """(codes [whole,128], scales [blocks]) in 64 bits."""
        x = self.rows[b][h, :, kv].double()
        parts = [code_block(x[j:j + self.block], self.e4m3) for j in range(0, self.whole(b), self.block)]
        if not parts:
            return x[:0], x.new_zeros(0)
        return torch.cat([c for c, _ in parts]), torch.stack([s.to(x.device) for _, s in parts])

    def values(self, b, h, kv):
        c, s = self.coded(b, h, kv)
        return torch.cat((c * s.repeat_interleave(self.block)[:, None], self.rows[b][h, self.whole(b):, kv].double()))


def attend(q, k, v, scale):
    """q f64 [128], k / v f64 [n,128] that it sees -> out, lse (base 2), mean of |v| under the weights, largest weight over the sum."""
    if k.shape[0] == 0:
        z = torch.zeros(128, dtype=torch.float64, device=q.device)
        return z, torch.tensor(float("-inf")), z, torch.zeros(1, dtype=torch.float64, device=q.device)
    s = (k @ q) * scale
    p = torch.softmax(s, 0)
    return p @ v, torch.logsumexp(s, 0) / torch.log(torch.tensor(2.0, dtype=torch.float64)), p @ v.abs(), p


def attention(ref, queries, scale):
    """queries bf16 [bs,T,Hq,128], the last T tokens -> out, lse, bound of the error that the kernel's roundings allow.

    The output's own rounding: 2^-8 of it.  A weight times the value's scale is rounded to fp16, 2^-11 of it, or, where it is far below the largest, by 2^-25 of a number from 2^-4 of the largest:
    2^-21 of the largest p_j amax_j for each row.  Scores are sums of 128 products in 32 bits, and the exponents' argument is rounded a few times: 140 * 2^-24 * sum |q k| scale moves every
    weight and the sum of weights by that share: the bound takes the largest over the rows, for numerator and denominator."""
    bs, T, Hq, _ = queries.shape
    H = ref.rows[0].shape[0]
    G = Hq // H
    out = torch.zeros(queries.shape, dtype=torch.float64, device=queries.device)
    lse = torch.full((bs, T, Hq), float("-inf"), dtype=torch.float64, device=queries.device)
    tol = torch.zeros_like(out)
    for b in range(bs):
        n = ref.rows[b].shape[1]
        for h in range(H):
            k, v = ref.values(b, h, 0), ref.values(b, h, 1)
            for t in range(T):
                last = n - T + t + 1
                if last <= 0:
                    continue
                for gq in range(h * G, (h + 1) * G):
                    q = queries[b, t, gq].double()
                    o, z, mean, p = attend(q, k[:last], v[:last], scale)
                    out[b, t, gq], lse[b, t, gq] = o, z
                    move = 140 * 2.0 ** -24 * float((k[:last].abs() @ q.abs()).max()) * scale
                    top = float((p * v[:last].abs().amax(-1)).max())   # (amax of the row's block is within a factor that the next line covers by all rows' largest)
                    top = max(top, float(p.max() * v[:last].abs().max()))
                    tol[b, t, gq] = 2.0 ** -8 * o.abs() + (2.0 ** -11 + 2 * move) * mean + last * 2.0 ** -21 * top
    return out, lse, tol
