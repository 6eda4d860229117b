"""Products with 4-bit weights: values of x far above the others of their group, and long products of several tokens.

Tolerances.  Products of a code and a bf16 value are exact.  A result is a path of fp32 additions, each off by at most a step (2^-23) of the
sum of absolute values so far: of a group, two for each sixteen columns; then one per group, one for each of sixteen warps, one for each of eight columns of
digits, whose absolute values together are at most three times those that they stand for.  With g columns in a group that is less than
d = 4 (g / 8 + I / g + 24) 2^-23 sum |x| |w|, where a weight's parts count one by one if there are offsets."""
import pytest
import torch

import many_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(seed, T, O, I, group, offsets):
    g = torch.Generator(device=DEV).manual_seed(seed)
    codes = torch.randint(0, 16, (O, I), generator=g, device=DEV).to(torch.uint8)
    scales = (torch.rand(O, I // group, generator=g, device=DEV) / I ** 0.5 + 1e-3).to(torch.bfloat16)
    off = (torch.randn(O, I // group, generator=g, device=DEV) / I ** 0.5).to(torch.bfloat16) if offsets else None
    x = torch.randn(T, I, generator=g, device=DEV).to(torch.bfloat16)
    return codes, scales, x, off


def check(codes, scales, x, off, gated):
    from pariskv_b200 import ops
    got = ops.gemv_w4(R.pack_w4(codes), scales, x, offsets=off, gated=gated)
    want, bound = [], []
    O, I = codes.shape
    group = I // scales.shape[1]
    for r in range(0, O, 16384):   # (a few GB of 64-bit weights at a time)
        s, c = scales[r:r + 16384].double().repeat_interleave(group, 1), codes[r:r + 16384].double()
        if off is not None:
            m = off[r:r + 16384].double().repeat_interleave(group, 1)
            w, parts = c * s + m, c * s.abs() + m.abs()
        else:
            w = (c - 8) * s
            parts = w.abs()
        want.append(x.double() @ w.t())
        bound.append(4 * (group / 8 + I / group + 24) * 2.0 ** -23 * (x.double().abs() @ parts.t()))
    y, d = torch.cat(want, 1), torch.cat(bound, 1)
    if gated:   # silu's slope is below 1.1; exp and the division of fp32 are good to 2^-20
        (g, u), (dg, du) = y.chunk(2, 1), d.chunk(2, 1)
        act = g * torch.sigmoid(g)
        y, d = act * u, 1.1 * dg * u.abs() + act.abs() * du + 1.1 * dg * du + 2.0 ** -20 * (act * u).abs()
    assert got.shape == y.shape and got.dtype == torch.bfloat16
    R.close(got, y, R.U * y.abs() + d * (1 + R.U))


def far_above(codes, scales, x, off, group, size):
    """In every group one value of every token `size` times the others', whose weight is zero in every row; next to it an ordinary one."""
    at = torch.arange(0, x.shape[1], group, device=DEV) + torch.arange(x.shape[1] // group, device=DEV) * 7 % group
    x[:, at] = size * x[:, at].sign()
    if off is not None:
        off.zero_()
    codes[:, at] = 0 if off is not None else 8


@pytest.mark.parametrize("size", [1e4, 1e6, 1e8])
@pytest.mark.parametrize("O,I,group,offsets,gated", [(2000, 4096, 128, False, False), (514, 1120, 32, True, True), (64, 17408, 64, False, True), (1030, 2048, 64, True, False),
                                                     (38000, 4096, 128, False, False), (76000, 1568, 32, True, True)])
def test_values_far_above_the_others_with_weights_of_zero(O, I, group, offsets, gated, size):
    """What a weight of zero meets adds nothing, however large it is."""
    for T in (1, 2, 3, 13):
        codes, scales, x, off = make(T + O, T, O, I, group, offsets)
        far_above(codes, scales, x, off, group, size)
        check(codes, scales, x, off, gated)


def test_a_value_far_above_the_others_in_a_row_that_counts_it():
    """The same value under other weights: its own product decides the result, to a rounding."""
    for T in (1, 2, 5):
        for O in (700, 38000):
            codes, scales, x, _ = make(T, T, O, 4096, 128, False)
            x[:, 777] = 1e6
            check(codes, scales, x, None, False)


@pytest.mark.parametrize("small", [2.0 ** -60, 2.0 ** -100])
def test_small_values(small):
    """Whole tokens near the lower end of the type's range."""
    for T in (1, 3):
        codes, scales, x, off = make(T, T, 152000, 1024, 64, False)
        check(codes, scales, (x.float() * small).to(torch.bfloat16), off, False)


@pytest.mark.parametrize("odd", [float("inf"), float("-inf"), float("nan")])
def test_a_single_token_that_is_not_finite(odd):
    from pariskv_b200 import ops
    for O in (300, 38000):
        codes, scales, x, off = make(3, 1, O, 4096, 64, True)
        x[0, 4000] = odd
        assert not ops.gemv_w4(R.pack_w4(codes), scales, x, offsets=off).isfinite().any()
