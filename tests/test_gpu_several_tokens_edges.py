"""Attention for several tokens over caches that hold infinities."""
import math

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


def _infinite_channels(out, want, tol, channels):
    rest = [i for i in range(128) if i not in channels]
    for c, sign in channels.items():
        assert (want[..., c] == sign * math.inf).all()
        assert (out[..., c] == sign * math.inf).all(), c
    R.close(out[..., rest], want[..., rest], tol[..., rest])


@pytest.mark.parametrize("T,G", [(1, 1), (1, 4), (2, 4), (3, 5), (8, 4), (9, 8), (61, 4)])
@pytest.mark.parametrize("n", [40, 3000])
def test_an_infinite_value_in_the_cache_comes_out(T, G, n):
    """Every token sees the row: the channel is infinite, the others are as without it.  Whole items and items that are cut."""
    from pariskv_b200 import ops
    r = rnd(T + n)
    keys, values, q, dk, dv = r(1, 2, n, 128), r(1, 2, n, 128), r(1, T, 2 * G, 128), r(1, T, 2, 128), r(1, T, 2, 128)
    values[:, :, 17, 5], values[:, :, n - 1, 9] = float("inf"), float("-inf")
    mask = torch.eye(T, dtype=torch.bool, device=DEV)[None]
    out = ops.tree_attention(q, keys, values, dk, dv, mask, i32([n]))
    want, tol, _, _ = R.tree(q, keys, values, dk, dv, mask, [n])
    _infinite_channels(out, want, tol, {5: 1, 9: -1})


@pytest.mark.parametrize("G,n", [(1, 3), (4, 3), (8, 90), (16, 3), (20, 90)])
def test_an_infinite_value_in_a_listed_block_comes_out(G, n):
    from pariskv_b200 import ops
    r = rnd(G + n)
    keys, values, q = r(1, 2, 6000, 128), r(1, 2, 6000, 128), r(1, 2, 2 * G, 128)
    values[:, :, 17, 5], values[:, :, 40, 9] = float("inf"), float("-inf")
    ids = torch.arange(n, dtype=torch.int32, device=DEV).expand(1, 2, 2, n).contiguous()
    out = ops.block_attention(q, keys, values, ids, i32([6000]), block=16)
    want, tol, _, _ = R.block_attention(q, keys, values, ids, [6000], 16)
    _infinite_channels(out, want, tol, {5: 1, 9: -1})


def test_results_over_two_sets_of_rows_are_joined_by_lse():
    """A cache in two parts, the drafts with the second; one part is empty for one sample."""
    from pariskv_b200 import dist, ops
    r = rnd(1)
    bs, T, H, G, n = 2, 5, 2, 4, 700
    keys, values, q, dk, dv = r(bs, H, n, 128), r(bs, H, n, 128), r(bs, T, H * G, 128), r(bs, T, H, 128), r(bs, T, H, 128)
    mask = torch.ones(1, T, T, dtype=torch.bool, device=DEV).tril()
    cut = [300, 0]
    first, second = i32(cut), i32([n - 300, n])
    tail_k, tail_v = keys.clone(), values.clone()
    tail_k[0, :, :n - 300], tail_v[0, :, :n - 300] = keys[0, :, 300:], values[0, :, 300:]
    parts = []
    for k, v, m, lengths in ((keys, values, torch.zeros_like(mask), first), (tail_k, tail_v, mask, second)):
        lse = torch.empty(bs, T, H * G, device=DEV)
        parts.append((ops.tree_attention(q, k, v, dk, dv, m, lengths, lse=lse), lse))
    packed = torch.stack([torch.cat((o.float().flatten(0, 1), lse.flatten(0, 1)[..., None]), -1) for o, lse in parts])
    out = dist.merge_gathered_partials(packed).view(bs, T, H * G, 128)
    want, tol, _, _ = R.tree(q, keys, values, dk, dv, mask, [n, n])
    # each part has been rounded to bf16 once
    R.close(out, want, 2 * tol + R.U * sum(o.double().abs() for o, _ in parts))
