"""Block selection where scores have few digits or none in 32 bits."""
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


@pytest.mark.parametrize("q_exp,k_exp", [(-70, -75), (-60, -66), (-78, -76), (-20, -120), (-130, -130)])
@pytest.mark.parametrize("nb,T", [(300, 1), (3000, 3)])
def test_scores_below_normal_numbers(nb, T, q_exp, k_exp):
    """Products of which 32 bits hold a few bits or none, while their sums in 64 bits, rounded to 32, differ."""
    from pariskv_b200 import ops
    r = rnd(nb - q_exp)
    bnd = (r(1, 1, nb, 2, 128).sort(3).values.float() * 2.0 ** k_exp).to(torch.bfloat16)
    q = (r(1, T, 4, 128).float() * 2.0 ** q_exp).to(torch.bfloat16)
    got = ops.select_blocks(q, bnd, i32([nb * 16]), 40, block=16)
    assert torch.equal(got.cpu(), R.select(q.cpu(), bnd.cpu(), [nb * 16], 40, 16, 1, 1))


def test_queries_of_zeros_take_the_lowest_blocks():
    from pariskv_b200 import ops
    bnd = rnd(3)(1, 2, 5000, 2, 128).sort(3).values
    q = torch.zeros(1, 2, 8, 128, dtype=torch.bfloat16, device=DEV)
    got = ops.select_blocks(q, bnd, i32([80000]), 6, block=16, sink_blocks=0)
    assert (got.cpu() == torch.tensor([0, 1, 2, 3, 4, 4999], dtype=torch.int32)).all()


@pytest.mark.parametrize("cap,block,T", [(65, 64, 4), (130, 64, 5), (1000, 16, 3), (128, 64, 2), (20001, 128, 7)])
def test_lengths_above_the_capacity(cap, block, T):
    """Selection puts the tokens where the attention does: at the last rows of the cache."""
    from pariskv_b200 import ops
    r = rnd(cap)
    keys, values, q = r(2, 2, cap, 128), r(2, 2, cap, 128), r(2, T, 4, 128)
    over, at_most = i32([cap + 100, cap]), i32([cap, cap])
    bnd = ops.block_bounds(keys, over, block=block)
    for n in (1, 2, 5):
        ids = ops.select_blocks(q, bnd, over, n, block=block, sink_blocks=0, cap=cap)
        assert torch.equal(ids.cpu(), R.select(q.cpu(), bnd.cpu(), [cap, cap], n, block, 0, 1))
        assert torch.equal(ids, ops.select_blocks(q, bnd, at_most, n, block=block, sink_blocks=0))
        out = ops.block_attention(q, keys, values, ids, over, block=block)
        want, tol, _, _ = R.block_attention(q, keys, values, ids, [cap, cap], block)
        R.close(out, want, tol)
        assert (out != 0).any(-1).all()   # (every token sees its own block)


def test_a_capacity_that_is_not_that_of_the_bounds():
    from pariskv_b200 import ops
    r = rnd(4)
    bnd, q, lengths = r(1, 1, 3, 2, 128), r(1, 1, 2, 128), i32([40])
    for cap in (32, 49, 0, -1, -5):
        with pytest.raises((RuntimeError, ValueError)):
            ops.select_blocks(q, bnd, lengths, 2, block=16, cap=cap)
