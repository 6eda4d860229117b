"""More arguments that the operators for several tokens a step refuse, on host tensors: no CUDA call is made for them."""
import pytest

from test_many_arguments import ATTEND, BOUNDS, SELECT, TREE, refused, z


@pytest.mark.parametrize("cap", [32, 49, 0, -2])
def test_a_capacity_that_is_not_that_of_the_bounds(cap):
    args = list(SELECT.values())
    refused("pk_select_blocks_ex", args[:4] + [cap] + args[4:], "cap must be")


@pytest.mark.parametrize("scale", [0.0, -0.1, float("nan"), float("inf"), 3.0e38, 2.4e38])
@pytest.mark.parametrize("name,args", [("pk_tree_attention", TREE), ("pk_block_attention", ATTEND)])
def test_a_scale_that_is_no_factor(name, args, scale):
    refused(name, list({**args, "scale": scale}.values()), "scale must be")


@pytest.mark.parametrize("out", [z(2, 1, 3, 2, 128).expand(2, 2, 3, 2, 128), z(1, 2, 3, 2, 128).expand(2, 2, 3, 2, 128), z(2, 2, 1, 2, 128).expand(2, 2, 3, 2, 128)])
def test_bounds_that_share_memory(out):
    refused("pk_block_bounds", list({**BOUNDS, "out": out}.values()), "must not share memory")
