"""More arguments that the operators for several tokens a step refuse, on host tensors: no CUDA call is made for them."""
import pytest

from test_many_arguments import SELECT, refused


@pytest.mark.parametrize("cap", [32, 49, 0, -2])
def test_a_capacity_that_is_not_that_of_the_bounds(cap):
    args = list(SELECT.values())
    refused("pk_select_blocks_ex", args[:4] + [cap] + args[4:], "cap must be")
