"""Long products of several tokens with 4-bit weights, where an SM has many stages: rows and columns that fill neither boxes nor units, x in one
piece and in several.  The tolerance is derived in test_gpu_gemv_w4_range.py."""
import pytest

from test_gpu_gemv_w4_range import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("O,I,group,offsets,gated", [(151936, 768, 128, False, False), (38017, 4096, 64, True, False), (76001, 1568, 32, True, False),
                                                     (75808, 2176, 128, True, True), (75790, 2208, 32, False, True), (19003, 8192, 64, False, False), (19003, 12416, 128, True, False)])
@pytest.mark.parametrize("T", [2, 3, 8, 9, 16])
def test_against_the_definition(T, O, I, group, offsets, gated):
    check(*make(T + O, T, O, I, group, offsets), gated)


def test_a_vocabulary_of_drafted_tokens():
    check(*make(5, 3, 151936, 4096, 128, False), False)
