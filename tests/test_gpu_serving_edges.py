"""The serving operators at the edges of what their entry points promise: lengths
and counts near 2^31, block ids outside the pool, calls on other streams."""
import pytest
import torch
from test_gpu_kv_cache import check_plan, make_step

pytestmark = pytest.mark.gpu

TOP = 2 ** 31 - 1


@pytest.mark.parametrize("block", [16, 128])
def test_plan_refuses_lengths_that_pass_31_bits(qg, cuda, block):
    """A refused request's rows get no slot, whatever its length, and their runs are
    counted where length and rows together pass 2^31."""
    table = [[0] * 4 for _ in range(4)]
    for have in (TOP, TOP - 7, TOP - 8, TOP - 200, 2 ** 30):
        check_plan(qg, [5, have, 3, have], [2, 300, 1, 40], table, [7, 8, 9], block, 343)
        check_plan(qg, [have], [1], [[0]], [7], block, 1)
    lens, new, table, free = make_step(21, 1500, 40, 3, block)
    lens[3], lens[1100], lens[1499] = TOP, TOP - 1, TOP - 5
    check_plan(qg, lens, new, table, free, block, sum(new))
