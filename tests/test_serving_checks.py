"""Refusals of the serving operators that are decided on the host (no GPU needed), beside
those of test_serving_abi.py."""

import pytest

M = 1 << 20  # plausible, aligned addresses that are never read, M apart


def plan(qg, block=64, requests=2, lens=M, news=2 * M, table=3 * M, width=4, free=4 * M, count=5 * M, tokens=5,
         lens_out=6 * M, starts=7 * M, slots=8 * M, positions=9 * M, runs=10 * M, counts=11 * M):
    return qg.lib().qgemm_kv_plan(block, requests, lens, news, table, width, free, count, tokens, lens_out, starts, slots,
                                  positions, runs, counts, None)


@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_plan_refuses_table_rows_past_31_bits(qg, block):
    """A granted request's length and positions are 32-bit numbers."""
    assert plan(qg, block=block, width=2 ** 31 // block) == qg.ERR_UNSUPPORTED_SHAPE
    assert plan(qg, block=block, width=2 ** 31 - 1) == qg.ERR_UNSUPPORTED_SHAPE
