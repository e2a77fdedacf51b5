"""Refusals of the serving operators that are decided on the host (no GPU needed), beside
those of test_serving_abi.py."""

import ctypes as C

import pytest
import torch
from test_serving_abi import Norm, cache

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


INPUTS = {"lens": 8, "news": 8, "table": 32, "count": 4}  # bytes that 2 requests, 4 table columns and 5 rows take
OUTPUTS = {"lens_out": 8, "starts": 12, "slots": 40, "positions": 20, "runs": 20, "counts": 16}


@pytest.mark.parametrize("out", list(OUTPUTS))
def test_plan_refuses_outputs_on_inputs_and_on_each_other(qg, out):
    """Blocks of the launch read the inputs while others write the outputs, so no output
    may share a byte with an input (counts[0] is the next call's free_count: not in the
    same call) nor with another output."""
    at = {"lens": M, "news": 2 * M, "table": 3 * M, "count": 5 * M, "lens_out": 6 * M, "starts": 7 * M, "slots": 8 * M,
          "positions": 9 * M, "runs": 10 * M, "counts": 11 * M}
    for other, size in {**INPUTS, **OUTPUTS}.items():
        if other == out:
            continue
        for shift in (0, size - 4, 4 - OUTPUTS[out]):  # equal, and one word shared at either end
            assert plan(qg, **{out: at[other] + shift}) == qg.ERR_INVALID_ARG, (other, shift)
            assert b"overlap" in qg.lib().qgemm_last_error_message(), (other, shift)
    assert plan(qg, **{out: 4 * M}) == qg.ERR_INVALID_ARG  # the free list, whose first entry may be read


def test_plan_bounded_refuses_a_negative_length(qg):
    args = [64, 2, M, 2 * M, 3 * M, 4, 4 * M, -1, 5 * M, 5, 6 * M, 7 * M, 8 * M, 9 * M, 10 * M, 11 * M, None]
    assert qg.lib().qgemm_kv_plan_bounded(*args) == qg.ERR_INVALID_ARG
    args[7], args[10] = 8, 4 * M + 28  # lens_out on the list's last entry
    assert qg.lib().qgemm_kv_plan_bounded(*args) == qg.ERR_INVALID_ARG
    assert b"overlap" in qg.lib().qgemm_last_error_message()


@pytest.mark.parametrize("off", [1, 4, 8, 15])
def test_attention_refuses_a_workspace_off_16_bytes(qg, off):
    """Tickets and vectors of four floats lie in it."""
    st = qg.lib().qgemm_kv_attention(C.byref(cache()), M, 8192, 128, 64, 2, 2 * M, 3 * M, 4 * M, 4, 3, 2, 0.1, 0, 1, 5 * M,
                                     None, 6 * M + off, 1 << 30, None)
    assert st == qg.ERR_WORKSPACE and b"16-byte" in qg.lib().qgemm_last_error_message()


def test_calls_refuse_a_host_cache(qg):
    """A KVCache of host tensors is a description; no call takes it."""
    k, s = torch.zeros((2, 1, 16, 64), dtype=torch.uint8), torch.zeros((2, 1), dtype=torch.uint8)
    c = qg.KVCache(qg.KV_E4M3, k, k.clone(), s, s.clone())
    x = torch.zeros((1, 1, 64), dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="the cache must be on a GPU"):
        qg.kv_append(c, x, x, torch.zeros(1, dtype=torch.int64), i)
    with pytest.raises(ValueError, match="the cache must be on a GPU"):
        qg.kv_attention(c, x, i, i[:1], i[None], 1)
    with pytest.raises(ValueError, match="the cache must be on a GPU"):
        qg.kv_attention(c, x, i, i[:1], i[None], 1, workspace=torch.zeros(4096, dtype=torch.uint8))


def test_a_caches_tensors_cannot_be_exchanged(qg):
    """The calls go by the pointers that the KVCache was made with, and its tensors keep
    that memory alive."""
    k, s = torch.zeros((2, 1, 16, 64), dtype=torch.uint8), torch.zeros((2, 1), dtype=torch.uint8)
    c = qg.KVCache(qg.KV_E4M3, k, k.clone(), s, s.clone())
    for name, value in (("k", k.clone()), ("v", k), ("k_scales", s), ("v_scales", s), ("type", qg.KV_INT8)):
        with pytest.raises(AttributeError):
            setattr(c, name, value)
        with pytest.raises(AttributeError):
            delattr(c, name)
    assert c.k is k and c.k_scales is s and c.type == qg.KV_E4M3
    c.k[0] = 5  # their contents can be changed
    assert c.values()[0].shape == (2, 1, 16, 64)


def test_norm_refuses_outputs_on_each_other_and_across_inputs(qg):
    """Only an element's own place may be written over: by residual_out for residual, by h
    for y, or for another input of the same layout and type."""
    def call(tokens=4, width=64, f32=0, y=M, residual=2 * M, post=3 * M, post_bias=None, gate=None, stride=0, pre=4 * M,
             pre_bias=None, out=5 * M, h=6 * M, kind=0):
        a = Norm(kind, tokens, width, f32, y, residual, post, post_bias, gate, stride, pre, pre_bias, 1.0, 1e-6, out, h)
        return qg.lib().qgemm_residual_norm(C.byref(a), None)

    row, whole = 64 * 2, 4 * 64 * 2
    for kw in (dict(h=5 * M), dict(h=5 * M + row), dict(h=5 * M - row), dict(f32=1, h=5 * M + 2 * whole - 16),  # on one another
               dict(h=M + row), dict(h=M - row), dict(out=2 * M + 16), dict(f32=1, out=2 * M - 16),         # shifted
               dict(f32=1, h=2 * M), dict(f32=1, out=M), dict(y=None, post=None, f32=1, h=2 * M),          # another type
               dict(out=3 * M), dict(h=4 * M + 112), dict(h=3 * M - whole + 16),                           # weights
               dict(tokens=1, out=4 * M), dict(tokens=1, h=3 * M), dict(kind=1, post_bias=7 * M, out=7 * M), dict(kind=1, pre_bias=7 * M, h=7 * M),
               dict(gate=7 * M, h=7 * M), dict(gate=7 * M, stride=72, out=7 * M), dict(gate=7 * M, stride=64, h=7 * M + row)):
        assert call(**kw) == qg.ERR_INVALID_ARG, kw
        assert b"overlap" in qg.lib().qgemm_last_error_message(), kw
