"""kv_attention where its host picks another kernel, row tile or split: both sides
of every such rule, against the 64-bit restatement and with the bounds of
test_gpu_kv_attention.py."""
import pytest
import serving_ref as R
import torch
from test_gpu_kv_attention import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", [0, 1])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens,new,group", [
    ([40 + 9 * i for i in range(40)], 2, 8),    # many pairs of 16 rows, short enough to stay whole
    ([900 - 13 * i for i in range(36)], 3, 4),  # longer: cut
    ([3, 700, 0, 1, 64] * 8, 2, 5),             # uneven, two rows for one token and for none
    ([130] * 32, 6, 8),                         # 48 rows: the last that decode takes at 128 dims
    ([10] * 300, 2, 6),
])
def test_two_row_tiles(qg, cuda, kv, d, lens, new, group):
    args = make(qg, kv, lens, [new] * len(lens), 16, 4, group, d, 7 * d + len(lens))
    check(qg, *args, new)


@pytest.mark.parametrize("kv", [0, 1])
@pytest.mark.parametrize("lens", [
    [300] * 200,                                     # whole pairs, longer than the mean share needs
    [620, 600, 5] * 70, [640] * 3, [641] * 64,       # at and past the longest that stays whole
    [575 - i for i in range(200)], [16] * 500, [1] * 700,
])
def test_whole_and_cut_pairs(qg, cuda, kv, lens):
    args = make(qg, kv, lens, [1] * len(lens), 32, 2, 3, 64, len(lens))
    check(qg, *args, 1)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [8, 9, 16, 17, 32, 33, 48, 49, 128, 129, 255, 256, 257])
def test_rows_on_both_sides_of_the_kernels(qg, cuda, d, rows):
    args = make(qg, rows % 2, [rows + 60, rows], [rows, rows], 32, 1, 1, d, rows)
    check(qg, *args, rows)
    check(qg, *args, rows, window=30)


def test_many_prompts_and_many_steps(qg, cuda):
    """More requests of both kinds than one launch of either kernel takes."""
    lens = [70 + (11 * i) % 60 for i in range(1300)]
    new = [65 if i % 4 == 0 else 1 for i in range(1300)]
    args = make(qg, 0, lens, new, 32, 1, 1, 64, 91)
    check(qg, *args, 65)


@pytest.mark.parametrize("kv", [0, 1])
def test_rows_left_over(qg, cuda, kv):
    """More rows than the requests bring: those that belong to none are left alone."""
    new = [1, 130, 20]
    c, q, starts, lens, table = make(qg, kv, [400, 500, 90], new, 64, 2, 4, 128, 95)
    total = sum(new)
    for pad in (7, 3 * 130 - total):  # the second is room enough for 130 rows of each
        wide = torch.cat([q, torch.full((pad, *q.shape[1:]), float("nan"), dtype=q.dtype, device="cuda")])
        out = torch.full_like(wide, 5.0)
        qg.kv_attention(c, wide, starts, lens, table, 130, out=out)
        assert (out[total:] == 5.0).all()
        want, _, mass, logit, floor = R.attention(kv, c.k, c.v, c.k_scales, c.v_scales, q, starts, lens, table, 128 ** -0.5)
        err = (out[:total].double() - want).abs()
        tol = want.abs() * 2.0 ** -8 + floor * 2.0 ** -35 + \
            mass * (2.0 ** -11 + 2.0 ** -20 + (2 * 128 * logit[..., None] + 500) * 2.0 ** -23)
        assert (err <= tol).all()


def test_fewer_rows_than_a_request_brings(qg, cuda):
    """max_new bounds the rows that are computed; the others are left alone."""
    c, q, starts, lens, table = make(qg, 0, [300, 200], [40, 3], 32, 2, 4, 64, 97)
    for most in (4, 20):
        out = torch.full_like(q, 5.0)
        qg.kv_attention(c, q, starts, lens, table, most, out=out)
        full = qg.kv_attention(c, q, starts, lens, table, 40)
        assert (out[most:40] == 5.0).all()
        assert float((out[:most].float() - full[:most].float()).abs().max()) < 0.05 * float(full.float().abs().max())
        assert (out[40:].float() - full[40:].float()).abs().max() < 0.05 * full.float().abs().max()
