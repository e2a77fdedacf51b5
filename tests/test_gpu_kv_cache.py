"""kv_plan and kv_append against plain restatements (tests/serving_ref.py).
Both are exact: whole numbers, and codes that round once from exact products,
so every comparison is for equality."""
import random

import pytest
import serving_ref as R
import torch

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def make_step(seed, requests, len_max, new_max, block, width=None, spare=None, new_min=0):
    """A random scheduler step: lists (lens, new, table, free)."""
    rng = random.Random(seed)
    lens = [rng.choice([0, rng.randint(0, len_max)]) for _ in range(requests)]
    new = [rng.choice([1, rng.randint(new_min, new_max)]) for _ in range(requests)]
    width = width or max(1, -(-(len_max + new_max) // block))
    held = [min(width, -(-x // block)) for x in lens]
    need = sum(-(-(x + n) // block) for x, n in zip(lens, new))
    ids = list(range(sum(held) + (need if spare is None else spare)))
    rng.shuffle(ids)
    table, at = [], 0
    for h in held:
        table.append(ids[at:at + h] + [0] * (width - h))
        at += h
    return lens, new, table, ids[at:]


def check_plan(qg, lens, new, table, free, block, tokens, count=None):
    count = len(free) if count is None else count
    want = R.plan(lens, new, table, free, count, block, tokens)
    tab = torch.tensor(table, dtype=torch.int32, device="cuda").reshape(len(lens), -1)
    p = qg.kv_plan(i32(lens), i32(new), tab, i32(free), i32([count]), block, tokens)
    got = (tab.tolist(), p.lens.tolist(), p.starts.tolist(), p.slots.tolist(), p.positions.tolist(), p.runs.tolist(),
           p.counts.tolist())
    for name, a, b in zip(("table", "lens", "starts", "slots", "positions", "runs", "counts"), got, want):
        assert a == b, name
    return p


@pytest.mark.parametrize("seed,requests,len_max,new_max,block", [
    (1, 1, 0, 1, 16), (2, 1, 500, 1, 64), (3, 7, 33, 40, 16), (4, 64, 8191, 1, 64), (5, 255, 100, 9, 32),
    (6, 1023, 60, 3, 16), (7, 1024, 300, 1, 128), (8, 1025, 40, 5, 16), (9, 2500, 20, 2, 32), (10, 3, 10, 5000, 64),
])
def test_plan(qg, cuda, seed, requests, len_max, new_max, block):
    lens, new, table, free = make_step(seed, requests, len_max, new_max, block)
    check_plan(qg, lens, new, table, free, block, sum(new))


def test_plan_spare_rows_and_no_requests(qg, cuda):
    lens, new, table, free = make_step(11, 5, 40, 6, 16)
    check_plan(qg, lens, new, table, free, 16, sum(new) + 300)
    check_plan(qg, [3, 16, 0], [0, 0, 0], [[0], [1], [2]], [5], 16, 0)
    p = qg.kv_plan(i32([]), i32([]), torch.zeros((0, 4), dtype=torch.int32, device="cuda"), i32([1]), i32([1]), 16, 3)
    assert p.slots.tolist() == [-1] * 3 and p.counts.tolist() == [1, 0, 0, 0] and p.starts.tolist() == [0]


@pytest.mark.parametrize("spare", [0, 1, 5, 17])
def test_plan_refuses_when_blocks_run_out(qg, cuda, spare):
    lens, new, table, free = make_step(12, 40, 70, 50, 16, spare=spare)
    p = check_plan(qg, lens, new, table, free, 16, sum(new))
    assert p.counts[3] > 0
    check_plan(qg, lens, new, table, free + [9, 9, 9], 16, sum(new), count=spare)  # the list may be longer


def test_plan_refuses_past_table_rows_and_negative(qg, cuda):
    lens, new, table, free = make_step(13, 30, 64, 40, 16, width=4, spare=200)
    check_plan(qg, lens, new, table, free, 16, sum(new))
    lens, new, table, free = make_step(14, 20, 30, 20, 16)
    for rows in (sum(new) - 1, sum(new) // 2, 1):
        check_plan(qg, lens, new, table, free, 16, rows)
    lens[3], new[5], new[6] = -1, -4, 0
    check_plan(qg, lens, new, table, free, 16, sum(max(n, 0) for n in new))


def test_plan_outputs_can_be_kept(qg, cuda):
    lens, new, table, free = make_step(15, 9, 90, 12, 32)
    tab = torch.tensor(table, dtype=torch.int32, device="cuda")
    args = (i32(lens), i32(new), tab, i32(free), i32([len(free)]), 32, sum(new))
    a = qg.kv_plan(*args)
    b = qg.kv_plan(*args, out=qg.kv_plan(*args))
    for f in ("starts", "lens", "slots", "positions", "runs", "counts"):
        assert torch.equal(getattr(a, f), getattr(b, f)), f


# ---- append -----------------------------------------------------------------------

def random_cache(qg, kv, blocks, block, heads, d, seed):
    g = torch.Generator().manual_seed(seed)
    c = qg.make_kv_cache(kv, blocks, block, heads, d)
    for t in (c.k, c.v):
        t.copy_(torch.randint(0, 256, t.shape, generator=g, dtype=torch.uint8))
        if kv == qg.KV_E4M3:
            t[(t & 0x7F) == 0x7F] = 0x11  # no NaN codes: appends never write them
        else:
            t[t == 0x80] = 0x81  # nor INT8's -128
    for t in (c.k_scales, c.v_scales):
        t.copy_(torch.randint(115, 130, t.shape, generator=g, dtype=torch.uint8))
    return c


def check_append(qg, cache, k, v, slots, runs):
    want = [t.cpu().clone() for t in (cache.k, cache.k_scales, cache.v, cache.v_scales)]
    R.append(want[0], want[1], k.cpu(), slots.cpu(), cache.type)
    R.append(want[2], want[3], v.cpu(), slots.cpu(), cache.type)
    qg.kv_append(cache, k, v, slots, runs)
    for name, a, b in zip(("k_scales", "v_scales"), (cache.k_scales, cache.v_scales), (want[1], want[3])):
        assert torch.equal(a.cpu(), b), name
    for name, a, b in zip(("k", "v"), (cache.k, cache.v), (want[0], want[2])):
        # -0 and 0 of E4M3 are the same value
        assert torch.equal(R.decode(a.cpu(), cache.type), R.decode(b, cache.type)), name


@pytest.mark.parametrize("kv", [0, 1])
@pytest.mark.parametrize("requests,len_max,new_max,block,heads,d", [
    (1, 0, 1, 16, 1, 64), (5, 40, 1, 16, 8, 128), (3, 100, 70, 64, 2, 128), (9, 30, 33, 32, 3, 64),
    (2, 300, 260, 128, 1, 128), (4, 20, 100, 16, 5, 64),
])
def test_append(qg, cuda, kv, requests, len_max, new_max, block, heads, d):
    lens, new, table, free = make_step(requests * 7 + d, requests, len_max, new_max, block, new_min=1)
    tab = torch.tensor(table, dtype=torch.int32, device="cuda")
    tokens = sum(new)
    p = qg.kv_plan(i32(lens), i32(new), tab, i32(free), i32([len(free)]), block, tokens)
    cache = random_cache(qg, kv, max(max(r) for r in tab.tolist()) + 1, block, heads, d, requests)
    g = torch.Generator().manual_seed(d + requests)
    # rows of a wider product, spread over many binades per row
    wide = torch.randn((tokens, 3, heads, d), generator=g) * torch.exp2(torch.randint(-12, 9, (tokens, 1, 1, 1), generator=g))
    wide = wide.to(torch.bfloat16).cuda()
    check_append(qg, cache, wide[:, 1], wide[:, 2], p.slots, p.runs)


@pytest.mark.parametrize("kv", [0, 1])
@pytest.mark.parametrize("d", [64, 128])
def test_append_token_by_token_matches_the_rule(qg, cuda, kv, d):
    """A block filled one token a call: its scale grows and its codes follow."""
    block, heads = 16, 2
    cache = random_cache(qg, kv, 3, block, heads, d, 5)
    g = torch.Generator().manual_seed(d)
    for i in range(20):
        x = (torch.randn((1, 2, heads, d), generator=g) * 2.0 ** (i // 3 - 4)).to(torch.bfloat16).cuda()
        slot = torch.tensor([(2 if i < block else 0) * block + i % block], dtype=torch.int64, device="cuda")
        check_append(qg, cache, x[:, 0], x[:, 1], slot, i32([0, 1]))


@pytest.mark.parametrize("kv", [0, 1])
def test_append_special_values(qg, cuda, kv):
    """Infinities saturate without setting the scale, NaN becomes 0, zero and
    tiny blocks take the lowest scale, the largest bf16 the highest."""
    heads, d, block = 1, 64, 16
    inf, nan, big, tiny = float("inf"), float("nan"), 3.3895e38, 1e-30
    rows = torch.zeros((10, heads, d))
    rows[0, 0, :4] = torch.tensor([inf, -inf, nan, 1.0])
    rows[1, 0, :3] = torch.tensor([nan, nan, nan])
    rows[2, 0, :3] = torch.tensor([big, -big, 1.0])
    rows[3, 0, :3] = torch.tensor([tiny, -tiny, 2 * tiny])
    rows[4, 0, :3] = torch.tensor([448.0, 449.0, 127.0])
    rows[5, 0, :3] = torch.tensor([127.0, 127.5, -128.0])
    rows[6, 0, :3] = torch.tensor([0.0, -0.0, 2.0 ** -64])
    rows[7, 0, :3] = torch.tensor([inf, inf, inf])
    rows[8, 0, :3] = torch.tensor([448.0, 1.75 * 2 ** -6, 2.0 ** -10])
    rows[9, 0, :3] = torch.tensor([126.5, 0.5, 1.5])
    x = rows.to(torch.bfloat16).cuda()
    cache = random_cache(qg, kv, 10, block, heads, d, 6)
    slots = torch.arange(10, dtype=torch.int64, device="cuda") * block  # a block each
    check_append(qg, cache, x, -x, slots, i32(list(range(11))))
    assert not cache.values()[0].isnan().any() or kv == 1


def test_append_skips_bad_slots_and_reads_strided_rows(qg, cuda):
    heads, d, block = 2, 128, 32
    for kv in (0, 1):
        cache = random_cache(qg, kv, 4, block, heads, d, 7)
        x = torch.randn((6, 5, heads, d), generator=torch.Generator().manual_seed(8)).to(torch.bfloat16).cuda()
        slots = torch.tensor([-1, 5, 6, 4 * block, 2 ** 40, 3 * block], dtype=torch.int64, device="cuda")
        check_append(qg, cache, x[:, 4], x[:, 0], slots, i32([0, 1, 3, 4, 5, 6, 6, 6]))
        k = x[:, :, 0].transpose(0, 1)[:3]  # rows closer together than a token's five parts
        check_append(qg, cache, k[:, :2], k[:, 2:4], torch.arange(3, device="cuda"), i32([0, 3]))


def test_cache_refusals(qg, cuda):
    with pytest.raises(ValueError, match="block must be"):
        c = qg.make_kv_cache(qg.KV_E4M3, 2, 24, 1, 64)
        x = torch.zeros((1, 1, 64), dtype=torch.bfloat16, device="cuda")
        qg.kv_append(c, x, x, torch.zeros(1, dtype=torch.int64, device="cuda"), i32([0, 1]))
    c = qg.make_kv_cache(qg.KV_E4M3, 2, 16, 2, 64)
    x = torch.zeros((3, 2, 65), dtype=torch.bfloat16, device="cuda")
    s, r = torch.zeros(3, dtype=torch.int64, device="cuda"), i32([0, 3])
    ok = x[:, :, :64].contiguous()
    for k, v in ((x, x), (x[:, :, :64], ok), (ok, ok[:2]), (ok.float(), ok), (ok[:, :1], ok)):
        with pytest.raises(ValueError):
            qg.kv_append(c, k, v, s, r)
    with pytest.raises(ValueError):
        qg.kv_append(c, ok, ok, s.int(), r)
    flat = torch.zeros(3 * 2 * 64 + 4, dtype=torch.bfloat16, device="cuda")[4:].view(3, 2, 64)
    with pytest.raises(ValueError, match="16-byte"):
        qg.kv_append(c, flat, ok, s, r)
    t = torch.zeros((3, 2), dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="lens_out"):
        p = qg.kv_plan(i32([0, 0, 0]), i32([1, 1, 1]), t, i32([1, 2, 3]), i32([3]), 16, 3)
        qg.kv_plan(p.lens, i32([1, 1, 1]), t, i32([1, 2, 3]), i32([3]), 16, 3, out=p)
    with pytest.raises(ValueError):
        qg.kv_plan(i32([0, 0]), i32([1, 1, 1]), t, i32([1]), i32([1]), 16, 3)
    with pytest.raises(ValueError):
        qg.kv_plan(i32([0, 0, 0]), i32([1, 1, 1]), t, i32([1]), i32([1]), 20, 3)
