"""kv_attention against a 64-bit restatement (tests/serving_ref.py).

Bounds, per output value with mass A = sum p |v| and per row with
S = max over tokens of scale * sum |q k|:
  * the score is a 32-bit sum of head_dim products: off by at most
    head_dim 2^-24 S, which moves every weight by that, twice (numerator and
    denominator);
  * a weight is rounded to f16: by 2^-11 of it, or by 2^-25, half f16's smallest
    step, where the largest weight of the row's share is at least 2^10; its
    exponential is off by less
    than 2^-21; sums of L weights in 32 bits by L 2^-24 at most;
  * the result is rounded to bf16 (8 significant bits): 2^-8 of it.
So |out - exact| <= 2^-8 |exact| + A (2^-11 + 2^-20 + (2 head_dim S + L) 2^-23)
+ 2^-35 F, where F = (largest p 2^ev) sum |v code|, and the lse by (head_dim S + L + 64) 2^-23 + 2^-22 |lse|.
"""
import math

import pytest
import serving_ref as R
import torch

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def make(qg, kv, lens, new, block, heads, group, d, seed, extra=3, q_mul=1.0, scales=(118, 123), nan_fill=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    held = [-(-x // block) for x in lens]
    blocks = sum(held) + extra
    c = qg.make_kv_cache(kv, blocks, block, heads, d)
    for t in (c.k, c.v):
        x = torch.randn(t.shape, generator=g, device="cuda")
        t.copy_((x * 90).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8) if kv == qg.KV_E4M3 else
                (x * 30).clamp(-127, 127).round().to(torch.int8).view(torch.uint8))
    for t in (c.k_scales, c.v_scales):
        t.copy_(torch.randint(scales[0], scales[1], t.shape, generator=g, device="cuda"))
    ids = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    width = max(held + [1]) + 1
    table = torch.full((len(lens), width), 2 ** 30, dtype=torch.int32, device="cuda")  # unused entries name nothing
    at = 0
    for r, (n, length) in enumerate(zip(held, lens)):
        table[r, :n] = ids[at:at + n]
        if nan_fill and n and length % block:  # what lies behind the last token must not matter
            last = int(ids[at + n - 1])
            c.k[last, :, length % block:] = 0x7F
            c.v[last, :, length % block:] = 0x7F if kv == qg.KV_E4M3 else 0x80
        at += n
    tokens = sum(new)
    wide = (torch.randn((tokens, heads * group + 2, d), generator=g, device="cuda") * q_mul).to(torch.bfloat16)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    return c, wide[:, 1:1 + heads * group], i32(starts), i32(lens), table


def check(qg, c, q, starts, lens, table, max_new, scale=None, window=0, causal=True, rows=None):
    d = q.shape[2]
    ws = qg.make_kv_workspace(c, q.shape[1], lens.numel(), q.shape[0], max_new)
    out, lse = qg.kv_attention(c, q, starts, lens, table, max_new, scale=scale, window=window, causal=causal, lse=True,
                               workspace=ws)
    again = qg.kv_attention(c, q, starts, lens, table, max_new, scale=scale, window=window, causal=causal,
                            workspace=ws)
    assert torch.equal(out.view(torch.int16), again.view(torch.int16)), "same call, other bits"
    want, wlse, mass, logit, floor = R.attention(c.type, c.k, c.v, c.k_scales, c.v_scales, q, starts, lens, table,
                                          d ** -0.5 if scale is None else scale, window, causal)
    n = int(lens.max())
    err = (out.double() - want).abs()
    tol = want.abs() * 2.0 ** -8 + mass * (2.0 ** -11 + 2.0 ** -20 + (2 * d * logit[..., None] + n) * 2.0 ** -23) + \
        floor * 2.0 ** -35
    assert (err <= tol).all(), f"off by {float((err / tol.clamp(min=1e-300)).max()):.3g} of the bound"
    empty = torch.isinf(wlse)
    assert torch.equal(torch.isinf(lse), empty)
    assert (out[empty] == 0).all()
    lerr = (lse.double() - wlse).abs()[~empty]
    ltol = ((d * logit + n + 64) * 2.0 ** -23 + wlse.abs() * 2.0 ** -22)[~empty]
    assert (lerr <= ltol).all(), f"lse off by {float((lerr / ltol).max()):.3g} of the bound"


@pytest.mark.parametrize("kv", [0, 1])
@pytest.mark.parametrize("lens,block,heads,group,d", [
    ([1], 16, 1, 1, 64), ([1], 64, 2, 8, 128), ([15, 16, 17], 16, 2, 4, 128), ([0, 1, 0, 33], 32, 1, 8, 64),
    ([2000], 64, 8, 8, 128), ([5000], 128, 1, 7, 128), ([700, 1, 64, 1300, 0, 129], 64, 3, 5, 64),
    ([333] * 40, 16, 4, 2, 64), ([100 + 7 * i for i in range(30)], 32, 8, 8, 128), ([900, 31], 16, 2, 16, 128),
    ([257], 64, 1, 71, 64), ([4096], 16, 1, 1, 64),
])
def test_decode(qg, cuda, kv, lens, block, heads, group, d):
    args = make(qg, kv, lens, [1] * len(lens), block, heads, group, d, 3 * d + len(lens))
    check(qg, *args, 1)


@pytest.mark.parametrize("kv", [0, 1])
@pytest.mark.parametrize("lens,new,block,heads,group,d,window", [
    ([40, 3, 500], [4, 3, 2], 16, 2, 4, 128, 0), ([40, 3, 500], [4, 3, 2], 16, 2, 4, 128, 20),
    ([300, 77], [1, 1], 64, 2, 8, 128, 1), ([300, 77, 5], [1, 1, 1], 32, 2, 8, 64, 64),
    ([200, 0, 90], [130, 0, 90], 64, 2, 4, 64, 0), ([200, 300, 90], [130, 1, 90], 64, 2, 4, 128, 50),
    ([517], [517], 32, 1, 8, 128, 0), ([517], [300], 16, 1, 3, 64, 100), ([2100, 64], [257, 64], 128, 2, 8, 128, 0),
    ([50, 2], [60, 5], 16, 1, 2, 128, 0),  # more rows than tokens: the first see nothing
    ([700, 800], [129, 128], 64, 1, 1, 128, 0), ([1000, 20, 999], [200, 1, 3], 32, 4, 7, 64, 0),
])
def test_several_rows(qg, cuda, kv, lens, new, block, heads, group, d, window):
    args = make(qg, kv, lens, new, block, heads, group, d, 5 * d + len(lens))
    check(qg, *args, max(new), window=window)
    if not window:
        check(qg, *args, max(new), causal=False)


@pytest.mark.parametrize("kv", [0, 1])
@pytest.mark.parametrize("new", [1, 5, 160])
def test_wide_scales_and_peaked_rows(qg, cuda, kv, new):
    """Block scales 40 binades apart, and logits whose softmax is one token."""
    args = make(qg, kv, [600, 170], [new, new], 16, 2, 4, 128, 21, scales=(95, 135))
    check(qg, *args, new, scale=2.0 ** -14)
    args = make(qg, kv, [600, 170], [new, new], 16, 2, 4, 128, 22, q_mul=20.0)
    check(qg, *args, new)
    check(qg, *args, new, scale=-0.05)
    args = make(qg, kv, [600, 170], [new, new], 16, 2, 4, 64, 23, q_mul=2.0 ** -100)
    check(qg, *args, new)
    args = make(qg, kv, [600, 170], [new, new], 16, 2, 4, 64, 24, q_mul=2.0 ** 60)
    check(qg, *args, new, scale=2.0 ** -63)


@pytest.mark.parametrize("new", [1, 40, 200])
def test_nan_query_rows_stay_their_own(qg, cuda, new):
    c, q, starts, lens, table = make(qg, 0, [500, 300], [new, new], 32, 2, 4, 128, 31)
    ref = qg.kv_attention(c, q, starts, lens, table, new)
    bad = q.clone()
    bad[0, 1, 3] = float("nan")
    bad[new, 5, 0] = float("inf")
    out = qg.kv_attention(c, bad, starts, lens, table, new)
    assert out[0, 1].isnan().all() and out[new, 5].isnan().any()
    keep = torch.ones(q.shape[:2], dtype=torch.bool, device="cuda")
    keep[0, 1] = keep[new, 5] = False
    assert torch.equal(out[keep].view(torch.int16), ref[keep].view(torch.int16))


def test_many_requests(qg, cuda):
    """More requests than one launch's prefix sums hold."""
    lens = [(37 * i) % 50 for i in range(4500)]
    args = make(qg, 1, lens, [1] * 4500, 16, 1, 2, 64, 41)
    check(qg, *args, 1)


def test_offsets_past_32_bits(qg, cuda):
    """Blocks near the end of a pool of more than 4 GiB of codes."""
    block, heads, d = 128, 8, 128
    blocks = 2 ** 32 // (block * heads * d) + 40
    c = qg.make_kv_cache(qg.KV_E4M3, blocks, block, heads, d)
    g = torch.Generator(device="cuda").manual_seed(51)
    ids = torch.tensor([blocks - 1, 3, blocks - 7, 2 ** 31 // (block * heads * d) + 1], device="cuda")
    table = ids.to(torch.int32)[None].contiguous()
    length = 4 * block
    x = torch.randn((length, 2, heads, d), generator=g, device="cuda").to(torch.bfloat16)
    slots = (ids[:, None] * block + torch.arange(block, device="cuda")).flatten()
    qg.kv_append(c, x[:, 0], x[:, 1], slots, i32([0, block, 2 * block, 3 * block, 4 * block]))
    for new in (1, 150):
        q = torch.randn((new, heads * 4, d), generator=g, device="cuda").to(torch.bfloat16)
        check(qg, c, q, i32([0, new]), i32([length]), table, new)


def test_other_stream_and_graph(qg, cuda):
    c, q, starts, lens, table = make(qg, 0, [300, 1100, 64], [1, 1, 1], 64, 2, 8, 128, 61)
    want = qg.kv_attention(c, q, starts, lens, table, 1)
    ws = qg.make_kv_workspace(c, q.shape[1], 3, 3, 1)
    out = torch.empty_like(want)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    qg.kv_attention(c, q, starts, lens, table, 1, out=out, workspace=ws, stream=s)
    s.synchronize()
    assert torch.equal(out, want)
    out.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qg.kv_attention(c, q, starts, lens, table, 1, out=out, workspace=ws)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_table_entries_outside_the_pool_read_as_zeros(qg, cuda):
    c, q, starts, lens, table = make(qg, 0, [64, 48], [1, 1], 16, 2, 4, 128, 71)
    table[0, 1], table[1, 0] = -5, c.k.shape[0]
    out = qg.kv_attention(c, q, starts, lens, table, 1)
    assert torch.isfinite(out.float()).all()


def test_attention_refusals(qg, cuda):
    c, q, starts, lens, table = make(qg, 0, [40, 20], [1, 1], 16, 2, 4, 64, 81)
    ws = qg.make_kv_workspace(c, 8, 2, 2, 1)
    with pytest.raises(qg.QGemmError, match="workspace"):
        qg.kv_attention(c, q, starts, lens, table, 1, workspace=ws[:-1])
    for args in ((q.float(), starts, lens, table), (q[:, :7], starts, lens, table), (q, starts[:2], lens, table),
                 (q, starts.long(), lens, table), (q, starts, lens, table[:1]), (q[:, :, :32], starts, lens, table)):
        with pytest.raises(ValueError):
            qg.kv_attention(c, *args, 1, workspace=ws)
    for kw in ({"scale": math.inf}, {"scale": math.nan}, {"window": -1}):
        with pytest.raises(ValueError):
            qg.kv_attention(c, q, starts, lens, table, 1, workspace=ws, **kw)
    assert qg.kv_attention(c, q[:0], i32([0, 0, 0]), lens, table, 1, workspace=ws).shape == (0, 8, 64)
