"""The serving operators at the edges of what their entry points promise: lengths
and counts near 2^31, block ids outside the pool, calls on other streams."""
import pytest
import serving_ref as R
import torch
from test_gpu_kv_attention import check, make
from test_gpu_kv_cache import check_plan, i32, make_step

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


@pytest.mark.parametrize("new", [
    [2 ** 30, 2 ** 30, 1], [TOP, TOP, 2, 1], [3, TOP, TOP, TOP, TOP, 1], [2 ** 30 - 1, 1, 1], [2, 2 ** 30, 2 ** 30 - 1, 4],
    [1] * 40 + [2 ** 30] * 6 + [1] * 40, [1] * 600 + [TOP] * 900 + [1],
])
def test_plan_refuses_counts_that_pass_30_bits(qg, cuda, new):
    """Row and block counts whose sums pass 2^30 and 2^31: starts stop at 2^30 and no
    request behind them is granted rows."""
    block, tokens = 16, 700
    lens = [(5 * i) % 16 for i in range(len(new))]
    table = [[3] * 2 for _ in new]
    free = list(range(10, 700))
    want = R.plan(lens, new, table, free, len(free), block, tokens)
    tab = torch.tensor(table, dtype=torch.int32, device="cuda")
    p = qg.kv_plan(i32(lens), i32(new), tab, i32(free), i32([len(free)]), block, tokens)
    assert tab.tolist() == want[0] and p.lens.tolist() == want[1]
    assert p.starts.tolist() == [min(s, 2 ** 30) for s in want[2]]
    assert p.slots.tolist() == want[3] and p.positions.tolist() == want[4]
    assert p.runs.tolist() == want[5] and p.counts.tolist() == want[6]


def test_plan_refuses_its_own_outputs_as_inputs(qg, cuda):
    lens, new, table, free = make_step(31, 9, 90, 12, 32)
    tab = torch.tensor(table, dtype=torch.int32, device="cuda")
    tokens = sum(new)

    def call(a, b, count, out):
        return qg.kv_plan(a, b, tab, i32(free), count, 32, tokens, out=out)

    p = call(i32(lens), i32(new), i32([len(free)]), None)
    for args in ((p.lens, i32(new), i32([3])), (i32(lens), p.lens, i32([3])), (i32(lens), i32(new), p.counts[:1]),
                 (i32(lens), i32(new), p.counts[3:]), (i32(lens), p.starts[1:], i32([3]))):
        with pytest.raises(ValueError, match="overlap"):
            call(*args, p)
    other = call(i32(lens), i32(new), i32([len(free)]), None)
    call(p.lens, i32(new), p.counts[:1], other)  # another plan's are inputs like any


@pytest.mark.parametrize("listed", [0, 1, 5, 60])
def test_plan_takes_no_block_past_the_free_list(qg, cuda, listed):
    """A free_count above the list's length counts as that length."""
    lens, new, table, free = make_step(41, 40, 70, 50, 16, spare=listed)
    want = R.plan(lens, new, table, free, listed, 16, sum(new))
    for count in (listed + 1, listed + 1000, TOP):
        tab = torch.tensor(table, dtype=torch.int32, device="cuda")
        p = qg.kv_plan(i32(lens), i32(new), tab, i32(free), i32([count]), 16, sum(new))
        assert tab.tolist() == want[0] and p.slots.tolist() == want[3] and p.counts.tolist() == want[6]


# ---- attention ----------------------------------------------------------------------

def within(out, lse, want, wlse, mass, logit, floor, d, most):
    """The bounds of test_gpu_kv_attention.py."""
    tol = want.abs() * 2.0 ** -8 + mass * (2.0 ** -11 + 2.0 ** -20 + (2 * d * logit[..., None] + most) * 2.0 ** -23) + \
        floor * 2.0 ** -35
    assert ((out.double() - want).abs() <= tol).all()
    if lse is not None:
        assert ((lse.double() - wlse).abs() <= (d * logit + most + 64) * 2.0 ** -23 + wlse.abs() * 2.0 ** -22).all()


def check_outside(qg, kv, lens, new, block, heads, group, d, seed, ids, fill=127):
    """kv_attention with some table entries outside the pool against a cache in which they
    name a block of zeros, with the bounds of test_gpu_kv_attention.py.  `fill`: the scale
    bytes of the pool's first block, which no request then uses."""
    c, q, starts, n, table = make(qg, kv, lens, [new] * len(lens), block, heads, group, d, seed)
    blocks = c.k.shape[0]
    c.k_scales[0] = c.v_scales[0] = fill
    table = torch.where(table == 0, 1, table)
    shadow = [torch.cat([x, torch.full_like(x[:1], y)]) for x, y in ((c.k, 0), (c.v, 0), (c.k_scales, 127), (c.v_scales, 127))]
    mapped, place = table.clone(), 0
    for r, length in enumerate(lens):
        for p in range(-(-length // block)):
            if (p + r) % 3 == 0:
                table[r, p] = ids[place % len(ids)] if ids[place % len(ids)] != "blocks" else blocks
                mapped[r, p] = blocks
                place += 1
    assert place >= len(ids)
    ws = qg.make_kv_workspace(c, q.shape[1], len(lens), q.shape[0], new)
    out, lse = qg.kv_attention(c, q, starts, n, table, new, lse=True, workspace=ws)
    within(out, lse, *R.attention(kv, *shadow, q, starts, n, mapped, d ** -0.5), d, max(lens))


OUTSIDE = [-1, -5, "blocks", TOP, -2 ** 31, -2 ** 30 - 1, -2 ** 30, -715827883, 2 ** 30]
WIDTHS = [(128, 1), (128, 2), (128, 150), (64, 1), (64, 2), (64, 150)]  # head_dim, rows a request brings


@pytest.mark.parametrize("kv", [0, 1])
@pytest.mark.parametrize("heads", [2, 3])
@pytest.mark.parametrize("d,new", WIDTHS)
def test_block_ids_far_outside_the_pool_read_as_zeros(qg, cuda, kv, heads, d, new):
    """Ids whose product with the heads wraps 32 bits to a place far behind the pool."""
    check_outside(qg, kv, [600, 170, 333], new, 16, heads, 4, d, 101, OUTSIDE)


@pytest.mark.parametrize("kv", [0, 1])
@pytest.mark.parametrize("fill", [0, 1, 60, 200, 254, 255])
@pytest.mark.parametrize("d,new", WIDTHS)
def test_block_ids_outside_the_pool_take_no_blocks_scale(qg, cuda, kv, fill, d, new):
    """Zeros whatever the scale bytes of the pool's first block are."""
    check_outside(qg, kv, [600, 170, 333], new, 32, 2, 4, d, 102, [-1, "blocks", -5, TOP], fill)


@pytest.mark.parametrize("new", [1, 100])
def test_a_workspace_belongs_to_the_calls_stream(qg, cuda, new):
    """What a call on another stream takes for itself is that stream's memory: the
    current stream does not get it when the call has returned."""
    c, q, starts, lens, table = make(qg, 0, [300, 1100, 64 + new], [new] * 3, 64, 2, 8, 128, 111)
    want = qg.kv_attention(c, q, starts, lens, table, new)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    ws = qg.make_kv_workspace(c, q.shape[1], 3, q.shape[0], new, stream=s)
    at, size = ws.data_ptr(), ws.numel()
    del ws
    again = torch.empty(size, dtype=torch.uint8, device="cuda")
    assert again.data_ptr() != at
    with torch.cuda.stream(s):
        assert torch.empty(size, dtype=torch.uint8, device="cuda").data_ptr() == at
    for _ in range(20):
        out = qg.kv_attention(c, q, starts, lens, table, new, stream=s)
        taken = [torch.full((size,), 255, dtype=torch.uint8, device="cuda") for _ in range(3)]
        s.synchronize()
        assert torch.equal(out, want)
        del taken


@pytest.mark.parametrize("lens,new,block,heads,group,d,seed,window,causal", [
    ([3, 3, 3, 4, 3, 3, 3, 4], [3] * 8, 32, 4, 16, 64, 795860, 0, False),
    ([3, 276, 26, 178], [162, 276, 26, 178], 128, 8, 4, 64, 183772, 0, False),
    ([408, 29, 399, 3], [408, 73, 399, 263], 16, 4, 12, 128, 303701, 274, True),
    ([2305, 373, 1611, 4, 836, 1224, 1684, 1454, 2083], [2, 4, 5, 4, 5, 2, 8, 7, 0], 128, 3, 16, 64, 736382, 297, True),
    ([2, 9, 40], [1, 1, 1], 16, 8, 8, 128, 5, 0, True),
])
def test_small_weights_beside_a_codes_zero(qg, cuda, lens, new, block, heads, group, d, seed, window, causal):
    """INT8 values that only small weights reach, the largest weight's code being 0: the
    step of an f16 weight is 2^-35 of the largest in both kernels."""
    check(qg, *make(qg, 1, lens, new, block, heads, group, d, seed, scales=(100, 130)), max(new), window=window,
          causal=causal)


@pytest.mark.parametrize("kv", [0, 1])
@pytest.mark.parametrize("d", [64, 128])
def test_rows_past_max_new_are_left_alone(qg, cuda, kv, d):
    """max_new bounds the rows that are computed, from each request's first on; those that
    are computed are at their own positions."""
    c, q, starts, lens, table = make(qg, kv, [300, 200, 7], [140, 3, 9], 32, 2, 4, d, 131)
    want, wlse, mass, logit, floor = R.attention(kv, c.k, c.v, c.k_scales, c.v_scales, q, starts, lens, table, d ** -0.5)
    first = torch.cat([torch.arange(n) for n in (140, 3, 9)]).to("cuda")
    empty = torch.isinf(wlse)
    for most in (1, 4, 12, 20, 139):
        out = torch.full_like(q, 5.0, memory_format=torch.contiguous_format)
        _, lse = qg.kv_attention(c, q, starts, lens, table, most, out=out, lse=True)
        some = first < most
        assert (out[~some] == 5.0).all()
        assert torch.equal(torch.isinf(lse[some]), empty[some]) and (out[some][empty[some]] == 0).all()
        see = some[:, None] & ~empty
        within(out[see], lse[see], want[see], wlse[see], mass[see], logit[see], floor[see], d, 300)


@pytest.mark.parametrize("kv", [0, 1])
@pytest.mark.parametrize("d", [64, 128])
def test_a_mixed_call_on_another_stream_and_in_a_graph(qg, cuda, kv, d):
    """Decoding requests beside prompt chunks, whose two kernels and join overlap, behind and
    in front of other calls: the same bits every time, within the bounds."""
    new = [1, 130, 1, 20, 300, 1, 2]
    c, q, starts, lens, table = make(qg, kv, [700, 500, 90, 64, 300, 1, 1500], new, 64, 2, 4, d, 141)
    tokens = sum(new)
    ws = qg.make_kv_workspace(c, 8, 7, tokens, 300)
    w = torch.ones(8 * d, dtype=torch.bfloat16, device="cuda")

    def call(out, stream=None):
        qg.kv_attention(c, q, starts, lens, table, 300, out=out, workspace=ws, stream=stream)
        return qg.residual_norm(None, out.flatten(1), pre=w, stream=stream)[1]

    want = torch.zeros((tokens, 8, d), dtype=torch.bfloat16, device="cuda")
    h = call(want)
    within(want, None, *R.attention(kv, c.k, c.v, c.k_scales, c.v_scales, q, starts, lens, table, d ** -0.5), d, 1500)
    out = torch.zeros_like(want)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for _ in range(5):
        got = [call(out, s) for _ in range(3)]
        s.synchronize()
        assert torch.equal(out, want) and all(torch.equal(x, h) for x in got)
        out.zero_()
        torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(3):
            got = call(out)
    for _ in range(5):
        out.zero_()
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(got, h)


# ---- where tensors lie ---------------------------------------------------------------

def each_on_the_host(args, kw):
    """The call's arguments with one tensor at a time on the host."""
    for i, t in enumerate(args):
        if isinstance(t, torch.Tensor):
            yield [*args[:i], t.cpu(), *args[i + 1:]], kw
    for n, t in kw.items():
        if isinstance(t, torch.Tensor):
            yield args, {**kw, n: t.cpu()}


def test_every_tensor_must_be_on_the_calls_gpu(qg, cuda):
    c, q, starts, lens, table = make(qg, 0, [40, 20], [1, 1], 16, 2, 4, 64, 121)
    ws = qg.make_kv_workspace(c, 8, 2, 2, 1)
    k = torch.zeros((2, 2, 64), dtype=torch.bfloat16, device="cuda")
    slots, runs = torch.tensor([0, 16], device="cuda"), i32([0, 1, 2])
    y, w = torch.zeros((2, 64), dtype=torch.bfloat16, device="cuda"), torch.ones(64, dtype=torch.bfloat16, device="cuda")
    calls = [
        (qg.kv_plan, [lens, i32([1, 1]), table, i32([7, 8]), i32([2]), 16, 2], {}),
        (qg.kv_append, [c, k, k.clone(), slots, runs], {}),
        (qg.kv_attention, [c, q, starts, lens, table, 1], {"out": torch.empty_like(q, memory_format=torch.contiguous_format),
                                                           "workspace": ws}),
        (qg.residual_norm, [y, y.clone()], {"post": w, "pre": w, "post_bias": w, "pre_bias": w, "gate": w, "kind": "layer",
                                            "residual_out": y.clone(), "h": y.clone()}),
    ]
    for f, args, kw in calls:
        f(*args, **kw)
        n = 0
        for a, b in each_on_the_host(args, kw):
            with pytest.raises(ValueError, match="GPU"):
                f(*a, **b)
            n += 1
        assert n >= 4
    plan = qg.kv_plan(*calls[0][1])
    plan.positions = plan.positions.cpu()
    with pytest.raises(ValueError, match="GPU"):
        qg.kv_plan(*calls[0][1], out=plan)
    host = qg.KVCache(qg.KV_E4M3, *(t.cpu() for t in (c.k, c.v, c.k_scales, c.v_scales)))
    with pytest.raises(ValueError, match="the cache must be on a GPU"):
        qg.kv_append(host, k, k, slots, runs)
    with pytest.raises(ValueError, match="the cache must be on a GPU"):
        qg.kv_attention(host, q, starts, lens, table, 1, workspace=ws)


# ---- calls behind one another ----------------------------------------------------------

@pytest.mark.parametrize("tokens,width", [(1, 8192), (700, 2880), (64, 16384)])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_norms_read_what_the_call_before_wrote(qg, cuda, tokens, width, kind):
    """A call is set up while the one before still runs; whatever it reads (stream, block,
    gate, weights) is what that call left."""
    g = torch.Generator(device="cuda").manual_seed(width)
    y, r = (torch.randn((tokens, width), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    w = (torch.randn(width, generator=g, device="cuda") * 0.1 + 1).to(torch.bfloat16)

    def chain(wait):
        a, h = qg.residual_norm(y, r, post=w, pre=w, kind=kind)
        for _ in range(6):
            wait()
            b, h2 = qg.residual_norm(h, a, post=w, pre=w, gate=h, alpha=0.5, kind=kind)      # block and gate
            wait()
            a, h = qg.residual_norm(h2, b, post=h2[-1], pre=b[0], gate=h2[0], kind=kind)     # weights
        return a, h

    want = chain(torch.cuda.synchronize)
    for _ in range(10):
        got = chain(lambda: None)
        for x, z in zip(got, want):
            assert torch.equal(x.view(torch.int16), z.view(torch.int16))


@pytest.mark.parametrize("tokens", [1, 37])
def test_norm_over_its_own_inputs(qg, cuda, tokens):
    """An output may be any input of its layout: the stream, the block or the gate."""
    g = torch.Generator(device="cuda").manual_seed(tokens)
    y, r, gate = (torch.randn((tokens, 520), generator=g, device="cuda").to(torch.bfloat16) for _ in range(3))
    w = (torch.randn(520, generator=g, device="cuda") * 0.1 + 1).to(torch.bfloat16)
    want, h = qg.residual_norm(y, r, post=w, pre=w, gate=gate)
    for a, b in ((1, 0), (0, 1), (2, 0), (1, 2), (0, 2)):
        x = [y.clone(), r.clone(), gate.clone()]
        got, got_h = qg.residual_norm(x[0], x[1], post=w, pre=w, gate=x[2], residual_out=x[a], h=x[b])
        assert torch.equal(got, want) and torch.equal(got_h, h)
        x = [y.clone(), r.clone(), gate.clone()]
        with pytest.raises(ValueError, match="overlap"):
            qg.residual_norm(x[0], x[1], post=w, pre=w, gate=x[2], residual_out=x[a], h=x[a])


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("news", [[1] * 9, [6] * 9, [150] * 9, [1, 150, 1, 1, 300, 1, 70, 1, 2], [1] * 300 + [90] * 4],
                         ids=["steps", "few", "prompts", "mixed", "many"])
def test_attention_reads_what_append_just_wrote(qg, cuda, news, d):
    """Steps without a wait between their calls give what the same calls give one by one;
    in a mixed step the two kernels of attention start beside one another."""
    block, heads, group, requests, tokens, new = 16, 2, 4, len(news), sum(news), max(news)
    g = torch.Generator(device="cuda").manual_seed(new)
    steps = 4
    x = torch.randn((steps, tokens, (group + 2) * heads, d), generator=g, device="cuda").to(torch.bfloat16)
    width = -(-steps * new // block)
    blocks = sum(-(-steps * n // block) for n in news) + 2

    def run(wait):
        c = qg.make_kv_cache(qg.KV_E4M3, blocks, block, heads, d)
        lens, table = i32([0] * requests), torch.zeros((requests, width), dtype=torch.int32, device="cuda")
        free, count = torch.arange(blocks, dtype=torch.int32, device="cuda"), i32([blocks])
        ws = qg.make_kv_workspace(c, heads * group, requests, tokens, new)
        outs = []
        for s in range(steps):
            q, k, v = x[s].split([group * heads, heads, heads], 1)
            p = qg.kv_plan(lens, i32(news), table, free, count, block, tokens)
            wait()
            qg.kv_append(c, k, v, p.slots, p.runs)
            wait()
            outs.append(qg.kv_attention(c, q, p.starts, p.lens, table, new, workspace=ws))
            wait()
            lens, count = p.lens, p.counts[:1]
        return outs

    want = run(torch.cuda.synchronize)
    for _ in range(5):
        for a, b in zip(run(lambda: None), want):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16))
