"""Measured cases of the serving operators around the W4A16 GEMM: the block
tables and slot maps of a paged 8-bit KV cache, the quantising append to it,
attention over it, and the norms around a block with its gate and residual.

``run`` computes each operator in its plain form (elementary torch operations
in 32 bits) or, with ``own`` set, through this package's entry points.
``exact`` restates the operators' definitions in 64 bits.

Cache layout: codes [blocks, heads, block, head_dim] in 8 bits (E4M3 or INT8)
and one E8M0 scale byte per (block, head), 2^(byte - 127), for K and for V.
Head counts and widths are those of the 70B-class (64 query / 8 KV heads of
128, width 8192), 8B-class (32 / 8 of 128, width 4096) and 2880-wide (64 / 8
of 64) models the GEMM benchmark takes its shapes from.
"""
import importlib
import math

import torch

own = False

E4M3_MAX, INT8_MAX = 448.0, 127.0
LOWEST_EXP = -64  # the smallest scale the cache holds is 2^-64

_package = None


def _qg():
    global _package
    if _package is None:
        _package = importlib.import_module("qgemm-mx_b200")
    return _package


# ---- cases --------------------------------------------------------------------

def _plan(name, requests, len_min, len_max, new_min, new_max, chunks, block):
    return {"name": name, "op": "plan", "requests": requests, "len_min": len_min, "len_max": len_max,
            "new_min": new_min, "new_max": new_max, "chunks": chunks, "block": block}


def _append(name, kv, requests, len_min, len_max, new_min, new_max, chunks, block, heads, head_dim):
    return {"name": name, "op": "append", "kv": kv, "requests": requests, "len_min": len_min, "len_max": len_max,
            "new_min": new_min, "new_max": new_max, "chunks": chunks, "block": block, "heads": heads,
            "head_dim": head_dim}


def _attend(name, kv, requests, len_min, len_max, new_min, new_max, chunks, block, q_heads, heads, head_dim, window,
            lse):
    return {"name": name, "op": "attend", "kv": kv, "requests": requests, "len_min": len_min, "len_max": len_max,
            "new_min": new_min, "new_max": new_max, "chunks": chunks, "block": block, "q_heads": q_heads,
            "heads": heads, "head_dim": head_dim, "window": window, "lse": lse}


def _norm(name, tokens, width, kind, gate, residual):
    return {"name": name, "op": "norm", "tokens": tokens, "width": width, "kind": kind, "gate": gate,
            "residual": residual}


def listed():
    return [
        # a decode step of 64 requests: one token each, a new block now and then
        _plan("plan decode 64", 64, 1, 8191, 1, 1, 0, 64),
        # a scheduler step that mixes 448 decoding requests with 64 prompt chunks
        _plan("plan mixed 512", 512, 0, 4095, 1, 512, 64, 16),
        # the K and V of one decode step of 64 requests
        _append("append decode 64 e4m3", "e4m3", 64, 1, 1023, 1, 1, 0, 64, 8, 128),
        # prompts of odd lengths, some behind cached tokens, in 16-token blocks
        _append("append ragged int8", "int8", 33, 0, 300, 1, 777, 5, 16, 8, 64),
        # chunks of four long prompts
        _append("append prompts e4m3", "e4m3", 4, 0, 1000, 4096, 4096, 4, 64, 8, 128),
        # one user's next token over a long context: latency
        _attend("attend decode 1", "e4m3", 1, 8192, 8192, 1, 1, 0, 64, 64, 8, 128, 0, False),
        # a full decode batch with ragged contexts: the ordinary serving step
        _attend("attend decode 64", "e4m3", 64, 129, 8192, 1, 1, 0, 64, 64, 8, 128, 0, False),
        # many short requests, sliding window, small blocks, one of them empty
        _attend("attend window int8", "int8", 200, 0, 1500, 1, 1, 0, 16, 64, 8, 64, 128, True),
        # a chunk of a long prompt against its cached beginning
        _attend("attend chunk 2048", "e4m3", 1, 8192, 8192, 2048, 2048, 1, 64, 32, 8, 128, 0, False),
        # decoding requests and prompt chunks in one call
        _attend("attend mixed int8", "int8", 16, 600, 4096, 1, 512, 3, 32, 64, 8, 64, 0, False),
        # the norms of one decode step of one request: latency
        _norm("norm 1 x 8192", 1, 8192, "rms", "none", "bf16"),
        # a prompt's worth of tokens, per-token gate, fp32 residual stream
        _norm("norm 6000 x 2880", 6000, 2880, "layer", "token", "f32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(["plan", "append", "append", "attend", "attend", "attend", "norm"])
        block = rng.choice([16, 32, 64, 128])
        kv = rng.choice(["e4m3", "int8"])
        q_heads, heads, head_dim = rng.choice([(64, 8, 128), (32, 8, 128), (64, 8, 64), (16, 16, 64), (12, 4, 128),
                                               (28, 4, 128), (8, 1, 64)])
        if op == "plan":
            r = _log_int(rng, 1, 2000)
            hi = _log_int(rng, 16, 8192)
            chunks = rng.choice([0, 0, rng.randint(0, min(r, 64))])
            c = _plan("", r, rng.choice([0, 1, hi // 2]), hi, rng.choice([0, 1, 1]), _log_int(rng, 2, 1024), chunks,
                      block)
        elif op == "append":
            r = _log_int(rng, 1, 600)
            chunks = rng.choice([0, rng.randint(0, min(r, 8))])
            c = _append("", kv, r, 0, _log_int(rng, 1, 1500), 1, _log_int(rng, 2, 4096), chunks, block, heads,
                        head_dim)
        elif op == "attend":
            form = rng.choice(["decode", "decode", "speculate", "chunk", "mixed"])
            window = rng.choice([0, 0, 0, _log_int(rng, 16, 2048)])
            hi = _log_int(rng, 40, 16384)
            lo = rng.choice([0, hi // 3, hi])
            if form == "decode":
                r, new_min, new_max, chunks = _log_int(rng, 1, 256), 1, 1, 0
            elif form == "speculate":
                r, chunks = _log_int(rng, 1, 128), 0
                new_min = new_max = rng.randint(2, 8)
            elif form == "chunk":
                r = rng.randint(1, 4)
                new_min, new_max, chunks = 1, _log_int(rng, 16, 2048), r
            else:
                r = rng.randint(2, 24)
                new_min, new_max, chunks = 1, _log_int(rng, 16, 512), rng.randint(1, 2)
            lo, hi = max(lo, new_min), max(hi, new_max)
            c = _attend("", kv, r, lo, hi, new_min, new_max, chunks, block, q_heads, heads, head_dim, window,
                        rng.random() < 0.3)
        else:
            c = _norm("", _log_int(rng, 1, 8192), rng.choice([2880, 4096, 8192, 8 * _log_int(rng, 8, 2048)]),
                      rng.choice(["rms", "layer"]), rng.choice(["none", "shared", "token"]),
                      rng.choice(["bf16", "f32"]))
        del c["name"]
        if 3072 in c.values() or not _affordable(c):
            continue
        return c


def _affordable(c):
    """No more than the largest listed case of its kind, in the plain form's
    padded memory too."""
    if c["op"] == "plan":
        return 0 < sum(_news(c)) <= 40000
    if c["op"] == "append":
        return sum(_news(c)) * c["heads"] * c["head_dim"] <= 16384 * 8 * 128
    if c["op"] == "attend":
        w = work(c)
        padded = c["requests"] * c["q_heads"] * max(_news(c)) * c["len_max"]
        pool = sum(_lens(c)) * c["heads"] * c["head_dim"]
        return w["bytes"] <= 5.6e8 and w["flops"] <= 2.4e11 and padded <= 6e8 and pool <= 2.8e8 and \
            c["requests"] * c["len_max"] * c["heads"] * c["head_dim"] <= 5.4e8
    return c["tokens"] * c["width"] <= 6000 * 2880


# ---- sizes a case stands for ---------------------------------------------------

def _spread(n, lo, hi):
    """n whole numbers evenly spread over [lo, hi]."""
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _news(c):
    """New tokens of each request: `chunks` of them, spread evenly over the
    batch, bring new_max down to half of it, the others new_min."""
    r, k = c["requests"], c["chunks"]
    news = [c["new_min"]] * r
    big = _spread(k, max(c["new_min"], c["new_max"] // 2), c["new_max"]) if k else []
    for i, n in enumerate(big):
        news[i * r // k] = n
    return news


def _lens(c):
    """Tokens in the cache: before the new ones for plan and append, all of
    them for attend.  Spread over the range in an order of its own."""
    r = c["requests"]
    lens = _spread(r, c["len_min"], c["len_max"])
    step = next(s for s in (7, 11, 13, 17, 19, 23, 29, 31, 37) if math.gcd(s, r) == 1)
    lens = [lens[(i * step + r - 1) % r] for i in range(r)]
    if c["op"] != "attend":
        return lens
    # a request holds its new tokens at least; only an empty one holds none
    return [x if n == 1 else max(x, n) for x, n in zip(lens, _news(c))]


def _blocks_of(tokens, block):
    return -(-tokens // block)


def work(case):
    c = case
    if c["op"] == "plan":
        t = sum(_news(c))
        # lengths in and out, starts; a slot and a position for each token
        return {"bytes": 4 * c["requests"] * 4 + 12 * t, "flops": 0}
    if c["op"] == "append":
        t = sum(_news(c))
        # K and V in bf16 and their codes
        return {"bytes": 2 * t * c["heads"] * c["head_dim"] * 3, "flops": 4 * t * c["heads"] * c["head_dim"]}
    if c["op"] == "attend":
        seen = pairs = 0
        for n, x in zip(_news(c), _lens(c)):
            w = c["window"] or x
            seen += min(x, w + n - 1)
            # query i of the last n sees min(position + 1, w) tokens
            first = max(0, x - n + 1)
            a, b = min(first, w), min(x, w)
            ramp = max(0, b - a)
            pairs += (a + b - 1) * ramp // 2 + b * (min(n, x) - ramp)
        t = sum(_news(c))
        cache = 2 * seen * c["heads"] * c["head_dim"]
        return {"bytes": cache + 4 * t * c["q_heads"] * c["head_dim"], "flops": 4 * pairs * c["q_heads"] * c["head_dim"]}
    t, d = c["tokens"], c["width"]
    stream = 2 if c["residual"] == "bf16" else 4
    gate = {"none": 0, "shared": 2 * d, "token": 2 * t * d}[c["gate"]]
    return {"bytes": t * d * (2 + 2 * stream + 2) + gate + 4 * d, "flops": 12 * t * d}


# ---- inputs ---------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _shuffled(values, g):
    return _i32(values)[torch.randperm(len(values), generator=g, device="cuda")]


def _random_cache(c, blocks, g):
    """A pool filled as a model fills it: normal values whose spread differs
    from head to head, quantised per block."""
    shape = (blocks, c["heads"], c["block"], c["head_dim"])
    out = []
    for _ in range(2):
        x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float16)
        if c["kv"] == "e4m3":
            codes = (x * 96).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)
            mid = -7
        else:
            codes = (x * 30).clamp_(-INT8_MAX, INT8_MAX).round_().to(torch.int8).view(torch.uint8)
            mid = -5
        scales = torch.randint(127 + mid - 1, 127 + mid + 2, shape[:2], generator=g, device="cuda").to(torch.uint8)
        out += [codes, scales]
    return {"k": out[0], "k_scales": out[1], "v": out[2], "v_scales": out[3]}


def _prepare_plan(c, seed):
    g = _generator(seed)
    news, lens, block = _news(c), _lens(c), c["block"]
    order = torch.randperm(c["requests"], generator=g, device="cuda")
    new, old = _i32(news)[order], _i32(lens)[order]
    width = _blocks_of(c["len_max"] + max(news), block)
    held = sum(_blocks_of(x, block) for x in lens)
    added = sum(_blocks_of(x + n, block) - _blocks_of(x, block) for x, n in zip(_lens(c), news))
    spare = _blocks_of(sum(news), block) + c["requests"] + 5
    ids = torch.randperm(held + added + spare, generator=g, device="cuda").to(torch.int32)
    have = (old + block - 1) // block
    first = torch.cumsum(have, 0) - have
    col = torch.arange(width, device="cuda", dtype=torch.int32)[None]
    at = (first[:, None] + col).clamp(max=len(ids) - 1)
    table = torch.where(col < have[:, None], ids[at.long()], torch.zeros_like(ids[:1])).contiguous()
    free = ids[held:].contiguous()
    return {"op": "plan", "lens": old, "new": new, "table": table, "free_list": free, "free_count": _i32([len(free)]),
            "block": block, "tokens": sum(news)}


def prepare(case, seed):
    c = case
    if c["op"] == "plan":
        return _prepare_plan(c, seed)
    g = _generator(seed)
    if c["op"] == "append":
        s = _prepare_plan(c, seed)
        blocks = int(s["free_list"].numel() + sum(_blocks_of(x, c["block"]) for x in _lens(c)))
        plan = _plan_plain(s)
        t, h, d = s["tokens"], c["heads"], c["head_dim"]
        # K and V are columns of the QKV product's output, so their tokens lie
        # three parts of a row apart
        qkv = torch.randn((t, 3, h, d), generator=g, device="cuda", dtype=torch.float32)
        qkv *= torch.exp(torch.randn((1, 3, h, d), generator=g, device="cuda"))
        qkv = qkv.to(torch.bfloat16)
        return {"op": "append", "kv": c["kv"], **_random_cache(c, blocks, g), "new_k": qkv[:, 1], "new_v": qkv[:, 2],
                "slots": plan[3], "runs": plan[5]}
    if c["op"] == "attend":
        order = torch.randperm(c["requests"], generator=g, device="cuda")
        new, lens = _i32(_news(c))[order], _i32(_lens(c))[order]
        width = max(1, _blocks_of(max(_lens(c)), c["block"]))
        held = sum(_blocks_of(x, c["block"]) for x in _lens(c))
        blocks = held + 3
        ids = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
        have = (lens + c["block"] - 1) // c["block"]
        first = torch.cumsum(have, 0) - have
        col = torch.arange(width, device="cuda", dtype=torch.int32)[None]
        at = (first[:, None] + col).clamp(max=blocks - 1)
        table = torch.where(col < have[:, None], ids[at.long()], torch.zeros_like(ids[:1])).contiguous()
        t = sum(_news(c))
        row = (c["q_heads"] + 2 * c["heads"]) * c["head_dim"]
        qkv = torch.randn((t, row), generator=g, device="cuda", dtype=torch.float32).to(torch.bfloat16)
        q = qkv[:, :c["q_heads"] * c["head_dim"]].unflatten(1, (c["q_heads"], c["head_dim"]))
        starts = torch.cat([_i32([0]), torch.cumsum(new, 0).to(torch.int32)])
        return {"op": "attend", "kv": c["kv"], **_random_cache(c, blocks, g), "q": q, "starts": starts, "lens": lens,
                "table": table, "max_new": max(_news(c)), "window": c["window"], "lse": c["lse"], "kept": {}}
    t, d = c["tokens"], c["width"]
    stream = torch.bfloat16 if c["residual"] == "bf16" else torch.float32

    def normal(*shape, scale=1.0, mean=0.0):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale + mean

    gate = {"none": None, "shared": (d,), "token": (t, d)}[c["gate"]]
    layer = c["kind"] == "layer"
    return {"op": "norm", "kind": c["kind"], "y": normal(t, d, scale=3.0, mean=0.1).to(torch.bfloat16),
            "residual": normal(t, d, scale=8.0).to(stream),
            "post": normal(d, scale=0.2, mean=1.0).to(torch.bfloat16),
            "pre": normal(d, scale=0.2, mean=1.0).to(torch.bfloat16),
            "post_bias": normal(d, scale=0.1).to(torch.bfloat16) if layer else None,
            "pre_bias": normal(d, scale=0.1).to(torch.bfloat16) if layer else None,
            "gate": None if gate is None else normal(*gate, scale=0.5, mean=0.5).to(torch.bfloat16),
            "alpha": 0.7, "eps": 1e-6}


# ---- one pass ---------------------------------------------------------------------

def run(state):
    s = state
    if own:
        return _OWN[s["op"]](s)
    return _PLAIN[s["op"]](s)


def _cache_out(s):
    kind = torch.float8_e4m3fn if s["kv"] == "e4m3" else torch.int8
    return s["k"].view(kind), s["v"].view(kind), s["k_scales"], s["v_scales"]


def _cache_own(s):
    qg = _qg()
    return qg.KVCache(qg.KV_E4M3 if s["kv"] == "e4m3" else qg.KV_INT8, s["k"], s["v"], s["k_scales"], s["v_scales"])


def _plan_own(s):
    p = _qg().kv_plan(s["lens"], s["new"], s["table"], s["free_list"], s["free_count"], s["block"], s["tokens"])
    return s["table"], p.lens, p.starts, p.slots, p.positions, p.runs, p.counts


def _append_own(s):
    _qg().kv_append(_cache_own(s), s["new_k"], s["new_v"], s["slots"], s["runs"])
    return _cache_out(s)


def _attend_own(s):
    qg = _qg()
    cache = _cache_own(s)
    if "workspace" not in s["kept"]:  # a serving loop keeps its workspace
        s["kept"]["workspace"] = qg.make_kv_workspace(cache, s["q"].shape[1], s["lens"].numel(), s["q"].shape[0],
                                                      s["max_new"])
    return qg.kv_attention(cache, s["q"], s["starts"], s["lens"], s["table"], s["max_new"], window=s["window"],
                           lse=s["lse"], workspace=s["kept"]["workspace"])


def _norm_own(s):
    return _qg().residual_norm(s["y"], s["residual"], post=s["post"], pre=s["pre"], post_bias=s["post_bias"],
                               pre_bias=s["pre_bias"], gate=s["gate"], alpha=s["alpha"], kind=s["kind"], eps=s["eps"])


_OWN = {"plan": _plan_own, "append": _append_own, "attend": _attend_own, "norm": _norm_own}


def _plan_plain(s):
    """Blocks for the requests' new tokens off the end of the free list, in
    request order while they last, and each token's slot."""
    lens, block, tokens, table = s["lens"], s["block"], s["tokens"], s["table"]
    requests, width = table.shape
    free, count = s["free_list"], s["free_count"]
    new = s["new"].clamp(min=0)
    starts = torch.zeros(requests + 1, dtype=torch.int32, device=lens.device)
    starts[1:] = torch.cumsum(new, 0)
    have = (lens + block - 1) // block
    need = (lens + new + block - 1) // block - have
    fits = have + need <= width
    need = torch.where(fits, need, torch.zeros_like(need))
    upto = torch.cumsum(need, 0).to(torch.int32)
    granted = fits & (starts[1:] <= tokens) & ((need == 0) | (upto <= count))
    need = torch.where(granted, need, torch.zeros_like(need))
    lens_out = torch.where(granted, lens + new, lens)
    col = torch.arange(width, device=lens.device, dtype=torch.int32)[None]
    off_end = (upto - need)[:, None] + col - have[:, None]
    fresh = (col >= have[:, None]) & (col < (have + need)[:, None])
    taken = free[(count - 1 - off_end).clamp(0, free.numel() - 1).long()]
    table.copy_(torch.where(fresh, taken, table))
    t = torch.arange(tokens, device=lens.device, dtype=torch.int32)
    total = starts[requests].clamp(max=tokens)
    r = torch.searchsorted(starts[1:].contiguous(), t, right=True).clamp(max=requests - 1)
    at = lens[r] + t - starts[r]
    lead = (t < total) & ((t == starts[r]) | (at % block == 0))
    good = (t < total) & granted[r]
    slots = table[r, (at // block).clamp(0, width - 1).long()].long() * block + at % block
    slots = torch.where(good, slots, torch.full_like(slots, -1))
    positions = torch.where(good, at, torch.full_like(at, -1))
    most = min(tokens, 2 * requests + tokens // block)
    runs = total.expand(most + 2).clone()
    where = torch.where(lead, torch.cumsum(lead, 0) - 1, torch.full_like(slots, most + 1))
    runs = runs.scatter_(0, where, t)[:most + 1]
    left = count[0] - torch.where(granted, upto, torch.zeros_like(upto)).amax().clamp(min=0)
    counts = torch.stack([left, lead.sum(), total, (~granted).sum()]).to(torch.int32)
    return table, lens_out, starts, slots, positions, runs, counts


def _needed_exp(amax, kv):
    """The smallest e with amax <= (largest code) * 2^e."""
    f, e = torch.frexp(amax)
    top, shift = (0.875, 9) if kv == "e4m3" else (0.9921875, 7)
    e = torch.where(f <= top, e - shift, e - shift + 1)
    return torch.where(amax > 0, e, torch.full_like(e, LOWEST_EXP)).clamp(min=LOWEST_EXP)


def _encode(x, kv):
    """x / scale to 8-bit codes: nearest, ties to even, saturating, NaN to 0."""
    x = torch.nan_to_num(x, nan=0.0, posinf=math.inf, neginf=-math.inf)
    if kv == "e4m3":
        return x.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)
    return x.clamp(-INT8_MAX, INT8_MAX).round().to(torch.int8).view(torch.uint8)


def _pow2(e):
    """2^e for whole e, by its bits: 0 below the smallest normal number."""
    return ((e.int() + 127).clamp(min=0) << 23).view(torch.float32)


def _decode(codes, kv):
    return codes.view(torch.float8_e4m3fn if kv == "e4m3" else torch.int8).float()


def _append_one(codes, scales, x, slots, runs, kv):
    block = codes.shape[2]
    x = x.float()
    page, at = slots // block, slots % block
    lead = runs[:-1].long()
    lead = torch.where(lead < runs[-1], lead, lead[0])  # entries past the last run repeat the first
    pages, old = page[lead], at[lead]
    size = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(-1)
    amax = torch.zeros(scales.shape, device=x.device).index_reduce_(0, page, size, "amax")[pages]
    was = scales[pages].int() - 127
    exp = _needed_exp(amax, kv)
    exp = torch.where(old[:, None] > 0, torch.maximum(exp, was), exp)
    shift = torch.where(old[:, None] > 0, was - exp, torch.zeros_like(exp))
    held = _decode(codes[pages], kv)
    moved = _encode(held * _pow2(shift)[:, :, None, None], kv)
    grown = (shift < 0)[:, :, None, None] & (torch.arange(block, device=x.device)[:, None] < old[:, None, None, None])
    codes[pages] = torch.where(grown, moved, codes[pages])
    scales[pages] = (exp + 127).to(torch.uint8)
    codes[page, :, at] = _encode(x * _pow2(127 - scales[page].int())[:, :, None], kv)


def _append_plain(s):
    _append_one(s["k"], s["k_scales"], s["new_k"], s["slots"], s["runs"], s["kv"])
    _append_one(s["v"], s["v_scales"], s["new_v"], s["slots"], s["runs"], s["kv"])
    return _cache_out(s)


def _gathered(codes, scales, table, kv):
    """The values of each request's blocks, [requests, heads, tokens, head_dim]."""
    at = table.long()
    x = _decode(codes[at], kv) * _pow2(scales[at].int() - 127)[..., None, None]
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3)


def _attend_plain(s):
    q, starts, lens, table, n = s["q"], s["starts"], s["lens"], s["table"], s["max_new"]
    tokens, q_heads, d = q.shape
    heads = s["k"].shape[1]
    requests = lens.numel()
    new = starts[1:] - starts[:-1]
    i = torch.arange(n, device=q.device)
    rows = (starts[:-1, None] + i).clamp(max=tokens - 1).long()
    qp = q[rows].float().unflatten(2, (heads, q_heads // heads)).permute(0, 2, 1, 3, 4)
    k = _gathered(s["k"], s["k_scales"], table, s["kv"])
    length = k.shape[2]
    score = (qp.flatten(2, 3) @ k.transpose(2, 3)).mul_(d ** -0.5).unflatten(2, (n, q_heads // heads))
    del k
    j = torch.arange(length, device=q.device)
    at = (lens - new)[:, None] + i
    seen = (j <= at[..., None]) & (j < lens[:, None, None])
    if s["window"]:
        seen &= j > at[..., None] - s["window"]
    score.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    v = _gathered(s["v"], s["v_scales"], table, s["kv"])
    v = torch.where((j < lens[:, None])[:, None, :, None], v, torch.zeros_like(v[:1, :1, :1]))
    out = (p.flatten(2, 3) @ v).unflatten(2, (n, q_heads // heads))
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    t = torch.arange(tokens, device=q.device, dtype=torch.int32)
    r = torch.searchsorted(starts[1:].contiguous(), t, right=True).clamp(max=requests - 1)
    flat = out.permute(0, 2, 1, 3, 4).flatten(2, 3)[r, (t - starts[r]).long()]
    if not s["lse"]:
        return flat.to(torch.bfloat16)
    lse = (top + total.log()).squeeze(-1).permute(0, 2, 1, 3).flatten(2, 3)[r, (t - starts[r]).long()]
    return flat.to(torch.bfloat16), lse


def _normed(x, weight, bias, kind, eps):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight.float()
    return x if bias is None else x + bias.float()


def _norm_plain(s):
    branch = _normed(s["y"].float(), s["post"], s["post_bias"], s["kind"], s["eps"])
    if s["gate"] is not None:
        branch = branch * s["gate"].float()
    stream = s["residual"].float() + s["alpha"] * branch
    h = _normed(stream, s["pre"], s["pre_bias"], s["kind"], s["eps"])
    return stream.to(s["residual"].dtype), h.to(torch.bfloat16)


_PLAIN = {"plan": _plan_plain, "append": _append_plain, "attend": _attend_plain, "norm": _norm_plain}


# ---- the definitions in 64 bits -----------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "plan":
        return None  # whole numbers throughout
    return _EXACT[s["op"]](s)


def _exact_codes(codes, scales, x, slots, kv):
    """The pool's code values with no rounding of what the call writes."""
    block = codes.shape[2]
    peak, low = (E4M3_MAX if kv == "e4m3" else INT8_MAX), 2.0 ** LOWEST_EXP
    value = codes.view(torch.float8_e4m3fn if kv == "e4m3" else torch.int8).double()
    where = slots.tolist()
    t = 0
    while t < len(where):
        page, off = divmod(where[t], block)
        n = 1
        while t + n < len(where) and off + n < block and where[t + n] == where[t] + n:
            n += 1
        rows = x[t:t + n].double().transpose(0, 1)
        least = rows.abs().amax((1, 2)).div(peak).clamp(min=low)
        scale = torch.exp2(torch.ceil(torch.log2(least)))
        if off:
            was = torch.exp2(scales[page].double() - 127)
            scale = torch.maximum(scale, was)
            value[page, :, :off] *= (was / scale)[:, None, None]
        value[page, :, off:off + n] = rows / scale[:, None, None]
        t += n
    return value


def _exact_append(s):
    if s["kv"] == "int8":  # whole numbers
        return None
    return (_exact_codes(s["k"], s["k_scales"], s["new_k"], s["slots"], s["kv"]),
            _exact_codes(s["v"], s["v_scales"], s["new_v"], s["slots"], s["kv"]), None, None)


def _exact_attend(s):
    q, starts, lens = s["q"], s["starts"].tolist(), s["lens"].tolist()
    q_heads, d = q.shape[1:]
    heads, block = s["k"].shape[1:3]
    kind = torch.float8_e4m3fn if s["kv"] == "e4m3" else torch.int8
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    for r, length in enumerate(lens):
        if not length:
            continue
        at = s["table"][r, :_blocks_of(length, block)].long()
        for h in range(heads):
            k, v = (s[x][at, h].view(kind).double() * torch.exp2(s[x + "_scales"][at, h].double() - 127)[:, None, None]
                    for x in ("k", "v"))
            k, v = k.flatten(0, 1)[:length], v.flatten(0, 1)[:length]
            mine = slice(h * q_heads // heads, (h + 1) * q_heads // heads)
            rows = q[starts[r]:starts[r + 1], mine].double()
            n = rows.shape[0]
            score = torch.einsum("ngd,td->ngt", rows, k) / math.sqrt(d)
            back = torch.arange(length - n, length, device=q.device)[:, None] - torch.arange(length, device=q.device)
            hidden = (back < 0) | (back >= s["window"]) if s["window"] else back < 0
            score.masked_fill_(hidden[:, None], -math.inf)
            z = torch.logsumexp(score, -1)
            lse[starts[r]:starts[r + 1], mine] = z
            p = torch.exp(score - z[..., None])
            out[starts[r]:starts[r + 1], mine] = torch.einsum("ngt,td->ngd", torch.nan_to_num(p), v)
    return (out, lse) if s["lse"] else out


def _exact_norm(s):
    def norm(x, w, b):
        if s["kind"] == "layer":
            x = x - x.mean(-1, keepdim=True)
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + s["eps"]) * w.double()
        return x if b is None else x + b.double()

    branch = norm(s["y"].double(), s["post"], s["post_bias"])
    branch = branch if s["gate"] is None else branch * s["gate"].double()
    stream = s["residual"].double() + s["alpha"] * branch
    return stream, norm(stream, s["pre"], s["pre_bias"])


_EXACT = {"append": _exact_append, "attend": _exact_attend, "norm": _exact_norm}
