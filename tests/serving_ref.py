"""Plain 64-bit restatements of the serving operators (paged 8-bit KV cache,
residual norms), with loops over requests, rows and blocks.  They run on any
device and share nothing with the kernels but the definitions."""
import math

import torch

E4M3, INT8 = 0, 1
QMAX = {E4M3: 448.0, INT8: 127.0}


def plan(lens, new, table, free, count, block, tokens):
    """Lists in, (table, lens, starts, slots, positions, runs, counts) out."""
    table = [list(r) for r in table]
    width = len(table[0]) if table else 0
    starts, out, refused, upto, used = [0], [], 0, 0, 0
    slots, positions, leads = [-1] * tokens, [-1] * tokens, []
    for r, (have, n) in enumerate(zip(lens, new)):
        n = max(n, 0)
        at, base = starts[-1], max(have, 0)
        held, last = -(-base // block), -(-(base + n) // block)
        fits = have >= 0 and last <= width
        need = last - held if fits else 0
        upto += need
        ok = fits and at + n <= tokens and (need == 0 or upto <= count)
        if ok:
            used = max(used, upto)
            for j in range(need):
                table[r][held + j] = free[count - 1 - (upto - need + j)]
        else:
            refused += 1
        for i in range(min(n, max(tokens - at, 0))):
            p = base + i
            if i == 0 or p % block == 0:
                leads.append(at + i)
            if ok:
                slots[at + i] = table[r][p // block] * block + p % block
                positions[at + i] = p
        out.append(base + n if ok else have)
        starts.append(at + n)
    total = min(starts[-1], tokens)
    most = min(tokens, 2 * len(lens) + tokens // block)
    runs = leads + [total] * (most + 1 - len(leads))
    return table, out, starts, slots, positions, runs, [count - used, len(leads), total, refused]


def needed_exp(amax, kv):
    """Smallest e >= -64 with amax <= QMAX 2^e (amax a float)."""
    e = -64
    while amax > QMAX[kv] * 2.0 ** e:
        e += 1
    return e


def encode(x, kv):
    """float64 values (divided by the scale) to 8-bit codes."""
    x = torch.where(torch.isnan(x), torch.zeros_like(x), x).clamp(-QMAX[kv], QMAX[kv])
    if kv == INT8:
        return x.round().to(torch.int8).view(torch.uint8)
    # nearest E4M3: grid 2^(e - 3) for |x| in [2^e, 2^(e + 1)), e >= -6; ties to even
    _, e = torch.frexp(x.abs())
    step = torch.exp2((e - 1).clamp(min=-6).double() - 3)
    return ((x / step).round() * step).float().to(torch.float8_e4m3fn).view(torch.uint8)


def decode(codes, kv):
    return codes.view(torch.float8_e4m3fn if kv == E4M3 else torch.int8).float().double()


def append(codes, scales, x, slots, kv):
    """In place on CPU tensors: one call's rows into codes / scales."""
    block = codes.shape[2]
    where = slots.tolist()
    t = 0
    while t < len(where):
        if where[t] < 0 or where[t] // block >= codes.shape[0]:
            t += 1
            continue
        page, off = divmod(where[t], block)
        n = 1
        while t + n < len(where) and off + n < block and where[t + n] == where[t] + n:
            n += 1
        for h in range(codes.shape[1]):
            rows = x[t:t + n, h].double()
            size = rows.abs()
            finite = size[torch.isfinite(size)]
            e = needed_exp(float(finite.max()) if finite.numel() else 0.0, kv)
            if off:
                was = int(scales[page, h]) - 127
                e = max(e, was)
                if e > was:
                    old = decode(codes[page, h, :off], kv)
                    codes[page, h, :off] = encode(old * 2.0 ** (was - e), kv)
            codes[page, h, off:off + n] = encode(rows * 2.0 ** -e, kv)
            scales[page, h] = e + 127
        t += n


def attention(kv, k, v, ks, vs, q, starts, lens, table, scale, window=0, causal=True):
    """float64 (out, lse, mass, logit, floor), the last three for error bounds:
    mass = sum p |v| per output value, logit = the largest sum |q k| scale per
    row, floor = (the row's largest p 2^ev) sum |v code|."""
    kind = torch.float8_e4m3fn if kv == E4M3 else torch.int8
    q_heads, d = q.shape[1:]
    heads, block = k.shape[1:3]
    group = q_heads // heads
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    mass = torch.zeros_like(out)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    logit = torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
    floor = torch.zeros_like(out)
    for r, length in enumerate(lens.tolist()):
        a, b = int(starts[r]), int(starts[r + 1])
        n, length = b - a, min(max(length, 0), table.shape[1] * block)
        if not n or not length:
            continue
        ids = table[r, :-(-length // block)].long()
        for h in range(heads):
            kk, vv = (c[ids, h].view(kind).float().double().flatten(0, 1)[:length] *
                      torch.exp2(s[ids, h].double() - 127).repeat_interleave(block)[:length, None]
                      for c, s in ((k, ks), (v, vs)))
            rows = q[a:b, h * group:(h + 1) * group].double()
            s = torch.einsum("ngd,td->ngt", rows, kk) * scale
            logit[a:b, h * group:(h + 1) * group] = \
                (torch.einsum("ngd,td->ngt", rows.abs(), kk.abs()) * abs(scale)).amax(-1)
            pos = torch.arange(length - n, length, device=q.device)[:, None]
            tok = torch.arange(length, device=q.device)[None]
            see = tok <= pos if causal else torch.ones_like(tok <= pos)
            if window:
                see = see & (tok > pos - window)
            s = s.masked_fill(~see[:, None], -math.inf)
            z = torch.logsumexp(s, -1)
            p = torch.exp(s - torch.where(torch.isinf(z), torch.zeros_like(z), z)[..., None])
            sl = (slice(a, b), slice(h * group, (h + 1) * group))
            out[sl] = torch.einsum("ngt,td->ngd", p, vv)
            mass[sl] = torch.einsum("ngt,td->ngd", p, vv.abs())
            lse[sl] = z
            ev = torch.exp2(vs[ids, h].double() - 127).repeat_interleave(block)[:length]
            floor[sl] = (p * ev).amax(-1, keepdim=True) * (vv / ev[:, None]).abs().sum(0)
    return out, lse, mass, logit, floor


def norm(x, w, b, kind, eps):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    return x if b is None else x + b.double()


def residual_norm(y, residual, post, pre, post_bias, pre_bias, gate, alpha, kind, eps):
    r = residual.double()
    if y is not None:
        z = y.double()
        if post is not None:
            z = norm(z, post, post_bias, kind, eps)
        if gate is not None:
            z = z * gate.double()
        r = r + alpha * z
    return r, None if pre is None else norm(r, pre, pre_bias, kind, eps)
