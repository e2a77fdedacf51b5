"""A decoder served with this package's operators: 4-bit products, a paged 8-bit
KV cache and the fused norms, with requests that come, are prefilled in chunks
beside others that decode, and go.

    python examples/serve_decode.py [--steps 64] [--kv e4m3|int8]

The weights are random: it shows the calls and their order, not a language.
Rotary embedding, SiLU and the choice of tokens are plain torch.
"""
import argparse
import importlib
import os
import sys
import time
from dataclasses import dataclass

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
qg = importlib.import_module("qgemm-mx_b200")


@dataclass
class Config:
    layers: int = 4
    width: int = 2048
    q_heads: int = 16
    heads: int = 4        # KV heads
    head_dim: int = 128
    inner: int = 5632
    vocab: int = 4000
    block: int = 64       # tokens in a cache block


class Decoder:
    """Random weights in MXFP4; norms around both halves of a layer, each with a
    residual scale, as residual_norm fuses them."""

    def __init__(self, c: Config, seed: int = 0):
        self.c = c
        g = torch.Generator(device="cuda").manual_seed(seed)

        def packed(n, k):
            return qg.pack_mxfp4(torch.randn((n, k), generator=g, device="cuda") * k ** -0.5)

        def norm():
            return (torch.randn(c.width, generator=g, device="cuda") * 0.1 + 1).to(torch.bfloat16)

        qkv = (c.q_heads + 2 * c.heads) * c.head_dim
        self.embedding = torch.randn((c.vocab, c.width), generator=g, device="cuda").to(torch.bfloat16)
        self.layers = [dict(qkv=packed(qkv, c.width), o=packed(c.width, c.q_heads * c.head_dim),
                            up=packed(2 * c.inner, c.width), down=packed(c.width, c.inner),
                            pre_attention=norm(), post_attention=norm(), pre_mlp=norm(), post_mlp=norm())
                       for _ in range(c.layers)]
        self.final = norm()
        self.head = packed(c.vocab, c.width)
        self.alpha = (2 * c.layers) ** -0.5
        self.rotation = 10000.0 ** (-torch.arange(c.head_dim // 2, device="cuda") * 2 / c.head_dim)

    def rotary(self, x, positions):
        angle = positions.clamp(min=0)[:, None].float() * self.rotation
        cos, sin = angle.cos()[:, None], angle.sin()[:, None]
        a, b = x.float().chunk(2, -1)
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1).to(torch.bfloat16)

    def __call__(self, tokens, plan, table, caches, max_new, workspace):
        """Logits of every row of the step; the step's K and V go into the caches."""
        c = self.c
        stream = self.embedding[tokens]
        first = self.layers[0]
        stream, h = qg.residual_norm(None, stream, pre=first["pre_attention"])
        for i, (w, cache) in enumerate(zip(self.layers, caches)):
            qkv = qg.gemm_w4a16(w["qkv"], h).unflatten(1, (c.q_heads + 2 * c.heads, c.head_dim))
            q = self.rotary(qkv[:, :c.q_heads], plan.positions)
            k = self.rotary(qkv[:, c.q_heads:c.q_heads + c.heads], plan.positions)
            qg.kv_append(cache, k, qkv[:, c.q_heads + c.heads:], plan.slots, plan.runs)
            attended = qg.kv_attention(cache, q, plan.starts, plan.lens, table, max_new, workspace=workspace)
            y = qg.gemm_w4a16(w["o"], attended.flatten(1))
            stream, h = qg.residual_norm(y, stream, post=w["post_attention"], pre=w["pre_mlp"], alpha=self.alpha)
            gate, up = qg.gemm_w4a16(w["up"], h).chunk(2, -1)
            y = qg.gemm_w4a16(w["down"], torch.nn.functional.silu(gate) * up)
            after = self.layers[i + 1]["pre_attention"] if i + 1 < c.layers else self.final
            stream, h = qg.residual_norm(y, stream, post=w["post_mlp"], pre=after, alpha=self.alpha)
        return qg.gemm_w4a16(self.head, h)


class Server:
    """Fixed places for requests: their lengths, block tables and the free list
    stay on the GPU; a step reads back the chosen tokens only."""

    def __init__(self, model: Decoder, places: int, max_tokens: int, blocks: int, kv: int):
        c = model.c
        self.model, self.places = model, places
        self.caches = [qg.make_kv_cache(kv, blocks, c.block, c.heads, c.head_dim) for _ in range(c.layers)]
        self.lens = torch.zeros(places, dtype=torch.int32, device="cuda")
        self.table = torch.zeros((places, -(-max_tokens // c.block)), dtype=torch.int32, device="cuda")
        self.free = torch.arange(blocks, dtype=torch.int32, device="cuda")
        self.free_count = torch.tensor([blocks], dtype=torch.int32, device="cuda")
        self.workspace = {}

    def step(self, tokens_by_place):
        """tokens_by_place: {place: token ids}.  Returns (plan, logits of all rows)."""
        news = [len(tokens_by_place.get(p, ())) for p in range(self.places)]
        rows = [t for p in range(self.places) for t in tokens_by_place.get(p, ())]
        new = torch.tensor(news, dtype=torch.int32, device="cuda")
        tokens = torch.tensor(rows, dtype=torch.int64, device="cuda")
        c = self.model.c
        plan = qg.kv_plan(self.lens, new, self.table, self.free, self.free_count, c.block, len(rows))
        key = max(news)
        if key not in self.workspace:
            self.workspace[key] = qg.make_kv_workspace(self.caches[0], c.q_heads, self.places, len(rows), key)
        logits = self.model(tokens, plan, self.table, self.caches, key, self.workspace[key])
        self.lens, self.free_count = plan.lens, plan.counts[:1].clone()
        return plan, logits

    def finish(self, place: int) -> None:
        """Gives a request's blocks back to the end of the free list."""
        n = -(-int(self.lens[place]) // self.model.c.block)
        count = int(self.free_count)
        self.free[count:count + n] = self.table[place, :n]
        self.free_count += n
        self.lens = self.lens.clone()
        self.lens[place] = 0


def serve(model: Decoder, prompts, steps: int, kv: int, places: int = 8, chunk: int = 256):
    """Runs the prompts to `steps` new tokens each, `places` at a time, prompts in
    chunks; returns the tokens of each."""
    longest = max(len(p) for p in prompts) + steps
    per = -(-longest // model.c.block)
    server = Server(model, places, longest, places * per + 1, kv)
    waiting = list(range(len(prompts)))
    running, out = {}, [[] for _ in prompts]  # place -> [request, tokens still to feed]
    while waiting or running:
        for p in range(places):
            if p not in running and waiting:
                r = waiting.pop(0)
                running[p] = [r, list(prompts[r])]
        fed = {p: todo[:chunk] for p, (_, todo) in running.items()}
        plan, logits = server.step(fed)
        last = (plan.starts[1:] - 1).clamp(min=0).long()
        chosen = logits[last].argmax(-1).tolist()
        for p in list(running):
            r, todo = running[p]
            del todo[:len(fed[p])]
            if todo:
                continue
            out[r].append(chosen[p])
            todo.append(chosen[p])
            if len(out[r]) == steps:
                server.finish(p)
                del running[p]
    return out


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--requests", type=int, default=12)
    ap.add_argument("--kv", choices=("e4m3", "int8"), default="e4m3")
    a = ap.parse_args()
    model = Decoder(Config())
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, model.c.vocab, (60 + 97 * i,), generator=g).tolist() for i in range(a.requests)]
    kv = qg.KV_E4M3 if a.kv == "e4m3" else qg.KV_INT8
    serve(model, prompts[:2], 2, kv)  # first use of the kernels
    torch.cuda.synchronize()
    t = time.perf_counter()
    out = serve(model, prompts, a.steps, kv)
    torch.cuda.synchronize()
    s = time.perf_counter() - t
    qg.umma_status()
    fed = sum(len(p) for p in prompts)
    print(f"{len(prompts)} requests, {fed} prompt tokens, {sum(map(len, out))} new tokens in {s:.2f} s")


if __name__ == "__main__":
    main()
