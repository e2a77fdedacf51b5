"""Serving operators around the W4A16 products: a paged KV cache in 8 bits
(block plan, quantising append, attention) and the norms around a block with
its gate and residual scale.  Thin layer over the C-ABI in
``include/qgemm_b200.h``, which states each operator's formula; everything
runs on the caller's stream and can be captured into a CUDA graph when the
workspace is passed in.  Imported when one of its names is first used; it needs
``_binding.so`` (`make -C qgemm-mx_b200/csrc binding`) beside the library.
"""
from __future__ import annotations

import os

import torch

from . import HERE, _check, _lib, _ptr, _stream

if not os.path.exists(os.path.join(HERE, "_binding.so")):
    raise ImportError(f"{HERE}/_binding.so is missing: build it with `make -C qgemm-mx_b200/csrc binding`")
from . import _binding as _b  # noqa: E402  csrc/binding.cpp

# cache types (qgemm_kv_type_t)
KV_E4M3, KV_INT8 = 0, 1
# norm kinds (qgemm_norm_kind_t)
NORM_KINDS = {"rms": 0, "layer": 1}


def _handle(stream):
    return None if stream is None else stream.cuda_stream


class KVCache:
    """A pool of blocks on the device.  ``k`` and ``v`` hold 8-bit codes
    (uint8 storage) [blocks, heads, block, head_dim], ``k_scales`` and
    ``v_scales`` one E8M0 byte per (block, head), 2^(byte - 127) with bytes of
    63 .. 249.  ``type`` is KV_E4M3 or KV_INT8.  The attributes cannot be set: the calls go by the
    pointers taken here."""
    __slots__ = ("_type", "_k", "_v", "_k_scales", "_v_scales", "_desc")

    def __init__(self, type: int, k: torch.Tensor, v: torch.Tensor, k_scales: torch.Tensor, v_scales: torch.Tensor):
        self._desc = _b.kv_cache(type, k, v, k_scales, v_scales)  # a qgemm_kv_cache_t, then its GPU
        self._type, self._k, self._v, self._k_scales, self._v_scales = type, k, v, k_scales, v_scales

    type = property(lambda self: self._type)
    k = property(lambda self: self._k)
    v = property(lambda self: self._v)
    k_scales = property(lambda self: self._k_scales)
    v_scales = property(lambda self: self._v_scales)

    def values(self) -> tuple[torch.Tensor, torch.Tensor]:
        """(K, V) as float32 [blocks, heads, block, head_dim], for inspection."""
        kind = torch.float8_e4m3fn if self.type == KV_E4M3 else torch.int8
        return tuple(c.view(kind).float() * torch.exp2(s.float() - 127)[..., None, None]
                     for c, s in ((self.k, self.k_scales), (self.v, self.v_scales)))


def make_kv_cache(type: int, blocks: int, block: int, heads: int, head_dim: int, device="cuda") -> KVCache:
    """A pool of `blocks` blocks of `block` tokens; its contents need no
    clearing (a block's first append sets its scale)."""
    shape = (blocks, heads, block, head_dim)
    k, v = (torch.empty(shape, dtype=torch.uint8, device=device) for _ in range(2))
    ks, vs = (torch.empty(shape[:2], dtype=torch.uint8, device=device) for _ in range(2))
    return KVCache(type, k, v, ks, vs)


class KVPlan:
    """What kv_plan computes for one step (qgemm_kv_plan's outputs):
    starts     int32 [requests + 1]: each request's rows of the step
    lens       int32 [requests]: lengths with the new tokens
    slots      int64 [tokens]: block * block size + place, -1 where there is none
    positions  int32 [tokens]: each row's position in its request, or -1
    runs       int32: first row of each run of rows that share a block, then end marks
    counts     int32 [4]: free blocks left, runs, rows, refused requests"""
    __slots__ = ("starts", "lens", "slots", "positions", "runs", "counts")

    def __init__(self, starts, lens, slots, positions, runs, counts):
        self.starts, self.lens, self.slots, self.positions, self.runs, self.counts = \
            starts, lens, slots, positions, runs, counts


def kv_plan(lens: torch.Tensor, new: torch.Tensor, table: torch.Tensor, free_list: torch.Tensor,
            free_count: torch.Tensor, block: int, tokens: int, out: KVPlan | None = None, stream=None) -> KVPlan:
    """Blocks, slots and positions of the `new` tokens of requests that hold
    `lens`; new block ids go into `table` [requests, width].  `tokens` is the
    step's row count (rows no request covers get slot -1).  A free_count past
    free_list's end counts as its length.  Nothing is read
    back: plan.counts[3] tells on the device how many requests were refused.
    With `out` (an earlier plan of the same sizes) nothing is allocated; lens,
    new and free_count must then not be that plan's own tensors."""
    kept = None if out is None else (out.starts, out.lens, out.slots, out.positions, out.runs, out.counts)
    st, *got = _b.kv_plan(lens, new, table, free_list, free_count, block, tokens, kept, _handle(stream))
    if st:
        _check(st, "kv_plan")
    return KVPlan(*got)


def kv_append(cache: KVCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, runs: torch.Tensor,
              stream=None) -> None:
    """Quantises the rows k, v (bf16 [tokens, heads, head_dim], rows may be
    slices of a QKV product) into the slots that kv_plan gave them."""
    st, = _b.kv_append(cache._desc, k, v, slots, runs, _handle(stream))
    if st:
        _check(st, "kv_append")


def kv_attention_workspace(cache: KVCache, q_heads: int, requests: int, tokens: int, max_new: int) -> int:
    return _lib.qgemm_kv_attention_workspace(cache._desc, q_heads, requests, tokens, max_new)


def make_kv_workspace(cache: KVCache, q_heads: int, requests: int, tokens: int, max_new: int,
                      stream=None) -> torch.Tensor:
    """Zeroed workspace for kv_attention calls of up to these sizes on `stream`
    (the current one), whose memory it is: allocated, cleared and, once dropped,
    given out again in that stream's order."""
    if not cache.k.is_cuda:
        raise ValueError("make_kv_workspace: the cache must be on a GPU")
    with torch.cuda.device(cache.k.device) if stream is None else torch.cuda.stream(stream):
        n = max(kv_attention_workspace(cache, q_heads, requests, tokens, max_new), 256)
        ws = torch.empty(n, dtype=torch.uint8, device=cache.k.device)
        _check(_lib.qgemm_workspace_init(_ptr(ws), n, _stream()), "workspace_init")
    return ws


def kv_attention(cache: KVCache, q: torch.Tensor, starts: torch.Tensor, lens: torch.Tensor, table: torch.Tensor,
                 max_new: int, scale: float | None = None, window: int = 0, causal: bool = True, lse: bool = False,
                 out: torch.Tensor | None = None, workspace: torch.Tensor | None = None, stream=None):
    """softmax(scale * q.K) . V over the cache: q bf16 [tokens, q_heads,
    head_dim], request r's rows starts[r] .. starts[r + 1] - 1 being the last
    of its lens[r] tokens.  scale defaults to head_dim ** -0.5; window > 0
    bounds how far back a row sees.  Returns out (bf16, as q), or (out, lse).
    Rows that no request brings, or past max_new of theirs, are not written."""
    if workspace is None:
        workspace = make_kv_workspace(cache, q.shape[1], lens.numel(), q.shape[0], max_new, stream)
    st, out, z = _b.kv_attention(cache._desc, q, starts, lens, table, max_new,
                                 cache._k.shape[3] ** -0.5 if scale is None else scale, window, causal, lse, out,
                                 workspace, _handle(stream))
    if st:
        _check(st, "kv_attention")
    return (out, z) if lse else out


def residual_norm(y: torch.Tensor | None, residual: torch.Tensor, post: torch.Tensor | None = None,
                  pre: torch.Tensor | None = None, post_bias: torch.Tensor | None = None,
                  pre_bias: torch.Tensor | None = None, gate: torch.Tensor | None = None, alpha: float = 1.0,
                  kind: str = "rms", eps: float = 1e-6, residual_out: torch.Tensor | None = None,
                  h: torch.Tensor | None = None, stream=None):
    """(residual + alpha * gate * N(y; post), N of that; pre): the end of one
    block and the beginning of the next.  y and h bf16 [tokens, width],
    residual bf16 or float32; gate [width] or [tokens, width].  A left-out
    post, gate or bias drops its factor; without pre, h is None; without y
    (the first block) residual is only normed.  residual_out may be residual
    and h may be y."""
    code = NORM_KINDS.get(kind)
    if code is None:
        raise ValueError("residual_norm: kind must be 'rms' or 'layer'")
    st, residual_out, h = _b.residual_norm(y, residual, post, pre, post_bias, pre_bias, gate, alpha, code, eps,
                                           residual_out, h, _handle(stream))
    if st:
        _check(st, "residual_norm")
    return residual_out, h
