"""Serving operators around the W4A16 products: a paged KV cache in 8 bits
(block plan, quantising append, attention) and the norms around a block with
its gate and residual scale.  Thin layer over the C-ABI in
``include/qgemm_b200.h``, which states each operator's formula; everything
runs on the caller's stream and can be captured into a CUDA graph when outputs
and workspace are passed in.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import torch

from . import _check, _lib, _ptr, _sig, _stream

_vp, _sz, _i32, _i64, _f32 = C.c_void_p, C.c_size_t, C.c_int32, C.c_int64, C.c_float

# cache types (qgemm_kv_type_t)
KV_E4M3, KV_INT8 = 0, 1
# norm kinds (qgemm_norm_kind_t)
NORM_KINDS = {"rms": 0, "layer": 1}


class _KVCache(C.Structure):
    _fields_ = [("type", _i32), ("block", _i32), ("heads", _i32), ("head_dim", _i32), ("blocks", _i64),
                ("k", _vp), ("v", _vp), ("k_scales", _vp), ("v_scales", _vp)]


class _ResidualNorm(C.Structure):
    _fields_ = [("kind", _i32), ("tokens", _i32), ("width", _i32), ("residual_f32", _i32), ("y", _vp),
                ("residual", _vp), ("post", _vp), ("post_bias", _vp), ("gate", _vp), ("gate_stride", _i64),
                ("pre", _vp), ("pre_bias", _vp), ("alpha", _f32), ("eps", _f32), ("residual_out", _vp), ("h", _vp)]


_sig("qgemm_kv_max_runs", _i32, [_i32, _i32, _i32])
_sig("qgemm_kv_plan", _i32, [_i32, _i32, _vp, _vp, _vp, _i32, _vp, _vp, _i32, _vp, _vp, _vp, _vp, _vp, _vp, _vp])
_sig("qgemm_kv_append", _i32, [C.POINTER(_KVCache), _vp, _vp, _i64, _i64, _i64, _i64, _i32, _vp, _vp, _i32, _vp])
_sig("qgemm_kv_attention_workspace", _sz, [C.POINTER(_KVCache), _i32, _i32, _i32, _i32])
_sig("qgemm_kv_attention", _i32, [C.POINTER(_KVCache), _vp, _i64, _i64, _i32, _i32, _vp, _vp, _vp, _i32, _i32, _i32, _f32,
                                  _i32, _i32, _vp, _vp, _vp, _sz, _vp])
_sig("qgemm_residual_norm", _i32, [C.POINTER(_ResidualNorm), _vp])


def _want(ok: bool, where: str, what: str) -> None:
    if not ok:
        raise ValueError(f"{where}: {what}")


@dataclass
class KVCache:
    """A pool of blocks on the device.  ``k`` and ``v`` hold 8-bit codes
    (uint8 storage) [blocks, heads, block, head_dim], ``k_scales`` and
    ``v_scales`` one E8M0 byte per (block, head), 2^(byte - 127)."""
    type: int
    k: torch.Tensor
    v: torch.Tensor
    k_scales: torch.Tensor
    v_scales: torch.Tensor

    def __post_init__(self):
        shape = self.k.shape
        for t in (self.k, self.v):
            _want(t.dim() == 4 and t.dtype == torch.uint8 and t.is_contiguous() and t.shape == shape, "KVCache",
                  "k and v must be contiguous uint8 tensors of one shape [blocks, heads, block, head_dim]")
        for t in (self.k_scales, self.v_scales):
            _want(t.dtype == torch.uint8 and t.is_contiguous() and t.shape == shape[:2], "KVCache",
                  "k_scales and v_scales must be contiguous uint8 [blocks, heads]")
        self._desc = _KVCache(self.type, shape[2], shape[1], shape[3], shape[0], self.k.data_ptr(),
                              self.v.data_ptr(), self.k_scales.data_ptr(), self.v_scales.data_ptr())

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


@dataclass
class KVPlan:
    """What kv_plan computes for one step (qgemm_kv_plan's outputs)."""
    starts: torch.Tensor     # int32 [requests + 1]: each request's rows of the step
    lens: torch.Tensor       # int32 [requests]: lengths with the new tokens
    slots: torch.Tensor      # int64 [tokens]: block * block size + place, -1 where there is none
    positions: torch.Tensor  # int32 [tokens]: each row's position in its request, or -1
    runs: torch.Tensor       # int32: first row of each run of rows that share a block, then end marks
    counts: torch.Tensor     # int32 [4]: free blocks left, runs, rows, refused requests


def _ints(t: torch.Tensor, where: str, what: str, dims: int = 1) -> None:
    _want(t.dtype == torch.int32 and t.dim() == dims and t.is_contiguous() and t.is_cuda, where,
          f"{what} must be a contiguous int32 CUDA tensor with {dims} dimension(s)")


def kv_plan(lens: torch.Tensor, new: torch.Tensor, table: torch.Tensor, free_list: torch.Tensor,
            free_count: torch.Tensor, block: int, tokens: int, out: KVPlan | None = None, stream=None) -> KVPlan:
    """Blocks, slots and positions of the `new` tokens of requests that hold
    `lens`; new block ids go into `table` [requests, width].  `tokens` is the
    step's row count (rows no request covers get slot -1).  Nothing is read
    back: plan.counts[3] tells on the device how many requests were refused."""
    requests = lens.numel()
    _ints(lens, "kv_plan", "lens")
    _ints(new, "kv_plan", "new")
    _ints(table, "kv_plan", "table", 2)
    _ints(free_list, "kv_plan", "free_list")
    _ints(free_count, "kv_plan", "free_count")
    _want(new.numel() == requests and table.shape[0] == requests and free_count.numel() == 1, "kv_plan",
          "new, table and free_count must have one entry per request, row per request, and one element")
    most = _lib.qgemm_kv_max_runs(requests, tokens, block)
    _want(most >= 0, "kv_plan", "block must be 16, 32, 64 or 128 and tokens not negative")
    if out is None:
        # one allocation for the int32 outputs
        sizes = (requests + 1, requests, tokens, most + 1, 4)
        starts, lens_out, positions, runs, counts = torch.empty(
            sum(sizes), dtype=torch.int32, device=lens.device).split(sizes)
        out = KVPlan(starts, lens_out, torch.empty(tokens, dtype=torch.int64, device=lens.device), positions, runs,
                     counts)
    else:
        _want(out.starts.numel() == requests + 1 and out.lens.numel() == requests and out.slots.numel() == tokens and
              out.positions.numel() == tokens and out.runs.numel() == most + 1 and out.counts.numel() == 4, "kv_plan",
              "out was made for other sizes")
    _check(_lib.qgemm_kv_plan(block, requests, lens.data_ptr(), new.data_ptr(), table.data_ptr(), table.shape[1],
                              free_list.data_ptr(), free_count.data_ptr(), tokens, out.lens.data_ptr(),
                              out.starts.data_ptr(), out.slots.data_ptr(), out.positions.data_ptr(),
                              out.runs.data_ptr(), out.counts.data_ptr(), _stream(stream)), "kv_plan")
    return out


def _rows(t: torch.Tensor, heads: int | None, head_dim: int, where: str, what: str) -> tuple[int, int]:
    """Checks bf16 [tokens, heads, head_dim] rows (any spacing of tokens and
    heads); returns the elements between tokens and between heads."""
    _want(t.dtype == torch.bfloat16 and t.dim() == 3 and t.is_cuda and t.shape[2] == head_dim and
          (heads is None or t.shape[1] == heads), where, f"{what} must be bf16 [tokens, heads, {head_dim}] on the GPU")
    a, b, c = t.stride()
    _want(c == 1 or t.numel() == 0, where, f"the head_dim values of {what} must lie together")
    return a, b


def kv_append(cache: KVCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, runs: torch.Tensor,
              stream=None) -> None:
    """Quantises the rows k, v (bf16 [tokens, heads, head_dim], rows may be
    slices of a QKV product) into the slots that kv_plan gave them."""
    d = cache._desc
    ks = _rows(k, d.heads, d.head_dim, "kv_append", "k")
    vs = _rows(v, d.heads, d.head_dim, "kv_append", "v")
    tokens = k.shape[0]
    _want(v.shape[0] == tokens and slots.dtype == torch.int64 and slots.numel() == tokens and slots.is_contiguous(),
          "kv_append", "k, v and int64 slots must have one row per token")
    _ints(runs, "kv_append", "runs")
    _want(runs.numel() >= 1, "kv_append", "runs must hold an end mark")
    _check(_lib.qgemm_kv_append(C.byref(d), k.data_ptr(), v.data_ptr(), *ks, *vs, tokens, slots.data_ptr(),
                                runs.data_ptr(), runs.numel() - 1, _stream(stream)), "kv_append")


def kv_attention_workspace(cache: KVCache, q_heads: int, requests: int, tokens: int, max_new: int) -> int:
    return _lib.qgemm_kv_attention_workspace(C.byref(cache._desc), q_heads, requests, tokens, max_new)


def make_kv_workspace(cache: KVCache, q_heads: int, requests: int, tokens: int, max_new: int,
                      stream=None) -> torch.Tensor:
    """Zeroed workspace for kv_attention calls of up to these sizes."""
    n = max(kv_attention_workspace(cache, q_heads, requests, tokens, max_new), 256)
    ws = torch.empty(n, dtype=torch.uint8, device=cache.k.device)
    _check(_lib.qgemm_workspace_init(_ptr(ws), n, _stream(stream)), "workspace_init")
    return ws


def kv_attention(cache: KVCache, q: torch.Tensor, starts: torch.Tensor, lens: torch.Tensor, table: torch.Tensor,
                 max_new: int, scale: float | None = None, window: int = 0, causal: bool = True, lse: bool = False,
                 out: torch.Tensor | None = None, workspace: torch.Tensor | None = None, stream=None):
    """softmax(scale * q.K) . V over the cache: q bf16 [tokens, q_heads,
    head_dim], request r's rows starts[r] .. starts[r + 1] - 1 being the last
    of its lens[r] tokens.  scale defaults to head_dim ** -0.5; window > 0
    bounds how far back a row sees.  Returns out (bf16, as q), or (out, lse)."""
    d = cache._desc
    strides = _rows(q, None, d.head_dim, "kv_attention", "q")
    tokens, q_heads = q.shape[0], q.shape[1]
    _ints(starts, "kv_attention", "starts")
    _ints(lens, "kv_attention", "lens")
    _ints(table, "kv_attention", "table", 2)
    requests = lens.numel()
    _want(starts.numel() == requests + 1 and table.shape[0] == requests, "kv_attention",
          "starts needs requests + 1 entries and table a row per request")
    if out is None:
        out = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
    else:
        _want(out.shape == q.shape and out.dtype == torch.bfloat16 and out.is_contiguous(), "kv_attention",
              "out must be contiguous bf16 of q's shape")
    z = torch.empty((tokens, q_heads), dtype=torch.float32, device=q.device) if lse else None
    if workspace is None:
        workspace = make_kv_workspace(cache, q_heads, requests, tokens, max_new, stream)
    _check(_lib.qgemm_kv_attention(C.byref(d), q.data_ptr(), *strides, q_heads, requests, starts.data_ptr(),
                                   lens.data_ptr(), table.data_ptr(), table.shape[1], tokens, max_new,
                                   d.head_dim ** -0.5 if scale is None else scale, window, causal, out.data_ptr(),
                                   0 if z is None else z.data_ptr(), workspace.data_ptr(), workspace.numel(),
                                   _stream(stream)), "kv_attention")
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
    where = "residual_norm"
    _want(kind in NORM_KINDS, where, "kind must be 'rms' or 'layer'")
    _want(residual.dim() == 2 and residual.dtype in (torch.bfloat16, torch.float32) and residual.is_contiguous() and
          residual.is_cuda, where, "residual must be contiguous bf16 or float32 [tokens, width] on the GPU")
    tokens, width = residual.shape
    stream_like = residual.dtype
    for t, what in ((y, "y"), (h, "h")):
        _want(t is None or (t.shape == residual.shape and t.dtype == torch.bfloat16 and t.is_contiguous()), where,
              f"{what} must be contiguous bf16 [tokens, width]")
    for t, what in ((post, "post"), (pre, "pre"), (post_bias, "post_bias"), (pre_bias, "pre_bias")):
        _want(t is None or (t.shape == (width,) and t.dtype == torch.bfloat16 and t.is_contiguous()), where,
              f"{what} must be contiguous bf16 [width]")
    gate_stride = 0
    if gate is not None:
        _want(gate.dtype == torch.bfloat16 and gate.is_cuda and gate.shape in ((width,), (tokens, width)) and
              (gate.stride(-1) == 1 or width == 1), where, "gate must be bf16 [width] or [tokens, width]")
        gate_stride = gate.stride(0) if gate.dim() == 2 else 0
    if y is not None and residual_out is None:
        residual_out = torch.empty_like(residual)
    elif y is None:
        residual_out = residual
    _want(residual_out.shape == residual.shape and residual_out.dtype == stream_like and
          residual_out.is_contiguous(), where, "residual_out must be like residual")
    if pre is not None and h is None:
        h = torch.empty(residual.shape, dtype=torch.bfloat16, device=residual.device)
    a = _ResidualNorm(NORM_KINDS[kind], tokens, width, stream_like == torch.float32,
                      *(0 if t is None else t.data_ptr() for t in (y, residual, post, post_bias, gate)), gate_stride,
                      *(0 if t is None else t.data_ptr() for t in (pre, pre_bias)), alpha, eps,
                      residual_out.data_ptr(), 0 if pre is None else h.data_ptr())
    _check(_lib.qgemm_residual_norm(C.byref(a), _stream(stream)), where)
    return residual_out, h if pre is not None else None
