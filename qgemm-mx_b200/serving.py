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


# The stream pointer of torch's current stream on a device: the calls below are
# short beside torch.cuda.current_stream().
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)
_i32t, _i64t, _u8t, _bf16, _f32t = torch.int32, torch.int64, torch.uint8, torch.bfloat16, torch.float32
_empty = torch.empty


def _on(t: torch.Tensor, stream) -> int:
    return _raw_stream(t.get_device()) if stream is None else stream.cuda_stream


def _bad(where: str, what: str):
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
        k, v, ks, vs = self.k, self.v, self.k_scales, self.v_scales
        shape = k.shape
        if not (len(shape) == 4 and v.shape == shape and k.dtype is _u8t and v.dtype is _u8t and k.is_contiguous() and
                v.is_contiguous()):
            _bad("KVCache", "k and v must be contiguous uint8 tensors of one shape [blocks, heads, block, head_dim]")
        if not (ks.shape == shape[:2] and vs.shape == shape[:2] and ks.dtype is _u8t and vs.dtype is _u8t and
                ks.is_contiguous() and vs.is_contiguous()):
            _bad("KVCache", "k_scales and v_scales must be contiguous uint8 [blocks, heads]")
        self._desc = _KVCache(self.type, shape[2], shape[1], shape[3], shape[0], k.data_ptr(), v.data_ptr(),
                              ks.data_ptr(), vs.data_ptr())
        self._ref = C.byref(self._desc)

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


def _ints(t: torch.Tensor, dims: int = 1) -> bool:
    return t.dtype is _i32t and t.dim() == dims and t.is_cuda and t.is_contiguous()


def kv_plan(lens: torch.Tensor, new: torch.Tensor, table: torch.Tensor, free_list: torch.Tensor,
            free_count: torch.Tensor, block: int, tokens: int, out: KVPlan | None = None, stream=None) -> KVPlan:
    """Blocks, slots and positions of the `new` tokens of requests that hold
    `lens`; new block ids go into `table` [requests, width].  `tokens` is the
    step's row count (rows no request covers get slot -1).  Nothing is read
    back: plan.counts[3] tells on the device how many requests were refused.
    With `out` (an earlier plan of the same sizes) nothing is allocated."""
    if not (_ints(lens) and _ints(new) and _ints(table, 2) and _ints(free_list) and _ints(free_count)):
        _bad("kv_plan", "lens, new, table [requests, width], free_list and free_count must be contiguous int32 CUDA tensors")
    requests, width = table.shape
    if not (lens.numel() == requests and new.numel() == requests and free_count.numel() == 1):
        _bad("kv_plan", "new, table and free_count must have one entry per request, row per request, and one element")
    most = _lib.qgemm_kv_max_runs(requests, tokens, block)
    if most < 0:
        _bad("kv_plan", "block must be 16, 32, 64 or 128 and tokens not negative")
    if out is None:
        dev = lens.device
        out = KVPlan(_empty(requests + 1, dtype=_i32t, device=dev), _empty(requests, dtype=_i32t, device=dev),
                     _empty(tokens, dtype=_i64t, device=dev), _empty(tokens, dtype=_i32t, device=dev),
                     _empty(most + 1, dtype=_i32t, device=dev), _empty(4, dtype=_i32t, device=dev))
    elif not (out.starts.numel() == requests + 1 and out.lens.numel() == requests and out.slots.numel() == tokens and
              out.positions.numel() == tokens and out.runs.numel() == most + 1 and out.counts.numel() == 4):
        _bad("kv_plan", "out was made for other sizes")
    st = _lib.qgemm_kv_plan(block, requests, lens.data_ptr(), new.data_ptr(), table.data_ptr(), width,
                            free_list.data_ptr(), free_count.data_ptr(), tokens, out.lens.data_ptr(),
                            out.starts.data_ptr(), out.slots.data_ptr(), out.positions.data_ptr(), out.runs.data_ptr(),
                            out.counts.data_ptr(), _on(lens, stream))
    if st:
        _check(st, "kv_plan")
    return out


def _rows(t: torch.Tensor, head_dim: int, where: str, what: str) -> tuple[int, int, int]:
    """Checks bf16 [tokens, heads, head_dim] rows (any spacing of tokens and
    heads); returns the heads, and the elements between tokens and heads."""
    if t.dtype is not _bf16 or t.dim() != 3 or not t.is_cuda or t.shape[2] != head_dim:
        _bad(where, f"{what} must be bf16 [tokens, heads, {head_dim}] on the GPU")
    a, b, c = t.stride()
    if c != 1 and t.numel():
        _bad(where, f"the head_dim values of {what} must lie together")
    return t.shape[1], a, b


def kv_append(cache: KVCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, runs: torch.Tensor,
              stream=None) -> None:
    """Quantises the rows k, v (bf16 [tokens, heads, head_dim], rows may be
    slices of a QKV product) into the slots that kv_plan gave them."""
    d = cache._desc
    kh, ka, kb = _rows(k, d.head_dim, "kv_append", "k")
    vh, va, vb = _rows(v, d.head_dim, "kv_append", "v")
    tokens = k.shape[0]
    if not (kh == d.heads and vh == kh and v.shape[0] == tokens and slots.dtype is _i64t and slots.numel() == tokens and
            slots.is_contiguous()):
        _bad("kv_append", "k, v (the cache's heads) and int64 slots must have one row per token")
    if not _ints(runs) or runs.numel() < 1:
        _bad("kv_append", "runs must be a contiguous int32 CUDA tensor with an end mark")
    st = _lib.qgemm_kv_append(cache._ref, k.data_ptr(), v.data_ptr(), ka, kb, va, vb, tokens, slots.data_ptr(),
                              runs.data_ptr(), runs.numel() - 1, _on(k, stream))
    if st:
        _check(st, "kv_append")


def kv_attention_workspace(cache: KVCache, q_heads: int, requests: int, tokens: int, max_new: int) -> int:
    return _lib.qgemm_kv_attention_workspace(cache._ref, q_heads, requests, tokens, max_new)


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
    head_dim = d.head_dim
    q_heads, qa, qb = _rows(q, head_dim, "kv_attention", "q")
    tokens, requests = q.shape[0], lens.numel()
    if not (_ints(starts) and _ints(lens) and _ints(table, 2)):
        _bad("kv_attention", "starts, lens and table [requests, width] must be contiguous int32 CUDA tensors")
    if not (starts.numel() == requests + 1 and table.shape[0] == requests):
        _bad("kv_attention", "starts needs requests + 1 entries and table a row per request")
    if out is None:
        out = _empty(q.shape, dtype=_bf16, device=q.device)
    elif not (out.shape == q.shape and out.dtype is _bf16 and out.is_contiguous()):
        _bad("kv_attention", "out must be contiguous bf16 of q's shape")
    z = _empty((tokens, q_heads), dtype=_f32t, device=q.device) if lse else None
    if workspace is None:
        workspace = make_kv_workspace(cache, q_heads, requests, tokens, max_new, stream)
    st = _lib.qgemm_kv_attention(cache._ref, q.data_ptr(), qa, qb, q_heads, requests, starts.data_ptr(),
                                 lens.data_ptr(), table.data_ptr(), table.shape[1], tokens, max_new,
                                 head_dim ** -0.5 if scale is None else scale, window, causal, out.data_ptr(),
                                 z.data_ptr() if lse else 0, workspace.data_ptr(), workspace.numel(), _on(q, stream))
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
    if not (residual.dim() == 2 and residual.dtype in (_bf16, _f32t) and residual.is_cuda and residual.is_contiguous()):
        _bad("residual_norm", "residual must be contiguous bf16 or float32 [tokens, width] on the GPU")
    shape = residual.shape
    tokens, width = shape
    for t in (y, h):
        if t is not None and not (t.dtype is _bf16 and t.shape == shape and t.is_contiguous()):
            _bad("residual_norm", "y and h must be contiguous bf16 [tokens, width]")
    for t in (post, pre, post_bias, pre_bias):
        if t is not None and not (t.dtype is _bf16 and t.dim() == 1 and t.numel() == width and t.is_contiguous()):
            _bad("residual_norm", "post, pre and their biases must be contiguous bf16 [width]")
    gate_stride = 0
    if gate is not None:
        if not (gate.dtype is _bf16 and gate.is_cuda and gate.shape in ((width,), shape) and
                (gate.stride(-1) == 1 or width == 1)):
            _bad("residual_norm", "gate must be bf16 [width] or [tokens, width]")
        gate_stride = gate.stride(0) if gate.dim() == 2 else 0
    code = NORM_KINDS.get(kind)
    if code is None:
        _bad("residual_norm", "kind must be 'rms' or 'layer'")
    if y is None:
        residual_out = residual
    elif residual_out is None:
        residual_out = _empty(shape, dtype=residual.dtype, device=residual.device)
    elif not (residual_out.shape == shape and residual_out.dtype is residual.dtype and residual_out.is_contiguous()):
        _bad("residual_norm", "residual_out must be like residual")
    if pre is None:
        h = None
    elif h is None:
        h = _empty(shape, dtype=_bf16, device=residual.device)
    a = _ResidualNorm(code, tokens, width, residual.dtype is _f32t, 0 if y is None else y.data_ptr(),
                      residual.data_ptr(), 0 if post is None else post.data_ptr(),
                      0 if post_bias is None else post_bias.data_ptr(), 0 if gate is None else gate.data_ptr(),
                      gate_stride, 0 if pre is None else pre.data_ptr(), 0 if pre_bias is None else pre_bias.data_ptr(),
                      alpha, eps, residual_out.data_ptr(), 0 if h is None else h.data_ptr())
    st = _lib.qgemm_residual_norm(C.byref(a), _on(residual, stream))
    if st:
        _check(st, "residual_norm")
    return residual_out, h
