"""Argument checks of the serving operators at the C-ABI, decided on the host before
any launch (no GPU needed), and their Python calls' refusals of what is not a
CUDA tensor."""
import ctypes as C

import pytest
import torch


class Cache(C.Structure):
    _fields_ = [("type", C.c_int32), ("block", C.c_int32), ("heads", C.c_int32), ("head_dim", C.c_int32),
                ("blocks", C.c_int64), ("k", C.c_void_p), ("v", C.c_void_p), ("ks", C.c_void_p), ("vs", C.c_void_p)]


class Norm(C.Structure):
    _fields_ = [("kind", C.c_int32), ("tokens", C.c_int32), ("width", C.c_int32), ("f32", C.c_int32), ("y", C.c_void_p),
                ("residual", C.c_void_p), ("post", C.c_void_p), ("post_bias", C.c_void_p), ("gate", C.c_void_p),
                ("gate_stride", C.c_int64), ("pre", C.c_void_p), ("pre_bias", C.c_void_p), ("alpha", C.c_float),
                ("eps", C.c_float), ("out", C.c_void_p), ("h", C.c_void_p)]


P = 1 << 20  # a plausible, aligned address that is never read


def cache(**kw):
    c = Cache(0, 64, 8, 128, 100, P, P, P, P)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


BAD_CACHES = [dict(type=2), dict(type=-1), dict(block=0), dict(block=24), dict(block=256), dict(heads=0),
              dict(heads=65536), dict(head_dim=96), dict(head_dim=256), dict(blocks=0), dict(blocks=2 ** 31),
              dict(k=None), dict(v=None), dict(ks=None), dict(vs=None), dict(k=P + 8), dict(v=P + 4)]


@pytest.mark.parametrize("bad", BAD_CACHES)
def test_bad_caches(qg, bad):
    lib, c = qg.lib(), cache(**bad)
    assert lib.qgemm_kv_append(C.byref(c), P, P, 1024, 128, 1024, 128, 4, P, P, 4, None) == qg.ERR_INVALID_ARG
    assert lib.qgemm_kv_attention(C.byref(c), P, 8192, 128, 64, 1, P, P, P, 4, 1, 1, 0.1, 0, 1, P, None, P, 1 << 30,
                                  None) == qg.ERR_INVALID_ARG
    assert lib.qgemm_kv_attention_workspace(C.byref(c), 64, 1, 1, 1) == 0


def test_append_refusals(qg):
    lib, c = qg.lib(), cache()

    def call(k=P, v=P, ks=1024, kh=128, vs=1024, vh=128, tokens=4, slots=P, runs=P, most=4):
        return lib.qgemm_kv_append(C.byref(c), k, v, ks, kh, vs, vh, tokens, slots, runs, most, None)

    for kw in (dict(k=None), dict(v=None), dict(slots=None), dict(runs=None), dict(k=P + 2), dict(v=P + 8), dict(ks=1025),
               dict(kh=4), dict(vs=-3), dict(vh=1), dict(tokens=-1), dict(tokens=2 ** 30), dict(most=-1)):
        assert call(**kw) == qg.ERR_INVALID_ARG, kw
    assert call(tokens=0) == qg.OK and call(most=0) == qg.OK  # nothing to do
    assert call(most=2 ** 30) == qg.ERR_UNSUPPORTED_SHAPE
    assert lib.qgemm_kv_append(None, P, P, 8, 8, 8, 8, 1, P, P, 1, None) == qg.ERR_INVALID_ARG


def test_attention_refusals(qg):
    lib, c = qg.lib(), cache()

    def call(q=P, qs=8192, qh=128, heads=64, requests=2, starts=P, lens=P, table=P, width=4, tokens=3, new=2, scale=0.1,
             window=0, out=P, ws=P, nbytes=1 << 30):
        return lib.qgemm_kv_attention(C.byref(c), q, qs, qh, heads, requests, starts, lens, table, width, tokens, new,
                                      scale, window, 1, out, None, ws, nbytes, None)

    for kw in (dict(q=None), dict(starts=None), dict(lens=None), dict(table=None), dict(out=None), dict(q=P + 2),
               dict(out=P + 8), dict(qs=8190), dict(qh=3), dict(heads=0), dict(heads=12), dict(requests=-1), dict(width=-1),
               dict(tokens=-1), dict(tokens=2 ** 30), dict(new=-1), dict(window=-1), dict(scale=float("nan")),
               dict(scale=float("inf"))):
        assert call(**kw) == qg.ERR_INVALID_ARG, kw
    for kw in (dict(requests=0), dict(tokens=0), dict(new=0)):
        assert call(**kw) == qg.OK, kw  # nothing to do
    assert call(width=2 ** 25) == qg.ERR_UNSUPPORTED_SHAPE


def test_plan_refusals(qg):
    lib = qg.lib()

    def call(block=64, requests=2, lens=P, news=P, table=P, width=4, free=P, count=P, tokens=5, lens_out=2 * P, starts=P,
             slots=P, positions=P, runs=P, counts=P):
        return lib.qgemm_kv_plan(block, requests, lens, news, table, width, free, count, tokens, lens_out, starts, slots,
                                 positions, runs, counts, None)

    for kw in (dict(block=0), dict(block=48), dict(requests=-1), dict(tokens=-1), dict(width=-1), dict(tokens=2 ** 30),
               dict(lens=None), dict(news=None), dict(table=None), dict(count=None), dict(lens_out=None), dict(starts=None),
               dict(slots=None), dict(positions=None), dict(runs=None), dict(counts=None), dict(lens_out=P)):
        assert call(**kw) == qg.ERR_INVALID_ARG, kw
    assert lib.qgemm_kv_max_runs(3, 100, 16) == 12 and lib.qgemm_kv_max_runs(64, 64, 64) == 64
    assert lib.qgemm_kv_max_runs(-1, 4, 16) == -1 and lib.qgemm_kv_max_runs(1, 4, 17) == -1


def test_norm_refusals(qg):
    lib = qg.lib()

    def call(**kw):
        a = Norm(0, 2, 64, 0, P, P, P, None, None, 0, P, None, 1.0, 1e-6, P, P)
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.qgemm_residual_norm(C.byref(a), None)

    for kw in (dict(kind=2), dict(tokens=-1), dict(width=0), dict(width=60), dict(width=16392), dict(eps=-1.0),
               dict(eps=float("nan")), dict(y=None), dict(residual=None), dict(out=None), dict(h=None), dict(post_bias=P),
               dict(pre_bias=P), dict(gate=P, gate_stride=4), dict(gate=P, gate_stride=-8), dict(y=P + 2), dict(h=P + 8),
               dict(residual=P + 4), dict(kind=1, post=None, post_bias=P), dict(y=None, post=None, pre=None)):
        assert call(**kw) == qg.ERR_INVALID_ARG, kw
    assert call(tokens=0) == qg.OK
    assert lib.qgemm_residual_norm(None, None) == qg.ERR_INVALID_ARG


def test_python_calls_refuse_host_tensors(qg):
    i = torch.zeros(2, dtype=torch.int32)
    x = torch.zeros((2, 8), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        qg.kv_plan(i, i, torch.zeros((2, 3), dtype=torch.int32), i, i[:1], 16, 2)
    with pytest.raises(ValueError, match="GPU"):
        qg.residual_norm(x, x, pre=x[0])
    k = torch.zeros((1, 1, 16, 64), dtype=torch.uint8)
    s = torch.zeros((1, 1), dtype=torch.uint8)
    c = qg.KVCache(qg.KV_E4M3, k, k, s, s)  # a description; the calls check where the rows are
    r = torch.zeros((1, 1, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        qg.kv_append(c, r, r, torch.zeros(1, dtype=torch.int64), i)
    for bad in ((k.float(), k, s, s), (k, k[..., :32], s, s), (k, k, s[0], s), (k, k.mT, s, s), (None, k, s, s)):
        with pytest.raises(ValueError):
            qg.KVCache(qg.KV_E4M3, *bad)
