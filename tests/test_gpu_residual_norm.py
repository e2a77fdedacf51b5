"""residual_norm against a 64-bit restatement (tests/serving_ref.py).

Bounds.  A row's sums run over at most 32 values in a thread, 5 shuffles and
16 warps: 53 additions of 2^-24 each; with the square root, the division and
the products the scaling factor is within 2^-17.  Centring a row leaves each
value off by 2^-17 of the row's largest value, which the norm divides by the
row's spread.  So N is off by 2^-17 (|N| + |w| max|x| / spread), the stream by
alpha |gate| times that plus 2^-22 (|r| + alpha |gate N|), and h by the same
rule again, with the stream's own error over its spread; bf16 (8
significant bits) adds 2^-8 of the value.
"""
import pytest
import serving_ref as R
import torch

pytestmark = pytest.mark.gpu


def spread(x, kind, eps):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    return torch.sqrt((x * x).mean(-1, keepdim=True) + eps)


def norm_tol(x, x_err, n, w, kind, eps):
    s = spread(x, kind, eps)
    return 2.0 ** -17 * (n.abs() + w.double().abs() * x.abs().amax(-1, keepdim=True) / s) + \
        2 * (w.double().abs() + n.abs()) * x_err.amax(-1, keepdim=True) / s


def check(qg, tokens, width, kind, gate, f32, post=True, pre=True, bias=False, y=True, alpha=0.7, eps=1e-5, seed=0,
          mean=0.1, inplace=False):
    g = torch.Generator(device="cuda").manual_seed(seed + width)

    def rand(*shape, scale=1.0, mean=0.0, dtype=torch.bfloat16):
        return (torch.randn(shape, generator=g, device="cuda") * scale + mean).to(dtype)

    yy = rand(tokens, width, scale=3, mean=mean) if y else None
    r = rand(tokens, width, scale=5, mean=mean, dtype=torch.float32 if f32 else torch.bfloat16)
    wpost = rand(width, scale=0.2, mean=1) if post and y else None
    wpre = rand(width, scale=0.2, mean=1) if pre else None
    bpost = rand(width) if bias and wpost is not None else None
    bpre = rand(width) if bias and wpre is not None else None
    gt = {"none": None, "shared": lambda: rand(width), "token": lambda: rand(tokens, width),
          "strided": lambda: rand(tokens, 3 * width)[:, width:2 * width]}[gate]
    gt = gt() if gt else None
    want_r, want_h = R.residual_norm(yy, r, wpost, wpre, bpost, bpre, gt, alpha, kind, eps)
    r0 = r.clone()
    kw = {"residual_out": r, "h": yy} if inplace else {}
    yd = yy.double() if y else None
    got_r, got_h = qg.residual_norm(yy, r, post=wpost, pre=wpre, post_bias=bpost, pre_bias=bpre, gate=gt, alpha=alpha,
                                    kind=kind, eps=eps, **kw)
    err = torch.zeros_like(want_r)
    if y:
        z = yd
        zerr = torch.zeros_like(z)
        if post:
            z = R.norm(yd, wpost, bpost, kind, eps)
            zerr = norm_tol(yd, zerr, z, wpost, kind, eps)
        f = abs(alpha) * (gt.double().abs() if gt is not None else 1.0)
        err = f * zerr + 2.0 ** -22 * (r0.double().abs() + f * z.abs())
        tol_r = err + (0 if f32 else 2.0 ** -8 * (want_r.abs() + err))
        assert ((got_r.double() - want_r).abs() <= tol_r).all()
    else:
        assert torch.equal(got_r, r0)
    if pre:
        tol = norm_tol(want_r, err, want_h, wpre, kind, eps)
        tol = tol + 2.0 ** -8 * (want_h.abs() + tol)
        assert ((got_h.double() - want_h).abs() <= tol).all()
    else:
        assert got_h is None


@pytest.mark.parametrize("tokens,width", [(1, 8), (1, 8192), (3, 16384), (5, 64), (33, 264), (7, 2880), (300, 4096),
                                          (1000, 248), (2, 8200), (149, 1000)])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_sizes(qg, cuda, tokens, width, kind):
    check(qg, tokens, width, kind, "none", False)
    check(qg, tokens, width, kind, "token", True, bias=kind == "layer", seed=1)


@pytest.mark.parametrize("gate", ["none", "shared", "token", "strided"])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("post,pre", [(True, True), (True, False), (False, True), (False, False)])
def test_parts(qg, cuda, gate, f32, post, pre):
    for kind in ("rms", "layer"):
        check(qg, 11, 520, kind, gate, f32, post=post, pre=pre, bias=kind == "layer")
        check(qg, 11, 520, kind, gate, f32, post=post, pre=pre, alpha=-1.5, inplace=True)


@pytest.mark.parametrize("f32", [False, True])
def test_first_block_norms_the_stream_only(qg, cuda, f32):
    for kind in ("rms", "layer"):
        check(qg, 9, 2880, kind, "none", f32, y=False)


def test_large_mean_and_zero_rows(qg, cuda):
    check(qg, 5, 4096, "layer", "none", True, mean=100.0)
    check(qg, 5, 4096, "rms", "none", True, mean=100.0)
    w = torch.ones(512, dtype=torch.bfloat16, device="cuda")
    z = torch.zeros((2, 512), dtype=torch.bfloat16, device="cuda")
    for kind in ("rms", "layer"):
        r, h = qg.residual_norm(z, z, post=w, pre=w, kind=kind)
        assert (r == 0).all() and (h == 0).all()


def test_rows_are_independent(qg, cuda):
    w = torch.ones(1024, dtype=torch.bfloat16, device="cuda")
    y = torch.randn((40, 1024), device="cuda").to(torch.bfloat16)
    r, h = qg.residual_norm(y, y, post=w, pre=w)
    bad = y.clone()
    bad[7, 3], bad[20, 5] = float("nan"), float("inf")
    r2, h2 = qg.residual_norm(bad, y, post=w, pre=w)
    keep = [i for i in range(40) if i not in (7, 20)]
    assert torch.equal(h2[keep], h[keep]) and h2[7].isnan().all() and h2[20].isnan().any()


def test_refusals(qg, cuda):
    def t(*s, dtype=torch.bfloat16):
        return torch.zeros(s, dtype=dtype, device="cuda")

    y, w = t(2, 64), t(64)
    for kw in (dict(kind="group"), dict(post_bias=w), dict(post=w, post_bias=w), dict(post=t(32)), dict(gate=t(3, 64)),
               dict(gate=w.float()), dict(eps=-1.0), dict(eps=float("nan"))):
        with pytest.raises(ValueError):
            qg.residual_norm(y, y, pre=w, **kw)
    for a, b in ((t(2, 60), t(2, 60)), (t(2, 16392), t(2, 16392)), (y, t(3, 64)), (y.float(), y), (None, y),
                 (t(2, 128)[:, ::2], y)):
        with pytest.raises(ValueError):
            qg.residual_norm(a, b)
    with pytest.raises(ValueError):
        qg.residual_norm(None, y, pre=w, gate=w)
    with pytest.raises(ValueError, match="16-byte"):
        qg.residual_norm(torch.zeros(132, dtype=torch.bfloat16, device="cuda")[4:].view(2, 64), y)
    r, h = qg.residual_norm(t(0, 64), t(0, 64), pre=w)
    assert r.shape == h.shape == (0, 64)
