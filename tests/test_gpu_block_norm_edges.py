"""The block norms against the 64-bit form with bounds from the arithmetic, many rows per CTA
on every form, and INT8 codes at ties.

Bounds, u = 2^-24.  Sums over a row go through at most 64 additions one after another (16
values a thread, then trees), so the mean square is within 64 u and its root's reciprocal
within 40 u with rsqrtf's 2 ulp.  With t = |a x| + |gate post(y) w_post| the terms of h, h is
within 48 u t; the second norm's root moves by 48 u k, k = rms(t) / rms(h) (spread(h) for a
layer norm), its mean by 64 u rms(t).  So out is within
    2^-17 r |w (1 + scale)| (t (1 + k) + rms(t)) + 2^-22 |shift|,  r = 1 / rms(h) or 1 / spread(h)
of the formula, and rounded once.  A second norm that took the rounded h would be off by 2^-9
of h, far more than that: INT8 row scales, which are fp32, would show it.
"""
import pytest
import torch

import ref64
from b200q import block_norm as bn

pytestmark = pytest.mark.gpu
DEV = "cuda"


def d(t):
    return None if t is None else t.to(DEV)


def make(rows, D, dtype, B, mod_dtype, seed):
    g = torch.Generator().manual_seed(seed)

    def r(*s):
        return torch.randn(*s, generator=g)

    return dict(x=(r(rows, D) * 3).to(dtype), y=r(rows, D).to(dtype), gate=r(B, D).to(mod_dtype),
                scale=(r(B, D) * 0.3).to(mod_dtype), shift=r(B, D).to(mod_dtype), weight=1 + 0.2 * r(D),
                post_weight=1 + 0.2 * r(D))


def reference(a, post_kind, kind, after, res=0.7, eps=1e-6):
    """(h, out, bound of out's fp32 error) in 64 bits."""
    rows, D = a["x"].shape

    def per_row(t):
        return t.double().repeat_interleave(rows // t.shape[0], 0)

    if after:
        h, out = ref64.block_norm(a["x"], a["y"], a["gate"], a["post_weight"], post_kind, res, a["weight"],
                                  a["scale"], a["shift"], kind, eps)
        t = (res * a["x"].double()).abs() + (h - res * a["x"].double()).abs()
    else:
        h, out = ref64.block_norm(a["x"], weight=a["weight"], scale=a["scale"], shift=a["shift"], kind=kind, eps=eps)
        t = h.abs()
    c = h - h.mean(-1, keepdim=True) if kind == "layer" else h
    r = 1 / ((c * c).mean(-1, keepdim=True) + eps).sqrt()
    rms_t = (t * t).mean(-1, keepdim=True).sqrt()
    k = rms_t * r
    w = (a["weight"].double() * (1 + per_row(a["scale"]))).abs()
    return h, out, 2.0 ** -17 * r * w * (t * (1 + k) + rms_t) + 2.0 ** -22 * per_row(a["shift"]).abs()


def run(a, post_kind, kind, after, quant, x=None, y=None, res=0.7):
    x, y = d(a["x"]) if x is None else x, d(a["y"]) if y is None else y
    pre = (d(a["weight"]), d(a["scale"]), d(a["shift"]), kind, 1e-6)
    if not after:
        return (None, *(bn.norm_modulate_quant_i8(x, *pre) if quant else (bn.norm_modulate(x, *pre),)))
    f = bn.gated_residual_norm_quant_i8 if quant else bn.gated_residual_norm
    return f(x, y, d(a["gate"]), d(a["post_weight"]), post_kind, res, *pre)


def compare(a, got, post_kind, kind, after, quant):
    h_ref, ref, tol = reference(a, post_kind, kind, after)
    if after:
        t = 0.7 * a["x"].double().abs() + (h_ref - 0.7 * a["x"].double()).abs()
        err = (got[0].double().cpu() - h_ref).abs()
        assert bool((err <= ref64.UNIT[a["x"].dtype] * h_ref.abs() + 48 * 2.0 ** -24 * t + 1e-7).all())
    if not quant:
        out = got[1].double().cpu()
        full = ref64.UNIT[a["x"].dtype] * ref.abs() + tol * 1.01 + 2.0 ** -25
        assert bool(((out - ref).abs() <= full).all()), f"worst {((out - ref).abs() / full).max().item():.3g}"
        return
    q, s = got[1].double().cpu(), got[2].double().cpu()
    top = ref.abs().amax(-1, keepdim=True)
    s_tol = tol.amax(-1, keepdim=True) / 127 + 2.0 ** -23 * top / 127
    assert bool(((s - top / 127).abs() <= s_tol).all())
    # the code is the nearest integer of a quotient of values this near to the reference's
    near = (tol + 127 * s_tol) / (top / 127) + 2.0 ** -16
    assert bool(((q - ref / (top / 127)).abs() <= 0.5 + near).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,B,D", [(3, 3, 5120), (3000, 3, 1024), (2997, 3, 1486), (2001, 3, 783), (900, 9, 5120),
                                      (4, 2, 9000)])
@pytest.mark.parametrize("post_kind,kind", [("rms", "layer"), ("layer", "rms"), ("none", "layer")])
@pytest.mark.parametrize("quant", [False, True])
def test_many_rows_and_modulations(native, dtype, rows, B, D, post_kind, kind, quant):
    """A CTA's rows meet another modulation in the middle; aligned rows, pairs, single values."""
    a = make(rows, D, dtype, B, torch.float32, D + rows)
    for after in (True, False):
        compare(a, run(a, post_kind, kind, after, quant), post_kind, kind, after, quant)


@pytest.mark.parametrize("D,off", [(1024, 2), (1024, 1), (1025, 0)])
@pytest.mark.parametrize("quant", [False, True])
def test_many_rows_of_views(native, D, off, quant):
    """Rows on pairs but not on 16 bytes, and on single values, thousands of them."""
    a = make(2400, D, torch.bfloat16, 3, torch.bfloat16, off)
    wide = torch.zeros(2400, D + 8, dtype=torch.bfloat16, device=DEV)
    wide[:, off:off + D] = d(a["x"])
    got = run(a, "rms", "layer", True, quant, x=wide[:, off:off + D])
    compare(a, got, "rms", "layer", True, quant)


# rows x D on each form: one row per CTA, persistent, pairs, single values, past 8192
FORMS = [(4, 512), (1500, 512), (1500, 510), (700, 511), (4, 510), (3, 9001)]


@pytest.mark.parametrize("rows,D", FORMS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_codes_at_ties(native, rows, D, dtype):
    """Half of the row's largest value is code 63.5, an exact tie: the code is what the
    rounded quotient gives, 64, for any largest value."""
    x = torch.zeros(rows, D)
    top = 1 + torch.arange(rows) % 128 / 128
    x[:, 0] = top
    x[:, 1], x[:, 2] = top / 2, -top / 2
    x[:, 3:9] = top[:, None] * torch.tensor([1 / 8, 3 / 8, -1 / 4, 7 / 8, 1 / 16, -5 / 16])
    x = x.to(dtype)
    q, s = bn.norm_modulate_quant_i8(d(x), kind="none")
    s_ref = x.float().abs().amax(-1, keepdim=True) / torch.tensor(127.0)
    assert torch.equal(s.cpu(), s_ref)
    assert torch.equal(q.cpu(), (x.float() / s_ref).round().to(torch.int8))


@pytest.mark.parametrize("rows,D", FORMS)
@pytest.mark.parametrize("power", [-100, -124, -130])
def test_codes_of_vanishing_rows(native, rows, D, power):
    """Rows so small that 1 / scale is not finite."""
    g = torch.Generator().manual_seed(D)
    x = ((torch.rand(rows, D, generator=g) * 2 - 1) * 2.0 ** -60).mul(2.0 ** (power + 60)).to(torch.bfloat16)
    q, s = bn.norm_modulate_quant_i8(d(x), kind="none")
    s_ref = x.float().abs().amax(-1, keepdim=True) / torch.tensor(127.0)
    assert torch.equal(s.cpu(), s_ref)
    ref = x.double() / s_ref.double()
    assert bool(((q.cpu().double() - ref).abs() <= 0.5 + 2.0 ** -16).all())
