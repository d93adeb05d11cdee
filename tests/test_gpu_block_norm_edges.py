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
