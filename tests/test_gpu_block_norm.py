"""The norms before and after a block on the GPU against the 64-bit form.

Bounds: one rounding of the output, plus fp32 arithmetic: a handful of operations
on values of at most the row's size and a sum over D (pairwise over threads), held
here to 2^-18 of the size of the terms that meet in the value.  INT8 codes are
within half a step of out / scale, with the same 2^-18 of the code range.
"""
import pytest
import torch

import ref64
from b200q import block_norm as bn

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(rows, D, dtype, B=1, mod_dtype=torch.float32, seed=0, mean=0.0):
    g = torch.Generator().manual_seed(seed)

    def r(*s):
        return torch.randn(*s, generator=g)

    return dict(x=(r(rows, D) * 3 + mean).to(dtype), y=(r(rows, D) + mean).to(dtype),
                gate=r(B, D).to(mod_dtype), scale=(r(B, D) * 0.3).to(mod_dtype),
                shift=r(B, D).to(mod_dtype), weight=1 + 0.2 * r(D), post_weight=1 + 0.2 * r(D))


def d(t):
    return None if t is None else t.to(DEV)


def close(out, ref, size):
    tol = ref64.UNIT[out.dtype] * ref.abs() + 2.0 ** -18 * size + 1e-7
    err = (out.double().cpu().reshape(ref.shape) - ref).abs()
    assert bool((err <= tol).all()), f"worst {(err / tol).max().item():.3g} of the bound"


def sizes(a, h_ref, out_ref, kind, post_kind):
    """The largest term that meets in each value: the row's largest entries."""
    size_h = (a["x"].double().abs().amax(-1, keepdim=True) + 1
              + 8 * a["gate"].double().abs().max() * a["y"].double().abs().amax(-1, keepdim=True))
    spread = h_ref.std(-1, unbiased=False, keepdim=True)
    rms = (h_ref * h_ref).mean(-1, keepdim=True).sqrt()
    amplify = size_h / (spread if kind == "layer" else rms).clamp(min=1e-3)
    return size_h, 8 * amplify * out_ref.abs().amax(-1, keepdim=True).clamp(min=1.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("post_kind", ["none", "rms", "layer"])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows,B,D", [(1, 1, 5120), (6, 3, 1), (10, 2, 33), (9, 9, 512), (14, 7, 4104),
                                      (4, 1, 8200), (2, 2, 32768), (3, 1, 32767)])
def test_after_and_before(native, dtype, post_kind, kind, rows, B, D):
    a = make(rows, D, dtype, B, dtype if D % 2 else torch.float32, seed=D)
    pw = None if post_kind == "none" else a["post_weight"]
    args = (a["gate"], pw, post_kind, 0.7, a["weight"], a["scale"], a["shift"], kind, 1e-6)
    h, out = bn.gated_residual_norm(d(a["x"]), d(a["y"]), *(d(t) if torch.is_tensor(t) else t for t in args))
    h_ref, out_ref = ref64.block_norm(a["x"], a["y"], *args)
    size_h, size_o = sizes(a, h_ref, out_ref, kind, post_kind)
    close(h, h_ref, size_h)
    if D > 1:
        close(out, out_ref, size_o)
    only = bn.gated_residual(d(a["x"]), d(a["y"]), d(a["gate"]), d(pw), post_kind, 0.7)
    assert torch.equal(only, h)


@pytest.mark.parametrize("kind", ["rms", "layer", "none"])
@pytest.mark.parametrize("D", [512, 1000, 5121])
def test_before_only_and_optional_operands(native, kind, D):
    a = make(5, D, torch.bfloat16)
    for w, sc, sh in ((None, None, None), (a["weight"], None, a["shift"]), (None, a["scale"], None)):
        out = bn.norm_modulate(d(a["x"]), d(w), d(sc), d(sh), kind, 1e-5)
        _, ref = ref64.block_norm(a["x"], weight=w, scale=sc, shift=sh, kind=kind, eps=1e-5)
        _, size = sizes(a, a["x"].double(), ref, kind, "none")
        close(out, ref, size)


def test_large_mean_layer_norm(native):
    """A mean far above the spread: the centred variance keeps its digits."""
    a = make(4, 4096, torch.float16, mean=300.0)
    out = bn.norm_modulate(d(a["x"]), kind="layer")
    _, ref = ref64.block_norm(a["x"], kind="layer")
    # x - mean carries 2^-24 of the mean, divided by the spread of 3
    tol = 2.0 ** -11 * ref.abs() + 4 * 300 / 3 * 2.0 ** -22
    assert bool(((out.double().cpu() - ref).abs() <= tol).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,B,D", [(7, 1, 1536), (12, 4, 259), (3, 1, 13824)])
@pytest.mark.parametrize("after", [False, True])
def test_int8_codes(native, dtype, rows, B, D, after):
    a = make(rows, D, dtype, B, seed=rows)
    if after:
        args = (a["gate"], a["post_weight"], "rms", 1.0, a["weight"], a["scale"], a["shift"], "layer")
        h, q, s = bn.gated_residual_norm_quant_i8(d(a["x"]), d(a["y"]), *(d(t) if torch.is_tensor(t) else t for t in args))
        h_ref, ref = ref64.block_norm(a["x"], a["y"], *args)
        assert torch.equal(h, bn.gated_residual(d(a["x"]), d(a["y"]), *(d(t) if torch.is_tensor(t) else t for t in args[:4])))
    else:
        q, s = bn.norm_modulate_quant_i8(d(a["x"]), d(a["weight"]), d(a["scale"]), d(a["shift"]), "layer")
        h_ref, ref = ref64.block_norm(a["x"], weight=a["weight"], scale=a["scale"], shift=a["shift"], kind="layer")
    assert q.shape == (rows, D) and q.dtype == torch.int8 and s.shape == (rows, 1)
    s_ref = ref.abs().amax(-1, keepdim=True) / 127
    amplify = (sizes(a, h_ref, ref, "layer", "rms")[0] / h_ref.std(-1, unbiased=False, keepdim=True)).max()
    rel = 8 * float(amplify) * 2.0 ** -18
    assert bool(((s.double().cpu() - s_ref).abs() <= rel * s_ref).all())
    assert bool(((q.double().cpu() - ref / s_ref).abs() <= 0.5 + 2 * 127 * rel).all())
    assert int(q.cpu().abs().max()) == 127


def test_codes_feed_the_int8_linear(native):
    """norm -> INT8 linear: the codes are what i8_matmul_nt_fused_cs takes."""
    a = make(40, 512, torch.bfloat16)
    q, s = bn.norm_modulate_quant_i8(d(a["x"]), d(a["weight"]))
    g = torch.Generator().manual_seed(5)
    w = torch.randint(-127, 128, (96, 512), generator=g, dtype=torch.int8)
    ws = torch.rand(96, generator=g) * 0.01
    out = native.i8_matmul_nt_fused_cs(q, d(w), s, d(ws))
    ref = (q.cpu().double() * s.cpu().double()) @ (w.double() * ws.double()[:, None]).t()
    assert bool(((out.double().cpu() - ref).abs() <= 2.0 ** -8 * ref.abs() + 1e-5).all())


def test_zero_and_nonfinite_rows(native):
    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    x[1], x[2, 5], x[3, 9] = 1.0, float("inf"), float("nan")
    out = bn.norm_modulate(x.to(DEV), eps=1e-6).cpu()
    assert bool((out[0] == 0).all()) and bool((out[1] == 1).all())
    assert bool(out[3].isnan().all())
    q, s = bn.norm_modulate_quant_i8(x.to(DEV))
    assert s[0].item() == 0 and bool((q[0] == 0).all()) and bool((q[1] == 127).all())
    assert bool(s[2:].isnan().all())


def test_strides_and_unaligned_rows(native):
    """Chunks of one [B, 6, D] modulation, x as a slice of a wider buffer, and
    operands off 16-byte boundaries give what contiguous ones do."""
    a = make(8, 520, torch.bfloat16, 2)
    ref = bn.gated_residual_norm(d(a["x"]), d(a["y"]), d(a["gate"]), None, "none", 1.0, d(a["weight"]),
                                 d(a["scale"]), d(a["shift"]), "layer")
    mods = torch.zeros(2, 6, 520)
    mods[:, 1], mods[:, 3], mods[:, 4] = a["gate"], a["scale"], a["shift"]
    m = mods.to(DEV)
    for off in (8, 3):
        wide = torch.zeros(8, 560, dtype=torch.bfloat16, device=DEV)
        wide[:, off:off + 520] = d(a["x"])
        got = bn.gated_residual_norm(wide[:, off:off + 520].view(8, 520) if off == 0 else wide[:, off:off + 520],
                                     d(a["y"]), m[:, 1], None, "none", 1.0, d(a["weight"]), m[:, 3], m[:, 4], "layer")
        for x, y, u in zip(got, ref, (0, 1)):
            # the element order of the sums differs between the two forms
            assert bool(((x.double() - y.double()).abs() <= 2.0 ** -7 * y.double().abs() + 2.0 ** -14).all())
    b3 = bn.norm_modulate(d(a["x"]).view(2, 4, 520), None, m[:, 3], m[:, 4])
    assert torch.equal(b3.view(8, 520), bn.norm_modulate(d(a["x"]), None, d(a["scale"]), d(a["shift"])))
    one = bn.norm_modulate(d(a["x"]), None, d(a["scale"][0]))
    assert torch.equal(one, bn.norm_modulate(d(a["x"]), None, d(a["scale"][:1])))


def test_many_rows_streams_and_ops(native):
    a = make(3001, 1024, torch.bfloat16)
    x, y = d(a["x"]), d(a["y"])
    h, out = bn.gated_residual_norm(x, y, d(a["gate"]))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        h2, out2 = torch.ops.b200q.gated_residual_norm(x, y, d(a["gate"]))
    side.synchronize()
    assert torch.equal(h, h2) and torch.equal(out, out2)
    h_ref, ref = ref64.block_norm(a["x"], a["y"], a["gate"])
    sh, so = sizes(a, h_ref, ref, "rms", "none")
    close(h, h_ref, sh)
    close(out, ref, so)
    assert bn.norm_modulate(x[:0]).shape == (0, 1024)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("post_kind", ["none", "layer"])
def test_rows_of_a_persistent_cta_stay_apart(native, quant, post_kind):
    """Tens of thousands of rows of very different sizes through persistent CTAs: each
    equals the same row computed alone, every time."""
    g = torch.Generator().manual_seed(11)
    rows, D = 30000, 1024
    size = torch.logspace(-2, 2, 97)[torch.randint(0, 97, (rows,), generator=g)][:, None]
    x = (torch.randn(rows, D, generator=g) * size).to(torch.bfloat16).to(DEV)
    y = (torch.randn(rows, D, generator=g) * size.flip(0)).to(torch.bfloat16).to(DEV)
    f = bn.gated_residual_norm_quant_i8 if quant else bn.gated_residual_norm
    args = (None, None, post_kind, 1.0, None, None, None, "layer")
    got = f(x, y, *args)
    # a few rows at a time: the form of one row per CTA
    pick = torch.arange(0, rows, 101)
    alone = [torch.cat(t) for t in zip(*(f(x[p], y[p], *args) for p in pick.split(200)))]
    for a, b in zip(got, alone):
        if a.dtype == torch.int8:
            assert int((a[pick].int() - b.int()).abs().max()) <= 1
        else:  # the sums' order differs between the forms
            assert bool(((a[pick].double() - b.double()).abs()
                         <= 2.0 ** -7 * b.double().abs() + 2.0 ** -13 * size.to(DEV)[pick]).all())
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(got, f(x, y, *args)))


def test_refusals(native):
    a = make(6, 64, torch.bfloat16, 2)
    x, y, g, w = d(a["x"]), d(a["y"]), d(a["gate"]), d(a["weight"])
    bad = [
        lambda: bn.norm_modulate(x.float()), lambda: bn.norm_modulate(x, kind="batch"),
        lambda: bn.norm_modulate(x.cpu()), lambda: bn.norm_modulate(x, w[:32]),
        lambda: bn.norm_modulate(x, w.double()), lambda: bn.norm_modulate(x, None, g[:, :32]),
        lambda: bn.norm_modulate(x[:5], None, g), lambda: bn.norm_modulate(x, None, g, g[:1]),
        lambda: bn.norm_modulate(x, None, g, g.bfloat16()), lambda: bn.norm_modulate(x, None, g.cpu()),
        lambda: bn.gated_residual(x, y[:3]), lambda: bn.gated_residual(x, y.half()),
        lambda: bn.norm_modulate(torch.zeros(2, 32769, dtype=torch.bfloat16, device=DEV)),
    ]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
