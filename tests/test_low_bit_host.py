"""CPU tests of the low-bit operators' host side: weight rounding, shapes, refusals
before any GPU is touched, and the integer forms the kernels rely on."""
import pytest
import torch

import ref64
from b200q import block_norm, kv8, w4


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_w4_quantize_layout(symmetric, group):
    g = torch.Generator().manual_seed(group)
    weight = torch.randn(6, 256, generator=g)
    w, s, z = w4.w4_quantize(weight, group, symmetric, torch.float32)
    assert w.shape == (6, 128) and w.dtype == torch.uint8 and s.shape == (6, 256 // group)
    assert (z is None) == symmetric
    codes = ref64.w4_codes(w)
    assert int(codes.min()) >= 0 and int(codes.max()) <= 15
    back = w4.w4_dequantize(w, s, z)
    assert torch.equal(back.double(), ref64.w4_weight(w, s, z).float().double())
    step = s.repeat_interleave(group, 1)
    # half a step, and as much again for a rounded zero point
    assert bool(((back - weight).abs() <= step * (0.501 if symmetric else 1.001)).all())


def test_w4_quantize_edges():
    w, s, z = w4.w4_quantize(torch.zeros(2, 64), 64)
    assert bool((w4.w4_dequantize(w, s, z) == 0).all())
    w, s, z = w4.w4_quantize(torch.full((2, 64), 3.0), 64, symmetric=False)
    assert bool(((w4.w4_dequantize(w, s, z) - 3.0).abs() < 1e-5).all())
    for bad in (torch.zeros(64), torch.zeros(2, 48), torch.zeros(2, 64, dtype=torch.int32)):
        with pytest.raises(RuntimeError):
            w4.w4_quantize(bad, 64)
    with pytest.raises(RuntimeError):
        w4.w4_quantize(torch.zeros(2, 256), 256)


def test_digits_hold_a_value():
    """v = p0 + p1 / 128 + p2 / 128^2 with int8 digits, as the kernels split |v| < 64."""
    g = torch.Generator().manual_seed(0)
    v = (torch.rand(100000, generator=g) * 2 - 1) * 63.99
    m = torch.tensor(12582912.0)
    a = (v + m) - m
    r = (v - a) * 128
    c = (r + m) - m
    e = ((r - c) * 128 + m) - m
    for d in (a, c, e):
        assert float(d.abs().max()) <= 64 and torch.equal(d, d.round())
    back = a.double() + c.double() / 128 + e.double() / 128 ** 2
    assert float((back - v.double()).abs().max()) <= 0.5 / 128 ** 2
    # the low byte of the sum with 1.5 * 2^23 is the digit in two's complement
    low = (v + m).view(torch.int32).to(torch.int8)
    assert torch.equal(low, a.to(torch.int8))


def test_nibbles_in_half_precision():
    """1024 + c and 1024 + 16 c from OR-ed nibbles; minus the zero point, exact."""
    c, z = torch.meshgrid(torch.arange(16), torch.arange(16), indexing="ij")
    low = (0x6400 | c).to(torch.int16).view(torch.float16)
    high = (0x6400 | (c << 4)).to(torch.int16).view(torch.float16)
    z0 = (0x6400 | z).to(torch.int16).view(torch.float16)
    z1 = ((0xD400 | (z << 4)) - 65536).to(torch.int16).view(torch.float16)
    want = (c - z).to(torch.float16)
    assert torch.equal(low - z0, want)
    assert torch.equal((high.float() / 16 + z1.float()).half(), want)


def test_codes_in_half_precision():
    """A sign-flipped byte OR-ed into 1024 is 1152 + code: exact for every code."""
    code = torch.arange(-128, 128)
    h = (0x6400 | ((code & 255) ^ 0x80)).to(torch.int16).view(torch.float16)
    assert torch.equal(h - torch.tensor(1152.0, dtype=torch.float16), code.half())


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    w, s, _ = w4.w4_quantize(torch.randn(8, 64), 64, True, torch.bfloat16)
    pool = (torch.zeros(2, 1, 16, 64, dtype=torch.int8),) * 2 + (torch.zeros(2, 1),) * 2
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    q = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16)
    for call in (lambda: w4.w4a16_linear(x, w, s), lambda: block_norm.norm_modulate(x),
                 lambda: block_norm.gated_residual(x, x),
                 lambda: kv8.kv8_append(q, q, *pool, table, lens),
                 lambda: kv8.kv8_gather(*pool, table, lens, lens, 4),
                 lambda: kv8.kv8_attention(q, *pool, table, lens)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(TypeError):
        w4.w4a16_linear(x, 3, s)


def test_fake_kernels_give_shapes():
    with torch._subclasses.FakeTensorMode():
        x = torch.empty(3, 5, 256, dtype=torch.bfloat16, device="cuda")
        w = torch.empty(96, 128, dtype=torch.uint8, device="cuda")
        s = torch.empty(96, 2, dtype=torch.bfloat16, device="cuda")
        o = torch.ops.b200q.w4a16_linear(x, w, s, None, None, "none", torch.float32)
        assert o.shape == (3, 5, 96) and o.dtype == torch.float32
        q, sc = torch.ops.b200q.norm_modulate_quant_i8(x)
        assert q.shape == (15, 256) and q.dtype == torch.int8 and sc.shape == (15, 1)
        h, n = torch.ops.b200q.gated_residual_norm(x, x)
        assert h.shape == x.shape == n.shape
        c = torch.empty(4, 2, 16, 64, dtype=torch.int8, device="cuda")
        cs = torch.empty(4, 2, device="cuda")
        t = torch.empty(3, 2, dtype=torch.int32, device="cuda")
        ln = torch.empty(3, dtype=torch.int32, device="cuda")
        qq = torch.empty(3, 6, 7, 64, dtype=torch.bfloat16, device="cuda")
        out, lse = torch.ops.b200q.kv8_attention(qq, c, c, cs, cs, t, ln)
        assert out.shape == (3, 6, 7, 64) and lse.shape == (3, 6, 7) and lse.dtype == torch.float32
        k, v = torch.ops.b200q.kv8_gather(c, c, cs, cs, t, ln, ln, 9)
        assert k.shape == v.shape == (3, 2, 9, 64)
