"""4-bit weight linears on the GPU against the 64-bit form.

Bounds, from the arithmetic alone: c - z and every product's operands are exact,
so a call of up to 32 tokens is off by its fp32 sums (2^-17 of sum |x||W| covers
K = 5120 additions in any order) and one output rounding; larger calls round each
weight to fp16 once (2^-11 of sum |x||W| at worst).  GELU's slope stays below 1.13.
"""
import pytest
import torch

import ref64
from b200q import w4

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(M, N, K, G, dtype, zeros, bias=False, scale_dtype=None, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g).to(dtype)
    w = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8)
    s = (torch.rand(N, K // G, generator=g) * 0.02 * spread + 1e-3).to(scale_dtype or dtype)
    z = torch.randint(0, 16, (N, K // G), generator=g, dtype=torch.uint8) if zeros else None
    b = torch.randn(N, generator=g).to(dtype) if bias else None
    return x, w, s, z, b


def dev(*ts):
    return tuple(None if t is None else t.to(DEV) for t in ts)


def check(out, x, w, s, z, b, act=None):
    ref, size = ref64.w4_linear(x, w, s, z, b, act)
    u = ref64.UNIT[out.dtype]
    tol = u * ref.abs() + 1.13 * size * (2.0 ** -17 + (2.0 ** -11 if x.shape[0] > 32 else 0)) + 1e-7
    err = (out.double().cpu() - ref).abs()
    assert bool((err <= tol).all()), f"worst {(err / tol).max().item():.3g} of the bound"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("M", [1, 3, 8, 9, 16, 17, 32, 33, 130])
def test_tokens_groups_types(native, dtype, G, zeros, M):
    x, w, s, z, b = make(M, 200, 1152, G, dtype, zeros, bias=True, seed=M + G)
    out = w4.w4a16_linear(*dev(x, w, s, z, b))
    assert out.dtype == dtype and out.shape == (M, 200)
    check(out, x, w, s, z, b)


@pytest.mark.parametrize("M,N,K,G", [(1, 1, 32, 32), (1, 17, 128, 128), (2, 5120, 5120, 128),
                                     (1, 1000, 13824, 64), (16, 515, 13824, 128), (5, 33, 96, 32),
                                     (300, 129, 160, 32), (257, 640, 2048, 128), (32, 64, 20480, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_shapes(native, M, N, K, G, dtype):
    x, w, s, z, b = make(M, N, K, G, dtype, True, seed=N)
    check(w4.w4a16_linear(*dev(x, w, s, z)), x, w, s, z, b)


@pytest.mark.parametrize("M,N,K,G", [(33, 131, 32, 32), (64, 128, 256, 128), (65, 1001, 544, 32), (128, 5120, 5120, 64),
                                     (129, 257, 5120, 128), (256, 1046, 1312, 32), (200, 515, 13824, 64),
                                     (700, 1131, 1536, 128)])
@pytest.mark.parametrize("scale_dtype", [torch.bfloat16, torch.float32])
def test_tiles_of_tokens(native, M, N, K, G, scale_dtype):
    """Tile edges in every direction; fp32 scales keep their bits; the same bits each time."""
    x, w, s, z, b = make(M, N, K, G, torch.bfloat16, True, bias=True, scale_dtype=scale_dtype, seed=M)
    d = dev(x, w, s, z, b)
    native.device_status(reset=True)
    out = w4.w4a16_linear(*d, "gelu_tanh")
    check(out, x, w, s, z, b, "gelu_tanh")
    for _ in range(20):
        assert torch.equal(w4.w4a16_linear(*d, "gelu_tanh"), out)
    assert native.device_status() == 0


@pytest.mark.parametrize("M", [50, 150])
def test_scales_far_apart_in_a_row(native, M):
    """Each group's weights keep their own bits next to groups 2^12 larger."""
    x, w, s, z, b = make(M, 48, 512, 64, torch.bfloat16, True, scale_dtype=torch.float32)
    s = s * torch.logspace(-12, 0, 8, base=2)
    x[:, 64:] = 0  # only the smallest group counts
    check(w4.w4a16_linear(*dev(x, w, s, z)), x, w, s, z, b)


@pytest.mark.parametrize("M", [4, 64])
@pytest.mark.parametrize("act", ["gelu_tanh", "gelu"])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_activations_and_out_types(native, M, act, out_dtype):
    x, w, s, z, b = make(M, 96, 512, 64, torch.bfloat16, False, bias=True, seed=3)
    out = w4.w4a16_linear(*dev(x, w, s, z, b), act, out_dtype)
    assert out.dtype == out_dtype
    check(out, x, w, s, z, b, act)


@pytest.mark.parametrize("scale_dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M", [2, 40])
def test_scale_types(native, scale_dtype, M):
    x, w, s, z, b = make(M, 64, 256, 64, torch.float16, True, scale_dtype=scale_dtype)
    check(w4.w4a16_linear(*dev(x, w, s, z)), x, w, s, z, b)


@pytest.mark.parametrize("M", [3, 48])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_strided_operands(native, M, dtype):
    """x as a slice whose rows are not 16-byte aligned, w as rows of a wider buffer."""
    x, w, s, z, b = make(M, 70, 512, 64, dtype, True)
    wide = torch.zeros(M, 520, dtype=dtype)
    wide[:, 3:515] = x
    wbig = torch.zeros(70, 512, dtype=torch.uint8)
    wbig[:, :256] = w
    xd, wd = wide.to(DEV)[:, 3:515], wbig.to(DEV)[:, :256]
    check(w4.w4a16_linear(xd, wd, *dev(s, z)), x, w, s, z, b)
    # a batch axis and a non-unit inner stride
    out = w4.w4a16_linear(x.t().contiguous().to(DEV).t().unsqueeze(0), *dev(w, s, z))
    assert out.shape == (1, M, 70)
    check(out[0], x, w, s, z, b)


@pytest.mark.parametrize("M", [1, 40])
@pytest.mark.parametrize("power", [-20, 20])
def test_extreme_magnitudes(native, M, power):
    """Scales and activations far from 1: neither route leaves its range."""
    x, w, s, z, b = make(M, 48, 256, 64, torch.bfloat16, True, scale_dtype=torch.float32)
    s = s * 2.0 ** power
    x = (x.float() * 2.0 ** (2 * power)).to(torch.bfloat16)
    out = w4.w4a16_linear(*dev(x, w, s, z), None, None, torch.float32)
    ref, size = ref64.w4_linear(x, w, s, z)
    tol = 2.0 ** -24 * ref.abs() + size * (2.0 ** -17 + (2.0 ** -11 if M > 32 else 0))
    assert bool(((out.double().cpu() - ref).abs() <= tol).all())


@pytest.mark.parametrize("M", [2, 40])
def test_nonfinite_rows_stay_theirs(native, M):
    x, w, s, z, b = make(M, 64, 256, 64, torch.bfloat16, False)
    bad = x.clone()
    bad[1, 7] = float("nan")
    out = w4.w4a16_linear(*dev(bad, w, s))
    assert bool(out[1].isnan().all())
    clean = w4.w4a16_linear(*dev(x, w, s))
    keep = [i for i in range(M) if i != 1]
    assert torch.equal(out[keep], clean[keep])


def test_zero_tokens_and_zero_scales(native):
    x, w, s, z, b = make(2, 64, 256, 64, torch.bfloat16, False, bias=True)
    assert w4.w4a16_linear(x[:0].to(DEV), *dev(w, s)).shape == (0, 64)
    for M in (2, 40):
        x = torch.ones(M, 256, dtype=torch.bfloat16)
        out = w4.w4a16_linear(x.to(DEV), w.to(DEV), torch.zeros_like(s).to(DEV), None, b.to(DEV))
        assert torch.equal(out.cpu(), b.expand(M, 64))


@pytest.mark.parametrize("M", [1, 16, 64])
def test_repeatable_and_on_another_stream(native, M):
    x, w, s, z, b = dev(*make(M, 1024, 2048, 128, torch.bfloat16, True))
    first = w4.w4a16_linear(x, w, s, z)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = [w4.w4a16_linear(x, w, s, z) for _ in range(3)]
    side.synchronize()
    assert all(torch.equal(first, a) for a in again)
    assert torch.equal(first, torch.ops.b200q.w4a16_linear(x, w, s, z))


def test_cuda_graph(native):
    x, w, s, z, b = dev(*make(2, 512, 1024, 64, torch.bfloat16, False))
    w4.w4a16_linear(x, w, s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = w4.w4a16_linear(x, w, s)
    x.mul_(2)
    graph.replay()
    assert torch.equal(out, w4.w4a16_linear(x, w, s))


def test_quantize_round_trip(native):
    g = torch.Generator().manual_seed(1)
    weight = torch.randn(80, 256, generator=g)
    for sym in (True, False):
        w, s, z = w4.w4_quantize(weight.to(DEV), 64, sym, torch.bfloat16)
        back = w4.w4_dequantize(w, s, z).cpu()
        step = s.float().cpu().repeat_interleave(64, 1)
        # half a step; the scale's own rounding to 8 bits moves up to 15 steps by 2^-8;
        # a rounded zero point can shift the range by another half
        assert bool(((back - weight).abs() <= step * (0.5 + 15 / 256 + (0 if sym else 0.5))).all())
        x = torch.randn(2, 256, generator=g).to(torch.bfloat16)
        check(w4.w4a16_linear(x.to(DEV), w, s, z), x, *(None if t is None else t.cpu() for t in (w, s, z)), None)


def test_refusals(native):
    x, w, s, z, b = dev(*make(2, 64, 256, 64, torch.bfloat16, True, bias=True))
    f = w4.w4a16_linear
    bad = [
        lambda: f(x.float(), w, s), lambda: f(x, w.to(torch.int8), s), lambda: f(x[:, :128], w, s),
        lambda: f(x, w, s[:, :3].contiguous()), lambda: f(x, w, s.t()), lambda: f(x, w, s.double()),
        lambda: f(x, w, s, z.int()), lambda: f(x, w, s, z[:32]), lambda: f(x, w, s, z, b[:5]),
        lambda: f(x, w, s, z, b, "relu"), lambda: f(x, w, s, z, b, None, torch.int8),
        lambda: f(x, w.cpu(), s), lambda: f(x.cpu(), w.cpu(), s.cpu()),
        lambda: f(x, w.reshape(-1)[8:8 + 63 * 128].reshape(63, 128), s[:63].contiguous()),
        lambda: f(x, w, s[:, :1].contiguous()),  # one group of 256
    ]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
    L = native.lib()
    out = torch.empty(40, 64, dtype=torch.bfloat16, device=DEV)
    x40 = torch.zeros(40, 256, dtype=torch.bfloat16, device=DEV)

    def abi(M=2, N=64, K=256, G=64, ldw=128, sdt=1, odt=0, xdt=0, wp=None, ws=0, wsb=0, xx=x):
        return L.b200q_w4a16_linear(xx.data_ptr(), xdt, 256, w.data_ptr() if wp is None else wp, ldw,
                                    s.data_ptr(), sdt, 0, G, 0, 0, 0, out.data_ptr(), odt, N, M, N, K,
                                    ws, wsb, torch.cuda.current_stream().cuda_stream)

    assert abi() == 0
    for kw in (dict(G=16), dict(G=256), dict(K=250), dict(ldw=120), dict(sdt=0), dict(odt=3),
               dict(xdt=2), dict(M=-1), dict(wp=0), dict(wp=w.data_ptr() + 4), dict(ldw=64)):
        assert abi(**kw) == 1, kw
    assert abi(M=40, xx=x40) == 4  # no workspace
    torch.cuda.synchronize()
