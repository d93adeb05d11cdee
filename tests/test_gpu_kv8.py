"""The paged 8-bit cache on the GPU against the 64-bit forms.

Bounds.  Append: scales are one fp32 division (2^-24 relative); a code is within
half a step of the 64-bit quotient plus fp32's share of it (2^-22 of 127).  Gather:
one product, one rounding.  Attention: P is rounded to fp16 (2^-11) and exponents
carry fp32's 2^-24 of scores up to about 64 in base 2, so out is off by at most
2^-10 of sum P|v| / sum P plus its own rounding, and lse by 2^-17.
"""
import math

import pytest
import torch

import ref64
from b200q import kv8

pytestmark = pytest.mark.gpu
DEV = "cuda"


def pool(B, H, T, D, nb, seed=0, spare=3):
    g = torch.Generator().manual_seed(seed)
    P = B * nb + spare
    table = torch.randperm(P, generator=g)[:B * nb].reshape(B, nb).to(torch.int32)
    c = [torch.randint(-127, 128, (P, H, T, D), generator=g).to(torch.int8) for _ in range(2)]
    s = [torch.rand(P, H, generator=g) * 0.02 + 0.005 for _ in range(2)]
    return c[0], c[1], s[0], s[1], table


def dev(*ts):
    return tuple(t.to(DEV) for t in ts)


def i32(*v):
    return torch.tensor(v, dtype=torch.int32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,D", [(16, 64), (32, 128), (64, 128), (128, 64), (128, 128)])
@pytest.mark.parametrize("S", [1, 5, 77])
def test_append(native, dtype, T, D, S):
    B, H, nb = 3, 2, 5 if T < 64 else 3
    kc, vc, ks, vs, table = pool(B, H, T, D, nb if T * nb > S + 40 else -(-(S + 40) // T), seed=S)
    start, counts = i32(0, T - 1, 37 % T), i32(S, S, max(S - 3, 0))
    g = torch.Generator().manual_seed(S + T)
    k, v = (torch.randn(B, H, S, D, generator=g).to(dtype) * f for f in (1.0, 4.0))
    k[0, 0] = 0  # an all-zero block: scale 0, codes 0
    d = dev(kc, vc, ks, vs, table)
    kv8.kv8_append(*dev(k, v), *d, *dev(start, counts))
    for x, c, s, c_new, s_new in ((k, kc, ks, d[0], d[2]), (v, vc, vs, d[1], d[3])):
        rc, rs = ref64.append(x, c, s, table, start, counts)
        assert bool(((s_new.cpu().double() - rs).abs() <= 2.0 ** -23 * rs).all())
        assert bool(((c_new.cpu().double() - rc).abs() <= 0.5 + 127 * 2.0 ** -22).all())
        untouched = (rc == c.double()) & (rc == rc.round())
        same = c_new.cpu() == c
        assert bool(same[untouched].all())
    k2, v2 = kv8.kv8_gather(*d, *dev(i32(0, 0, 0), start + counts), int((start + counts).max()), torch.float32)
    for b in range(B):
        n = int(start[b] + counts[b])
        got = ref64.read(d[0].cpu(), d[2].cpu(), table, b, 0, n)
        assert bool(((k2[b, :, :n].cpu().double() - got).abs() <= 2.0 ** -24 * got.abs()).all())
        assert bool((k2[b, :, n:] == 0).all()) and bool((v2[b, :, n:] == 0).all())


def test_append_in_steps_is_close_to_at_once(native):
    """Token by token the scale grows and codes are requantized: each growth adds at
    most half a step of the final scale."""
    g = torch.Generator().manual_seed(2)
    k = torch.randn(1, 2, 20, 64, generator=g).to(torch.bfloat16)
    cache = kv8.KV8Cache(1, 2, 64, 32, block=32, device=DEV)
    for i in range(20):
        cache.append(k[:, :, i:i + 1].to(DEV), k[:, :, i:i + 1].to(DEV))
    assert cache.lens.tolist() == [20]
    got = cache.values(20, torch.float32)[0].cpu()
    step = cache.k_scale.cpu()[0][None, :, None, None]
    grew = sum(bool((k[0, h, i].abs().max() > k[0, h, :i].abs().max()).item())
               for h in range(2) for i in range(1, 20))
    assert bool(((got - k.float()).abs() <= step * (0.5 + 0.5 * grew)).all())
    assert torch.equal(cache.k_scale.cpu()[0], k[0].float().abs().amax((1, 2)) / torch.full((2,), 127.0))


def test_append_strides_and_nonfinite(native):
    """A [B, S, H, D] projection's transposed view; a NaN makes its block NaN and no other."""
    kc, vc, ks, vs, table = dev(*pool(2, 2, 16, 64, 4))
    g = torch.Generator().manual_seed(0)
    qkv = torch.randn(2, 20, 6, 64, generator=g).to(torch.bfloat16).to(DEV)
    k, v = qkv[:, :, 2:4].transpose(1, 2), qkv[:, :, 4:].transpose(1, 2)
    start = i32(0, 16).to(DEV)
    a = [t.clone() for t in (kc, vc, ks, vs)]
    kv8.kv8_append(k, v, *a, table, start)
    b = [t.clone() for t in (kc, vc, ks, vs)]
    kv8.kv8_append(k.contiguous(), v.contiguous(), *b, table, start)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    k = k.clone()
    k[0, 0, 3, 5], k[1, 1, 18, 0] = float("nan"), float("inf")
    kv8.kv8_append(k, v, kc, vc, ks, vs, table, start)
    back = kv8.kv8_gather(kc, vc, ks, vs, table, start, i32(20, 20).to(DEV), 20, torch.float32)[0]
    bad = torch.zeros(2, 2, 20, dtype=torch.bool)
    bad[0, 0, :16], bad[1, 1, 16:] = True, True
    finite = back.isfinite().all(-1).cpu()
    assert bool(finite[~bad].all()) and not bool(finite[bad].any())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_gather_ranges(native, dtype):
    kc, vc, ks, vs, table = pool(3, 2, 16, 64, 5)
    first, counts = i32(0, 13, 40), i32(0, 50, 40)
    k, v = kv8.kv8_gather(*dev(kc, vc, ks, vs, table, first, counts), 50, dtype)
    for b in range(3):
        n = int(counts[b])
        for got, c, s in ((k, kc, ks), (v, vc, vs)):
            ref = ref64.read(c, s, table, b, int(first[b]), n)
            tol = (ref64.UNIT[dtype] + 2.0 ** -24) * ref.abs()
            assert bool(((got[b, :, :n].cpu().double() - ref).abs() <= tol).all())
            assert bool((got[b, :, n:] == 0).all())


def run_attention(q, c, lens, causal, max_len=None, scale=None):
    out, lse = kv8.kv8_attention(q.to(DEV), *dev(*c), lens.to(DEV), causal, scale, max_len)
    ref, lse_ref, size = ref64.attention(q, *c, lens, causal, scale)
    tol = ref64.UNIT[q.dtype] * ref.abs() + 2.0 ** -10 * size + 1e-7
    err = (out.double().cpu() - ref).abs()
    assert bool((err <= tol).all()), f"worst {(err / tol).max().item():.3g} of the bound"
    empty = lse_ref == -math.inf
    assert torch.equal(lse.cpu() == -math.inf, empty)
    assert bool((out.cpu()[empty] == 0).all())
    seen = ~empty
    assert bool(((lse.double().cpu() - lse_ref)[seen].abs() <= 2.0 ** -17 * (1 + lse_ref[seen].abs())).all())
    return out, lse


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,D", [(16, 64), (64, 128), (128, 64), (32, 128)])
@pytest.mark.parametrize("H,G,Tq", [(1, 1, 1), (2, 5, 1), (1, 8, 4), (2, 3, 7), (1, 16, 3), (3, 2, 40)])
@pytest.mark.parametrize("causal", [True, False])
def test_attention(native, dtype, T, D, H, G, Tq, causal):
    """Ragged lengths with an empty sequence, one shorter than its queries, ones
    ending inside a page and inside a 16-token tile."""
    c = pool(5, H, T, D, -(-260 // T), seed=T + G)
    g = torch.Generator().manual_seed(Tq)
    q = torch.randn(5, H * G, Tq, D, generator=g).to(dtype)
    run_attention(q, c, i32(0, 1, 3, 131, 256), causal)


@pytest.mark.parametrize("max_len", [None, 1, 700, 4096])
def test_attention_splits(native, max_len):
    """Long lengths are split over CTAs and joined; the plan's hint changes nothing
    but the order of the sums."""
    c = pool(2, 1, 64, 128, 64, seed=9)
    g = torch.Generator().manual_seed(1)
    q = torch.randn(2, 4, 2, 128, generator=g).to(torch.float16)
    run_attention(q, c, i32(4095, 17), True, max_len)


def test_attention_scales_spread(native):
    """Block scales over six decades (a zero one among them) and scores up to +-60."""
    kc, vc, ks, vs, table = pool(1, 2, 16, 64, 16, seed=4)
    vs = torch.logspace(-6, 0, vs.numel()).reshape(vs.shape)[torch.randperm(vs.shape[0])]
    vs[int(table[0, 3])] = 0.0
    ks = ks * 3
    q = torch.randn(1, 4, 3, 64).to(torch.bfloat16) * 2
    run_attention(q, (kc, vc, ks, vs, table), i32(250), True)
    run_attention(q, (kc, vc, torch.zeros_like(ks), vs, table), i32(250), False)
    run_attention(q, (kc, vc, ks, torch.zeros_like(vs), table), i32(250), False)
    run_attention(q * 2.0 ** -60, (kc, vc, ks * 2.0 ** 40, vs, table), i32(99), False, scale=2.0 ** 18)


def test_attention_ignores_what_is_past_the_length(native):
    """Codes past the length and pages past it (NaN scales, bad page numbers) do not matter."""
    kc, vc, ks, vs, table = pool(1, 1, 16, 64, 8, seed=6)
    q = torch.randn(1, 2, 1, 64).to(torch.bfloat16)
    base = kv8.kv8_attention(q.to(DEV), *dev(kc, vc, ks, vs, table), i32(37).to(DEV))
    for i in range(3, 8):
        ks[int(table[0, i])] = vs[int(table[0, i])] = float("nan")
    kc[int(table[0, 2]), :, 5:] = 99
    vc[int(table[0, 2]), :, 5:] = -99
    table[0, 3:] = 10 ** 6
    native.device_status(reset=True)
    again = kv8.kv8_attention(q.to(DEV), *dev(kc, vc, ks, vs, table), i32(37).to(DEV))
    assert torch.equal(base[0], again[0]) and torch.equal(base[1], again[1])
    assert native.device_status() == 0


def test_attention_nonfinite(native):
    """A NaN in q makes its row NaN and no other; a block of NaN scale the rows that see it."""
    c = pool(1, 2, 16, 64, 4, seed=7)
    q = torch.randn(1, 4, 2, 64).to(torch.bfloat16)
    clean = kv8.kv8_attention(q.to(DEV), *dev(*c), i32(50).to(DEV))
    q2 = q.clone()
    q2[0, 1, 0, 3] = float("nan")
    out, lse = kv8.kv8_attention(q2.to(DEV), *dev(*c), i32(50).to(DEV))
    hit = torch.zeros(1, 4, 2, dtype=torch.bool, device=DEV)
    hit[0, 1, 0] = True
    assert bool(out[hit].isnan().all()) and bool(lse[hit].isnan().all())
    assert torch.equal(out[~hit], clean[0][~hit])
    c[3][int(c[4][0, 1]), 1] = float("nan")
    out, _ = kv8.kv8_attention(q.to(DEV), *dev(*c), i32(50).to(DEV))
    assert bool(out[:, 2:].isnan().all()) and torch.equal(out[:, :2], clean[0][:, :2])


@pytest.mark.parametrize("G,Tq", [(2, 3), (3, 5), (5, 8), (6, 40)])
def test_attention_small_weights_keep_their_bits(native, G, Tq):
    """Block scales over six decades: where the largest weight's code is near zero the
    small ones make the value.  And a block of vanishing values (scale 1e-30)."""
    kc, vc, ks, vs, table = pool(1, 2, 16, 64, 16, seed=4)
    for seed in range(12):
        g = torch.Generator().manual_seed(seed)
        vs = torch.logspace(-6, 0, vs.numel())[torch.randperm(vs.numel(), generator=g)].reshape(vs.shape)
        vs[int(table[0, 3])] = 1e-30
        q = torch.randn(1, 2 * G, Tq, 64, generator=g).to(torch.bfloat16) * 2
        run_attention(q, (kc, vc, ks * 3, vs, table), i32(250), True)


@pytest.mark.parametrize("H,G,Tq", [(2, 5, 129), (2, 8, 9), (2, 8, 1)])
def test_attention_repeats_bit_for_bit(native, H, G, Tq):
    """Many launches of a pipelined kernel, other work in between: the same bits each
    time, and no wait ever ran out."""
    c = dev(*pool(3, H, 64, 128, 30, seed=12))
    q = torch.randn(3, H * G, Tq, 128).to(torch.float16).to(DEV)
    lens = i32(1900, 1333, 700).to(DEV)
    native.device_status(reset=True)
    first = kv8.kv8_attention(q, *c, lens)
    noise = torch.randn(1 << 20, device=DEV)
    for i in range(300):
        if i % 3 == 0:
            noise.mul_(1.0001)
        again = kv8.kv8_attention(q, *c, lens)
        if i % 20 == 0:
            assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    assert torch.equal(first[0], again[0])
    assert native.device_status() == 0


def test_append_ties(native):
    """x = half of the block's largest value is code 63.5, an exact tie: it rounds as
    the quotient does, to 64."""
    kc, vc, ks, vs, table = dev(*pool(1, 1, 16, 64, 1))
    x = torch.zeros(1, 1, 16, 64, dtype=torch.float16)
    for i in range(16):
        x[0, 0, i, 0] = 1.0 + i / 16
    top = x.amax()
    x[0, 0, :, 1] = top / 2
    x[0, 0, :, 2] = -top / 2
    d = x.to(DEV)
    kv8.kv8_append(d, d, kc, vc, ks, vs, table, i32(0).to(DEV))
    codes = kc[int(table[0, 0]), 0].cpu()
    s = (top.float() / torch.tensor(127.0))
    want = (x[0, 0].float() / s).round().clamp(-127, 127).to(torch.int8)
    assert torch.equal(codes, want)


def test_bad_pages_are_flagged_and_skipped(native):
    """Out-of-range page numbers inside the length: checked in the kernels, no access."""
    kc, vc, ks, vs, table = pool(1, 1, 16, 64, 4, seed=8)
    q = torch.randn(1, 1, 1, 64).to(torch.bfloat16).to(DEV)
    bad = table.clone()
    bad[0, 1], bad[0, 2] = -1, 1 << 20
    d = dev(kc, vc, ks, vs)
    before = [t.clone() for t in d]
    native.device_status(reset=True)
    out, _ = kv8.kv8_attention(q, *d, bad.to(DEV), i32(64).to(DEV))
    assert native.device_status(reset=True) == 2
    assert bool(out.isfinite().all())
    x = torch.randn(1, 1, 8, 64).to(torch.bfloat16).to(DEV)
    kv8.kv8_append(x, x, *d, bad.to(DEV), i32(18).to(DEV))
    assert native.device_status(reset=True) == 2
    assert all(torch.equal(x, y) for x, y in zip(before, d))
    kv8.kv8_append(x, x, *d, table.to(DEV), i32(62).to(DEV))  # runs past the table
    assert native.device_status(reset=True) == 2
    k, _ = kv8.kv8_gather(*d, bad.to(DEV), i32(16).to(DEV), i32(16).to(DEV), 16)
    assert native.device_status(reset=True) == 2 and bool((k == 0).all())


def test_query_strides_streams_graph(native):
    c = dev(*pool(2, 2, 32, 128, 8, seed=3))
    lens = i32(200, 77).to(DEV)
    qkv = torch.randn(2, 3, 10, 128).to(torch.bfloat16).to(DEV)
    q = qkv[:, :, :6].transpose(1, 2)  # [B, 6, 3, D] view
    out, lse = kv8.kv8_attention(q, *c, lens)
    assert out.transpose(1, 2).is_contiguous()
    out2, lse2 = torch.ops.b200q.kv8_attention(q.contiguous(), *c, lens)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        out3, _ = kv8.kv8_attention(q, *c, lens)
    side.synchronize()
    assert torch.equal(out, out3)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out4, _ = kv8.kv8_attention(q, *c, lens)
    lens += 9
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out4, kv8.kv8_attention(q, *c, lens)[0])


def test_long_cache_offsets(native):
    """A pool of more than 2^31 bytes of codes: pages near its end are reached."""
    P, H, T, D = 40000, 8, 64, 128
    k = torch.zeros(P, H, T, D, dtype=torch.int8, device=DEV)
    assert k.numel() > 2 ** 31
    s = torch.ones(P, H, device=DEV)
    table = torch.tensor([[P - 1, 0, P - 2]], dtype=torch.int32, device=DEV)
    x = torch.randn(1, H, 150, D, device=DEV).to(torch.bfloat16)
    v = torch.zeros_like(k)
    vs = s.clone()
    kv8.kv8_append(x, x, k, v, s, vs, table, i32(0).to(DEV))
    small = [torch.stack([t[P - 1], t[0], t[P - 2]]) for t in (k, v, s, vs)]
    t3 = torch.tensor([[0, 1, 2]], dtype=torch.int32, device=DEV)
    q = torch.randn(1, H, 1, D, device=DEV).to(torch.bfloat16)
    a = kv8.kv8_attention(q, k, v, s, vs, table, i32(150).to(DEV))
    b = kv8.kv8_attention(q, *small, t3, i32(150).to(DEV))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    back = kv8.kv8_gather(k, v, s, vs, table, i32(0).to(DEV), i32(150).to(DEV), 150, torch.float32)[0]
    assert bool(((back - x.float()).abs() <= 0.51 * x.float().abs().max() / 127 + 1e-6).all())


def test_refusals(native):
    kc, vc, ks, vs, table = dev(*pool(2, 2, 16, 64, 4))
    lens = i32(20, 30).to(DEV)
    q = torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16, device=DEV)
    k = torch.zeros(2, 2, 3, 64, dtype=torch.bfloat16, device=DEV)
    c = (kc, vc, ks, vs, table)

    def but(i, t):
        return c[:i] + (t,) + c[i + 1:]

    f, a, g = kv8.kv8_attention, kv8.kv8_append, kv8.kv8_gather
    bad = [
        lambda: f(q.float(), *c, lens), lambda: f(q[:, :3], *c, lens), lambda: f(q[..., :32], *c, lens),
        lambda: f(q[:1], *c, lens), lambda: f(q, *c, lens.long()), lambda: f(q, *c, lens[:1]),
        lambda: f(q, *c, lens.cpu()), lambda: f(q.cpu(), *c, lens), lambda: f(q, *but(0, kc.to(torch.uint8)), lens),
        lambda: f(q, *but(1, vc[:5]), lens), lambda: f(q, *but(2, ks.double()), lens),
        lambda: f(q, *but(3, vs.t()), lens), lambda: f(q, *but(4, table.long()), lens),
        lambda: f(q, *but(0, kc.transpose(1, 2)), lens), lambda: f(q[0], *c, lens),
        lambda: f(q, kc[:, :, :8].contiguous(), vc[:, :, :8].contiguous(), ks, vs, table, lens),
        lambda: f(q, *c, lens, max_len=-1),
        lambda: a(k.float(), k.float(), *c, lens), lambda: a(k, k[:, :1], *c, lens),
        lambda: a(k[:1], k[:1], *c, lens), lambda: a(k, k, *c, lens, lens[:1]), lambda: a(k, k, *c, lens.float()),
        lambda: g(*c, lens, lens, -1), lambda: g(*c, lens, lens, 3, torch.int8),
    ]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
    assert f(q[:, :, :0], *c, lens)[0].shape == (2, 4, 0, 64)
    a(k[:, :, :0], k[:, :, :0], *c, lens)
    assert g(*c, lens, lens, 0)[0].shape == (2, 2, 0, 64)
