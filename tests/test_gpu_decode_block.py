"""The low-bit operators together: DecodeBlock against a 64-bit block.

Eight values in a row are rounded to bf16 on the way through the block (2^-9 rms each
of their own size), so what the block adds to h is off by about sqrt(8) 2^-9 of its
size, 0.6%; 2% is allowed.  The attention of the 64-bit block reads the values that
the cache holds, so the cache's own 8-bit rounding is not part of the difference.
"""
import pytest
import torch

import ref64
from b200q import kv8, w4
from b200q.decode_block import DecodeBlock

pytestmark = pytest.mark.gpu
DEV = "cuda"
H, N, HD, D, F, R = 6, 2, 128, 512, 640, 32


@pytest.fixture(scope="module")
def block():
    g = torch.Generator().manual_seed(7)

    def r(*s, f=1.0):
        return (torch.randn(*s, generator=g) * f).to(DEV)

    weights = {"qkv": r((H + 2 * N) * HD, D, f=D ** -0.5), "out": r(D, H * HD, f=(H * HD) ** -0.5),
               "up": r(2 * F, D, f=D ** -0.5), "down": r(D, F, f=F ** -0.5)}
    norms = {n: 1 + 0.1 * r(D) for n in ("pre_attn", "post_attn", "pre_mlp", "post_mlp")}
    norms |= {n: 1 + 0.1 * r(HD) for n in "qk"}
    return DecodeBlock(weights, norms, H, N, gate_attn=r(D, f=0.3), gate_mlp=r(D, f=0.3))


def freqs(B, first, T):
    at = torch.arange(first, first + T, dtype=torch.float64)[:, None]
    ang = at * torch.pow(10000.0, -torch.arange(R, dtype=torch.float64) / R)
    f = torch.stack((ang.cos(), -ang.sin(), ang.sin(), ang.cos()), -1).reshape(T, R, 2, 2)
    return f.to(torch.bfloat16).repeat(B, 1, 1, 1).to(DEV).contiguous()


def added_64(block, h, cache, fr, seen):
    """What a 64-bit block adds to h; the cache already holds the new tokens."""
    B, T, _ = h.shape

    def lin(x, name):
        w, s, z = block.w[name]
        return x @ w4.w4_dequantize(w, s, z).double().cpu().t()

    def rope(x, weight):
        y = ref64.unit_rows(x, "rms", block.eps) * weight.double().cpu()
        a, b, f = y[..., :R], y[..., R:2 * R], fr.double().cpu().view(B, 1, T, R, 2, 2)
        turned = [f[..., 0, 0] * a + f[..., 0, 1] * b, f[..., 1, 0] * a + f[..., 1, 1] * b]
        return torch.cat((*turned, y[..., 2 * R:]), -1)

    n = {k: v.double().cpu() for k, v in block.norm.items()}
    x = h.double().cpu()
    qkv = lin(ref64.unit_rows(x, "rms", block.eps) * n["pre_attn"], "qkv").view(B, T, H + 2 * N, HD)
    q, k = (rope(t.transpose(1, 2), n[s]) for t, s in ((qkv[:, :, :H], "q"), (qkv[:, :, H:H + N], "k")))
    keys, values = (t.double().cpu() for t in cache.values(seen, torch.float32))
    # the cache holds this call's keys to half a step of their block's scale, and bf16
    step = cache.k_scale.double().cpu().max() * 0.51 + 2.0 ** -7 * k.abs().max()
    assert float((keys[:, :, seen - T:] - k).abs().max()) <= step
    s = q @ keys.repeat_interleave(H // N, 1).transpose(-1, -2) * HD ** -0.5
    hide = torch.arange(seen)[None] > seen - T + torch.arange(T)[:, None]
    p = torch.softmax(s.masked_fill(hide, -torch.inf), -1)
    o = (p @ values.repeat_interleave(H // N, 1)).transpose(1, 2).reshape(B, T, H * HD)
    attn = ref64.unit_rows(lin(o, "out"), "rms", block.eps) * n["post_attn"] * block.gate_attn.double().cpu()
    a = ref64.unit_rows(x + attn, "rms", block.eps) * n["pre_mlp"]
    gate, up = lin(a, "up").chunk(2, -1)
    mlp = ref64.unit_rows(lin(gate * torch.sigmoid(gate) * up, "down"), "rms", block.eps) * n["post_mlp"]
    return attn + mlp * block.gate_mlp.double().cpu()


def close(out, h, ref):
    got = out.double().cpu() - h.double().cpu()
    # h itself is stored twice (after each half), 2^-9 rms of its size
    tol = 0.02 * float(ref.norm()) + 2 * 2.0 ** -9 * float(h.double().norm())
    assert float((got - ref).norm()) <= tol


def test_prompt_then_tokens(native, block):
    """A prompt of 37 tokens, then single tokens, two sequences."""
    g = torch.Generator().manual_seed(1)
    cache = kv8.KV8Cache(2, N, HD, 64, block=16, device=DEV)
    h = torch.randn(2, 37, D, generator=g).to(torch.bfloat16).to(DEV)
    out = block(h, cache, freqs(2, 0, 37))
    close(out, h, added_64(block, h, cache, freqs(2, 0, 37), 37))
    for i in range(37, 41):
        h = torch.randn(2, 1, D, generator=g).to(torch.bfloat16).to(DEV)
        out = block(h, cache, freqs(2, i, 1))
        close(out, h, added_64(block, h, cache, freqs(2, i, 1), i + 1))
    assert cache.lens.tolist() == [41, 41]
    assert native.device_status() == 0


def test_step_in_a_cuda_graph(native, block):
    """A captured one-token step advances the cache at every replay, as eager steps do."""
    g = torch.Generator().manual_seed(2)
    tokens = torch.randn(5, 1, 1, D, generator=g).to(torch.bfloat16).to(DEV)
    tables = [freqs(1, i, 1) for i in range(5)]
    eager = kv8.KV8Cache(1, N, HD, 32, block=16, device=DEV)
    want = [block(tokens[i], eager, tables[i]) for i in range(5)]
    cache = kv8.KV8Cache(1, N, HD, 32, block=16, device=DEV)
    x, fr = tokens[0].clone(), tables[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block(x, cache, fr)
    torch.cuda.current_stream().wait_stream(side)
    cache.lens.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block(x, cache, fr)
    for i in range(5):
        x.copy_(tokens[i])
        fr.copy_(tables[i])
        graph.replay()
        assert torch.equal(out, want[i])
    assert torch.equal(cache.lens, eager.lens)
