"""The paged 8-bit cache at the edges of its kernels: values that are not finite, scales far
from 1, prompts of many rows, counts that do not fit (bounds as in test_gpu_kv8.py)."""
import math

import pytest
import torch

import ref64
from b200q import kv8
from test_gpu_kv8 import dev, i32, pool, run_attention

pytestmark = pytest.mark.gpu
DEV = "cuda"
# query heads per cache head and tokens on each attention kernel: up to 8 rows, up to 16, up
# to 128, more
ROWS = [(2, 2), (4, 3), (5, 8), (6, 40)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("start", [0, 5])
def test_an_infinite_value_makes_its_block_nan(native, dtype, sign, start):
    """Every token of the block, those already there among them; no other block."""
    g = torch.Generator().manual_seed(start)
    kc, vc, ks, vs, table = dev(*pool(1, 2, 16, 64, 4))
    k, v = (torch.randn(1, 2, 40, 64, generator=g).to(dtype) for _ in range(2))
    k[0, 0, 3, 7], v[0, 1, 20, 1] = sign * math.inf, sign * math.inf
    kv8.kv8_append(*dev(k, v), kc, vc, ks, vs, table, i32(start).to(DEV))
    n = start + 40
    back = kv8.kv8_gather(kc, vc, ks, vs, table, i32(0).to(DEV), i32(n).to(DEV), n, torch.float32)
    for x, h, at in ((back[0], 0, start + 3), (back[1], 1, start + 20)):
        bad = torch.zeros(2, n, dtype=torch.bool, device=DEV)
        bad[h, at // 16 * 16:at // 16 * 16 + 16] = True
        assert bool(x[0][bad].isnan().all()) and bool(x[0][~bad].isfinite().all())


@pytest.mark.parametrize("G,Tq", ROWS)
@pytest.mark.parametrize("D", [64, 128])
def test_attention_over_an_infinite_key(native, G, Tq, D):
    """A row that sees the key's block is NaN, whatever the sign of its products; rows that do
    not see it are what they were."""
    g = torch.Generator().manual_seed(G)
    kc, vc, ks, vs, table = dev(*pool(1, 2, 16, D, 8, seed=G))
    q = torch.randn(1, 2 * G, Tq, D, generator=g).to(torch.float16).to(DEV)
    k, v = (torch.randn(1, 2, 1, D, generator=g).to(torch.float16).to(DEV) for _ in range(2))
    n = 81  # the block of the last token holds no other
    lens = i32(n).to(DEV)
    kv8.kv8_append(k, v, kc, vc, ks, vs, table, i32(n - 1).to(DEV))
    clean, clean_lse = kv8.kv8_attention(q, kc, vc, ks, vs, table, lens)
    for sign in (1, -1):
        k[0, 1, 0, 3] = sign * math.inf
        kv8.kv8_append(k, v, kc, vc, ks, vs, table, i32(n - 1).to(DEV))
        out, lse = kv8.kv8_attention(q, kc, vc, ks, vs, table, lens)
        hit = torch.zeros(1, 2 * G, Tq, dtype=torch.bool, device=DEV)
        hit[:, G:, -1] = True  # causal: the last query alone sees position n - 1
        assert bool(out[hit].isnan().all()) and bool(lse[hit].isnan().all())
        assert torch.equal(out[~hit], clean[~hit]) and torch.equal(lse[~hit], clean_lse[~hit])
    # a scale that is already infinite in the pool
    ks[int(table[0, 1]), 0] = math.inf
    out, lse = kv8.kv8_attention(q, kc, vc, ks, vs, table, lens)
    assert bool(out[:, :G].isnan().all()) and bool(lse[:, :G].isnan().all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("G,Tq", ROWS)
def test_infinite_query(native, dtype, G, Tq):
    """An infinity in q: its scores are infinite with the keys' signs, or NaN, so its row is NaN,
    also where every one of them is -inf; a row that sees nothing stays 0 and -inf."""
    c = pool(2, 1, 16, 64, 6, seed=3)
    c[0][..., 5] = -c[0][..., 5].abs().clamp(min=1)  # every key is negative there
    g = torch.Generator().manual_seed(2)
    q = torch.randn(2, G, Tq, 64, generator=g).to(dtype)
    lens = i32(90, 0)
    clean, clean_lse = kv8.kv8_attention(q.to(DEV), *dev(*c), lens.to(DEV), False)
    q[:, 0, 0, 5] = math.inf
    out, lse = kv8.kv8_attention(q.to(DEV), *dev(*c), lens.to(DEV), False)
    hit = torch.zeros(2, G, Tq, dtype=torch.bool, device=DEV)
    hit[0, 0, 0] = True
    assert bool(out[hit].isnan().all()) and bool(lse[hit].isnan().all())
    assert torch.equal(out[~hit], clean[~hit]) and torch.equal(lse[~hit], clean_lse[~hit])


@pytest.mark.parametrize("G,Tq", ROWS)
@pytest.mark.parametrize("power", [-20, -40, -60])
def test_a_block_of_zero_values_beside_small_ones(native, G, Tq, power):
    """A block whose values are all zero counts in the softmax's sum alone: the weights of the
    other blocks keep their bits however small those blocks' scales are."""
    kc, vc, ks, vs, table = pool(1, 2, 16, 64, 16, seed=G)
    vs = vs * 2.0 ** power
    vs[int(table[0, 2])] = 0.0
    g = torch.Generator().manual_seed(Tq)
    q = torch.randn(1, 2 * G, Tq, 64, generator=g).to(torch.bfloat16)
    d = dev(kc, vc, ks, vs, table)
    out, lse = kv8.kv8_attention(q.to(DEV), *d, i32(250).to(DEV))
    ref, lse_ref, size = ref64.attention(q, kc, vc, ks, vs, table, i32(250), True)
    tol = ref64.UNIT[q.dtype] * ref.abs() + 2.0 ** -10 * size
    err = (out.double().cpu() - ref).abs()
    assert bool((err <= tol).all()), f"worst {(err / tol).max().item():.3g} of the bound"
    assert bool(((lse.double().cpu() - lse_ref).abs() <= 2.0 ** -17 * (1 + lse_ref.abs())).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16])
@pytest.mark.parametrize("power", [-100, -120, -130])
def test_append_of_vanishing_values(native, dtype, power):
    """Codes are the rounded quotients also where the scale's reciprocal is not finite."""
    g = torch.Generator().manual_seed(1)
    x = (torch.rand(1, 1, 16, 64, generator=g) * 2 - 1)
    x = (x * 2.0 ** power).to(dtype) if power > -126 else (x * 2.0 ** -100).mul(2.0 ** (power + 100)).to(dtype)
    kc, vc, ks, vs, table = dev(*pool(1, 1, 16, 64, 1))
    kv8.kv8_append(*dev(x, x), kc, vc, ks, vs, table, i32(0).to(DEV))
    page = int(table[0, 0])
    s = ks[page, 0].cpu()
    assert torch.equal(s, (x.float().abs().max() / torch.tensor(127.0)))
    want = (x[0, 0].double() / s.double())
    assert bool(((kc[page, 0].cpu().double() - want).abs() <= 0.5 + 2.0 ** -16).all())


@pytest.mark.parametrize("Hq,H,Tq", [(64, 8, 16384), (40, 8, 26300), (1, 1, 131)])
def test_prompts_of_many_rows(native, Hq, H, Tq):
    """The number of a call's 16-row tiles is no limit: what runs is tiles of 256 rows."""
    c = pool(1, H, 16, 64, 3, seed=1)
    g = torch.Generator().manual_seed(Tq)
    q = torch.randn(1, Hq, Tq, 64, generator=g).to(torch.bfloat16)
    run_attention(q, c, i32(37), True)
    run_attention(q[:, :, :500], c, i32(37), False)


@pytest.mark.parametrize("H,G,Tq", [(65535, 1, 17), (960, 1, 18000)])
def test_row_tiles_and_heads_past_65535(native, H, G, Tq):
    """Heads x row tiles of a call go past what one axis of a grid holds in its y and z."""
    D, T = 64, 16
    kc = torch.randint(-127, 128, (1, H, T, D), dtype=torch.int8, device=DEV)
    vc = torch.randint(-127, 128, (1, H, T, D), dtype=torch.int8, device=DEV)
    ks, vs = (torch.full((1, H), 0.01, device=DEV) for _ in range(2))
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    q = torch.randn(1, H * G, Tq, D, dtype=torch.float16, device=DEV)
    out, lse = kv8.kv8_attention(q, kc, vc, ks, vs, table, i32(9).to(DEV), False)
    for h in (0, H // 2, H - 1):
        k, v = (t[0, h, :9].double() * 0.01 for t in (kc, vc))
        p = torch.softmax(q[0, h * G].double() @ k.t() * D ** -0.5, -1)
        ref, size = p @ v, p @ v.abs()
        err = (out[0, h * G].double() - ref).abs()
        assert bool((err <= 2.0 ** -11 * ref.abs() + 2.0 ** -10 * size + 1e-7).all())


def test_counts_outside_the_tokens_given(native):
    """counts above S write S tokens and negative ones none: the lengths say the same."""
    cache = kv8.KV8Cache(3, 1, 64, 64, block=16, device=DEV)
    x = torch.randn(3, 1, 5, 64).to(torch.bfloat16).to(DEV)
    cache.append(x, x, i32(9, -2, 3).to(DEV))
    assert cache.lens.tolist() == [5, 0, 3]
    cache.append(x[:, :, :2], x[:, :, :2])
    assert cache.lens.tolist() == [7, 2, 5]
    k = cache.values(9, torch.float32)[0]
    assert bool((k[0, :, 7:] == 0).all()) and bool((k[0, :, :7].abs().amax(-1) > 0).all())


# ---- the widest forms against 64 bits
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,G,Tq", [(2, 5, 129), (1, 4, 33), (1, 3, 43), (1, 17, 1), (2, 1, 40)])
@pytest.mark.parametrize("causal", [True, False])
def test_row_tiles_over_split_lengths(native, D, H, G, Tq, causal):
    """Both tile kernels with their lengths split over CTAs, ragged, one shorter than its
    queries and one empty."""
    c = pool(4, H, 64, D, 18, seed=D + G)
    g = torch.Generator().manual_seed(Tq)
    q = torch.randn(4, H * G, Tq, D, generator=g).to(torch.float16)
    run_attention(q, c, i32(1100, 20, 641, 0), causal)


@pytest.mark.parametrize("H,G,Tq", [(20, 2, 70), (10, 1, 100)])
def test_more_tiles_than_places(native, H, G, Tq):
    """More CTAs than SMs: sequences start by length, equal and empty ones among them."""
    lens = i32(300, 900, 0, 900, 17, 900, 640, 300)
    c = pool(8, H, 64, 128, 15, seed=G)
    g = torch.Generator().manual_seed(Tq)
    q = torch.randn(8, H * G, Tq, 128, generator=g).to(torch.bfloat16)
    run_attention(q, c, lens, True)


@pytest.mark.parametrize("D,G,Tq", [(128, 5, 700), (64, 1, 513), (128, 1, 1025)])
def test_prompt_into_an_empty_cache(native, D, G, Tq):
    """append, then attention of the same tokens: every row sees itself and what is before."""
    g = torch.Generator().manual_seed(Tq)
    k, v = (torch.randn(1, 2, Tq, D, generator=g).to(torch.bfloat16) for _ in range(2))
    q = torch.randn(1, 2 * G, Tq, D, generator=g).to(torch.bfloat16)
    cache = kv8.KV8Cache(1, 2, D, Tq, block=32, device=DEV)
    cache.append(*dev(k, v))
    pool_ = tuple(t.cpu() for t in cache.pool)
    run_attention(q, pool_, i32(Tq), True)
