"""4-bit weight linears at the edges of their kernels, against the 64-bit form (bounds as in
test_gpu_w4a16.py)."""
import pytest
import torch

import ref64
from b200q import w4
from test_gpu_w4a16 import check, dev, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N", [1, 31, 129, 1003, 4149])
@pytest.mark.parametrize("M", [97, 128, 191, 256])
def test_last_rows_of_a_tile_over_several_columns(native, M, N):
    """N off a multiple of 32: some lanes of a warp have no row to store while the warp goes
    on to more tokens.  One K slice (the epilogue's stores) and several (partial sums)."""
    for K in (256, 4096):
        x, w, s, z, b = make(M, N, K, 64, torch.bfloat16, True, bias=True, seed=N + M)
        native.device_status(reset=True)
        out = w4.w4a16_linear(*dev(x, w, s, z, b), "gelu_tanh")
        check(out, x, w, s, z, b, "gelu_tanh")
        assert native.device_status() == 0


def bound(out, ref, size, exact):
    u = ref64.UNIT[out.dtype]
    return u * ref.abs() + size * (2.0 ** -17 + (0 if exact else 2.0 ** -11))


def large(M, power):
    """bf16 values up to 2^power and some with weights that keep the output in range, exactly
    representable ones (whose lower digits are zero) and others."""
    x, w, s, z, b = make(M, 48, 256, 64, torch.bfloat16, True)
    s = (s.float() * 2.0 ** -20).to(torch.bfloat16)
    x[0] = torch.sign(x[0].float()).to(torch.bfloat16)
    return (x.float() * 2.0 ** power).to(torch.bfloat16), w, s, z


@pytest.mark.parametrize("M", [1, 2, 3, 8, 9])
@pytest.mark.parametrize("power", [100, 110, 117, 124])
def test_large_activations_of_few_tokens(native, M, power):
    x, w, s, z = large(M, power)
    out = w4.w4a16_linear(*dev(x, w, s, z), None, None, torch.float32)
    ref, size = ref64.w4_linear(x, w, s, z)
    assert bool(((out.double().cpu() - ref).abs() <= bound(out, ref, size, True)).all())


@pytest.mark.parametrize("M,N", [(40, 48), (130, 48), (300, 48), (300, 45)])
@pytest.mark.parametrize("power", [100, 110, 117, 124])
def test_large_activations_of_many_tokens(native, M, N, power):
    x, w, s, z = large(M, power)
    w, s, z = w[:N].contiguous(), s[:N].contiguous(), z[:N].contiguous()
    out = w4.w4a16_linear(*dev(x, w, s, z), None, None, torch.float32)
    ref, size = ref64.w4_linear(x, w, s, z)
    assert bool(((out.double().cpu() - ref).abs() <= bound(out, ref, size, False)).all())


@pytest.mark.parametrize("M", [40, 300])
def test_small_activations_and_large_scales(native, M):
    """The other way round: rows near the smallest normal number, scales far above 1."""
    x, w, s, z = large(M, -110)
    s = (s.float() * 2.0 ** 60).to(torch.bfloat16)
    out = w4.w4a16_linear(*dev(x, w, s, z), None, None, torch.float32)
    ref, size = ref64.w4_linear(x, w, s, z)
    assert bool(((out.double().cpu() - ref).abs() <= bound(out, ref, size, False)).all())


# (M, K, G) around the longest K whose slice of x fits beside the rings, and past the tile
# kernel's fallback
@pytest.mark.parametrize("M,K,G", [(32, 41984, 32), (32, 42016, 32), (17, 53248, 32), (32, 53248, 32),
                                   (24, 56352, 32), (32, 53312, 64), (32, 57472, 128), (32, 200000, 32),
                                   (1, 200000, 32), (9, 300032, 128)])
def test_long_rows_of_few_tokens(native, M, K, G):
    x, w, s, z, b = make(M, 40, K, G, torch.bfloat16, True, seed=M)
    out = w4.w4a16_linear(*dev(x, w, s, z), None, None, torch.float32)
    ref, size = ref64.w4_linear(x, w, s, z)
    # fp32 sums: 2^-17 covers 5120 additions in any order, a slice and the join at most
    # K / 32 / G + 64 here
    exact = K < 190000
    assert bool(((out.double().cpu() - ref).abs() <= bound(out, ref, size, exact)).all())


@pytest.mark.parametrize("dtype,scale_dtype", [(torch.bfloat16, torch.float32), (torch.float16, torch.bfloat16),
                                               (torch.bfloat16, torch.float16), (torch.float16, torch.float32)])
@pytest.mark.parametrize("M", [1, 2, 3])
def test_scales_of_another_type_split_k_too(native, dtype, scale_dtype, M):
    """Scales that are not of x's type take the slice kernel, whose few tiles at one token
    need K split over CTAs to fill the GPU: the product and the join are two launches."""
    x, w, s, z, b = make(M, 1024, 2048, 64, dtype, True, scale_dtype=scale_dtype)
    d = dev(x, w, s, z)
    before = native.launch_count()
    out = w4.w4a16_linear(*d)
    assert native.launch_count() - before == 2
    check(out, x, w, s, z, b)


@pytest.mark.parametrize("M", [12, 100, 300])
def test_infinity_beside_large_values(native, M):
    """A row's infinity decides its outputs' sign; finite values of any size beside it do
    not make infinities of their own."""
    x, w, s, z, b = make(M, 64, 256, 64, torch.bfloat16, False)
    x[3] = x[3].float().mul(1e30).to(torch.bfloat16)
    x[3, 9] = float("inf")
    out = w4.w4a16_linear(*dev(x, w, s))
    W = ref64.w4_weight(w, s)[:, 9]
    want = torch.where(W == 0, torch.nan, torch.sign(W) * torch.inf)
    got = out[3].double().cpu()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got[~want.isnan()], want[~want.isnan()])
