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
