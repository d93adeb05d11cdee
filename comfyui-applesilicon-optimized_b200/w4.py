"""4-bit weight-only linears: ``out = act(x . W^T + bias)`` with
``W[n, k] = scales[n, k // G] * (code[n, k] - zeros[n, k // G])``.

Weight layout (what ``w4_quantize`` gives and ``w4a16_linear`` takes): ``w``
[N, K/2] uint8, two codes per byte along K (even k in the low nibble); ``scales``
[N, K/G] bf16/f16/f32; ``zeros`` [N, K/G] uint8 in 0..15, or None for 8.  The
group size G = K / scales.shape[1] is 32, 64 or 128.

Next to the FP8 weight-only linear (``torch.ops.b200q.w8a16_linear``) this halves
the bytes of a small-token call, whose time is its weight stream.  Also
registered as ``torch.ops.b200q.w4a16_linear``.
"""
import torch

from ._patches import _native
from ._patches._native import TAG, _BIAS_DT

GROUPS = (32, 64, 128)


def w4_quantize(weight, group=128, symmetric=True, scale_dtype=None):
    """Round a [N, K] float weight to 4 bits, group by group along K.

    Symmetric: scale = max|w| / 7, zero point 8 (zeros is None).  Otherwise scale
    = (max - min) / 15 over the group widened to hold 0, and a zero point of its
    own.  Returns (w, scales, zeros) in the layout of ``w4a16_linear``.  A one-time
    step at load, on the weight's own device, in torch."""
    if weight.dim() != 2 or not weight.is_floating_point():
        raise RuntimeError(f"{TAG} w4_quantize expects a 2-D float weight, got "
                           f"{tuple(weight.shape)} {weight.dtype}")
    N, K = weight.shape
    if group not in GROUPS or K % group:
        raise RuntimeError(f"{TAG} w4_quantize: group must be one of {GROUPS} and divide K={K}")
    if scale_dtype is None:
        scale_dtype = weight.dtype if weight.dtype in _BIAS_DT else torch.float32
    wg = weight.float().reshape(N, K // group, group)
    if symmetric:
        s = wg.abs().amax(-1, keepdim=True) / 7
    else:
        lo, hi = wg.amin(-1, keepdim=True).clamp(max=0), wg.amax(-1, keepdim=True).clamp(min=0)
        s = (hi - lo) / 15
    scales = s.to(scale_dtype)
    s = scales.float()
    s = torch.where(s > 0, s, torch.ones_like(s))
    z = torch.full_like(s, 8.0) if symmetric else (-lo / s).round().clamp(0, 15)
    c = ((wg / s).round() + z).clamp(0, 15).to(torch.uint8).reshape(N, K // 2, 2)
    packed = (c[..., 0] | (c[..., 1] << 4)).contiguous()
    zeros = None if symmetric else z.to(torch.uint8).reshape(N, K // group).contiguous()
    return packed, scales.reshape(N, K // group).contiguous(), zeros


def w4_dequantize(w, scales, zeros=None):
    """The fp32 [N, K] weight that (w, scales, zeros) stands for (torch, any device)."""
    N = w.shape[0]
    c = torch.stack((w & 15, w >> 4), -1).reshape(N, scales.shape[1], -1).float()
    z = 8.0 if zeros is None else zeros.float().unsqueeze(-1)
    return ((c - z) * scales.float().unsqueeze(-1)).reshape(N, -1)


def w4a16_linear(x, w, scales, zeros=None, bias=None, act=None, out_dtype=None):
    """x [..., K] bf16/f16 -> act(x . W^T + bias) [..., N] in ``out_dtype`` (x's type).

    act: None / "none", "gelu_tanh" or "gelu".  Up to 256 tokens run on kernels that
    read the 4-bit weight as stored (up to 32 with exact products, above that with each
    weight rounded to fp16's 11 bits); more decode it once per call, rounded alike, for
    the 16-bit tile GEMM.  One and two tokens are fastest with scales of x's type.  A
    token that holds an infinity or NaN gives infinities or NaN and no other token does
    (of one or two tokens: NaN in either case)."""
    f = _w4a16 or _load()
    return f(x, w, scales, zeros, bias, act, out_dtype)


_w4a16 = None


def _load():
    global _w4a16
    _w4a16 = _native.bindings().w4a16_linear
    return _w4a16


_LIB = torch.library.Library("b200q", "FRAGMENT")
_LIB.define("w4a16_linear(Tensor x, Tensor w, Tensor scales, Tensor? zeros=None, "
            "Tensor? bias=None, str act='none', ScalarType? out_dtype=None) -> Tensor")
_LIB.impl("w4a16_linear", w4a16_linear, "CUDA")
torch.library.register_fake(
    "b200q::w4a16_linear",
    lambda x, w, s, z=None, b=None, act="none", od=None: x.new_empty(
        (*x.shape[:-1], w.shape[0]), dtype=od or x.dtype), lib=_LIB)
