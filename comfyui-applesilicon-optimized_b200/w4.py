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
from ._patches._native import ACTS, TAG, _BIAS_DT, _DT

GROUPS = (32, 64, 128)
_raw_stream = torch._C._cuda_getCurrentRawStream


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

    act: None / "none", "gelu_tanh" or "gelu".  Up to 32 tokens run on a kernel
    that reads the 4-bit weight as stored; more decode it once per call for the
    16-bit tile GEMM."""
    dt = x.dtype
    xdt = _DT.get(dt)
    if xdt is None or xdt == 2:
        raise RuntimeError(f"{TAG} w4a16 expects bf16/f16 activations, got {dt}")
    K = x.shape[-1]
    N, half = w.shape if w.dim() == 2 else (0, 0)
    if w.dtype != torch.uint8 or 2 * half != K or w.stride(1) != 1:
        raise RuntimeError(f"{TAG} w4a16: w must be uint8 [N, K/2] with K={K} and unit inner "
                           f"stride, got {w.dtype} {tuple(w.shape)}")
    if w.data_ptr() % 16 or w.stride(0) % 16:
        raise RuntimeError(f"{TAG} w4a16: the rows of w must start on 16-byte boundaries")
    sdt = _BIAS_DT.get(scales.dtype)
    if sdt is None or scales.dim() != 2 or scales.shape[0] != N or not scales.is_contiguous():
        raise RuntimeError(f"{TAG} w4a16: scales must be contiguous bf16/f16/f32 [N, K/G], got "
                           f"{scales.dtype} {tuple(scales.shape)}")
    groups = scales.shape[1]
    G = K // groups if groups else 0
    if G not in GROUPS or G * groups != K:
        raise RuntimeError(f"{TAG} w4a16: K={K} in {groups} groups; the group size must be one "
                           f"of {GROUPS}")
    if zeros is not None and (zeros.dtype != torch.uint8 or zeros.shape != scales.shape
                              or not zeros.is_contiguous()):
        raise RuntimeError(f"{TAG} w4a16: zeros must be contiguous uint8 of scales' shape")
    code = xdt if out_dtype is None else _DT.get(out_dtype)
    if code is None:
        raise RuntimeError(f"{TAG} unsupported out dtype {out_dtype}")
    if act not in ACTS:
        raise RuntimeError(f"{TAG} unknown activation {act!r}")
    dev = x.device
    if dev.type != "cuda":
        raise RuntimeError(f"{TAG} expected CUDA tensors, got {dev}")
    for t in (w, scales, zeros, bias):
        if t is not None and t.device != dev:
            raise RuntimeError(f"{TAG} w4a16: tensors on {dev} and {t.device}")
    x2 = x if x.dim() == 2 else x.reshape(-1, K)
    M = x2.shape[0]
    if x2.stride(1) != 1 or (M > 1 and x2.stride(0) < K):
        x2 = x2.contiguous()
    bdt, bp = 0, 0
    if bias is not None:
        if bias.numel() != N:
            raise RuntimeError(f"{TAG} bias numel {bias.numel()} != N {N}")
        bias = bias.contiguous()
        if bias.dtype not in _BIAS_DT:
            bias = bias.float()
        bdt, bp = _BIAS_DT[bias.dtype], bias.data_ptr()
    L = _native.lib()
    with _native.device_of(dev):
        ldx = x2.stride(0) if M > 1 else K
        wsb = L.b200q_w4a16_workspace_size(M, N, K)
        work, wp = None, 0
        if wsb:
            work = torch.empty(wsb, dtype=torch.uint8, device=dev)
            wp = work.data_ptr()
            if xdt == 1 and (x2.data_ptr() % 16 or ldx % 8):
                x2 = x2.clone(memory_format=torch.contiguous_format)
                ldx = K
        out = torch.empty((*x.shape[:-1], N), dtype=out_dtype or dt, device=dev)
        st = L.b200q_w4a16_linear(
            x2.data_ptr(), xdt, ldx, w.data_ptr(), w.stride(0), scales.data_ptr(), sdt,
            0 if zeros is None else zeros.data_ptr(), G, bp, bdt, ACTS[act], out.data_ptr(), code,
            N, M, N, K, wp, wsb, _raw_stream(dev.index))
        if st:
            _native._check(st)
    return out


_LIB = torch.library.Library("b200q", "FRAGMENT")
_LIB.define("w4a16_linear(Tensor x, Tensor w, Tensor scales, Tensor? zeros=None, "
            "Tensor? bias=None, str act='none', ScalarType? out_dtype=None) -> Tensor")
_LIB.impl("w4a16_linear", w4a16_linear, "CUDA")
torch.library.register_fake(
    "b200q::w4a16_linear",
    lambda x, w, s, z=None, b=None, act="none", od=None: x.new_empty(
        (*x.shape[:-1], w.shape[0]), dtype=od or x.dtype), lib=_LIB)
