"""The norms before and after a transformer block, fused with the block's gate,
the residual scale and the next block's modulation:

    after:   h   = residual_scale * residual + gate * (norm_post(y) * post_weight)
    before:  out = norm(h) * weight * (1 + scale) + shift

``kind`` / ``post_kind``: "rms", "layer" or "none".  Rows are the last axis;
``gate``, ``scale`` and ``shift`` are [B, D] (or [D]) with the rows split evenly
over B in order, so [B, T, D] activations take the [B, D] chunks of a DiT block's
modulation as they are, and B = rows gives every token its own.  Each is optional.

One pass over the rows; statistics, gate, residual and modulation in fp32, each
output rounded once.  The ``_quant_i8`` forms return the INT8 codes and row scales
that the INT8 linears take (``torch.ops.b200q.i8_matmul_nt_fused_cs``), quantized
from the unrounded output: no 16-bit activation is written in between.

Also registered under the same names in ``torch.ops.b200q``.
"""
import torch

from ._patches import _native
from ._patches._native import TAG, _BIAS_DT, _DT

KINDS = {"none": 0, "rms": 1, "layer": 2}
MAX_D = 32768  # B200Q_NORM_MAX_D
_raw_stream = torch._C._cuda_getCurrentRawStream


def _rows(t, D, name):
    """[..., D] as (tensor, row stride) over its flattened rows."""
    if t.is_contiguous():
        return t, D
    t2 = t.reshape(-1, D)
    if t2.stride(1) != 1 or (t2.shape[0] > 1 and t2.stride(0) < D):
        t2 = t2.contiguous()
    return t2, t2.stride(0) if t2.shape[0] > 1 else D


def _vector(t, D, dev, name):
    if t is None:
        return 0, 0
    if t.numel() != D or t.dtype not in _BIAS_DT or t.device != dev or (t.dim() != 1):
        raise RuntimeError(f"{TAG} {name} must be bf16/f16/f32 [{D}] on {dev}, got {t.dtype} "
                           f"{tuple(t.shape)} on {t.device}")
    if t.stride(0) != 1:
        raise RuntimeError(f"{TAG} {name} must have unit stride")
    return t.data_ptr(), _BIAS_DT[t.dtype]


def _run(x, y, gate, post_weight, post_kind, residual_scale, weight, scale, shift, kind, eps,
         quant, want_h, want_out):
    dt = x.dtype
    code = _DT.get(dt)
    if code is None or code == 2:
        raise RuntimeError(f"{TAG} block norms expect bf16/f16 activations, got {dt}")
    if kind not in KINDS or post_kind not in KINDS:
        raise RuntimeError(f"{TAG} norm kind must be one of {tuple(KINDS)}, got {kind!r}, "
                           f"{post_kind!r}")
    dev = x.device
    if dev.type != "cuda":
        raise RuntimeError(f"{TAG} expected CUDA tensors, got {dev}")
    if x.dim() == 0 or not 0 < x.shape[-1] <= MAX_D:
        raise RuntimeError(f"{TAG} block norms take rows of 1 to {MAX_D} values, got "
                           f"{tuple(x.shape)}")
    D = x.shape[-1]
    rows = x.numel() // D
    x2, ldx = _rows(x, D, "x")
    yp = ldy = 0
    if y is not None:
        if y.shape != x.shape or y.dtype != dt or y.device != dev:
            raise RuntimeError(f"{TAG} y must match the residual: {tuple(x.shape)} {dt} on {dev}, "
                               f"got {tuple(y.shape)} {y.dtype} on {y.device}")
        y, ldy = _rows(y, D, "y")
        yp = y.data_ptr()
    pw, pwt = _vector(post_weight, D, dev, "post_weight")
    w, wt = _vector(weight, D, dev, "weight")
    mods, mdt, per, ptrs = None, 0, max(rows, 1), []
    for name, t in (("gate", gate), ("scale", scale), ("shift", shift)):
        if t is None:
            ptrs.append((0, 0))
            continue
        if (t.dim() not in (1, 2) or t.shape[-1] != D or t.dtype not in _BIAS_DT
                or t.device != dev or t.stride(-1) != 1):
            raise RuntimeError(f"{TAG} {name} must be bf16/f16/f32 [B, {D}] with unit inner "
                               f"stride on {dev}, got {t.dtype} {tuple(t.shape)} on {t.device}")
        b = t.shape[0] if t.dim() == 2 else 1
        if mods is None:
            mods, mdt = b, _BIAS_DT[t.dtype]
            if b == 0 or rows % b:
                raise RuntimeError(f"{TAG} {rows} rows do not split over {b} rows of {name}")
            per = max(rows // b, 1)
        elif b != mods or _BIAS_DT[t.dtype] != mdt:
            raise RuntimeError(f"{TAG} gate, scale and shift must agree in type and rows")
        ld = t.stride(0) if b > 1 else D
        if ld < D:  # a row expanded over the batch
            t = t.contiguous()
            ld = D
        ptrs.append((t.data_ptr(), ld, t))
    L = _native.lib()
    with _native.device_of(dev):
        h = torch.empty(x.shape, dtype=dt, device=dev) if want_h else None
        out = q = s = None
        if want_out and quant:
            q = torch.empty((rows, D), dtype=torch.int8, device=dev)
            s = torch.empty((rows, 1), dtype=torch.float32, device=dev)
        elif want_out:
            out = torch.empty(x.shape, dtype=dt, device=dev)
        st = L.b200q_block_norm(
            x2.data_ptr(), ldx, yp, ldy, code, KINDS[post_kind], pw, pwt, ptrs[0][0], ptrs[0][1],
            residual_scale, KINDS[kind], w, wt, ptrs[1][0], ptrs[1][1], ptrs[2][0], ptrs[2][1],
            mdt, per, eps, 0 if h is None else h.data_ptr(), D,
            0 if out is None else out.data_ptr(), D, 0 if q is None else q.data_ptr(), D,
            0 if s is None else s.data_ptr(), rows, D, _raw_stream(dev.index))
        if st:
            _native._check(st)
    return h, out, q, s


def norm_modulate(x, weight=None, scale=None, shift=None, kind="rms", eps=1e-6):
    """The norm before a block: norm(x) * weight * (1 + scale) + shift, like x."""
    return _run(x, None, None, None, "none", 1.0, weight, scale, shift, kind, eps, False, False,
                True)[1]


def norm_modulate_quant_i8(x, weight=None, scale=None, shift=None, kind="rms", eps=1e-6):
    """``norm_modulate`` as INT8: (codes [rows, D], scales [rows, 1] fp32)."""
    return _run(x, None, None, None, "none", 1.0, weight, scale, shift, kind, eps, True, False,
                True)[2:]


def gated_residual(residual, y, gate=None, post_weight=None, post_kind="none",
                   residual_scale=1.0, eps=1e-6):
    """The end of a block: residual_scale * residual + gate * (norm_post(y) * post_weight)."""
    return _run(residual, y, gate, post_weight, post_kind, residual_scale, None, None, None,
                "none", eps, False, True, False)[0]


def gated_residual_norm(residual, y, gate=None, post_weight=None, post_kind="none",
                        residual_scale=1.0, weight=None, scale=None, shift=None, kind="rms",
                        eps=1e-6):
    """``gated_residual`` and the next block's ``norm_modulate`` in one pass: (h, out)."""
    return _run(residual, y, gate, post_weight, post_kind, residual_scale, weight, scale, shift,
                kind, eps, False, True, True)[:2]


def gated_residual_norm_quant_i8(residual, y, gate=None, post_weight=None, post_kind="none",
                                 residual_scale=1.0, weight=None, scale=None, shift=None,
                                 kind="rms", eps=1e-6):
    """``gated_residual_norm`` with INT8 codes out: (h, codes [rows, D], scales [rows, 1])."""
    r = _run(residual, y, gate, post_weight, post_kind, residual_scale, weight, scale, shift, kind,
             eps, True, True, True)
    return r[0], r[2], r[3]


_LIB = torch.library.Library("b200q", "FRAGMENT")


def _register():
    pre = "Tensor? weight=None, Tensor? scale=None, Tensor? shift=None, str kind='rms', float eps=1e-06"
    post = ("Tensor residual, Tensor y, Tensor? gate=None, Tensor? post_weight=None, "
            "str post_kind='none', float residual_scale=1.0")

    def codes(x):
        rows = x.numel() // x.shape[-1]
        return (x.new_empty((rows, x.shape[-1]), dtype=torch.int8),
                x.new_empty((rows, 1), dtype=torch.float32))

    for fn, schema, fake in (
            (norm_modulate, f"(Tensor x, {pre}) -> Tensor", lambda x, *a, **k: torch.empty_like(x)),
            (norm_modulate_quant_i8, f"(Tensor x, {pre}) -> (Tensor, Tensor)",
             lambda x, *a, **k: codes(x)),
            (gated_residual, f"({post}, float eps=1e-06) -> Tensor",
             lambda x, *a, **k: torch.empty_like(x)),
            (gated_residual_norm, f"({post}, {pre}) -> (Tensor, Tensor)",
             lambda x, *a, **k: (torch.empty_like(x), torch.empty_like(x))),
            (gated_residual_norm_quant_i8, f"({post}, {pre}) -> (Tensor, Tensor, Tensor)",
             lambda x, *a, **k: (torch.empty_like(x), *codes(x)))):
        name = fn.__name__
        _LIB.define(name + schema)
        _LIB.impl(name, fn, "CUDA")
        torch.library.register_fake(f"b200q::{name}", fake, lib=_LIB)


_register()
