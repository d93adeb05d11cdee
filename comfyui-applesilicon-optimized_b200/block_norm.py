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

_block_norm = None


def _run(*args):
    """bindings.block_norm: x, y, gate, post_weight, post_kind, residual_scale, weight,
    scale, shift, kind, eps, quant, want_out."""
    global _block_norm
    if _block_norm is None:
        _block_norm = _native.bindings().block_norm
    return _block_norm(*args)


def norm_modulate(x, weight=None, scale=None, shift=None, kind="rms", eps=1e-6):
    """The norm before a block: norm(x) * weight * (1 + scale) + shift, like x."""
    return _run(x, None, None, None, "none", 1.0, weight, scale, shift, kind, eps, False, True)


def norm_modulate_quant_i8(x, weight=None, scale=None, shift=None, kind="rms", eps=1e-6):
    """``norm_modulate`` as INT8: (codes [rows, D], scales [rows, 1] fp32)."""
    return _run(x, None, None, None, "none", 1.0, weight, scale, shift, kind, eps, True, True)


def gated_residual(residual, y, gate=None, post_weight=None, post_kind="none",
                   residual_scale=1.0, eps=1e-6):
    """The end of a block: residual_scale * residual + gate * (norm_post(y) * post_weight)."""
    return _run(residual, y, gate, post_weight, post_kind, residual_scale, None, None, None,
                "none", eps, False, False)


def gated_residual_norm(residual, y, gate=None, post_weight=None, post_kind="none",
                        residual_scale=1.0, weight=None, scale=None, shift=None, kind="rms",
                        eps=1e-6):
    """``gated_residual`` and the next block's ``norm_modulate`` in one pass: (h, out)."""
    return _run(residual, y, gate, post_weight, post_kind, residual_scale, weight, scale, shift,
                kind, eps, False, True)


def gated_residual_norm_quant_i8(residual, y, gate=None, post_weight=None, post_kind="none",
                                 residual_scale=1.0, weight=None, scale=None, shift=None,
                                 kind="rms", eps=1e-6):
    """``gated_residual_norm`` with INT8 codes out: (h, codes [rows, D], scales [rows, 1])."""
    return _run(residual, y, gate, post_weight, post_kind, residual_scale, weight, scale, shift,
                kind, eps, True, True)


_LIB = torch.library.Library("b200q", "FRAGMENT")


def _register():
    pre = "Tensor? weight=None, Tensor? scale=None, Tensor? shift=None, str kind='rms', float eps=1e-06"
    post = ("Tensor residual, Tensor y, Tensor? gate=None, Tensor? post_weight=None, "
            "str post_kind='none', float residual_scale=1.0")

    def like(x):  # contiguous, whatever x's strides
        return x.new_empty(x.shape)

    def codes(x):
        rows = x.numel() // x.shape[-1]
        return (x.new_empty((rows, x.shape[-1]), dtype=torch.int8),
                x.new_empty((rows, 1), dtype=torch.float32))

    for fn, schema, fake in (
            (norm_modulate, f"(Tensor x, {pre}) -> Tensor", lambda x, *a, **k: like(x)),
            (norm_modulate_quant_i8, f"(Tensor x, {pre}) -> (Tensor, Tensor)",
             lambda x, *a, **k: codes(x)),
            (gated_residual, f"({post}, float eps=1e-06) -> Tensor",
             lambda x, *a, **k: like(x)),
            (gated_residual_norm, f"({post}, {pre}) -> (Tensor, Tensor)",
             lambda x, *a, **k: (like(x), like(x))),
            (gated_residual_norm_quant_i8, f"({post}, {pre}) -> (Tensor, Tensor, Tensor)",
             lambda x, *a, **k: (like(x), *codes(x)))):
        name = fn.__name__
        _LIB.define(name + schema)
        _LIB.impl(name, fn, "CUDA")
        torch.library.register_fake(f"b200q::{name}", fake, lib=_LIB)


_register()
