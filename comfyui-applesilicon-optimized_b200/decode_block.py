"""A transformer block with 4-bit weights and an 8-bit key/value cache, step by step.

``DecodeBlock`` runs the low-bit operators together as a serving loop does: prompts
and single tokens go through the same call, and nothing is read back to the host, so
a one-token step can be captured in a CUDA graph.

    a   = norm(h)                                      block_norm.norm_modulate
    qkv = a . Wqkv^T                                   w4.w4a16_linear
    q, k = RoPE(rmsnorm(q)), RoPE(rmsnorm(k))          torch.ops.b200q.rms_rope_partial_
    cache <- k, v                                      kv8.kv8_append
    o   = attention(q, cache) . Wo^T                   kv8.kv8_attention, w4.w4a16_linear
    h, a = h + gate_a * norm(o), next norm             block_norm.gated_residual_norm
    m   = silu(gate) * up of a . Wup^T                 w4, torch.ops.b200q.silu_mul_split
    h   = h + gate_m * norm(m . Wdown^T)               w4, block_norm.gated_residual
"""
import torch

from . import block_norm, kv8, w4
from ._patches import _native


class DecodeBlock:
    """One block: ``heads`` query heads of 128 over ``kv_heads``, bf16 activations.

    Weights come as [N, K] float tensors and are rounded to 4 bits once, here.
    ``weights``: qkv [(heads + 2 kv_heads) * 128, D], out [D, heads * 128], up [2F, D]
    (gate rows, then up rows), down [D, F].  ``norms``: pre_attn, post_attn, pre_mlp,
    post_mlp [D] and q, k [128] (fp32 norm weights).  ``gate_attn``, ``gate_mlp`` [D] or
    None scale what a block adds to the residual stream."""

    HEAD_DIM = 128

    def __init__(self, weights, norms, heads, kv_heads, gate_attn=None, gate_mlp=None,
                 group=128, symmetric=True, eps=1e-6):
        if heads % kv_heads:
            raise ValueError("heads must be a multiple of kv_heads")
        self.heads, self.kv_heads, self.eps = heads, kv_heads, eps
        self.w = {n: w4.w4_quantize(t, group, symmetric, torch.bfloat16)
                  for n, t in weights.items()}
        self.norm = norms
        self.gate_attn, self.gate_mlp = gate_attn, gate_mlp

    def linear(self, x, name, bias=None):
        return w4.w4a16_linear(x, *self.w[name], bias)

    def rope(self, qk, freqs):
        """RMSNorm and split-half RoPE of qk [B, T, heads + kv_heads, 128] -> q, k
        [B, heads, T, 128].  The kernel works in place on two equal tensors at a time:
        each of the heads / kv_heads groups of q, and k, as [B, kv_heads, T, 128]."""
        B, T, n, d = qk.shape[0], qk.shape[1], self.kv_heads, self.HEAD_DIM
        G = self.heads // n
        x = torch.empty((G + 1 + (G + 1) % 2, B, n, T, d), dtype=qk.dtype, device=qk.device)
        x[:G] = qk[:, :, :self.heads].view(B, T, n, G, d).permute(3, 0, 2, 1, 4)
        x[G] = qk[:, :, self.heads:].transpose(1, 2)
        weights = [self.norm["q"]] * G + [self.norm["k"]] * 2
        for i in range(0, x.shape[0], 2):  # (an even count: a spare one is not read)
            _native.rms_rope_partial_(x[i], x[i + 1], freqs, weights[i], weights[i + 1], self.eps)
        return x[:G].permute(1, 2, 0, 3, 4).reshape(B, self.heads, T, d), x[G]

    def __call__(self, h, cache, freqs):
        """h [B, T, D] bf16 -> h after the block; k and v of the T tokens go into
        ``cache`` (a kv8.KV8Cache) behind what it holds."""
        B, T, D = h.shape
        H, n, d = self.heads, self.kv_heads, self.HEAD_DIM
        a = block_norm.norm_modulate(h, self.norm["pre_attn"], eps=self.eps)
        qkv = self.linear(a, "qkv").view(B, T, H + 2 * n, d)
        q, k = self.rope(qkv[:, :, :H + n], freqs)
        cache.append(k, qkv[:, :, H + n:].transpose(1, 2))
        o = cache.attention(q).transpose(1, 2).reshape(B, T, H * d)
        h, a = block_norm.gated_residual_norm(
            h, self.linear(o, "out"), self.gate_attn, self.norm["post_attn"], "rms", 1.0,
            self.norm["pre_mlp"], eps=self.eps)
        up = self.linear(a, "up").view(B * T, -1)
        m = _native.silu_mul_split(up).view(B, T, -1)
        return block_norm.gated_residual(h, self.linear(m, "down"), self.gate_mlp,
                                         self.norm["post_mlp"], "rms", 1.0, self.eps)
