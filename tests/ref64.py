"""Plain 64-bit forms of the low-bit decode operators, on the CPU."""
import math

import torch

# Largest relative error of one rounding to the type.
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def w4_codes(w):
    """[N, K/2] bytes -> [N, K] codes."""
    return torch.stack((w & 15, w >> 4), -1).reshape(w.shape[0], -1)


def w4_weight(w, scales, zeros=None):
    c = w4_codes(w).double()
    G = c.shape[1] // scales.shape[1]
    z = torch.full(scales.shape, 8.0, dtype=torch.float64) if zeros is None else zeros.double()
    return (c - z.repeat_interleave(G, 1)) * scales.double().repeat_interleave(G, 1)


def gelu_tanh(y):
    return y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))


def gelu_erf(y):
    return 0.5 * y * torch.erfc(-y / math.sqrt(2))


def w4_linear(x, w, scales, zeros=None, bias=None, act=None):
    """(out, sum |x||W|) in 64 bits."""
    W = w4_weight(w, scales, zeros)
    y = x.double() @ W.t()
    if bias is not None:
        y = y + bias.double()
    size = x.double().abs() @ W.abs().t()
    return {"gelu_tanh": gelu_tanh, "gelu": gelu_erf}.get(act, lambda v: v)(y), size


def unit_rows(v, kind, eps):
    if kind == "none":
        return v
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    return v / ((v * v).mean(-1, keepdim=True) + eps).sqrt()


def block_norm(x, y=None, gate=None, post_weight=None, post_kind="none", residual_scale=1.0,
               weight=None, scale=None, shift=None, kind="rms", eps=1e-6):
    """(h, out) of rows [R, D]; gate, scale, shift [B, D] with R split evenly over B."""
    def per_row(t):
        t = t.double().reshape(-1, x.shape[-1])
        return t.repeat_interleave(x.shape[0] // t.shape[0], 0)

    h = x.double()
    if y is not None:
        u = unit_rows(y.double(), post_kind, eps)
        u = u if post_weight is None else u * post_weight.double()
        h = residual_scale * h + (u if gate is None else u * per_row(gate))
    o = unit_rows(h, kind, eps)
    o = o if weight is None else o * weight.double()
    o = o if scale is None else o * (1 + per_row(scale))
    return h, (o if shift is None else o + per_row(shift))


def append(x, codes, scale, table, start, counts):
    """Sequence by sequence: new codes before rounding [pages, H, T, D] (64 bits)
    and scales, from the cache's state before the call."""
    T = codes.shape[2]
    c, s = codes.double(), scale.double()
    for b in range(x.shape[0]):
        p, n, done = int(start[b]), int(counts[b]), 0
        while done < n:
            page, at = int(table[b, (p + done) // T]), (p + done) % T
            take = min(T - at, n - done)
            part = x[b, :, done:done + take].double()
            before = s[page] if at else torch.zeros(x.shape[1], dtype=torch.float64)
            new = torch.maximum(before, part.abs().amax((1, 2)) / 127)
            d = torch.where(new > 0, new, torch.ones_like(new))[:, None, None]
            c[page, :, :at] = c[page, :, :at] * (before[:, None, None] / d)
            c[page, :, at:at + take] = part / d
            s[page] = new
            done += take
    return c, s


def read(codes, scale, table, b, first, n):
    """Values [H, n, D] of tokens first .. first + n - 1 of sequence b."""
    T = codes.shape[2]
    out = torch.zeros(codes.shape[1], n, codes.shape[3], dtype=torch.float64)
    for i in range(n):
        page, at = int(table[b, (first + i) // T]), (first + i) % T
        out[:, i] = codes[page, :, at].double() * scale[page].double()[:, None]
    return out


def attention(q, codes_k, codes_v, scale_k, scale_v, table, lens, causal, sm=None):
    """(out, lse, sum P |v| / sum P)."""
    B, Hq, Tq, D = q.shape
    H = codes_k.shape[1]
    G = Hq // H
    sm = D ** -0.5 if sm is None else sm
    out = torch.zeros(B, Hq, Tq, D, dtype=torch.float64)
    size = torch.zeros_like(out)
    lse = torch.full((B, Hq, Tq), -math.inf, dtype=torch.float64)
    for b in range(B):
        n = int(lens[b])
        if n == 0:
            continue
        k, v = (read(c, s, table, b, 0, n) for c, s in ((codes_k, scale_k), (codes_v, scale_v)))
        k, v = k.repeat_interleave(G, 0), v.repeat_interleave(G, 0)
        s = q[b].double() @ k.transpose(1, 2) * sm
        if causal:
            see = torch.arange(n)[None] <= n - Tq + torch.arange(Tq)[:, None]
            s = torch.where(see, s, torch.full_like(s, -math.inf))
        m = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
        total = p.sum(-1, keepdim=True)
        d = torch.where(total == 0, torch.ones_like(total), total)
        out[b], size[b] = p @ v / d, p @ v.abs() / d
        lse[b] = (m + total.log()).squeeze(-1)
    return out, lse, size
