"""Measured cases of the low-bit decode operators: 4-bit weight linears, the
norms before and after a block with gate and residual scale, and the paged
8-bit KV cache (append, read back, attention).

``run`` computes an operator in elementary torch operations in 32 bits where
``own`` is false, and calls the pack's public functions where it is true.
``exact`` gives the same outputs in 64 bits from the definitions.

Sizes: 5120 and 13824 are the widths of the Wan-shaped block that ``bench.py``
runs (65,520 tokens); the cache sizes are generic (128-wide heads, 64-token
blocks).
"""
import importlib.util
import math
import os
import sys

import torch

own = False

DEV = "cuda"
_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _pack():
    """The pack, imported from its directory under the name ``b200q``."""
    mod = sys.modules.get("b200q")
    if mod is None:
        os.environ.setdefault("B200Q_NO_BOOTSTRAP", "1")
        d = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                         "comfyui-applesilicon-optimized_b200")
        spec = importlib.util.spec_from_file_location("b200q", os.path.join(d, "__init__.py"),
                                                      submodule_search_locations=[d])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["b200q"] = mod
        spec.loader.exec_module(mod)
    return mod


# ------------------------------------------------------------------ cases
def listed():
    return [
        # 4-bit weight linears
        # the attention output projection of one decoded token: the smallest call
        {"name": "w4 out, 1 token", "op": "w4", "m": 1, "k": 5120, "n": 5120, "group": 128,
         "zeros": False, "bias": False, "act": "none", "dtype": "bf16"},
        # the up projection of one decoded token, zero points and a fused bias + GELU
        {"name": "w4 up, 1 token", "op": "w4", "m": 1, "k": 5120, "n": 13824, "group": 64,
         "zeros": True, "bias": True, "act": "gelu_tanh", "dtype": "bf16"},
        # the down projection of a batch of 16 sequences in fp16
        {"name": "w4 down, 16 tokens", "op": "w4", "m": 16, "k": 13824, "n": 5120, "group": 128,
         "zeros": True, "bias": True, "act": "none", "dtype": "f16"},
        # the up projection of a ragged prompt: tensor-bound
        {"name": "w4 up, 2047 tokens", "op": "w4", "m": 2047, "k": 5120, "n": 13824, "group": 128,
         "zeros": False, "bias": True, "act": "gelu_tanh", "dtype": "bf16"},
        # norms before and after a block
        # one decoded token: post norm, gate, residual and the next block's norm in one call
        {"name": "norm after+before, 1 row", "op": "norm", "batch": 1, "tokens": 1, "dim": 5120,
         "after": True, "post": "rms", "pre": "rms", "mods": "same", "quant": False,
         "dtype": "bf16"},
        # the whole Wan-shaped sequence: gate and residual, then LayerNorm with fp32 modulation
        {"name": "norm after+before, 65520 rows", "op": "norm", "batch": 2, "tokens": 32760,
         "dim": 5120, "after": True, "post": "none", "pre": "layer", "mods": "f32", "quant": False,
         "dtype": "bf16"},
        # the norm in front of an INT8 linear, its codes and scales straight out, ragged rows
        {"name": "norm before, int8 out", "op": "norm", "batch": 3, "tokens": 1367, "dim": 5120,
         "after": False, "post": "none", "pre": "layer", "mods": "same", "quant": True,
         "dtype": "bf16"},
        # the 8-bit cache: write, then read the touched blocks back
        # one new token for each of 64 sequences
        {"name": "kv8 append, 64 x 1", "op": "append", "batch": 64, "tokens": 1, "count_min": 1,
         "start_min": 0, "start_max": 4095, "heads": 8, "dim": 128, "block": 64, "dtype": "bf16"},
        # two ragged prompts written at once behind what is there already
        {"name": "kv8 append, 2 x 8191", "op": "append", "batch": 2, "tokens": 8191,
         "count_min": 5003, "start_min": 0, "start_max": 1000, "heads": 8, "dim": 128, "block": 64,
         "dtype": "f16"},
        # attention over the cache
        # one sequence, one token: too few rows to fill the GPU without splitting the length
        {"name": "kv8 attention, 1 x 1", "op": "attention", "batch": 1, "q_tokens": 1,
         "len_min": 8193, "len_max": 8193, "kv_heads": 8, "group": 5, "dim": 128, "block": 64,
         "causal": True, "dtype": "bf16"},
        # a ragged serving batch up to 32768 tokens, one of them still empty
        {"name": "kv8 attention, 32 x 1", "op": "attention", "batch": 32, "q_tokens": 1,
         "len_min": 0, "len_max": 32767, "kv_heads": 8, "group": 8, "dim": 128, "block": 64,
         "causal": True, "dtype": "bf16"},
        # a chunk of a prompt against what is cached
        {"name": "kv8 attention, 4 x 129", "op": "attention", "batch": 4, "q_tokens": 129,
         "len_min": 4001, "len_max": 12001, "kv_heads": 8, "group": 5, "dim": 128, "block": 64,
         "causal": True, "dtype": "f16"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["w4", "norm", "append", "attention"])
    dt = rng.choice(["bf16", "f16"])
    if op == "w4":
        g = rng.choice([32, 64, 128])
        return {"op": op, "m": _log(rng, 1, 2000), "k": g * _log(rng, -(-1024 // g), 13824 // g),
                "n": _log(rng, 1000, 5120), "group": g, "zeros": rng.random() < 0.5,
                "bias": rng.random() < 0.5, "act": rng.choice(["none", "gelu_tanh"]), "dtype": dt}
    if op == "norm":
        after = rng.random() < 0.6
        return {"op": op, "batch": rng.choice([1, 2, 3]), "tokens": _log(rng, 1, 20000),
                "dim": rng.choice([8 * _log(rng, 64, 640), _log(rng, 512, 5120)]), "after": after,
                "post": rng.choice(["none", "rms", "layer"]) if after else "none",
                "pre": rng.choice(["rms", "layer"]), "mods": rng.choice(["same", "f32"]),
                "quant": rng.random() < 0.4, "dtype": dt}
    if op == "append":
        t = _log(rng, 1, 6000)
        return {"op": op, "batch": rng.randint(1, 4) if t > 64 else rng.randint(1, 64),
                "tokens": t, "count_min": rng.randint(t // 2, t), "start_min": 0,
                "start_max": rng.randint(0, 2000), "heads": rng.choice([1, 2, 8]),
                "dim": rng.choice([64, 128]), "block": rng.choice([16, 32, 64, 128]), "dtype": dt}
    t = rng.choice([1, 1, 2, 5, 17, 65])
    hi = _log(rng, 70, 30000)
    heads = rng.choice([1, 2, 4, 8])
    return {"op": op, "batch": rng.randint(1, 16 if t < 16 else 4), "q_tokens": t,
            "len_min": rng.randint(0, hi), "len_max": hi, "kv_heads": heads,
            "group": rng.choice([1, 2, 3, 4, 7, 8]), "dim": rng.choice([64, 128]),
            "block": rng.choice([16, 32, 64, 128]), "causal": rng.random() < 0.7, "dtype": dt}


def _spread(lo, hi, n):
    """n whole numbers from lo to hi: the batch's lengths or positions."""
    return [lo + (hi - lo) * i // max(n - 1, 1) if n > 1 else hi for i in range(n)]


def _cdiv(a, b):
    return -(-a // b)


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    dt = _DT[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    def shuffled(values):
        order = torch.randperm(len(values), generator=g, device=DEV)
        return torch.tensor(values, dtype=torch.int32, device=DEV)[order].contiguous()

    st = {"case": case}
    if case["op"] == "w4":
        m, k, n, G = case["m"], case["k"], case["n"], case["group"]
        # a checkpoint's weight: N(0, 0.02) rounded to 4 bits group by group
        w = (randn(n, k) * 0.02).view(n, k // G, G)
        if case["zeros"]:
            lo, hi = w.amin(-1, keepdim=True), w.amax(-1, keepdim=True)
            s = ((hi - lo) / 15).to(dt).float()
            z = (-lo / s).round().clamp(0, 15)
            st["zeros"] = z.view(n, k // G).to(torch.uint8)
        else:
            s, z = (w.abs().amax(-1, keepdim=True) / 7).to(dt).float(), 8.0
            st["zeros"] = None
        c = ((w / s).round() + z).clamp(0, 15).to(torch.uint8).view(n, k // 2, 2)
        st["w"] = (c[..., 0] | (c[..., 1] << 4)).contiguous()
        st["scales"] = s.view(n, k // G).to(dt)
        st["x"] = randn(m, k).to(dt)
        st["bias"] = (randn(n) * 0.1).to(dt) if case["bias"] else None
    elif case["op"] == "norm":
        b, t, d = case["batch"], case["tokens"], case["dim"]
        mdt = torch.float32 if case["mods"] == "f32" else dt
        # the modulation of a block comes as one [batch, 3, dim] tensor
        mods = (randn(b, 3, d) * 0.3).to(mdt)
        st["scale"], st["shift"], st["gate"] = mods[:, 0], mods[:, 1], mods[:, 2]
        st["weight"] = 1 + 0.1 * randn(d)
        st["post_weight"] = 1 + 0.1 * randn(d)
        # a residual stream with a few large channels
        st["x"] = (randn(b, t, d) * (1 + 8 * (randn(d) > 2.5))).to(dt)
        st["y"] = (randn(b, t, d) * 0.7).to(dt) if case["after"] else None
    elif case["op"] == "append":
        B, S, H, D, T = (case[k] for k in ("batch", "tokens", "heads", "dim", "block"))
        start = _spread(case["start_min"], case["start_max"], B)
        nb = _cdiv(case["start_max"] + S, T)
        pages = B * nb
        st["table"] = torch.randperm(pages, generator=g, device=DEV).to(torch.int32).view(B, nb)
        st["start"] = shuffled(start)
        st["counts"] = shuffled(_spread(case["count_min"], S, B))
        st["k"], st["v"] = randn(B, H, S, D).to(dt), randn(B, H, S, D).to(dt)
        for x in "kv":
            st[x + "_codes"] = torch.randint(-127, 128, (pages, H, T, D), generator=g, device=DEV,
                                             dtype=torch.int8)
            st[x + "_scale"] = 0.01 + 0.02 * torch.rand(pages, H, generator=g, device=DEV)
        # what is read back: the touched blocks, from their first token on
        st["first"] = (st["start"] // T * T).to(torch.int32)
        st["rcounts"] = (st["start"] + st["counts"] - st["first"]).to(torch.int32)
        st["rmax"] = T - 1 + S
    else:
        B, Tq, H, D, T = (case[k] for k in ("batch", "q_tokens", "kv_heads", "dim", "block"))
        nb = max(1, _cdiv(case["len_max"], T))
        pages = B * nb
        st["table"] = torch.randperm(pages, generator=g, device=DEV).to(torch.int32).view(B, nb)
        st["lens"] = shuffled(_spread(case["len_min"], case["len_max"], B))
        st["q"] = randn(B, H * case["group"], Tq, D).to(dt)
        for x in "kv":
            c = torch.empty(pages, H, T, D, dtype=torch.int8, device=DEV)
            for i in range(0, pages, 4096):  # N(0, 32) codes, as a block's largest value gets 127
                c[i:i + 4096] = (randn(*c[i:i + 4096].shape) * 32).clamp_(-127, 127).round_()
            st[x + "_codes"] = c
            st[x + "_scale"] = 0.02 + 0.02 * torch.rand(pages, H, generator=g, device=DEV)
    return st


# ------------------------------------------------------------------ the pack's calls
def _run_own(st):
    case, b = st["case"], _pack()
    if case["op"] == "w4":
        from b200q import w4
        return w4.w4a16_linear(st["x"], st["w"], st["scales"], st["zeros"], st["bias"], case["act"])
    if case["op"] == "norm":
        from b200q import block_norm
        if not case["after"]:
            f = block_norm.norm_modulate_quant_i8 if case["quant"] else block_norm.norm_modulate
            out = f(st["x"], st["weight"], st["scale"], st["shift"], case["pre"], 1e-6)
            return _values(out, st["x"]) if case["quant"] else out
        f = (block_norm.gated_residual_norm_quant_i8 if case["quant"]
             else block_norm.gated_residual_norm)
        post_weight = None if case["post"] == "none" else st["post_weight"]
        out = f(st["x"], st["y"], st["gate"], post_weight, case["post"], 0.9, st["weight"],
                st["scale"], st["shift"], case["pre"], 1e-6)
        return (out[0], _values(out[1:], st["x"])) if case["quant"] else out
    from b200q import kv8
    if case["op"] == "append":
        kv8.kv8_append(st["k"], st["v"], st["k_codes"], st["v_codes"], st["k_scale"],
                       st["v_scale"], st["table"], st["start"], st["counts"])
        k, v = kv8.kv8_gather(st["k_codes"], st["v_codes"], st["k_scale"], st["v_scale"],
                              st["table"], st["first"], st["rcounts"], st["rmax"], st["k"].dtype)
        return {"k": k, "v": v, "k_scale": st["k_scale"], "v_scale": st["v_scale"]}
    return kv8.kv8_attention(st["q"], st["k_codes"], st["v_codes"], st["k_scale"], st["v_scale"],
                             st["table"], st["lens"], case["causal"], max_len=case["len_max"])


def _values(qs, x):
    """What the 8-bit codes stand for, in the activation's type (one launch)."""
    return torch.mul(qs[0], qs[1], out=torch.empty(qs[0].shape, dtype=x.dtype, device=x.device))


# ------------------------------------------------------------------ the plain forms
def _plain_w4(st):
    x, w, s, case = st["x"], st["w"], st["scales"].float(), st["case"]
    n, G = w.shape[0], case["group"]
    c = torch.stack((w & 15, w >> 4), -1).view(n, -1, G).float()
    z = 8.0 if st["zeros"] is None else st["zeros"].float().unsqueeze(-1)
    y = x.float() @ ((c - z) * s.unsqueeze(-1)).view(n, -1).t()
    if st["bias"] is not None:
        y = y + st["bias"].float()
    if case["act"] == "gelu_tanh":
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    return y.to(x.dtype)


def _plain_unit(v, kind):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    return v if kind == "none" else v * torch.rsqrt((v * v).mean(-1, keepdim=True) + 1e-6)


def _plain_norm(st):
    case, x, d = st["case"], st["x"], st["case"]["dim"]
    h = x.float()
    if case["after"]:
        y = _plain_unit(st["y"].float(), case["post"])
        if case["post"] != "none":
            y = y * st["post_weight"]
        h = 0.9 * h + st["gate"].float().unsqueeze(1) * y
    o = _plain_unit(h, case["pre"]) * st["weight"]
    o = o * (1 + st["scale"].float().unsqueeze(1)) + st["shift"].float().unsqueeze(1)
    if case["quant"]:
        o = o.view(-1, d)
        s = o.abs().amax(-1, keepdim=True) / 127
        o = _values(((o / s).round().clamp(-127, 127).to(torch.int8), s), x)
    else:
        o = o.to(x.dtype)
    return (h.to(x.dtype), o) if case["after"] else o


def _plain_store(x, codes, scale, st):
    """Writes x [B, H, S, D] into the cache's blocks, all touched blocks at once."""
    B, H, S, D = x.shape
    T, start, cnt = codes.shape[2], st["start"].long(), st["counts"].long()
    nb = _cdiv(T - 1 + S, T)
    b0, off = start // T, start % T
    j = torch.arange(nb * T, device=DEV)
    src = j - off[:, None]                                      # [B, nb*T] the new token there
    new = ((src >= 0) & (src < cnt[:, None])).view(B, nb, 1, T, 1)
    old = (src < 0).view(B, nb, 1, T, 1)
    idx = src.clamp(0, S - 1)[:, None, :, None].expand(B, H, nb * T, D)
    xb = x.float().gather(2, idx).view(B, H, nb, T, D).transpose(1, 2)  # [B, nb, H, T, D]
    blk = (b0[:, None] + torch.arange(nb, device=DEV)).clamp(max=st["table"].shape[1] - 1)
    page = st["table"].long().gather(1, blk)                    # [B, nb]
    oc, held = codes[page].float(), old.any(3).view(B, nb, 1)
    os_ = torch.where(held, scale[page], 0.0)                   # [B, nb, H]
    amax = torch.where(new, xb.abs(), 0.0).amax((3, 4))
    ns = torch.maximum(os_, amax / torch.full_like(amax, 127.0))
    div = torch.where(ns > 0, ns, 1.0)[..., None, None]
    c = torch.where(new, xb / div, oc * (os_[..., None, None] / div))
    c = torch.where(new | old, c.round().clamp(-127, 127), oc).to(torch.int8)
    hit = new.any(3).view(B, nb)                                # blocks with a new token
    codes[page[hit]] = c[hit]
    scale[page[hit]] = ns[hit]


def _plain_read(codes, scale, table, first, counts, rmax, dt):
    T, H, D = codes.shape[2], codes.shape[1], codes.shape[3]
    B, nb = table.shape[0], _cdiv(rmax, T)
    blk = (first.long()[:, None] // T + torch.arange(nb, device=DEV)).clamp(max=table.shape[1] - 1)
    page = table.long().gather(1, blk)
    x = codes[page].float() * scale[page][..., None, None]
    x = x.transpose(1, 2).reshape(B, H, nb * T, D)[:, :, :rmax]
    live = torch.arange(rmax, device=DEV) < counts[:, None]
    return torch.where(live[:, None, :, None], x, 0.0).to(dt)


def _plain_append(st):
    _plain_store(st["k"], st["k_codes"], st["k_scale"], st)
    _plain_store(st["v"], st["v_codes"], st["v_scale"], st)
    where = (st["table"], st["first"], st["rcounts"], st["rmax"], st["k"].dtype)
    return {"k": _plain_read(st["k_codes"], st["k_scale"], *where),
            "v": _plain_read(st["v_codes"], st["v_scale"], *where),
            "k_scale": st["k_scale"], "v_scale": st["v_scale"]}


def _plain_attention(st):
    q, case, table, lens = st["q"].float(), st["case"], st["table"].long(), st["lens"]
    B, Hq, Tq, D = q.shape
    H, T = case["kv_heads"], case["block"]
    L = table.shape[1] * T
    k = (st["k_codes"][table].float() * st["k_scale"][table][..., None, None]).transpose(1, 2)
    k = k.reshape(B, H, L, D)
    s = q.view(B, H, -1, D) @ k.transpose(-1, -2) / math.sqrt(D)
    del k
    last = lens[:, None] - (Tq if case["causal"] else 1)        # the last position query 0 sees
    last = last + (torch.arange(Tq, device=DEV) if case["causal"] else torch.zeros(Tq, device=DEV))
    see = torch.arange(L, device=DEV) <= last[:, :, None]       # [B, Tq, L]
    s = torch.where(see[:, None, None], s.view(B, H, -1, Tq, L), -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.where(see[:, None, None], torch.exp(s - m), 0.0)
    total = p.sum(-1, keepdim=True)
    v = (st["v_codes"][table].float() * st["v_scale"][table][..., None, None]).transpose(1, 2)
    v = torch.where(torch.arange(L, device=DEV)[:, None] < lens[:, None, None, None],
                    v.reshape(B, H, L, D), 0.0)
    o = p.view(B, H, -1, L) @ v / torch.where(total > 0, total, 1.0).view(B, H, -1, 1)
    lse = torch.where(total > 0, m + torch.log(total), -math.inf)
    return o.view(B, Hq, Tq, D).to(st["q"].dtype), lse.view(B, Hq, Tq)


def run(state):
    if own:
        return _run_own(state)
    return {"w4": _plain_w4, "norm": _plain_norm, "append": _plain_append,
            "attention": _plain_attention}[state["case"]["op"]](state)


# ------------------------------------------------------------------ work
def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "w4":
        m, k, n, G = case["m"], case["k"], case["n"], case["group"]
        by = (n * k // 2 + n * (k // G) * (es + case["zeros"]) + es * (m * k + m * n)
              + es * n * case["bias"])
        return {"bytes": by, "flops": 2 * m * n * k}
    if case["op"] == "norm":
        e = case["batch"] * case["tokens"] * case["dim"]
        out = e * (1 + 1 + es if case["quant"] else es)  # codes written, read for their values
        mods = (2 + case["after"]) * case["batch"] * case["dim"] * (4 if case["mods"] == "f32" else es)
        by = e * es * (3 if case["after"] else 1) + out + mods
        return {"bytes": by, "flops": e * (14 if case["after"] else 8)}
    B, D, T = case["batch"], case["dim"], case["block"]
    if case["op"] == "append":
        H, S = case["heads"], case["tokens"]
        new = sum(_spread(case["count_min"], S, B)) * H * D * 2
        back = B * (T - 1 + S) * H * D * 2 * es
        return {"bytes": new * (es + 2) + back, "flops": 4 * new}
    H, Tq, G = case["kv_heads"], case["q_tokens"], case["group"]
    lens = _spread(case["len_min"], case["len_max"], B)
    seen = sum(max(0, n - Tq + 1 + i) if case["causal"] else n for n in lens for i in range(Tq))
    tok, blocks = sum(lens), sum(_cdiv(n, T) for n in lens)
    by = 2 * tok * H * D + 8 * blocks * H + B * H * G * Tq * (2 * es * D + 4)
    return {"bytes": by, "flops": 4 * seen * H * G * D}


# ------------------------------------------------------------------ 64 bits
def _f64(t):
    return None if t is None else t.to(torch.float64)


def _exact_w4(st):
    w, s, case = st["w"].to(torch.int64), _f64(st["scales"]), st["case"]
    n, half = w.shape
    codes = torch.empty(n, 2 * half, dtype=torch.float64, device=DEV)
    codes[:, 0::2] = (w % 16).double()
    codes[:, 1::2] = (w // 16).double()
    zero = torch.full_like(s, 8.0) if st["zeros"] is None else _f64(st["zeros"])
    G = case["group"]
    weight = (codes - zero.repeat_interleave(G, 1)) * s.repeat_interleave(G, 1)
    y = torch.einsum("mk,nk->mn", _f64(st["x"]), weight)
    if st["bias"] is not None:
        y += _f64(st["bias"])
    if case["act"] == "gelu_tanh":
        u = 2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)
        y = y * torch.sigmoid(u)  # (1 + tanh(u/2)) / 2
    return y


def _exact_unit(v, kind):
    if kind == "none":
        return v
    if kind == "rms":
        return v / (v.pow(2).sum(-1, keepdim=True) / v.shape[-1] + 1e-6).sqrt()
    return (v - v.mean(-1, keepdim=True)) / (v.var(-1, keepdim=True, unbiased=False) + 1e-6).sqrt()


def _exact_norm(st):
    case = st["case"]
    hs, outs = [], []
    for b in range(case["batch"]):
        h = _f64(st["x"][b])
        if case["after"]:
            y = _exact_unit(_f64(st["y"][b]), case["post"])
            y = y * _f64(st["post_weight"]) if case["post"] != "none" else y
            h = 0.9 * h + _f64(st["gate"][b]) * y
        o = _exact_unit(h, case["pre"]) * _f64(st["weight"]) * (1 + _f64(st["scale"][b]))
        o += _f64(st["shift"][b])
        if case["quant"]:
            s = o.abs().amax(-1, keepdim=True) / 127
            o = (o / s).round() * s
        hs.append(h)
        outs.append(o)
    out = torch.cat(outs) if case["quant"] else torch.stack(outs)
    return (torch.stack(hs), out) if case["after"] else out


def _exact_append(st):
    """Sequence by sequence and block by block, on the host."""
    T = st["k_codes"].shape[2]
    got = {}
    for x in "kv":
        codes, scale = _f64(st[x + "_codes"]).cpu(), _f64(st[x + "_scale"]).cpu()
        new, table = _f64(st[x]).cpu(), st["table"].cpu().tolist()
        B, H, _, D = new.shape
        back = torch.zeros(B, H, st["rmax"], D, dtype=torch.float64)
        for b, (p0, n) in enumerate(zip(st["start"].tolist(), st["counts"].tolist())):
            done = 0
            while done < n:
                pos = p0 + done
                page, at = table[b][pos // T], pos % T
                take = min(T - at, n - done)
                part = new[b, :, done:done + take]
                before = scale[page] if at else torch.zeros(H, dtype=torch.float64)
                s = torch.maximum(before, part.abs().amax((1, 2)) / 127)
                d = torch.where(s > 0, s, 1.0)[:, None, None]
                codes[page, :, :at] = (codes[page, :, :at] * (before[:, None, None] / d)).round()
                codes[page, :, at:at + take] = (part / d).round()
                scale[page] = s
                done += take
            first, n_back = st["first"][b].item(), st["rcounts"][b].item()
            for i in range(0, n_back, T):
                page, take = table[b][(first + i) // T], min(T, n_back - i)
                back[b, :, i:i + take] = codes[page, :, :take] * scale[page][:, None, None]
        got[x], got[x + "_scale"] = back, scale
    return got


def _exact_attention(st):
    case, q = st["case"], _f64(st["q"])
    B, Hq, Tq, D = q.shape
    G = case["group"]
    out = torch.zeros_like(q)
    lse = torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device=DEV)
    for b, n in enumerate(st["lens"].tolist()):
        pages = st["table"][b].long()[:_cdiv(n, case["block"])]
        for h in range(case["kv_heads"] if n else 0):
            k, v = ((_f64(st[x + "_codes"][pages, h]) * _f64(st[x + "_scale"][pages, h])
                     [:, None, None]).reshape(-1, D)[:n] for x in "kv")
            s = torch.einsum("gtd,ld->gtl", q[b, h * G:(h + 1) * G], k) * D ** -0.5
            if case["causal"]:
                at = torch.arange(n, device=DEV)
                hide = at[None] > (n - Tq + torch.arange(Tq, device=DEV))[:, None]
                s = s.masked_fill(hide, -math.inf)
            e = torch.logsumexp(s, -1)
            p = torch.exp(s - torch.where(torch.isfinite(e), e, 0.0)[..., None])
            out[b, h * G:(h + 1) * G] = p @ v
            lse[b, h * G:(h + 1) * G] = e
    return out, lse


def exact(case, seed):
    return {"w4": _exact_w4, "norm": _exact_norm, "append": _exact_append,
            "attention": _exact_attention}[case["op"]](prepare(case, seed))
