"""A paged 8-bit key/value cache and the attention that reads it.

``k_codes``, ``v_codes`` [pages, heads, T, D] int8 hold the tokens' values in pages
of T tokens (16, 32, 64 or 128; D 64 or 128), ``k_scale``, ``v_scale`` [pages, heads]
fp32 one scale for each page and head: value = code * scale.  ``block_table``
[B, max_blocks] int32 gives the page of each block of T tokens of a sequence.

* ``kv8_append`` writes new tokens behind each sequence's length.  A block's scale
  only grows: it becomes max(its scale so far, max|new| / 127), and codes already
  there are requantized when it does.
* ``kv8_gather`` reads tokens back as 16-bit or fp32 values.
* ``kv8_attention`` is softmax(q K^T) V over the cache, for one query token or
  many, causal or not, with grouped heads.
* ``KV8Cache`` owns the pool, the tables and the lengths of a batch.

Lengths, positions and tables live on the GPU and nothing is read back, so a
decode step can be captured in a CUDA graph.  Page numbers are checked on the
device: a bad one sets bit 1 of the device status word (``_native.device_status``)
and its tokens are skipped.  Also registered in ``torch.ops.b200q``.
"""
import ctypes

import torch

from ._patches import _native
from ._patches._native import TAG, _DT

BLOCKS = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)
_raw_stream = torch._C._cuda_getCurrentRawStream
_Strides = ctypes.c_int64 * 3


def _cache_args(kc, vc, ks, vs, table, B):
    """Checks a cache; the arguments that the native calls share."""
    if kc.dim() != 4 or kc.shape != vc.shape or kc.dtype != torch.int8 or vc.dtype != torch.int8 \
            or not kc.is_contiguous() or not vc.is_contiguous():
        raise RuntimeError(f"{TAG} kv8: k_codes and v_codes must be contiguous int8 [pages, heads, "
                           f"T, D], got {tuple(kc.shape)} {kc.dtype}, {tuple(vc.shape)} {vc.dtype}")
    P, H, T, D = kc.shape
    if T not in BLOCKS or D not in HEAD_DIMS or P < 1 or H < 1:
        raise RuntimeError(f"{TAG} kv8: pages of {T} tokens x {D}; T must be one of {BLOCKS} and "
                           f"D one of {HEAD_DIMS}")
    if ks.shape != (P, H) or vs.shape != (P, H) or ks.dtype != torch.float32 \
            or vs.dtype != torch.float32 or not ks.is_contiguous() or not vs.is_contiguous():
        raise RuntimeError(f"{TAG} kv8: k_scale and v_scale must be contiguous fp32 "
                           f"[{P}, {H}], got {tuple(ks.shape)}, {tuple(vs.shape)}")
    if table.dim() != 2 or table.dtype != torch.int32 or table.shape[0] != B \
            or table.shape[1] < 1 or table.stride(1) != 1:
        raise RuntimeError(f"{TAG} kv8: block_table must be int32 [{B}, max_blocks], got "
                           f"{table.dtype} {tuple(table.shape)}")
    dev = kc.device
    if dev.type != "cuda":
        raise RuntimeError(f"{TAG} expected CUDA tensors, got {dev}")
    if vc.device != dev or ks.device != dev or vs.device != dev or table.device != dev:
        raise RuntimeError(f"{TAG} kv8: the cache's tensors are on different devices")
    nb = table.shape[1]
    ld = table.stride(0) if B > 1 else nb
    if ld < nb:
        raise RuntimeError(f"{TAG} kv8: block_table rows overlap")
    return (P, H, T, D, table.data_ptr(), ld, nb), dev


def _per_seq(t, B, dev, name):
    if t.shape != (B,) or t.dtype != torch.int32 or t.device != dev or not t.is_contiguous():
        raise RuntimeError(f"{TAG} kv8: {name} must be contiguous int32 [{B}] on {dev}, got "
                           f"{t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _tokens(t, shape, dt, dev, name):
    """A [B, heads, S, D] operand with unit inner stride and 16-byte rows."""
    if tuple(t.shape) != shape or t.dtype != dt or t.device != dev:
        raise RuntimeError(f"{TAG} kv8: {name} must be {shape} {dt} on {dev}, got "
                           f"{tuple(t.shape)} {t.dtype} on {t.device}")
    a, b, c, d = t.stride()
    if d != 1 or (a | b | c) % 8 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def kv8_append(k, v, k_codes, v_codes, k_scale, v_scale, block_table, start, counts=None):
    """Write k, v [B, heads, S, D] (bf16/f16) into the cache, in place: the first
    counts[b] (all S without counts) tokens of sequence b go to positions start[b],
    start[b] + 1, ...  Sequences must not share a page that is written."""
    if k.dim() != 4:
        raise RuntimeError(f"{TAG} kv8: k must be [B, heads, S, D], got {tuple(k.shape)}")
    B, _, S, _ = k.shape
    args, dev = _cache_args(k_codes, v_codes, k_scale, v_scale, block_table, B)
    dt = k.dtype
    code = _DT.get(dt)
    if code is None or code == 2:
        raise RuntimeError(f"{TAG} kv8_append expects bf16/f16 keys and values, got {dt}")
    shape = (B, args[1], S, args[3])
    k, v = _tokens(k, shape, dt, dev, "k"), _tokens(v, shape, dt, dev, "v")
    sp = _per_seq(start, B, dev, "start")
    cp = 0 if counts is None else _per_seq(counts, B, dev, "counts")
    with _native.device_of(dev):
        st = _native.lib().b200q_kv8_append(
            k.data_ptr(), v.data_ptr(), code, B, S, _Strides(*k.stride()[:3]),
            _Strides(*v.stride()[:3]), k_codes.data_ptr(), v_codes.data_ptr(), k_scale.data_ptr(),
            v_scale.data_ptr(), *args, sp, cp, _raw_stream(dev.index))
        if st:
            _native._check(st)


def kv8_gather(k_codes, v_codes, k_scale, v_scale, block_table, first, counts, max_count,
               out_dtype=torch.bfloat16):
    """k, v [B, heads, max_count, D]: the values of tokens first[b] .. first[b] +
    counts[b] - 1 of each sequence, zeros behind them."""
    B = block_table.shape[0]
    args, dev = _cache_args(k_codes, v_codes, k_scale, v_scale, block_table, B)
    code = _DT.get(out_dtype)
    if code is None or max_count < 0:
        raise RuntimeError(f"{TAG} kv8_gather: out dtype {out_dtype}, max_count {max_count}")
    fp, cp = _per_seq(first, B, dev, "first"), _per_seq(counts, B, dev, "counts")
    with _native.device_of(dev):
        shape = (B, args[1], max_count, args[3])
        k = torch.empty(shape, dtype=out_dtype, device=dev)
        v = torch.empty(shape, dtype=out_dtype, device=dev)
        st = _native.lib().b200q_kv8_gather(
            k_codes.data_ptr(), v_codes.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), *args,
            fp, cp, k.data_ptr(), v.data_ptr(), code, B, max_count, _raw_stream(dev.index))
        if st:
            _native._check(st)
    return k, v


def kv8_attention(q, k_codes, v_codes, k_scale, v_scale, block_table, lens, causal=True,
                  scale=None, max_len=None):
    """softmax(scale * q K^T) V over the first lens[b] tokens of each sequence.

    q [B, Hq, Tq, D] bf16/f16, any strides with unit inner one; Hq a multiple of the
    cache's heads.  causal: query i of Tq sits at position lens[b] - Tq + i and sees
    positions up to its own.  scale: 1 / sqrt(D) by default.  max_len: an upper
    bound of lens when the host knows one; only the plan depends on it.  Returns
    (out [B, Hq, Tq, D], stored token-major, and lse [B, Hq, Tq] fp32); a row that
    sees nothing gives 0 and -inf."""
    if q.dim() != 4:
        raise RuntimeError(f"{TAG} kv8: q must be [B, heads, Tq, D], got {tuple(q.shape)}")
    B, Hq, Tq, D = q.shape
    args, dev = _cache_args(k_codes, v_codes, k_scale, v_scale, block_table, B)
    dt = q.dtype
    code = _DT.get(dt)
    if code is None or code == 2:
        raise RuntimeError(f"{TAG} kv8_attention expects bf16/f16 queries, got {dt}")
    H = args[1]
    if Hq % H or D != args[3] or Hq == 0:
        raise RuntimeError(f"{TAG} kv8: {Hq} query heads of {D} over {H} cache heads of {args[3]}")
    q = _tokens(q, (B, Hq, Tq, D), dt, dev, "q")
    lp = _per_seq(lens, B, dev, "lens")
    cap = args[2] * args[6]
    max_len = cap if max_len is None else min(int(max_len), cap)
    if max_len < 0:
        raise RuntimeError(f"{TAG} kv8: max_len {max_len}")
    L = _native.lib()
    with _native.device_of(dev):
        out = torch.empty((B, Tq, Hq, D), dtype=dt, device=dev).transpose(1, 2)
        lse = torch.empty((B, Hq, Tq), dtype=torch.float32, device=dev)
        wsb = L.b200q_kv8_attention_workspace_size(B, Hq, H, Tq, D, max_len)
        work = torch.empty(wsb, dtype=torch.uint8, device=dev) if wsb else None
        st = L.b200q_kv8_attention(
            q.data_ptr(), code, B, Hq, Tq, _Strides(*q.stride()[:3]), k_codes.data_ptr(),
            v_codes.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), *args, lp, max_len,
            bool(causal), D ** -0.5 if scale is None else scale, out.data_ptr(),
            _Strides(*out.stride()[:3]), lse.data_ptr(), 0 if work is None else work.data_ptr(),
            wsb, _raw_stream(dev.index))
        if st:
            _native._check(st)
    return out, lse


class KV8Cache:
    """Pool, tables and lengths of a batch of sequences.

    Pages are handed out in order, ``max_blocks`` per sequence; the tensors are
    plain attributes, so a caller with its own page allocator may rewrite
    ``table``.  ``append`` and ``attention`` leave all state on the GPU."""

    def __init__(self, batch, heads, head_dim, max_len, block=64, device="cuda"):
        nb = -(-max_len // block)
        self.max_len = nb * block
        shape = (batch * nb, heads, block, head_dim)
        self.k_codes = torch.zeros(shape, dtype=torch.int8, device=device)
        self.v_codes = torch.zeros(shape, dtype=torch.int8, device=device)
        self.k_scale = torch.zeros(shape[:2], dtype=torch.float32, device=device)
        self.v_scale = torch.zeros(shape[:2], dtype=torch.float32, device=device)
        self.table = torch.arange(batch * nb, dtype=torch.int32, device=device).view(batch, nb)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)

    @property
    def pool(self):
        return self.k_codes, self.v_codes, self.k_scale, self.v_scale, self.table

    def append(self, k, v, counts=None):
        """Add k, v [B, heads, S, D] behind what is there and advance the lengths."""
        kv8_append(k, v, *self.pool, self.lens, counts)
        self.lens += k.shape[2] if counts is None else counts

    def attention(self, q, causal=True, scale=None, max_len=None):
        """out [B, Hq, Tq, D] over everything appended so far."""
        return kv8_attention(q, *self.pool, self.lens, causal, scale, max_len or self.max_len)[0]

    def values(self, max_count=None, out_dtype=torch.bfloat16):
        """The cached k, v [B, heads, max_count, D], zeros behind each length."""
        return kv8_gather(*self.pool, torch.zeros_like(self.lens), self.lens,
                          self.max_len if max_count is None else max_count, out_dtype)


_LIB = torch.library.Library("b200q", "FRAGMENT")


def _register():
    pool = "Tensor{} k_codes, Tensor{} v_codes, Tensor{} k_scale, Tensor{} v_scale, Tensor block_table"
    _LIB.define("kv8_append(Tensor k, Tensor v, " + pool.format("(a!)", "(b!)", "(c!)", "(d!)")
                + ", Tensor start, Tensor? counts=None) -> ()")
    _LIB.define("kv8_gather(" + pool.format("", "", "", "") + ", Tensor first, Tensor counts, "
                "int max_count, ScalarType out_dtype=15) -> (Tensor, Tensor)")
    _LIB.define("kv8_attention(Tensor q, " + pool.format("", "", "", "") + ", Tensor lens, "
                "bool causal=True, float? scale=None, int? max_len=None) -> (Tensor, Tensor)")
    _LIB.impl("kv8_append", kv8_append, "CUDA")
    _LIB.impl("kv8_gather", kv8_gather, "CUDA")
    _LIB.impl("kv8_attention", kv8_attention, "CUDA")

    def fake_gather(kc, vc, ks, vs, table, first, counts, max_count, out_dtype=torch.bfloat16):
        shape = (table.shape[0], kc.shape[1], max_count, kc.shape[3])
        return kc.new_empty(shape, dtype=out_dtype), kc.new_empty(shape, dtype=out_dtype)

    def fake_attention(q, kc, vc, ks, vs, table, lens, causal=True, scale=None, max_len=None):
        B, Hq, Tq, D = q.shape
        return (q.new_empty((B, Tq, Hq, D)).transpose(1, 2),
                q.new_empty((B, Hq, Tq), dtype=torch.float32))

    torch.library.register_fake("b200q::kv8_append", lambda *a, **k: None, lib=_LIB)
    torch.library.register_fake("b200q::kv8_gather", fake_gather, lib=_LIB)
    torch.library.register_fake("b200q::kv8_attention", fake_attention, lib=_LIB)


_register()
