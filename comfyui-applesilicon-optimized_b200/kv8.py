"""A paged 8-bit key/value cache and the attention that reads it.

``k_codes``, ``v_codes`` [pages, heads, T, D] int8 hold the tokens' values in pages
of T tokens (16, 32, 64 or 128; D 64 or 128), ``k_scale``, ``v_scale`` [pages, heads]
fp32 one scale (not negative) for each page and head: value = code * scale.  ``block_table``
[B, max_blocks] int32 gives the page of each block of T tokens of a sequence.

* ``kv8_append`` writes new tokens behind each sequence's length.  A block's scale
  only grows: it becomes max(its scale so far, max|new| / 127), and codes already
  there are requantized when it does.  An infinity or NaN makes its block's scale
  NaN: the block reads back as NaN, and so do the rows of attention that see it.
* ``kv8_gather`` reads tokens back as 16-bit or fp32 values.
* ``kv8_attention`` is softmax(q K^T) V over the cache, for one query token or
  many, causal or not, with grouped heads.
* ``KV8Cache`` owns the pool, the tables and the lengths of a batch.

Lengths, positions and tables live on the GPU and nothing is read back, so a
decode step can be captured in a CUDA graph.  Page numbers are checked on the
device: a bad one sets bit 1 of the device status word (``_native.device_status``)
and its tokens are skipped.  Also registered in ``torch.ops.b200q``.
"""
import torch

from ._patches import _native

_calls = None


def _load():
    global _calls
    b = _native.bindings()
    _calls = (b.kv8_append, b.kv8_gather, b.kv8_attention)
    return _calls


def kv8_append(k, v, k_codes, v_codes, k_scale, v_scale, block_table, start, counts=None):
    """Write k, v [B, heads, S, D] (bf16/f16) into the cache, in place: the first
    counts[b] (all S without counts, at most S) tokens of sequence b go to positions start[b],
    start[b] + 1, ...  Sequences must not share a page that is written."""
    (_calls or _load())[0](k, v, k_codes, v_codes, k_scale, v_scale, block_table, start, counts)


def kv8_gather(k_codes, v_codes, k_scale, v_scale, block_table, first, counts, max_count,
               out_dtype=torch.bfloat16):
    """k, v [B, heads, max_count, D]: the values of tokens first[b] .. first[b] +
    counts[b] - 1 of each sequence, zeros behind them."""
    return (_calls or _load())[1](k_codes, v_codes, k_scale, v_scale, block_table, first, counts,
                                  max_count, out_dtype)


def kv8_attention(q, k_codes, v_codes, k_scale, v_scale, block_table, lens, causal=True,
                  scale=None, max_len=None):
    """softmax(scale * q K^T) V over the first lens[b] tokens of each sequence.

    q [B, Hq, Tq, D] bf16/f16, any strides with unit inner one; Hq a multiple of the
    cache's heads.  causal: query i of Tq sits at position lens[b] - Tq + i and sees
    positions up to its own.  scale: 1 / sqrt(D) by default.  max_len: an upper
    bound of lens when the host knows one; only the plan depends on it.  Returns
    (out [B, Hq, Tq, D], stored token-major, and lse [B, Hq, Tq] fp32); a row that
    sees nothing gives 0 and -inf."""
    return (_calls or _load())[2](q, k_codes, v_codes, k_scale, v_scale, block_table, lens, causal,
                                  scale, max_len)


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
        """Add k, v [B, heads, S, D] behind what is there (sequence b: its first counts[b],
        at most S and none below 0) and advance the lengths."""
        kv8_append(k, v, *self.pool, self.lens, counts)
        self.lens += k.shape[2] if counts is None else counts.clamp(0, k.shape[2])

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
