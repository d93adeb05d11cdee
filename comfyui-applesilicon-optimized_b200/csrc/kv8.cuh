// A paged 8-bit key/value cache: int8 codes [pages, heads, T, D] and one fp32
// scale per (page, head), value = code * scale.  A page is a block of T tokens;
// block_table[b][i] is the page of sequence b's tokens [i*T, (i+1)*T).
//
//   append     writes new tokens behind each sequence's length.  A block's scale
//              is max(its scale so far if it holds tokens, max|new| / 127): it
//              only grows, and codes already there are requantized when it does.
//   gather     reads a range of tokens back as 16-bit / fp32 values.
//   attention  softmax(q K^T) V over the cache.
//
// Page numbers come from device memory and are checked against the pool before
// any access; a bad one sets the status word's bit 1 and its tokens are skipped.
#pragma once

#include "digits.cuh"
#include "numerics.cuh"
#include "ptx.cuh"

namespace b200q {

struct Kv8Cache {
  int8_t *k, *v;           // [pages, heads, T, D]
  float *ks, *vs;          // [pages, heads]
  const int32_t* table;    // [B, max_blocks]
  int64_t ld_table;
  int max_blocks, pages, heads, T, D, log_t;
};

// Page of block `blk` of sequence b, or -1 (flagged) if the table holds no page there.
__device__ __forceinline__ int kv8_page(const Kv8Cache& c, int b, int blk) {
  if (blk < 0 || blk >= c.max_blocks) {
    atomicOr(&g_device_status, kStatusBadArgument);
    return -1;
  }
  const int p = __ldg(c.table + b * c.ld_table + blk);
  if (p < 0 || p >= c.pages) {
    atomicOr(&g_device_status, kStatusBadArgument);
    return -1;
  }
  return p;
}

// ---------------------------------------------------------------- append
struct Kv8AppendArgs {
  Kv8Cache c;
  const void *k, *v;  // [B, heads, S, D], unit inner stride, 16-byte aligned rows
  int64_t kb, kh, kt, vb, vh, vt;  // strides in elements
  const int32_t* start;   // [B] tokens already in the cache
  const int32_t* counts;  // [B] new tokens (<= S), or null: S each
  int B, S;
};

constexpr int kKvThreads = 256;

// One CTA per (block, head, sequence, K or V).  NV: 8-value vectors a thread
// holds (T * D <= 2048 * NV).  Bound: HBM; the quotient x / scale is a product with
// the scale's reciprocal and one correction by its remainder, which gives the rounded
// quotient (16-bit values are often exact ties, half of the block's largest among them),
// and the nearest integer is the low byte of its sum with 1.5 * 2^23: the divide's
// branches and the clamping cost twice the memory's time.  Two prompts of 8191 tokens, 8
// heads: 26 us, 0.60 of the copy rate (issue 63%); one token for each of 64 sequences 4 us.
template <typename T, int NV>
__global__ void __launch_bounds__(kKvThreads) kv8_append_kernel(const Kv8AppendArgs a) {
  __shared__ uint32_t wmax[kKvThreads / 32];
  griddep_wait();
  griddep_launch_dependents();
  const Kv8Cache& c = a.c;
  const bool is_v = blockIdx.z & 1;
  const int b = blockIdx.z >> 1, h = blockIdx.y, tid = threadIdx.x;
  const int start = a.start[b];
  const int count = min(a.counts ? a.counts[b] : a.S, a.S);
  if (start < 0 || count <= 0) return;
  const int blk = (start >> c.log_t) + blockIdx.x;
  const int64_t first = static_cast<int64_t>(blk) << c.log_t;  // the block's first position
  const int64_t end = static_cast<int64_t>(start) + count;
  if (first >= end) return;
  const int page = kv8_page(c, b, blk);
  if (page < 0) return;
  const int old = static_cast<int>(first < start ? start - first : 0);  // tokens already there
  const int upto = static_cast<int>(end - first < c.T ? end - first : c.T);
  const int ldv = c.D == 128 ? 4 : 3, dv = 1 << ldv;  // vectors per token
  const T* src = static_cast<const T*>(is_v ? a.v : a.k) + b * (is_v ? a.vb : a.kb) + h * (is_v ? a.vh : a.kh);
  const int64_t st = is_v ? a.vt : a.kt;
  int8_t* codes = (is_v ? c.v : c.k) + (static_cast<int64_t>(page) * c.heads + h) * (static_cast<int64_t>(c.T) * c.D);
  float* scale = (is_v ? c.vs : c.ks) + static_cast<int64_t>(page) * c.heads + h;

  uint4 raw[NV];
  uint32_t top = 0;  // largest |x| as bits: NaN and infinities sort above
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int i = (old * dv) + tid + k * kKvThreads;
    if (i < upto * dv) {
      const int tok = i >> ldv;
      raw[k] = __ldg(reinterpret_cast<const uint4*>(src + (first + tok - start) * st + (i & (dv - 1)) * 8));
      const uint32_t u[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) top = max(top, max(u[j] & 0x7FFFu, (u[j] >> 16) & 0x7FFFu));
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((tid & 31) == 0) wmax[tid >> 5] = top;
  const float before = old > 0 ? *scale : 0.0f;
  __syncthreads();  // also: every thread has read the old scale
#pragma unroll
  for (int i = 0; i < kKvThreads / 32; ++i) top = max(top, wmax[i]);
  const uint16_t tb = static_cast<uint16_t>(top);
  const float amax = to_float<T>(*reinterpret_cast<const T*>(&tb));
  const float grown = __fdiv_rn(amax, 127.0f);
  // an infinity or NaN on either side makes the scale NaN, so that the block reads back as NaN
  // (codes times inf would be infinities whose signs say nothing)
  const float most = before > grown || before != before ? before : grown;
  const float s = most <= 3.402823466e38f ? most : __uint_as_float(0x7FC00000u);
  if (tid == 0) *scale = s;
  // a zero scale's block holds zeros, a NaN one's codes do not matter; below 2^-100 the remainder
  // and then the reciprocal leave fp32's range, and the quotient is divided out
  const float inv = s >= 0x1p-100f ? __fdiv_rn(1.0f, s) : 0.0f;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int i = (old * dv) + tid + k * kKvThreads;
    if (i < upto * dv) {
      const uint32_t u[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
      uint32_t o[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint16_t e = static_cast<uint16_t>(u[j >> 1] >> (16 * (j & 1)));
        const float x = to_float<T>(*reinterpret_cast<const T*>(&e)), y = x * inv;
        o[j] = __float_as_uint(fmaf(fmaf(-y, s, x), inv, y) + 12582912.0f);
      }
      *reinterpret_cast<uint2*>(codes + i * 8) =
          make_uint2(low_bytes(o[0], o[1], o[2], o[3]), low_bytes(o[4], o[5], o[6], o[7]));
    }
  }
  if (s > 0.0f && s < 0x1p-100f) {  // a loop of its own behind: in the one above it took 5% of every call
#pragma unroll 1
    for (int i = old * dv + tid; i < upto * dv; i += kKvThreads) {
      const T* x = src + (first + (i >> ldv) - start) * st + (i & (dv - 1)) * 8;
#pragma unroll 1
      for (int j = 0; j < 8; ++j)
        codes[i * 8 + j] = static_cast<int8_t>(__float_as_uint(__fdiv_rn(to_float<T>(x[j]), s) + 12582912.0f));
    }
  }
  if (old > 0 && s != before) {
    const float ratio = s > 0.0f ? __fdiv_rn(before, s) : 0.0f;
    for (int i = tid; i < old * dv; i += kKvThreads) {
      __align__(8) int8_t o[8];
      *reinterpret_cast<uint2*>(o) = *reinterpret_cast<const uint2*>(codes + i * 8);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float f = rintf(__fmul_rn(static_cast<float>(o[j]), ratio));
        o[j] = static_cast<int8_t>(fminf(fmaxf(f, -127.0f), 127.0f));
      }
      *reinterpret_cast<uint2*>(codes + i * 8) = *reinterpret_cast<const uint2*>(o);
    }
  }
}

// ---------------------------------------------------------------- gather
struct Kv8GatherArgs {
  Kv8Cache c;
  void *k, *v;            // [B, heads, S, D] contiguous
  int out_dtype;          // kOutBF16 / kOutF16 / kOutF32
  const int32_t* first;   // [B]
  const int32_t* counts;  // [B] tokens to read (<= S); the rest of S is zeroed
  int B, S;
};

// Four vectors of 8 codes per thread, their loads in flight together; grid (vectors of
// a head, heads, 2 B).  Bound: HBM (two times 8191 tokens, 8 heads: 16 us, 0.94 of the copy
// rate).
constexpr int kGatherVecs = 4;
__global__ void __launch_bounds__(kKvThreads) kv8_gather_kernel(const Kv8GatherArgs a) {
  griddep_wait();
  griddep_launch_dependents();
  const Kv8Cache& c = a.c;
  const bool is_v = blockIdx.z & 1;
  const int b = blockIdx.z >> 1, h = blockIdx.y, ldv = c.D == 128 ? 4 : 3;
  const int first = a.first[b];
  const int count = first >= 0 ? a.counts[b] : 0;
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * (kKvThreads * kGatherVecs) + threadIdx.x;
  const int8_t* codes = is_v ? c.v : c.k;
  const float* scales = is_v ? c.vs : c.ks;
  uint2 raw[kGatherVecs];
  float s[kGatherVecs];
#pragma unroll
  for (int u = 0; u < kGatherVecs; ++u) {
    const int64_t i = i0 + u * kKvThreads;
    const int64_t tok = i >> ldv;
    raw[u] = make_uint2(0, 0);
    s[u] = 0.0f;
    if (tok < a.S && tok < count) {
      const int64_t pos = first + tok;
      const int page = kv8_page(c, b, static_cast<int>(pos >> c.log_t));
      if (page >= 0) {
        const int64_t at = static_cast<int64_t>(page) * c.heads + h;
        s[u] = __ldg(scales + at);
        raw[u] = __ldg(reinterpret_cast<const uint2*>(codes + (((at << c.log_t) + (pos & (c.T - 1))) << (ldv + 3)) +
                                                      ((i & ((1 << ldv) - 1)) << 3)));
      }
    }
  }
  void* out = is_v ? a.v : a.k;
  const int64_t base = ((static_cast<int64_t>(b) * c.heads + h) * a.S) << (ldv + 3);
#pragma unroll
  for (int u = 0; u < kGatherVecs; ++u) {
    const int64_t i = i0 + u * kKvThreads;
    if ((i >> ldv) >= a.S) break;
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t w = j < 4 ? raw[u].x : raw[u].y;
      f[j] = __fmul_rn(static_cast<float>(static_cast<int8_t>(w >> (8 * (j & 3)))), s[u]);
    }
    const int64_t dst = base + (i << 3);
    if (a.out_dtype == kOutF32) {
      float4* p = reinterpret_cast<float4*>(static_cast<float*>(out) + dst);
      p[0] = make_float4(f[0], f[1], f[2], f[3]);
      p[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        o[j] = a.out_dtype == kOutBF16 ? pack_bf16x2(f[2 * j], f[2 * j + 1]) : pack_f16x2(f[2 * j], f[2 * j + 1]);
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + dst) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

// ---------------------------------------------------------------- attention
// Rows: the G query heads of a key/value head and their Tq tokens are packed as
// rows r = token * G + head of one matrix, 16 rows per MMA (m16n8k16, fp16
// operands, fp32 accumulation).  int8 codes are exact in fp16: with the sign bit
// flipped a byte OR-ed into the mantissa of 1024 is 1152 + code, and subtracting
// 1152 is exact.  q is scaled by the power of two of its row's largest |q| and
// is then exact in fp16 (bf16: down to 2^-17 of the row's maximum, within 2^-25
// of it below).
//
// Softmax, online, base 2.  With sigma = q.k_code * ks * scale * log2 e and vs the
// block's V scale, the weights kept are P = 2^(sigma + log2 vs - m) <= 2^15, m the
// running maximum of that exponent less 15; then
//   out = sum P * v_code / sum P / vs,
// so V's scales cost one add per score instead of a pass over the accumulators,
// and P fits fp16 whatever the scales are: P's fp16 rounding (2^-11 relative,
// 2^-40 of the row's largest weight at least) is the only one before the
// output's.  A block with vs = 0 adds its P / 2^-80 to the sum only, as if vs were 2^-80.
//
// Layout, D = 128: lane (g, t) loads 32 consecutive bytes (quarter t) of K token
// g, and 16 bytes (eighth g) of V tokens 2t, 2t+1, 2t+8, 2t+9: every load of the
// warp covers whole 128-byte rows.  The order of d inside the K product is free
// (q is permuted alike), and V's columns come out as d = 16 g + i for tile i, so
// a lane ends with 32 consecutive d of its rows.
struct Kv8AttnArgs {
  Kv8Cache c;
  const void* q;  // [B, Hq, Tq, D] strides qb, qh, qt
  int q_f16;
  int64_t qb, qh, qt;
  void* out;  // [B, Hq, Tq, D] strides ob, oh, ot
  int64_t ob, oh, ot;
  float* lse;     // [B, Hq, Tq] contiguous
  float* part_o;  // [splits][B*Hq*Tq][D] fp32 (splits > 1)
  float* part_ml; // [splits][B*Hq*Tq][2]: m (base 2), l
  const int32_t* lens;
  int B, Hq, G, Tq, causal, splits;
  int longest_first;  // (row tiles) start CTAs in the order of their sequences' lengths
  float scale_log2;  // softmax scale * log2 e
};

constexpr int kAttnBox = 64;          // rows of a TMA box at most
constexpr int kAttnMaxSplits = 64;    // joined by the join kernel
constexpr int kAttnStages = 4;

constexpr int kAttnWarps = 4;                        // consumer warps
constexpr int kAttnThreads = (kAttnWarps + 1) * 32;  // and a producer warp

// The CTA's ring: stages of 64 tokens of K and V, brought by TMA with the row
// swizzle; 16-token tile w of a stage belongs to consumer warp w.  meta: per tile
// {ks, log2 vs, 1 / vs, state}, state 0 = skip (bad page), 1 = ok, 2 = V is 0.
template <int D, int ST = kAttnStages>
struct AttnRing {
  uint8_t k[ST][16 * kAttnWarps * D];
  uint8_t v[ST][16 * kAttnWarps * D];
  float4 meta[ST][kAttnWarps];
  uint64_t full[ST], empty[ST];
  int abort;
};
template <int D>
constexpr int attn_smem_bytes() {
  return static_cast<int>(sizeof(AttnRing<D>)) + 1024;
}
template <int D>
__device__ __forceinline__ AttnRing<D>* attn_ring() {
  extern __shared__ uint8_t attn_smem[];  // the swizzle pattern is anchored at 1024 bytes
  return reinterpret_cast<AttnRing<D>*>((reinterpret_cast<uintptr_t>(attn_smem) + 1023) & ~uintptr_t(1023));
}
// `readers`: warps that release a stage.
template <int D, int ST>
__device__ __forceinline__ void attn_ring_init(AttnRing<D, ST>* ring, const CUtensorMap* tk, const CUtensorMap* tv,
                                               int readers = kAttnWarps) {
  if (threadIdx.x == 0) {
    tma_prefetch_desc(tk);
    tma_prefetch_desc(tv);
    for (int i = 0; i < ST; ++i) {
      mbar_init(&ring->full[i], 2);  // the copies and the meta words
      mbar_init(&ring->empty[i], readers);
    }
    ring->abort = 0;
    fence_mbarrier_init();
  }
  __syncthreads();
}
// Byte offset of 16-byte chunk `ch` of token row `row`, XOR-swizzled so that the
// K reads (rows g, chunks of quarter t) and the V reads (rows 2t, chunk g) of a
// warp are both free of bank conflicts (D = 64: V's 8-byte reads 2-way).
template <int D>
__device__ __forceinline__ int attn_at(int row, int ch) {
  return D == 128 ? row * 128 + ((ch ^ (row & 7)) << 4) : row * 64 + ((ch ^ ((row >> 1) & 3)) << 4);
}

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t hsub2_1152(uint32_t a) {
  const uint32_t k = 0x64806480u;  // 1152, 1152
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&k));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// Bytes 0,1 (lo) / 2,3 (hi) of a sign-flipped word as two exact fp16 values.
__device__ __forceinline__ uint32_t i8_lo(uint32_t w) { return hsub2_1152(__byte_perm(w, 0x64646464u, 0x4140)); }
__device__ __forceinline__ uint32_t i8_hi(uint32_t w) { return hsub2_1152(__byte_perm(w, 0x64646464u, 0x4342)); }

// Value of q as fp16 bits after scaling, from bf16 / fp16 bits.
__device__ __forceinline__ uint32_t q_pair(uint32_t raw, int f16, float inv) {
  float a, b;
  if (f16) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&raw));
    a = f.x;
    b = f.y;
  } else {
    a = __uint_as_float(raw << 16);
    b = __uint_as_float(raw & 0xFFFF0000u);
  }
  return pack_f16x2(a * inv, b * inv);
}

// Whether a row whose largest |q| has these bits is finite.  Every score of one that is not is
// an infinity or NaN, so its softmax is NaN: its scores are made NaN, as -inf would be masked.
__device__ __forceinline__ bool q_finite(uint32_t top, int f16) { return top < (f16 ? 0x7C00u : 0x7F80u); }

// A row's m is its largest exponent less this: P <= 2^15 uses fp16's whole range, so
// weights down to 2^-29 of the largest keep all their bits (P <= 1 loses bits below
// 2^-14, which shows where blocks' V scales lie far apart).
constexpr float kAttnHead = 15.0f;

// log-sum-exp pieces of two halves of a row: (m, l) and the factors of each side.
__device__ __forceinline__ float safe_ex2_diff(float m, float top) {
  return m == -INFINITY ? 0.0f : ex2_approx(m - top);
}

// The producer warp: chunks c0 .. c1 - 1 (64 tokens each) of (sequence b, head h).
// Lane i looks up tile i % 4 of chunk i / 4 of the next eight chunks at once (page,
// scales, their logarithm and inverse), then the chunks go out one by one: a box of
// min(T, 64) rows per page.  Tiles at or past `tiles` are not fetched.  The first
// stages' copies start before the scales are waited for: a stage is full after two
// arrivals, the copies' and the one behind its meta words.
template <int D, int ST>
__device__ __forceinline__ void attn_produce(const Kv8AttnArgs& a, const CUtensorMap* tk, const CUtensorMap* tv,
                                             AttnRing<D, ST>* ring, int b, int h, int c0, int c1, int tiles) {
  const Kv8Cache& c = a.c;
  const int lane = threadIdx.x & 31;
  const int box = c.T < kAttnBox ? c.T : kAttnBox;
  const int per_box = box >> 4;  // tiles
  int n = 0;                     // chunks issued
  bool live = true;
  for (int base = c0; base < c1 && live; base += 32 / kAttnWarps) {
    const int tile = base * kAttnWarps + lane, pos = tile << 4;
    int page = -1;
    if (tile < tiles && (base + (lane / kAttnWarps)) < c1) page = kv8_page(c, b, pos >> c.log_t);
    const int64_t at = static_cast<int64_t>(page < 0 ? 0 : page) * c.heads + h;
    float ks = __ldg(c.ks + at);
    const float vs = __ldg(c.vs + at);
    // scores of an infinite scale are NaN, never the -inf of a masked position
    if (!(fabsf(ks) <= 3.402823466e38f)) ks = __uint_as_float(0x7FC00000u);
    const bool lead = page >= 0 && (lane & (per_box - 1)) == 0;
    const unsigned leads = __ballot_sync(0xffffffffu, lead);
    const int y = static_cast<int>(at * c.T) + (pos & (c.T - 1));
    auto copy = [&](int i, int s) {
      if (lane == 0)
        mbar_arrive_expect_tx(&ring->full[s], 2 * D * box * __popc((leads >> (kAttnWarps * i)) & ((1u << kAttnWarps) - 1u)));
      __syncwarp();
      if ((lane / kAttnWarps) == i && lead) {
        tma_load_2d(tk, &ring->full[s], ring->k[s] + (lane % kAttnWarps) * 16 * D, 0, y);
        tma_load_2d(tv, &ring->full[s], ring->v[s] + (lane % kAttnWarps) * 16 * D, 0, y);
      }
    };
    const int many = min(32 / kAttnWarps, c1 - base);
    if (n == 0)
      for (int i = 0; i < min(many, ST); ++i) copy(i, i);
    // below 2^-80 (values under 2^-73) a block counts as one of zeros at scale 2^-80: P / vs must
    // not overflow, and its weights, which reach the sum alone, must not raise m and with it
    // take the bits of weights whose blocks' scales are small but not zero
    float4 meta = make_float4(ks, -80.0f, 0x1p80f, 2.0f);
    if (!(fabsf(vs) < 0x1p-80f)) meta = make_float4(ks, log2f(vs), 1.0f / vs, 1.0f);
    if (page < 0) meta = make_float4(0.0f, 0.0f, 1.0f, 0.0f);
    for (int i = 0; i < many; ++i, ++n) {
      const int s = n % ST;
      if (n >= ST) {
        if (!mbar_wait_warp(&ring->empty[s], ((n / ST) - 1) & 1, &ring->abort)) {
          live = false;
          break;
        }
        copy(i, s);
      }
      if ((lane / kAttnWarps) == i) ring->meta[s][lane % kAttnWarps] = meta;
      __syncwarp();
      if (lane == 0) mbar_arrive(&ring->full[s]);
    }
  }
  if (!live && lane == 0) {  // gave up: let the copies in flight land before the CTA ends
    for (int i = n > ST ? n - ST : 0; i < n; ++i)
      mbar_wait_drain(&ring->full[i % ST], (i / ST) & 1);
  }
}
// This lane's K words of a 16-token tile: tokens g and g + 8, quarter t.
template <int D>
__device__ __forceinline__ void attn_read_k(const uint8_t* k, int g, int t, uint32_t (&kw)[2][D / 16]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int j = 0; j < D / 64; ++j) {
      const uint4 v = *reinterpret_cast<const uint4*>(k + attn_at<D>(8 * i + g, t * (D / 64) + j));
      kw[i][4 * j] = v.x; kw[i][4 * j + 1] = v.y; kw[i][4 * j + 2] = v.z; kw[i][4 * j + 3] = v.w;
    }
  }
}
// Its V words: tokens 2t, 2t+1, 2t+8, 2t+9, eighth g.
template <int D>
__device__ __forceinline__ void attn_read_v(const uint8_t* vp, int g, int t, uint32_t (&vw)[4][D / 32]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = 2 * t + (i & 1) + 8 * (i >> 1);
    if constexpr (D == 128) {
      const uint4 v = *reinterpret_cast<const uint4*>(vp + attn_at<D>(row, g));
      vw[i][0] = v.x; vw[i][1] = v.y; vw[i][2] = v.z; vw[i][3] = v.w;
    } else {
      const uint2 v = *reinterpret_cast<const uint2*>(vp + attn_at<D>(row, g >> 1) + (g & 1) * 8);
      vw[i][0] = v.x; vw[i][1] = v.y;
    }
  }
}

// Where the warps leave their rows: R rows of D values per warp in the ring's
// memory (its last stage has been read).  Row stride and the skew by d / 16 (D =
// 64: d / 8) spread a warp's writes, rows 2t x d = (D / 8) g, over the banks.
template <int D, int R>
struct AttnOut {
  static constexpr int kStride = D + 20;
  float o[kAttnWarps][R][kStride];
  static __device__ __forceinline__ int at(int d) { return d + d / (D / 8); }
};
// Joins the warps in order and stores the rows, or hands the CTA's partial to the
// join kernel.  ml: (m, l) of each warp and row; each warp's o is already scaled to
// the CTA's maximum.  Called by all threads, for rows 0 .. rows - 1.
template <int D, int R>
__device__ __forceinline__ void attn_epilogue(const Kv8AttnArgs& a, const AttnOut<D, R>* buf,
                                              const float (&ml)[kAttnWarps][R][2], float (&fin)[R][2], int b,
                                              int h, int split, int rows) {
  __syncthreads();
  if (threadIdx.x < R) {
    const int r = threadIdx.x;
    float m = ml[0][r][0], l = 0.0f;
#pragma unroll
    for (int w = 1; w < kAttnWarps; ++w) m = fmaxf(m, ml[w][r][0]);
#pragma unroll
    for (int w = 0; w < kAttnWarps; ++w) l += ml[w][r][1] * safe_ex2_diff(ml[w][r][0], m);
    fin[r][0] = m;
    fin[r][1] = l;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < rows * D; e += kAttnThreads) {
    const int r = e / D, d = e - r * D, ds = AttnOut<D, R>::at(d);
    const int ti = r / a.G, hi = h * a.G + (r - ti * a.G);
    const int64_t flat = (static_cast<int64_t>(b) * a.Hq + hi) * a.Tq + ti;
    const float m = fin[r][0], l = fin[r][1];
    float x = 0.0f;
#pragma unroll
    for (int w = 0; w < kAttnWarps; ++w) x += buf->o[w][r][ds];
    if (a.splits > 1) {
      const int64_t at = static_cast<int64_t>(split) * a.B * a.Hq * a.Tq + flat;
      a.part_o[at * D + d] = x;
      if (d == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(m, l);
      continue;
    }
    x = l == 0.0f ? 0.0f : x / l;
    const int64_t at = b * a.ob + hi * a.oh + ti * a.ot + d;
    if (a.q_f16) static_cast<__half*>(a.out)[at] = __float2half_rn(x);
    else static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(x);
    if (d == 0) a.lse[flat] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
  }
}
// Positions that token ti of Tq sees.
__device__ __forceinline__ int attn_limit(const Kv8AttnArgs& a, int len, int ti) {
  return a.causal ? min(max(len - a.Tq + ti + 1, 0), len) : len;
}

template <int D>
__global__ void __launch_bounds__(kAttnThreads)
    kv8_attn_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                    const Kv8AttnArgs a) {
  constexpr int KS = D / 16;   // k16 steps of the K product
  constexpr int KW = D / 16;   // 32-bit words per lane and K token (D / 4 bytes)
  constexpr int VW = D / 32;   // words per lane and V token (D / 8 bytes)
  constexpr int NV = D / 8;    // n8 tiles of the output
  __shared__ float sm_ml[kAttnWarps][16][2];
  __shared__ float sm_fin[16][2];
  AttnRing<D>* ring = attn_ring<D>();
  attn_ring_init(ring, &tk, &tv);
  griddep_wait();
  griddep_launch_dependents();
  const Kv8Cache& c = a.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int split = blockIdx.x, b = blockIdx.z;
  const int rows = a.G * a.Tq, h = blockIdx.y;  // at most 16 rows
  const int cap = c.max_blocks << c.log_t;
  const int len = min(max(a.lens[b], 0), cap);

  // rows g and g + 8 of this lane: how many positions each sees
  int lim[2];
  int64_t q_at[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = min(g + 8 * i, rows - 1);
    const int ti = r / a.G, hi = h * a.G + (r - ti * a.G);
    lim[i] = attn_limit(a, len, ti);
    q_at[i] = b * a.qb + hi * a.qh + ti * a.qt;
  }
  // the tile's last row sees the most, its first the least
  const int lim_max = attn_limit(a, len, (rows - 1) / a.G), lim_min = attn_limit(a, len, 0);
  const int tiles = (lim_max + 15) >> 4;  // 16-token tiles to visit
  const int chunks = (tiles + kAttnWarps - 1) / kAttnWarps;
  const int c0 = static_cast<int>(static_cast<int64_t>(chunks) * split / a.splits);
  const int c1 = static_cast<int>(static_cast<int64_t>(chunks) * (split + 1) / a.splits);

  // ---- q fragments, scaled to fp16
  uint32_t qf[KS][4];
  float sc[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint16_t* src = static_cast<const uint16_t*>(a.q) + q_at[i] + t * (D / 4);
    uint32_t raw[KS * 2];
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(src) + j);
      raw[4 * j] = v.x; raw[4 * j + 1] = v.y; raw[4 * j + 2] = v.z; raw[4 * j + 3] = v.w;
    }
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < KS * 2; ++j) top = max(top, max(raw[j] & 0x7FFFu, (raw[j] >> 16) & 0x7FFFu));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    float inv = 1.0f, up = 1.0f;
    if (!a.q_f16) {
      const int ex = min(max(static_cast<int>(top >> 7), 1), 253);
      inv = __uint_as_float(static_cast<uint32_t>(254 - ex) << 23);
      up = __uint_as_float(static_cast<uint32_t>(ex) << 23);
    }
    sc[i] = q_finite(top, a.q_f16) ? a.scale_log2 * up : __uint_as_float(0x7FC00000u);
#pragma unroll
    for (int j = 0; j < KS; ++j) {
      qf[j][i] = q_pair(raw[2 * j], a.q_f16, inv);
      qf[j][i + 2] = q_pair(raw[2 * j + 1], a.q_f16, inv);
    }
  }

  float o[NV][4];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

  if (warp == kAttnWarps) attn_produce(a, &tk, &tv, ring, b, h, c0, c1, tiles);
  for (int n = 0; warp < kAttnWarps && n < c1 - c0; ++n) {
    const int s_ = n % kAttnStages;
    if (!mbar_wait_warp(&ring->full[s_], (n / kAttnStages) & 1, &ring->abort)) break;
    const float4 meta = ring->meta[s_][warp];
    if (meta.w == 0.0f) {
      __syncwarp();
      if (lane == 0) mbar_arrive(&ring->empty[s_]);
      continue;
    }
    uint32_t kw[2][KW], vw[4][VW];
    attn_read_k<D>(ring->k[s_] + warp * 16 * D, g, t, kw);
    const int pos = ((c0 + n) * kAttnWarps + warp) << 4;
    const bool zero_v = meta.w == 2.0f;
    const float lv = meta.y, iv = meta.z;
    const float ksc[2] = {meta.x * sc[0], meta.x * sc[1]};

    // ---- scores of 16 tokens
    float s[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] = 0.0f;
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        const uint32_t w = kw[i][j] ^ 0x80808080u;
        mma_f16(s[i], qf[j], i8_lo(w), i8_hi(w));
      }
    }
    const bool mask = pos + 16 > lim_min;
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = j >> 1;
        s[i][j] = fmaf(s[i][j], ksc[r], lv);
        if (mask && pos + 8 * i + 2 * t + (j & 1) >= lim[r]) s[i][j] = -INFINITY;
        top[r] = fmaxf(top[r], s[i][j]);
      }
    float corr[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
      const float mn = fmaxf(m[r], top[r] - kAttnHead);
      corr[r] = safe_ex2_diff(m[r], mn);
      m[r] = mn;
      l[r] *= corr[r];
    }
    uint32_t pf[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float p[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = j >> 1;
        // a masked score is exactly -inf; a NaN one (NaN q or scales) stays NaN
        p[j] = s[i][j] == -INFINITY ? 0.0f : ex2_approx(s[i][j] - m[r]);
        l[r] = fmaf(p[j], iv, l[r]);
      }
      pf[2 * i] = zero_v ? 0u : pack_f16x2(p[0], p[1]);
      pf[2 * i + 1] = zero_v ? 0u : pack_f16x2(p[2], p[3]);
    }
    if (__any_sync(0xffffffffu, corr[0] != 1.0f || corr[1] != 1.0f)) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        o[i][0] *= corr[0]; o[i][1] *= corr[0];
        o[i][2] *= corr[1]; o[i][3] *= corr[1];
      }
    }
    attn_read_v<D>(ring->v[s_] + warp * 16 * D, g, t, vw);
    __syncwarp();
    if (lane == 0) mbar_arrive(&ring->empty[s_]);
    // ---- P V: tiles 4w .. 4w+3 come from word w of the four tokens
#pragma unroll
    for (int w = 0; w < VW; ++w) {
      const uint32_t ta = vw[0][w] ^ 0x80808080u, tb = vw[1][w] ^ 0x80808080u;
      const uint32_t tc = vw[2][w] ^ 0x80808080u, td = vw[3][w] ^ 0x80808080u;
      const uint32_t ab0 = __byte_perm(ta, tb, 0x5140), ab1 = __byte_perm(ta, tb, 0x7362);
      const uint32_t cd0 = __byte_perm(tc, td, 0x5140), cd1 = __byte_perm(tc, td, 0x7362);
      mma_f16(o[4 * w], pf, i8_lo(ab0), i8_lo(cd0));
      mma_f16(o[4 * w + 1], pf, i8_hi(ab0), i8_hi(cd0));
      mma_f16(o[4 * w + 2], pf, i8_lo(ab1), i8_lo(cd1));
      mma_f16(o[4 * w + 3], pf, i8_hi(ab1), i8_hi(cd1));
    }
  }

  // ---- join the warps (in order), then store or hand over the partial
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    if (t == 0 && warp < kAttnWarps) {
      sm_ml[warp][g + 8 * r][0] = m[r];
      sm_ml[warp][g + 8 * r][1] = l[r];
    }
  }
  __syncthreads();
  AttnOut<D, 16>* buf = reinterpret_cast<AttnOut<D, 16>*>(ring->k);
  static_assert(sizeof(AttnOut<D, 16>) <= sizeof(ring->k) + sizeof(ring->v), "");
  if (warp < kAttnWarps) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float mt = sm_ml[0][g + 8 * r][0];
#pragma unroll
      for (int w = 1; w < kAttnWarps; ++w) mt = fmaxf(mt, sm_ml[w][g + 8 * r][0]);
      const float f = safe_ex2_diff(m[r], mt);
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)  // tile i, column 2t + j is d = (D / 8) (2t + j) + i
          buf->o[warp][g + 8 * r][AttnOut<D, 16>::at((2 * t + j) * (D / 8) + i)] = o[i][2 * r + j] * f;
    }
  }
  attn_epilogue<D, 16>(a, buf, sm_ml, sm_fin, b, h, split, rows);
}

// ---- up to 8 rows per key/value head (one token of up to 8 grouped heads)
//
// q.K on the integer tensor path: q's row, scaled by a power of two 2^-E to
// |v| < 64, is three int8 digits v = p0 + p1 / 128 + p2 / 128^2 (within 2^-21 of
// 2^E), and K's codes are the other operand as they are stored: no instruction
// converts them.  Rows 0-7 of an m16n8k32 MMA hold p0 and rows 8-15 p1 of the 8
// rows, a second MMA p2.  The int32 accumulators start at the bits of 1.5 * 2^23,
// so a subtraction turns each sum (|sum| <= 64 * 127 * 128 < 2^20) into its fp32
// value exactly.
//
// P V is computed transposed, V^T (16 d x 16 tokens) as the MMA's rows and P as its
// 8 columns: half the MMAs and accumulators of the 16-row form.
//
// Bound: HBM for long caches.  32 sequences of 0 to 32767 tokens, 8 heads of 8 rows, D 128:
// 198 to 202 us in a captured graph, 0.82 of the measured copy, 214 (0.77) among eager calls;
// one sequence of 8193 tokens, 5 rows: 9.8 us (11.2), of which the splits' join and two
// launches' latency are half.
__device__ __forceinline__ void mma_s8_start(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  const int z = 0x4B400000;
  asm(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%10,%10,%10};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(z));
}
__device__ __forceinline__ void mma_s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <int D>
__global__ void __launch_bounds__(kAttnThreads, 3)
    kv8_attn8_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                     const Kv8AttnArgs a) {
  constexpr int KS = D / 32;   // k32 steps of the K product
  constexpr int VW = D / 32;   // words per lane and V token
  constexpr int NM = D / 16;   // m16 tiles of the output
  __shared__ float sm_ml[kAttnWarps][8][2];
  __shared__ float sm_fin[8][2];
  AttnRing<D>* ring = attn_ring<D>();
  attn_ring_init(ring, &tk, &tv);
  griddep_wait();
  griddep_launch_dependents();
  const Kv8Cache& c = a.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int split = blockIdx.x, b = blockIdx.z, rows = a.G * a.Tq, h = blockIdx.y;
  const int len = min(max(a.lens[b], 0), c.max_blocks << c.log_t);
  const int lim = attn_limit(a, len, min(g, rows - 1) / a.G);
  const int lim_max = attn_limit(a, len, (rows - 1) / a.G), lim_min = attn_limit(a, len, 0);
  const int tiles = (lim_max + 15) >> 4;
  const int chunks = (tiles + kAttnWarps - 1) / kAttnWarps;
  const int c0 = static_cast<int>(static_cast<int64_t>(chunks) * split / a.splits);
  const int c1 = static_cast<int>(static_cast<int64_t>(chunks) * (split + 1) / a.splits);
  if (warp == kAttnWarps) attn_produce(a, &tk, &tv, ring, b, h, c0, c1, tiles);

  // ---- q digits of row g, quarter t: each warp makes its share of the words
  __shared__ uint32_t sm_q[3][D / 16][32];
  uint32_t q01[KS][4], q2[KS][2];
  float sc = 0.0f;
  if (warp < kAttnWarps) {
    const int r = min(g, rows - 1), ti = r / a.G, hi = h * a.G + (r - ti * a.G);
    const uint16_t* src = static_cast<const uint16_t*>(a.q) + b * a.qb + hi * a.qh + ti * a.qt + t * (D / 4);
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(src) + j);
      const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) top = max(top, max(u[i] & 0x7FFFu, (u[i] >> 16) & 0x7FFFu));
    }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    float down, up;
    digit_scale(top, a.q_f16, &down, &up);
    sc = a.scale_log2 * up;
    for (int j = warp; j < D / 16; j += kAttnWarps) {  // 4 values: word j of the lane's K bytes
      const uint2 u2 = *reinterpret_cast<const uint2*>(src + 4 * j);
      const uint32_t u[2] = {u2.x, u2.y};
      uint32_t p[3][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint16_t e = static_cast<uint16_t>(u[i >> 1] >> (16 * (i & 1)));
        const float v = a.q_f16 ? __half2float(*reinterpret_cast<const __half*>(&e))
                                : __uint_as_float(static_cast<uint32_t>(e) << 16);
        digits3(v * down, p[0][i], p[1][i], p[2][i]);
      }
#pragma unroll
      for (int i = 0; i < 3; ++i) sm_q[i][j][lane] = low_bytes(p[i][0], p[i][1], p[i][2], p[i][3]);
    }
    named_bar_sync(1, 32 * kAttnWarps);
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      q01[j >> 1][2 * (j & 1)] = sm_q[0][j][lane];
      q01[j >> 1][2 * (j & 1) + 1] = sm_q[1][j][lane];
      q2[j >> 1][j & 1] = sm_q[2][j][lane];
    }
  }

  float o[NM][4];
#pragma unroll
  for (int i = 0; i < NM; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;
  float m = -INFINITY, l = 0.0f;

  for (int n = 0; warp < kAttnWarps && n < c1 - c0; ++n) {
    const int s_ = n % kAttnStages;
    if (!mbar_wait_warp(&ring->full[s_], (n / kAttnStages) & 1, &ring->abort)) break;
    const float4 meta = ring->meta[s_][warp];
    if (meta.w == 0.0f) {
      __syncwarp();
      if (lane == 0) mbar_arrive(&ring->empty[s_]);
      continue;
    }
    uint32_t kw[2][D / 16], vw[4][VW];
    attn_read_k<D>(ring->k[s_] + warp * 16 * D, g, t, kw);
    const bool zero_v = meta.w == 2.0f;
    const float lv = meta.y, iv = meta.z, ksc = meta.x * sc;
    float s[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      int d01[4], d2[4];
      mma_s8_start(d01, q01[0], kw[i][0], kw[i][1]);
      const uint32_t z0[4] = {q2[0][0], 0u, q2[0][1], 0u};
      mma_s8_start(d2, z0, kw[i][0], kw[i][1]);
#pragma unroll
      for (int j = 1; j < KS; ++j) {
        mma_s8(d01, q01[j], kw[i][2 * j], kw[i][2 * j + 1]);
        const uint32_t zj[4] = {q2[j][0], 0u, q2[j][1], 0u};
        mma_s8(d2, zj, kw[i][2 * j], kw[i][2 * j + 1]);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float f0 = __int_as_float(d01[j]) - 12582912.0f, f1 = __int_as_float(d01[j + 2]) - 12582912.0f,
                    f2 = __int_as_float(d2[j]) - 12582912.0f;
        s[2 * i + j] = fmaf(fmaf(fmaf(f2, 0.0078125f, f1), 0.0078125f, f0), ksc, lv);
      }
    }
    const int pos = ((c0 + n) * kAttnWarps + warp) << 4;
    if (pos + 16 > lim_min) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (pos + 8 * (i >> 1) + 2 * t + (i & 1) >= lim) s[i] = -INFINITY;
    }
    float top = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    top -= kAttnHead;
    if (__any_sync(0xffffffffu, top > m)) {
      const float mn = fmaxf(m, top);
      const float corr = safe_ex2_diff(m, mn);
      m = mn;
      l *= corr;
      // the accumulators' columns are rows 2t and 2t + 1
      const float c0 = __shfl_sync(0xffffffffu, corr, 8 * t), c1 = __shfl_sync(0xffffffffu, corr, 8 * t + 4);
#pragma unroll
      for (int i = 0; i < NM; ++i) {
        o[i][0] *= c0; o[i][1] *= c1;
        o[i][2] *= c0; o[i][3] *= c1;
      }
    }
    float p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)  // a masked score is exactly -inf; a NaN one stays NaN
      p[i] = s[i] == -INFINITY ? 0.0f : ex2_approx(s[i] - m);
    l = fmaf((p[0] + p[1]) + (p[2] + p[3]), iv, l);
    const uint32_t pb0 = zero_v ? 0u : pack_f16x2(p[0], p[1]), pb1 = zero_v ? 0u : pack_f16x2(p[2], p[3]);
    attn_read_v<D>(ring->v[s_] + warp * 16 * D, g, t, vw);
    __syncwarp();
    if (lane == 0) mbar_arrive(&ring->empty[s_]);
#pragma unroll
    for (int w = 0; w < VW; ++w) {
      const uint32_t ta = vw[0][w] ^ 0x80808080u, tb = vw[1][w] ^ 0x80808080u;
      const uint32_t tc = vw[2][w] ^ 0x80808080u, td = vw[3][w] ^ 0x80808080u;
      const uint32_t ab0 = __byte_perm(ta, tb, 0x5140), ab1 = __byte_perm(ta, tb, 0x7362);
      const uint32_t cd0 = __byte_perm(tc, td, 0x5140), cd1 = __byte_perm(tc, td, 0x7362);
      const uint32_t a0[4] = {i8_lo(ab0), i8_hi(ab0), i8_lo(cd0), i8_hi(cd0)};
      const uint32_t a1[4] = {i8_lo(ab1), i8_hi(ab1), i8_lo(cd1), i8_hi(cd1)};
      mma_f16(o[2 * w], a0, pb0, pb1);
      mma_f16(o[2 * w + 1], a1, pb0, pb1);
    }
  }

  // ---- join the warps (in order), then store or hand over the partial
  l += __shfl_xor_sync(0xffffffffu, l, 1);
  l += __shfl_xor_sync(0xffffffffu, l, 2);
  if (t == 0 && warp < kAttnWarps) {
    sm_ml[warp][g][0] = m;
    sm_ml[warp][g][1] = l;
  }
  __syncthreads();
  AttnOut<D, 8>* buf = reinterpret_cast<AttnOut<D, 8>*>(ring->k);
  if (warp < kAttnWarps) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float mt = sm_ml[0][2 * t + j][0];
#pragma unroll
      for (int w = 1; w < kAttnWarps; ++w) mt = fmaxf(mt, sm_ml[w][2 * t + j][0]);
      const float f = safe_ex2_diff(sm_ml[warp][2 * t + j][0], mt);
#pragma unroll
      for (int i = 0; i < NM; ++i)
#pragma unroll
        for (int r = 0; r < 2; ++r)  // tile i: this lane's rows g and g + 8 are d = (D / 8) g + 2 i and + 1
          buf->o[warp][2 * t + j][AttnOut<D, 8>::at(g * (D / 8) + 2 * i + r)] = o[i][2 * r + j] * f;
    }
  }
  attn_epilogue<D, 8>(a, buf, sm_ml, sm_fin, b, h, split, rows);
}

// Joins up to 8 splits of each row, one warp per row.
template <int D>
__global__ void __launch_bounds__(256) kv8_attn_join_few_kernel(const Kv8AttnArgs a) {
  constexpr int VL = D / 32;  // values per lane
  griddep_wait();
  griddep_launch_dependents();
  const int64_t rows = static_cast<int64_t>(a.B) * a.Hq * a.Tq;
  const int64_t flat = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (flat >= rows) return;
  const int lane = threadIdx.x & 31;
  float2 ml = make_float2(-INFINITY, 0.0f);
  if (lane < a.splits) ml = *reinterpret_cast<const float2*>(a.part_ml + (lane * rows + flat) * 2);
  float x[8][VL];
#pragma unroll
  for (int s = 0; s < 8; ++s)
    if (s < a.splits) {
      const float* p = a.part_o + (s * rows + flat) * D + lane * VL;
      if constexpr (VL == 4) {
        const float4 v = *reinterpret_cast<const float4*>(p);
        x[s][0] = v.x; x[s][1] = v.y; x[s][2] = v.z; x[s][3] = v.w;
      } else {
        const float2 v = *reinterpret_cast<const float2*>(p);
        x[s][0] = v.x; x[s][1] = v.y;
      }
    }
  float top = ml.x;
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  top = __shfl_sync(0xffffffffu, top, 0);
  const float f = safe_ex2_diff(ml.x, top);
  float lt = 0.0f, acc[VL];
#pragma unroll
  for (int i = 0; i < VL; ++i) acc[i] = 0.0f;
#pragma unroll
  for (int s = 0; s < 8; ++s) {
    const float fs = __shfl_sync(0xffffffffu, f, s), ls = __shfl_sync(0xffffffffu, ml.y, s);
    if (s < a.splits) {
      lt = fmaf(ls, fs, lt);
#pragma unroll
      for (int i = 0; i < VL; ++i) acc[i] = fmaf(x[s][i], fs, acc[i]);
    }
  }
  const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;
  const int ti = static_cast<int>(flat % a.Tq);
  const int64_t bh = flat / a.Tq, b = bh / a.Hq, hi = bh - b * a.Hq;
  uint16_t* dst = static_cast<uint16_t*>(a.out) + b * a.ob + hi * a.oh + ti * a.ot + lane * VL;
#pragma unroll
  for (int i = 0; i < VL; i += 2)
    *reinterpret_cast<uint32_t*>(dst + i) = a.q_f16 ? pack_f16x2(acc[i] * inv, acc[i + 1] * inv)
                                                    : pack_bf16x2(acc[i] * inv, acc[i + 1] * inv);
  if (lane == 0) a.lse[flat] = lt == 0.0f ? -INFINITY : (top + log2f(lt)) * 0.6931471805599453f;
}

// Joins up to 64 splits of a row: one CTA per row.  Every warp weighs all splits
// (lane i has splits i and i + 32) and sums every kJoinWarps-th split's D values;
// the warps' sums are added in order.  All loads are independent of one another.
constexpr int kJoinWarps = 8;
template <int D>
__global__ void __launch_bounds__(kJoinWarps * 32) kv8_attn_join_kernel(const Kv8AttnArgs a) {
  constexpr int VL = D / 32;  // values per lane
  __shared__ float sums[kJoinWarps][D];
  griddep_wait();
  griddep_launch_dependents();
  const int64_t flat = blockIdx.x, rows = gridDim.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (lane + 32 * i < a.splits) {
      const float2 v = *reinterpret_cast<const float2*>(a.part_ml + ((lane + 32 * i) * rows + flat) * 2);
      m[i] = v.x;
      l[i] = v.y;
    }
  float x[kAttnMaxSplits / kJoinWarps][VL];
#pragma unroll
  for (int k = 0; k < kAttnMaxSplits / kJoinWarps; ++k) {
    const int s = warp + kJoinWarps * k;
    if (s < a.splits) {
      const float* p = a.part_o + (s * rows + flat) * D + lane * VL;
      if constexpr (VL == 4) {
        const float4 v = *reinterpret_cast<const float4*>(p);
        x[k][0] = v.x; x[k][1] = v.y; x[k][2] = v.z; x[k][3] = v.w;
      } else {
        const float2 v = *reinterpret_cast<const float2*>(p);
        x[k][0] = v.x; x[k][1] = v.y;
      }
    }
  }
  float top = fmaxf(m[0], m[1]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float f[2] = {safe_ex2_diff(m[0], top), safe_ex2_diff(m[1], top)};
  float lt = l[0] * f[0] + l[1] * f[1];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) lt += __shfl_xor_sync(0xffffffffu, lt, o);
  float acc[VL];
#pragma unroll
  for (int i = 0; i < VL; ++i) acc[i] = 0.0f;
#pragma unroll
  for (int k = 0; k < kAttnMaxSplits / kJoinWarps; ++k) {
    const int s = warp + kJoinWarps * k;
    const float fs = __shfl_sync(0xffffffffu, k < 32 / kJoinWarps ? f[0] : f[1], s & 31);
    if (s < a.splits) {
#pragma unroll
      for (int i = 0; i < VL; ++i) acc[i] = fmaf(x[k][i], fs, acc[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < VL; ++i) sums[warp][lane * VL + i] = acc[i];
  __syncthreads();
  if (threadIdx.x < D) {
    float o = 0.0f;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) o += sums[w][threadIdx.x];
    o = lt == 0.0f ? 0.0f : o / lt;
    const int ti = static_cast<int>(flat % a.Tq);
    const int64_t bh = flat / a.Tq, b = bh / a.Hq, hi = bh - b * a.Hq;
    const int64_t at = b * a.ob + hi * a.oh + ti * a.ot + threadIdx.x;
    if (a.q_f16) static_cast<__half*>(a.out)[at] = __float2half_rn(o);
    else static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(o);
    if (threadIdx.x == 0) a.lse[flat] = lt == 0.0f ? -INFINITY : (top + log2f(lt)) * 0.6931471805599453f;
  }
}

}  // namespace b200q
