// Attention over the paged 8-bit cache for many rows per key/value head (a prompt's
// chunk, or many grouped heads): 128 packed rows (token * G + head) per CTA on the
// tensor cores' tcgen05 MMAs, fp16 operands, fp32 accumulators in TMEM.
//
// The mathematics is that of kv8.cuh: codes are exact in fp16, q's rows are scaled by
// a power of two, the weights are P = 2^(sigma + log2 vs - m) and the sum of P / vs
// divides at the end.  m starts 7 below a row's largest exponent and is only raised when
// that has grown by more than 8 (P <= 2^15 fits fp16), so the accumulator in TMEM is
// rarely rescaled.
//
// A CTA has RT row tiles of 128 (2 when there are more than 128 rows: K and V are
// then widened once for 256 rows).  Per 64-token stage:
//   warps 0 .. 4 RT - 1   softmax, one thread per row: S from TMEM, P back over it
//   the next four         int8 -> fp16: K and V as 64 x D tiles, rows of 128 bytes with
//                         the 128-byte swizzle
//   then                  the TMA producer (the ring of kv8.cuh)
//   and                   the MMAs, one thread: S[128 x 64] = Q K^T (both K-major), then
//                         O[128 x D] += P V with P from TMEM and V as the N-major
//                         operand its rows are (no transpose)
// S has two buffers: stage j + 1's scores are computed while stage j's softmax runs.
// RT = 2 takes an SM's whole TMEM and double-buffers the fp16 tiles; RT = 1 puts two
// CTAs on an SM.  Four chunks of 129 tokens (5 rows each) over 4001 to 12001: 186 us, 0.28
// of the measured GEMM rate (one 128-row tile per CTA 253 us; sequences in any order 201).
// A prompt into an empty cache, 40 heads over 8: 512 tokens 27 us, 2048 193 us, 8192 1.24 ms
// (0.34), 32768 16.6 ms (0.41).
// Bound: the chain scores -> softmax -> P V of a stage, above all the scores, whose MMAs of
// 64 columns read q's tile from shared memory for each stage: with an eighth of them 201
// became 152 us; without conversion 188, exponentials 195, rescaling 190.
#pragma once

#include "kv8.cuh"

namespace b200q {

constexpr int kPfRows = 128;
constexpr int pf_threads(int rt) { return 128 * rt + 192; }
constexpr int pf_stages(int rt) { return rt == 2 ? 4 : 2; }

template <int D, int RT>
struct PfSmem {
  static constexpr int NB = RT;                   // fp16 tiles of K and of V
  AttnRing<D, pf_stages(RT)> ring;
  alignas(1024) uint8_t q[RT][kPfRows * D * 2];   // D / 64 atoms of 128 rows x 128 bytes
  alignas(1024) uint8_t k[NB][64 * D * 2];        // D / 64 atoms of 64 rows x 128 bytes
  alignas(1024) uint8_t v[NB][64 * D * 2];
  uint64_t k_full[NB], k_empty[NB], v_full[NB], v_empty[NB];
  // the last P V has its own: the last scores only say that the last but one's is issued,
  // and one parity cannot tell "two to go" from "done"
  uint64_t o_done[RT], o_last[RT];
  // by S buffer: one side may be a whole stage ahead of the other, and a wait tells only
  // the last phase from the one before
  uint64_t s_full[RT][2], p_full[RT][2];
  uint32_t tmem;
};
template <int D, int RT>
constexpr int pf_smem_bytes() {
  return static_cast<int>(sizeof(PfSmem<D, RT>)) + 1024;
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void pf_tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void pf_tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// D(tmem) (+)= A(tmem) x B(smem desc), kind::f16, one thread.
__device__ __forceinline__ void pf_umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// Descriptor of an N-major operand in the same tiles: rows of 64 values of N (128
// bytes, swizzled), 8-row groups of K 1024 bytes apart (the stride field), 64-value
// atoms of N `atom` bytes apart (the leading field).
__device__ __forceinline__ uint64_t pf_nmajor_desc(uint32_t smem_addr, uint32_t atom) {
  return (make_sw128_desc(smem_addr) & ~(uint64_t(0x3FFF) << 16)) | (uint64_t((atom >> 4) & 0x3FFFu) << 16);
}

// 16 int8 codes as 16 fp16 values.
__device__ __forceinline__ void pf_widen(const uint4& c, uint4& lo, uint4& hi) {
  const uint32_t w[4] = {c.x ^ 0x80808080u, c.y ^ 0x80808080u, c.z ^ 0x80808080u, c.w ^ 0x80808080u};
  lo = make_uint4(i8_lo(w[0]), i8_hi(w[0]), i8_lo(w[1]), i8_hi(w[1]));
  hi = make_uint4(i8_lo(w[2]), i8_hi(w[2]), i8_lo(w[3]), i8_hi(w[3]));
}
// Widens a 64 x D tile with 128 threads (x = 0 .. 127).  Eight lanes take four chunks
// of rows r and r ^ 5: with the two swizzles neither the reads nor the writes collide.
template <int D>
__device__ __forceinline__ void pf_convert(const uint8_t* src, uint8_t* dst, int x) {
  constexpr int HALVES = D / 64;  // groups of four 16-byte chunks per row
#pragma unroll
  for (int it = 0; it < 2 * HALVES; ++it) {
    const int c = (x & 3) + 4 * (it % HALVES);
    const int idx = (x >> 3) + 16 * (it / HALVES);
    const int row = (idx >> 2) * 8 + ((idx & 3) ^ (((x >> 2) & 1) * 5));
    uint4 lo, hi;
    pf_widen(*reinterpret_cast<const uint4*>(src + attn_at<D>(row, c)), lo, hi);
    uint8_t* to = dst + ((2 * c) >> 3) * (64 * 128) + row * 128;
    *reinterpret_cast<uint4*>(to + ((((2 * c) & 7) ^ (row & 7)) << 4)) = lo;
    *reinterpret_cast<uint4*>(to + ((((2 * c + 1) & 7) ^ (row & 7)) << 4)) = hi;
  }
}

// The sequence of this CTA.  CTAs start in grid order, and long ones that start last leave SMs
// idle: longest first (the four chunks above: 201 -> 185 us).  Called by whole warps.
__device__ __forceinline__ int attn_sequence(const Kv8AttnArgs& a) {
  const int z = blockIdx.z, lane = threadIdx.x & 31;
  if (!a.longest_first) return z;
  const int len = lane < a.B ? a.lens[lane] : 0;
  int rank = 0;
  for (int i = 0; i < a.B; ++i) {
    const int other = __shfl_sync(0xffffffffu, len, i);
    rank += other > len || (other == len && i < lane);
  }
  return __ffs(__ballot_sync(0xffffffffu, lane < a.B && rank == z)) - 1;
}

template <int D, int RT>
__global__ void __launch_bounds__(128 * RT + 192, RT == 2 ? 1 : 2)
    kv8_prefill_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                       const Kv8AttnArgs a) {
  extern __shared__ uint8_t smem_raw[];
  using Smem = PfSmem<D, RT>;
  constexpr int NB = Smem::NB, ST = RT == 2 ? 4 : 2;
  constexpr int kSoft = 4 * RT;            // softmax warps
  constexpr uint32_t kCols = 256 * RT;     // TMEM: S at 128 r + 64 (stage & 1), O at 128 (RT + r)
  Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  AttnRing<D, ST>* ring = &sm.ring;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < NB; ++i) {
      mbar_init(&sm.k_full[i], 4);  // warps
      mbar_init(&sm.v_full[i], 4);
      mbar_init(&sm.k_empty[i], 1);
      mbar_init(&sm.v_empty[i], 1);
    }
    for (int i = 0; i < RT; ++i) {
      for (int j = 0; j < 2; ++j) {
        mbar_init(&sm.p_full[i][j], 4);
        mbar_init(&sm.s_full[i][j], 1);
      }
      mbar_init(&sm.o_done[i], 1);
      mbar_init(&sm.o_last[i], 1);
    }
  }
  if (warp == kSoft + 5) {
    tmem_alloc(&sm.tmem, kCols);
    tmem_relinquish();
  }
  attn_ring_init(ring, &tk, &tv, kSoft + 4);  // softmax warps and converters; ends with a barrier
  griddep_wait();
  griddep_launch_dependents();

  const Kv8Cache& c = a.c;
  // grid (splits * heads * row tiles, 1, B): a prompt's heads x tiles go past what y holds
  const int split = blockIdx.x % a.splits, b = attn_sequence(a), rows = a.G * a.Tq;
  const int row_tiles = (rows + kPfRows * RT - 1) / (kPfRows * RT), tile = blockIdx.x / a.splits;
  const int h = tile / row_tiles, r0 = (tile - h * row_tiles) * (kPfRows * RT);
  const int len = min(max(a.lens[b], 0), c.max_blocks << c.log_t);
  const int last = min(r0 + kPfRows * RT, rows) - 1;
  const int lim_max = attn_limit(a, len, last / a.G), lim_min = attn_limit(a, len, r0 / a.G);
  const int tiles = (lim_max + 15) >> 4, chunks = (tiles + 3) >> 2;
  const int c0 = static_cast<int>(static_cast<int64_t>(chunks) * split / a.splits);
  const int c1 = static_cast<int>(static_cast<int64_t>(chunks) * (split + 1) / a.splits);
  const int n_tiles = c1 - c0;
  volatile int* abort = &ring->abort;

  // ---- Q: one row per softmax thread, scaled to fp16, K-major tile
  float sc = 0.0f;
  int lim = 0, ti = 0, hi = 0;
  if (warp < kSoft) {
    const int r = min(r0 + tid, rows - 1), row = tid & 127;
    uint8_t* qs = sm.q[tid >> 7];
    ti = r / a.G;
    hi = h * a.G + (r - ti * a.G);
    lim = attn_limit(a, len, ti);
    const uint16_t* src = static_cast<const uint16_t*>(a.q) + b * a.qb + hi * a.qh + ti * a.qt;
    float inv = 1.0f, up = 1.0f;
    uint32_t top = 0;
    if (!a.q_f16) {
#pragma unroll 4
      for (int j = 0; j < D / 8; ++j) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(src) + j);
        const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, max(u[i] & 0x7FFFu, (u[i] >> 16) & 0x7FFFu));
      }
      const int ex = min(max(static_cast<int>(top >> 7), 1), 253);
      inv = __uint_as_float(static_cast<uint32_t>(254 - ex) << 23);
      up = __uint_as_float(static_cast<uint32_t>(ex) << 23);
    }
#pragma unroll 4
    for (int j = 0; j < D / 8; ++j) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(src) + j);
      if (a.q_f16) {
        const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, max(u[i] & 0x7FFFu, (u[i] >> 16) & 0x7FFFu));
      }
      *reinterpret_cast<uint4*>(qs + (j >> 3) * (kPfRows * 128) + row * 128 + (((j & 7) ^ (row & 7)) << 4)) =
          make_uint4(q_pair(v.x, a.q_f16, inv), q_pair(v.y, a.q_f16, inv), q_pair(v.z, a.q_f16, inv),
                     q_pair(v.w, a.q_f16, inv));
    }
    sc = q_finite(top, a.q_f16) ? a.scale_log2 * up : __uint_as_float(0x7FC00000u);
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem;

  float m = -INFINITY, l = 0.0f;
  if (warp == kSoft + 4) {
    attn_produce(a, &tk, &tv, ring, b, h, c0, c1, tiles);
  } else if (warp == kSoft + 5) {
    if (lane == 0) {
      constexpr uint32_t iqk = kind_idesc<MmaKind::F16>(kPfRows, 64);
      constexpr uint32_t ipv = kind_idesc<MmaKind::F16>(kPfRows, D) | (1u << 16);  // B is N-major
      auto scores = [&](int j) {
        const int kb = j % NB;
        if (!mbar_wait(&sm.k_full[kb], (j / NB) & 1, abort)) return false;
        tc_fence_after();
        const uint64_t dk = make_sw128_desc(smem_u32(sm.k[kb]));
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          // stage j - 2's P V still reads P from this buffer until it has completed: only
          // MMAs on one accumulator are ordered by themselves
          if (j >= 2 && !mbar_wait(&sm.o_done[r], j & 1, abort)) return false;
          const uint64_t dq = make_sw128_desc(smem_u32(sm.q[r]));
#pragma unroll
          for (int s = 0; s < D / 16; ++s)
            umma_ss<MmaKind::F16>(tmem + 128 * r + 64 * (j & 1), dq + (s >> 2) * (kPfRows * 128 >> 4) + (s & 3) * 2,
                                  dk + (s >> 2) * (64 * 128 >> 4) + (s & 3) * 2, iqk, s > 0);
          umma_commit(&sm.s_full[r][j & 1]);
        }
        umma_commit(&sm.k_empty[kb]);
        return true;
      };
      bool live = n_tiles > 0 && scores(0);
      for (int j = 0; live && j < n_tiles; ++j) {
        if (j + 1 < n_tiles && !scores(j + 1)) break;
        const int vb = j % NB;
        live = mbar_wait(&sm.v_full[vb], (j / NB) & 1, abort);
        const uint64_t dv = pf_nmajor_desc(smem_u32(sm.v[vb]), 64 * 128);
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          live = live && mbar_wait(&sm.p_full[r][j & 1], (j >> 1) & 1, abort);
          if (live) {
            tc_fence_after();
            const uint32_t tm_p = tmem + 128 * r + 64 * (j & 1);
#pragma unroll
            for (int s = 0; s < 4; ++s)
              pf_umma_ts(tmem + 128 * (RT + r), tm_p + s * 8, dv + s * (16 * 128 >> 4), ipv, j > 0 || s > 0);
            umma_commit(j + 1 < n_tiles ? &sm.o_done[r] : &sm.o_last[r]);
          }
        }
        if (live) umma_commit(&sm.v_empty[vb]);
      }
    }
    __syncwarp();
  } else if (warp >= kSoft) {
    const int x = tid - 128 * RT;
    for (int j = 0; j < n_tiles; ++j) {
      const int s = j % ST, nb = j % NB;
      if (!mbar_wait_warp(&ring->full[s], (j / ST) & 1, abort)) break;
      if (j >= NB && !mbar_wait_warp(&sm.k_empty[nb], (j / NB - 1) & 1, abort)) break;
      pf_convert<D>(ring->k[s], sm.k[nb], x);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.k_full[nb]);
      if (j >= NB && !mbar_wait_warp(&sm.v_empty[nb], (j / NB - 1) & 1, abort)) break;
      pf_convert<D>(ring->v[s], sm.v[nb], x);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&sm.v_full[nb]);
        mbar_arrive(&ring->empty[s]);
      }
    }
  } else {
    const int rt = warp >> 2;  // this warp's row tile; it may touch lanes 32 (warp % 4) ..
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tm_o = tmem + 128 * (RT + rt) + lane_base;
    const bool idle = r0 + 32 * warp >= rows;
    for (int j = 0; j < n_tiles; ++j) {
      const int st = j % ST;
      if (!mbar_wait_warp(&ring->full[st], (j / ST) & 1, abort)) break;
      float4 meta[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) meta[i] = ring->meta[st][i];
      __syncwarp();
      if (lane == 0) mbar_arrive(&ring->empty[st]);
      const uint32_t tm_s = tmem + 128 * rt + 64 * (j & 1) + lane_base;
      if (!mbar_wait_warp(&sm.s_full[rt][j & 1], (j >> 1) & 1, abort)) break;
      if (idle) {  // no row of this warp is stored: its lanes of P may hold anything
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_full[rt][j & 1]);
        continue;
      }
      tc_fence_after();
      uint32_t s0[32], s1[32];
      tmem_ld32(tm_s, s0);
      tmem_ld32(tm_s + 32, s1);
      tmem_ld_wait();
      const int pos = (c0 + j) * 64;
      // exponents: fma(S, ks * sc, log2 vs); a bad page's are -inf
      float ksc[4], add[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ksc[i] = meta[i].w == 0.0f ? 0.0f : meta[i].x * sc;
        add[i] = meta[i].w == 0.0f ? -INFINITY : meta[i].y;
      }
      float top = -INFINITY;
      const bool plain = pos + 64 <= lim_min && a.scale_log2 >= 0.0f;
      if (plain) {  // every row sees all 64: a sub-tile's largest S has its largest exponent
        auto largest = [&](const uint32_t (&r)[32], int half) {
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            float x = __uint_as_float(r[16 * q]);
#pragma unroll
            for (int i = 1; i < 16; ++i) x = fmaxf(x, __uint_as_float(r[16 * q + i]));
            top = fmaxf(top, fmaf(x, ksc[2 * half + q], add[2 * half + q]));
          }
        };
        largest(s0, 0);
        largest(s1, 1);
      } else {
        auto score = [&](uint32_t (&r)[32], int half) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const int q = half * 2 + (i >> 4);
            float x = fmaf(__uint_as_float(r[i]), ksc[q], add[q]);
            if (pos + half * 32 + i >= lim) x = -INFINITY;
            top = fmaxf(top, x);
            r[i] = __float_as_uint(x);
          }
        };
        score(s0, 0);
        score(s1, 1);
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // they are exponents now
          ksc[i] = 1.0f;
          add[i] = 0.0f;
        }
      }
      if (__any_sync(0xffffffffu, top > m + kAttnHead)) {
        const float mn = fmaxf(m, top - (kAttnHead - 8.0f));
        const float corr = safe_ex2_diff(m, mn);
        m = mn;
        l *= corr;
        if (j > 0) {
          if (!mbar_wait_warp(&sm.o_done[rt], (j - 1) & 1, abort)) break;  // the last P V
          tc_fence_after();
#pragma unroll 1
          for (int q = 0; q < D / 16; ++q) {
            uint32_t o[16];
            tmem_ld16(tm_o + 16 * q, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
            pf_tmem_st16(tm_o + 16 * q, o);
          }
          pf_tmem_st_wait();
        }
      }
      // P = 2^(exponent - m); -inf gives 0 whatever m is
      const float mf = m == -INFINITY ? 0.0f : m;
      auto weigh = [&](const uint32_t (&r)[32], int half) {
        uint32_t p[16];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int u = 2 * half + q;
          const float shift = add[u] - mf;
          const bool zero = meta[u].w == 2.0f;
          float sum = 0.0f;
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const float px = ex2_approx(fmaf(__uint_as_float(r[16 * q + i]), ksc[u], shift));
            const float py = ex2_approx(fmaf(__uint_as_float(r[16 * q + i + 1]), ksc[u], shift));
            sum += px + py;
            p[8 * q + (i >> 1)] = zero ? 0u : pack_f16x2(px, py);
          }
          l = fmaf(sum, meta[u].z, l);
        }
        pf_tmem_st16(tm_s + 16 * half, p);
      };
      weigh(s0, 0);
      weigh(s1, 1);
      pf_tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.p_full[rt][j & 1]);
    }
    // ---- O: the last P V has to complete; every lane stores its own row
    const bool good = n_tiles == 0 || mbar_wait_warp(&sm.o_last[rt], 0, abort);
    tc_fence_after();
    const bool stored = r0 + tid < rows && good;
    const int64_t flat = (static_cast<int64_t>(b) * a.Hq + hi) * a.Tq + ti;
    const int64_t part = static_cast<int64_t>(split) * a.B * a.Hq * a.Tq + flat;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint16_t* out = static_cast<uint16_t*>(a.out) + b * a.ob + hi * a.oh + ti * a.ot;
#pragma unroll 1
    for (int q = 0; q < D / 32; ++q) {
      uint32_t o[32];
      if (n_tiles > 0) {
        tmem_ld32(tm_o + 32 * q, o);
        tmem_ld_wait();
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = 0u;
      }
      if (stored && a.splits > 1) {
        float4* to = reinterpret_cast<float4*>(a.part_o + part * D + 32 * q);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          to[i] = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]), __uint_as_float(o[4 * i + 2]),
                              __uint_as_float(o[4 * i + 3]));
      } else if (stored) {
        uint4* to = reinterpret_cast<uint4*>(out + 32 * q);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float x = __uint_as_float(o[8 * i + 2 * k]) * inv, y = __uint_as_float(o[8 * i + 2 * k + 1]) * inv;
            w[k] = a.q_f16 ? pack_f16x2(x, y) : pack_bf16x2(x, y);
          }
          to[i] = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      __syncwarp();  // the next load wants the whole warp
    }
    if (stored) {
      if (a.splits > 1) *reinterpret_cast<float2*>(a.part_ml + part * 2) = make_float2(m, l);
      else a.lse[flat] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kSoft + 5) tmem_dealloc(tmem, kCols);
}

}  // namespace b200q
