// The 4-bit linear for tens to hundreds of tokens on the tcgen05 MMAs, without a decoded
// copy of the weight: 128 weight rows x TN tokens per CTA, K cut into slices when there
// are fewer tiles than SMs.
//
//   D[128 x TN] += A[128 x 64] B[64 x TN] per 64-code stage, fp16 operands, fp32 in TMEM
//   A: the weight, s * (c - z) * 2^-e with 2^e the power of two of the row's largest |s|
//      less 11 (so at most 15 * 2^12), decoded from the ring straight into TMEM: lane n of
//      the MMA's A operand is row n, so a thread decodes its own row and needs only its
//      own scales.  c - z is exact; its product with s is rounded once, to fp16's 11 bits
//      (an fp32 s is two fp16 parts: c * hi + c * lo in one FMA).
//   B: x as fp16 rows (a power of two per row taken out), brought by TMA.  A word's eight
//      codes decode as pairs (i, i + 4), so x's columns are stored in that order.
//
// Warps 0 .. 15 decode (four teams, a stage each in turn) and store the result; warp 16
// brings x, warp 18 the codes and the scales; warp 17 issues the MMAs.
//
// Bound: per stage and SM, x's TN * 128 bytes from L2 (64 bytes a cycle) against the MMAs'
// 2 * TN cycles and the decode.  K 5120, N 13824, 64 tokens: 50 us, 11 of them the operand
// kernel, 0.33 us per stage of which half stays with decode and MMAs taken out (x from L2
// into 108 SMs); 256 tokens: 63 us.  K 13824, N 5120, 200 tokens: 56 us.
#pragma once

#include "kv8_prefill.cuh"
#include "w4a16.cuh"

namespace b200q {

// ---------------------------------------------------------------- operands
// x16: fp16 rows with columns in pair order, x_pow their powers of two; sz [groups][ldn]:
// {hi | lo << 16, w4_zero} of each row's group, zeros past N and K; w_pow [N].
struct W4TilePrepareArgs {
  const void* x;
  int64_t ldx;
  int x_f16, x_vec, M, K;
  __half* x16;
  float* x_pow;
  const void* scales;
  int scale_dtype;
  const uint8_t* zeros;
  int N, KG, groups, ldn;  // KG = K / G; groups: a whole number of stages; ldn: N up to 128
  uint2* sz;
  float* w_pow;
  int scale_blocks, group_blocks;  // the first blocks: (rows, groups); the rest take a token row each
};

constexpr int kW4PrepRows = 32, kW4PrepGroups = 64;  // of a block

__global__ void __launch_bounds__(256) w4_tile_prepare_kernel(const W4TilePrepareArgs a) {
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (static_cast<int>(blockIdx.x) < a.scale_blocks) {
    __shared__ float inv_s[kW4PrepRows];
    __shared__ uint2 turns[2][kW4PrepRows][33];
    const int n0 = (blockIdx.x / a.group_blocks) * kW4PrepRows, gb = blockIdx.x % a.group_blocks;
    float m[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // of rows warp + 8 r
#pragma unroll 4
    for (int i = lane; i < a.KG; i += 32)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        m[r] = fmaxf(m[r], fabsf(load_scale(a.scales, a.scale_dtype,
                                            static_cast<int64_t>(min(n0 + warp + 8 * r, a.N - 1)) * a.KG + i)));
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = warp + 8 * r;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m[r] = fmaxf(m[r], __shfl_xor_sync(0xffffffffu, m[r], o));
      // 2^(127 - ex + 11) and its inverse are both normal
      const int ex = min(max(static_cast<int>(__float_as_uint(m[r]) >> 23), 12), 253);
      if (lane == 0) {
        inv_s[row] = __uint_as_float(static_cast<uint32_t>(265 - ex) << 23);
        if (gb == 0 && n0 + row < a.N) a.w_pow[n0 + row] = __uint_as_float(static_cast<uint32_t>(ex - 11) << 23);
      }
    }
    __syncwarp();
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int g0 = gb * kW4PrepGroups + 32 * half;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = warp + 8 * r;
        uint2 v = make_uint2(0, 0);
        if (n0 + row < a.N && g0 + lane < a.KG) {
          const int64_t at = static_cast<int64_t>(n0 + row) * a.KG + g0 + lane;
          const float s = load_scale(a.scales, a.scale_dtype, at) * inv_s[row];
          const __half hi = __float2half_rn(s);
          const float rest = s - __half2float(hi);  // (inf and NaN: hi carries them)
          const __half lo = __float2half_rn(fabsf(rest) <= 4.0f ? rest : 0.0f);
          v.x = __half_as_ushort(hi) | (static_cast<uint32_t>(__half_as_ushort(lo)) << 16);
          v.y = w4_zero(a.zeros ? __ldg(a.zeros + at) & 15u : 8u);
        }
        turns[half][row][lane] = v;
      }
    }
    __syncthreads();
    for (int g = warp; g < kW4PrepGroups; g += 8) {
      const int at = gb * kW4PrepGroups + g;
      if (at < a.groups) a.sz[static_cast<int64_t>(at) * a.ldn + n0 + lane] = turns[g >> 5][lane][g & 31];
    }
    return;
  }
  const int64_t m = blockIdx.x - a.scale_blocks;
  const uint16_t* row = static_cast<const uint16_t*>(a.x) + m * a.ldx;
  const int pieces = a.K >> 3;
  auto piece = [&](int p, uint32_t (&e)[4]) {
    if (a.x_vec) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(row + p * 8));
      e[0] = v.x; e[1] = v.y; e[2] = v.z; e[3] = v.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) e[j] = __ldg(row + p * 8 + 2 * j) | (uint32_t(__ldg(row + p * 8 + 2 * j + 1)) << 16);
    }
  };
  float inv = 1.0f, pow = 1.0f;
  if (!a.x_f16) {  // as in w4_prepare_kernel
    uint32_t top = 0;
#pragma unroll 4
    for (int p = threadIdx.x; p < pieces; p += 256) {
      uint32_t e[4];
      piece(p, e);
#pragma unroll
      for (int j = 0; j < 4; ++j) top = max(top, max(e[j] & 0x7FFFu, (e[j] >> 16) & 0x7FFFu));
    }
    __shared__ uint32_t tops[8];
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) tops[warp] = top;
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, tops[lane & 7]);
    const int ex = min(max(static_cast<int>(top >> 7), 1), 253);
    inv = __uint_as_float(static_cast<uint32_t>(254 - ex) << 23);
    pow = __uint_as_float(static_cast<uint32_t>(ex) << 23);
  }
  if (threadIdx.x == 0) a.x_pow[m] = pow;
  uint4* dst = reinterpret_cast<uint4*>(a.x16 + m * a.K);
#pragma unroll 4
  for (int p = threadIdx.x; p < pieces; p += 256) {
    uint32_t e[4];
    piece(p, e);
    if (!a.x_f16) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        e[j] = pack_f16x2(__uint_as_float(e[j] << 16) * inv, __uint_as_float(e[j] & 0xFFFF0000u) * inv);
    }
    dst[p] = make_uint4(__byte_perm(e[0], e[2], 0x5410), __byte_perm(e[0], e[2], 0x7632),
                        __byte_perm(e[1], e[3], 0x5410), __byte_perm(e[1], e[3], 0x7632));
  }
}

// v * a * b for powers of two a and b, the smaller first: x's row at 2^110 and then a scale of
// 2^-10 would leave fp32's range on the way to a value inside it.  (What the smaller one, at
// least 2^-126, takes off a subnormal product is below 2^-24 of the row's terms.)
__device__ __forceinline__ float times_powers(float v, float a, float b) { return v * fminf(a, b) * fmaxf(a, b); }

// ---------------------------------------------------------------- the product
struct W4TileArgs {
  const uint2* sz;
  int64_t ldn;
  const float *w_pow, *x_pow;
  float* part;  // [slices][M][N] fp32, or null: one slice, the epilogue runs here
  int M, N, slots, log_g, slices;  // slots of 256 codes
};

constexpr int kW4Teams = 4;  // of four warps: one per 64-code stage of a slot
constexpr int kW4TileThreads = (4 * kW4Teams + 3) * 32;
constexpr int w4_tile_stages(int tn) { return tn == 256 ? 4 : tn == 128 ? 6 : 8; }
// The weight's ring: 256 codes of 128 rows per slot, in 128-byte boxes (boxes of 32 bytes, 64
// codes, kept the copy engine at twice the time).  It has its own warp: behind x's waits it
// ran one slot ahead, 2 us per slot.
constexpr int w4_tile_slots(int tn) { return tn == 256 ? 3 : tn == 128 ? 5 : 6; }
template <int TN>
struct W4TileSmem {
  static constexpr int ST = w4_tile_stages(TN), SL = w4_tile_slots(TN);
  alignas(1024) uint8_t x[ST][TN * 128];  // 128-byte swizzle
  alignas(1024) uint8_t w[SL][128 * 128];
  alignas(16) uint2 sz[SL][8][128];
  uint64_t full[ST], decoded[ST], empty[ST], w_full[SL], w_empty[SL], done;
  uint32_t tmem;
  int abort;
};
template <int TN>
constexpr int w4_tile_smem_bytes() {
  return static_cast<int>(sizeof(W4TileSmem<TN>)) + 1024;
}

// LO: scales have a second part (fp32 ones).
template <int TN, bool LO>
__global__ void __launch_bounds__(kW4TileThreads)
    w4_tile_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tw, const W4TileArgs a,
                   const EpiArgs ep) {
  extern __shared__ uint8_t smem_raw[];
  using Smem = W4TileSmem<TN>;
  constexpr int ST = Smem::ST, SL = Smem::SL;
  constexpr uint32_t kCols = 512;  // D: TN columns from 0, A: 32 per stage from 256
  Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    tma_prefetch_desc(&tx);
    tma_prefetch_desc(&tw);
    for (int i = 0; i < ST; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.decoded[i], 4);  // a team's warps
      mbar_init(&sm.empty[i], 1);
    }
    for (int i = 0; i < SL; ++i) {
      mbar_init(&sm.w_full[i], 1);
      mbar_init(&sm.w_empty[i], 4 * kW4Teams);
    }
    mbar_init(&sm.done, 1);
    sm.abort = 0;
    fence_mbarrier_init();
  }
  if (warp == 4 * kW4Teams + 1) {
    tmem_alloc(&sm.tmem, kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem;
  griddep_wait();
  griddep_launch_dependents();

  const int slice = blockIdx.x % a.slices, n0 = (blockIdx.x / a.slices) * 128;
  const int k0 = static_cast<int>(static_cast<int64_t>(a.slots) * slice / a.slices);
  const int slots = static_cast<int>(static_cast<int64_t>(a.slots) * (slice + 1) / a.slices) - k0, count = 4 * slots;
  volatile int* abort = &sm.abort;

  if (warp == 4 * kW4Teams) {
    int issued = 0;
    for (int j = 0; j < count; ++j) {
      const int s = j % ST;
      if (j >= ST && !mbar_wait_warp(&sm.empty[s], (j / ST - 1) & 1, abort)) break;
      issued = j + 1;
      if (lane == 0) {
        mbar_arrive_expect_tx(&sm.full[s], TN * 128);
        tma_load_2d(&tx, &sm.full[s], sm.x[s], (4 * k0 + j) * 128, 0);
      }
    }
    if (lane == 0)  // whatever happened: the copies in flight land before the CTA ends
      for (int i = max(issued - ST, 0); i < issued; ++i) mbar_wait_drain(&sm.full[i % ST], (i / ST) & 1);
    __syncwarp();
  } else if (warp == 4 * kW4Teams + 2) {
    const int per = 256 >> a.log_g;  // scale groups per slot
    int issued = 0;
    for (int i = 0; i < slots; ++i) {
      const int s = i % SL;
      if (i >= SL && !mbar_wait_warp(&sm.w_empty[s], (i / SL - 1) & 1, abort)) break;
      issued = i + 1;
      if (lane == 0) {
        mbar_arrive_expect_tx(&sm.w_full[s], 16384 + per * 1024);
        tma_load_2d(&tw, &sm.w_full[s], sm.w[s], (k0 + i) * 128, n0);
        for (int q = 0; q < per; ++q)
          bulk_load(sm.sz[s][q], a.sz + (static_cast<int64_t>(k0 + i) * per + q) * a.ldn + n0, 1024, &sm.w_full[s]);
      }
    }
    if (lane == 0)
      for (int i = max(issued - SL, 0); i < issued; ++i) mbar_wait_drain(&sm.w_full[i % SL], (i / SL) & 1);
    __syncwarp();
  } else if (warp == 4 * kW4Teams + 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = kind_idesc<MmaKind::F16>(128, TN);
      bool live = true;
      for (int j = 0; live && j < count; ++j) {
        const int s = j % ST;
        live = mbar_wait(&sm.full[s], (j / ST) & 1, abort) && mbar_wait(&sm.decoded[s], (j / ST) & 1, abort);
        if (!live) break;
        tc_fence_after();
        const uint64_t dx = make_sw128_desc(smem_u32(sm.x[s]));
#pragma unroll
        for (int i = 0; i < 4; ++i)
          pf_umma_ts(tmem, tmem + 256 + 32 * s + 8 * i, dx + 2 * i, idesc, j > 0 || i > 0);
        umma_commit(&sm.empty[s]);
      }
      if (live) umma_commit(&sm.done);
    }
    __syncwarp();
  } else {
    const int team = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    bool live = true;
    for (int j = team; j < count; j += kW4Teams) {
      const int i = j >> 2, ws = i % SL, s = j % ST;
      if (!mbar_wait_warp(&sm.w_full[ws], (i / SL) & 1, abort) ||
          (j >= ST && !mbar_wait_warp(&sm.empty[s], (j / ST - 1) & 1, abort))) {
        live = false;
        break;
      }
      const uint8_t* src = sm.w[ws] + row * 128;
      const int c = 2 * (j & 3), swz = row & 7;
      const uint4 u0 = *reinterpret_cast<const uint4*>(src + ((c ^ swz) << 4));
      const uint4 u1 = *reinterpret_cast<const uint4*>(src + (((c + 1) ^ swz) << 4));
      const uint32_t words[8] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w};
      uint32_t out[32];
      uint32_t hi = 0, lo = 0, z0 = 0, z1 = 0;
      auto group = [&](int q) {
        const uint2 v = sm.sz[ws][(((j & 3) * 64) >> a.log_g) + q][row];
        hi = __byte_perm(v.x, 0, 0x1010);
        lo = __byte_perm(v.x, 0, 0x3232);
        z0 = __byte_perm(v.y, 0, 0x1010);
        z1 = __byte_perm(v.y, 0, 0x3232);
      };
      group(0);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i == 4 && a.log_g == 5) group(1);
        uint32_t p[4];
        w4_decode(words[i], z0, z1, p);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const __half2 c = *reinterpret_cast<const __half2*>(&p[q]), h = *reinterpret_cast<const __half2*>(&hi);
          __half2 r;
          if (LO) r = __hfma2(c, h, __hmul2(c, *reinterpret_cast<const __half2*>(&lo)));
          else r = __hmul2(c, h);
          out[4 * i + q] = *reinterpret_cast<const uint32_t*>(&r);
        }
      }
      tc_fence_after();
      const uint32_t at = tmem + 256 + 32 * s + lanes;
      const uint32_t half0[16] = {out[0], out[1], out[2],  out[3],  out[4],  out[5],  out[6],  out[7],
                                  out[8], out[9], out[10], out[11], out[12], out[13], out[14], out[15]};
      const uint32_t half1[16] = {out[16], out[17], out[18], out[19], out[20], out[21], out[22], out[23],
                                  out[24], out[25], out[26], out[27], out[28], out[29], out[30], out[31]};
      pf_tmem_st16(at, half0);
      pf_tmem_st16(at + 16, half1);
      pf_tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&sm.decoded[s]);
        mbar_arrive(&sm.w_empty[ws]);
      }
    }
    // ---- store: lane = weight row; the teams share the tokens
    live = live && mbar_wait_warp(&sm.done, 0, abort);
    tc_fence_after();
    if (live) {
      const int n = n0 + row;
      const float wp = n < a.N ? __ldg(a.w_pow + n) : 1.0f;
      // through shared memory (the ring is free), so that the epilogue's code is there once
      float* buf = reinterpret_cast<float*>(sm.x) + warp * (16 * 32) + lane;
#pragma unroll 1
      for (int c = team * 16; c < TN; c += 16 * kW4Teams) {
        const int many = min(16, a.M - c);
        if (many <= 0) break;
        uint32_t r[16];
        tmem_ld16(tmem + lanes + c, r);
        tmem_ld_wait();
        const float xp = __ldg(a.x_pow + min(c + (lane & 15), a.M - 1));
#pragma unroll
        for (int i = 0; i < 16; ++i) buf[i * 32] = times_powers(__uint_as_float(r[i]), __shfl_sync(0xffffffffu, xp, i), wp);
        if (n < a.N) {
          if (a.part) {
            float* to = a.part + (static_cast<int64_t>(slice) * a.M + c) * a.N + n;
#pragma unroll 8
            for (int i = 0; i < many; ++i) to[static_cast<int64_t>(i) * a.N] = buf[i * 32];
          } else {
#pragma unroll 4
            for (int i = 0; i < many; ++i) store_out(ep, c + i, n, epi_scaled(buf[i * 32], 1.0f, 1.0f, 1.0f, ep, n));
          }
        }
        __syncwarp();  // the next load wants the whole warp
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 4 * kW4Teams + 1) tmem_dealloc(tmem, kCols);
}

}  // namespace b200q
