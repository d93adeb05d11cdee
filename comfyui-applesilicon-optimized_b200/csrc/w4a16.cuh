// 4-bit weight-only linear with group scales: up to 32 tokens, and the operands of the
// decoded form for more than 256 (w4_tile.cuh has what lies between):
//   out[m,n] = act( sum_k x[m,k] * s[n,k/G] * (c[n,k] - z[n,k/G]) + b[n] )
// c: unsigned 4-bit codes, two per byte along K (even k in the low nibble);
// s: one scale per row and group of G codes; z: one zero point (0..15) per row
// and group, 8 when absent.
//
// Mathematics.  Inside a group the scale is a constant, so the group's sum is
// taken over the exact integers c - z, and one fp32 multiply-add per group
// joins it to the row's accumulator:  acc += s * sum_{k in group} x_k (c_k - z).
// c - z is exact in fp16: OR-ing a nibble into the mantissa of 1024 gives 1024 + c,
// and subtracting 1024 + z is exact.  Products and sums run on warp MMAs (m16n8k16,
// fp32 accumulation) with 16 weight rows as the MMA's rows and 8 tokens as its
// columns.  A bf16 token row is scaled by the power of two of its largest |x| and is
// then exact in fp16 down to 2^-17 of it, within 2^-25 of it below; nothing else is
// rounded before the output.
//
// Layout.  The order of k inside a group is free as long as both operands
// agree.  Lane (g, t) = (lane / 4, lane % 4) takes the G/4 codes of its quarter t
// of the group for rows g and g + 8 as they are stored; pair i of an 8-code word w
// is (w >> 4i) & 0x000F000F = codes i and i + 4.  x is staged in shared memory in
// that order (8 values as 0 4 1 5 2 6 3 7; quarter-major), so one 16-byte shared
// load feeds two MMAs, and the row pitch is 64 modulo 128 bytes, which makes those
// loads free of bank conflicts.  Few tokens take an integer form of the same sums.
#pragma once

#include <type_traits>

#include "digits.cuh"
#include "numerics.cuh"
#include "ptx.cuh"

namespace b200q {

constexpr int kW4Warps = 8;  // warps that split a row tile's K in the integer kernel

__device__ __forceinline__ float load_scale(const void* p, int dtype, int64_t i) {
  if (dtype == kBiasBF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  if (dtype == kBiasF16) return __half2float(static_cast<const __half*>(p)[i]);
  return static_cast<const float*>(p)[i];
}
// A scale as its raw bits, and their value.
__device__ __forceinline__ uint32_t load_scale_bits(const void* p, int dtype, uint32_t i) {
  return dtype == kBiasF32 ? __ldg(static_cast<const uint32_t*>(p) + i)
                           : static_cast<uint32_t>(__ldg(static_cast<const uint16_t*>(p) + i));
}
__device__ __forceinline__ float scale_value(uint32_t bits, int dtype) {
  if (dtype == kBiasF32) return __uint_as_float(bits);
  if (dtype == kBiasBF16) return __uint_as_float(bits << 16);
  const uint16_t h = static_cast<uint16_t>(bits);
  return __half2float(*reinterpret_cast<const __half*>(&h));
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ int rev3(int r) { return ((r & 1) << 2) | (r & 2) | ((r >> 2) & 1); }

// This lane's LW words of group q (of a stage) of row g, from a ring stage: 128 bytes
// per row, 16-byte chunks XOR-swizzled by rev3(row & 7) (`swz`, rows 8 apart alike).
template <int LW>
__device__ __forceinline__ void w4_words(const uint8_t* buf, int g, int t, int q, int swz, uint32_t (&w)[LW]) {
  if constexpr (LW == 4) {
    const uint4 u = *reinterpret_cast<const uint4*>(buf + g * 128 + (((q * 4 + t) ^ swz) << 4));
    w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
  } else if constexpr (LW == 2) {
    const uint2 u = *reinterpret_cast<const uint2*>(buf + g * 128 + (((q * 2 + (t >> 1)) ^ swz) << 4) + (t & 1) * 8);
    w[0] = u.x; w[1] = u.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(buf + g * 128 + ((q ^ swz) << 4) + t * 4);
  }
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same with a zero accumulator.
__device__ __forceinline__ void mma_f16_start(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
// (a & mask) | bits in one instruction (the compiler makes two of it).
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t mask, uint32_t bits) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "r"(mask), "r"(bits));
  return r;
}
// Nibbles become fp16 by their place in the mantissa of a constant power of two, a published
// method (Kim, Henry, Fahim and Awadalla, "Who Says Elephants Can't Run: Bringing Large Scale
// MoE Models into Cloud Scale Production", 2022).
// A row's zero point for w4_decode: 1024 + z (low half) and -(64 + z) as fp16.
__device__ __forceinline__ uint32_t w4_zero(uint32_t z) { return 0xD4006400u | (z << 20) | z; }

// The four exact fp16 pairs (c_i - z, c_{i+4} - z) of one 8-code word, from its row's
// pairs z0 = (1024 + z) twice and z1 = -(64 + z) twice: a low nibble OR-ed into 1024
// is 1024 + c, the nibble above it 1024 + 16 c (one shift per word).
__device__ __forceinline__ void w4_decode(uint32_t w, uint32_t z0, uint32_t z1, uint32_t (&p)[4]) {
  const uint32_t m = 0x64006400u, sixteenth = 0x2C002C00u;
  const uint32_t v = w >> 8;
  const uint32_t a[4] = {and_or(w, 0x000F000Fu, m), and_or(w, 0x00F000F0u, m), and_or(v, 0x000F000Fu, m),
                         and_or(v, 0x00F000F0u, m)};
  const __half2 h0 = *reinterpret_cast<const __half2*>(&z0), h1 = *reinterpret_cast<const __half2*>(&z1);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 x = *reinterpret_cast<const __half2*>(&a[i]);
    const __half2 r = i & 1 ? __hfma2(x, *reinterpret_cast<const __half2*>(&sixteenth), h1) : __hsub2(x, h0);
    p[i] = *reinterpret_cast<const uint32_t*>(&r);
  }
}

// ---------------------------------------------------------------- up to 32 tokens
// x does not fit one CTA's shared memory whole, so K is cut into slices: a CTA keeps
// its slice of x and its warps, each on its own, go through 16-row tiles of the
// weight's slice (persistent, no barrier after x is staged).  With more than one
// slice the fp32 sums go to the workspace, [slice][token][row], and w4_join_kernel
// adds them in slice order.  Rings as in the integer kernel below: 128 bytes per row
// and stage, scales travelling along.
//
// Bound: the instructions per weight word (unpacking, 2 MMAs per 8 tokens) and the ring's
// latency.  16 tokens, K 13824, N 5120: 21 us, 1.7 TB/s of codes; 32 tokens, K 5120, N
// 13824: 30 us.  TMA boxes instead of cp.async were slower (one issuer per CTA).
constexpr int kWsWarps = 16;
constexpr int kWsStages = 3;  // issue() relies on three

struct W4SliceArgs {
  const void* x;         // [M, K] bf16 / fp16
  int64_t ldx;           // elements
  int x_f16;
  const uint8_t* w;      // [N, K / 2]
  int64_t ldw;           // bytes
  const void* scales;    // [N, K / G]
  int scale_dtype;       // kBiasBF16 / kBiasF16 / kBiasF32
  const uint8_t* zeros;  // [N, K / G] or null (8)
  float* part;           // [slices][M][N], or null: one slice, the epilogue runs here
  int M, N, K;
  int x_vec;             // rows of x are 16-byte aligned
  int slices, parts;     // grid = slices * parts
};

// Shared bytes per token row for a slice of `k` codes: 64 modulo 128.
__host__ __device__ __forceinline__ int ws_pitch(int k) { return 2 * k + ((2 * k & 127) == 64 ? 0 : 64); }
__host__ __device__ __forceinline__ int ws_smem_bytes(int M, int k_slice, int G) {
  return kWsWarps * kWsStages * (2048 + (256 / G) * 16 * 8) + M * ws_pitch(k_slice);
}

// LW = G / 32 words per lane, row and group; NT = 8-token columns.
template <int LW, int NT>
__global__ void __launch_bounds__(kWsWarps * 32) w4_slice_kernel(const W4SliceArgs a, const EpiArgs ep) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float x_pow[8 * NT];
  constexpr int G = 32 * LW;
  constexpr int GS = 8 / LW;  // groups per stage
  constexpr int SL = GS / 2;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int slice = blockIdx.x % a.slices, part = blockIdx.x / a.slices;
  const int KG = a.K / G;
  const int g0 = static_cast<int>(int64_t(KG) * slice / a.slices);
  const int ng = static_cast<int>(int64_t(KG) * (slice + 1) / a.slices) - g0;
  const int spt = (ng + GS - 1) / GS;
  const int pitch = ws_pitch((KG + a.slices - 1) / a.slices * G);
  uint8_t* ring = smem + warp * (kWsStages * 2048);
  float2* sz = reinterpret_cast<float2*>(smem + kWsWarps * kWsStages * 2048) + warp * (kWsStages * GS * 16);
  uint8_t* xsm = smem + kWsWarps * kWsStages * (2048 + GS * 16 * 8);
  const int tiles = (a.N + 15) / 16;
  const int tile0 = part * kWsWarps + warp, tile_step = a.parts * kWsWarps;

  griddep_wait();
  griddep_launch_dependents();

  // ---- the ring: lane copies chunk lane % 8 of rows lane / 8 + 4 j, and loads entries
  // e = lane + 32 k = (group e / 16, row e % 16) of the stage's scales
  int it_tile = tile0, it_stage = 0, it_slot = 0;
  const int cp_row = lane >> 3, cp_ch = lane & 7;
  uint32_t s_next[2][SL], z_next[2][SL];  // of the last stage asked for, and the one before
#pragma unroll
  for (int k = 0; k < SL; ++k) s_next[0][k] = z_next[0][k] = s_next[1][k] = z_next[1][k] = 0;
  const uint8_t* src0 = nullptr;
  auto aim = [&]() {
    src0 = a.w + static_cast<int64_t>(it_tile * 16 + cp_row) * a.ldw + g0 * (LW * 16) + cp_ch * 16;
  };
  aim();
  const uint32_t dst0 = smem_u32(ring) + cp_row * 128;
  auto issue = [&]() {
    {  // the scales asked for two steps ago have arrived by now: the stage read next
      float2* to = sz + (it_slot == kWsStages - 1 ? 0 : it_slot + 1) * (GS * 16);
#pragma unroll
      for (int k = 0; k < SL; ++k) {
        to[lane + 32 * k] = make_float2(scale_value(s_next[1][k], a.scale_dtype),
                                          __uint_as_float(w4_zero(z_next[1][k] & 15u)));
        s_next[1][k] = s_next[0][k];
        z_next[1][k] = z_next[0][k];
      }
    }
    if (it_tile < tiles) {
      if (it_stage * 8 + cp_ch < ng * LW) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          // rows past N repeat row N - 1
          const int over = min(a.N - 1 - (it_tile * 16 + cp_row + 4 * j), 0);
          cp_async16(dst0 + 512 * j + it_slot * 2048 + ((cp_ch ^ rev3((cp_row + 4 * j) & 7)) << 4),
                     src0 + static_cast<int64_t>(4 * j + over) * a.ldw + it_stage * 128);
        }
      }
#pragma unroll
      for (int k = 0; k < SL; ++k) {
        const int e = lane + 32 * k;
        const int n = min(it_tile * 16 + e % 16, a.N - 1);
        const uint32_t at = static_cast<uint32_t>(n) * KG + g0 + min(it_stage * GS + e / 16, ng - 1);
        s_next[0][k] = load_scale_bits(a.scales, a.scale_dtype, at);
        z_next[0][k] = a.zeros ? __ldg(a.zeros + at) : 8;
      }
      if (++it_stage == spt) {
        it_stage = 0;
        it_tile += tile_step;
        aim();
      }
    }
    it_slot = it_slot == kWsStages - 1 ? 0 : it_slot + 1;
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kWsStages - 1; ++i) issue();

  // ---- stage x[:, slice] in fragment order: warp w takes tokens w, w + 16, ..., 256
  // pieces of 8 values (8 per lane, all in flight) at a time.  A bf16 row longer than
  // that is read once more, for its largest |x|.
  {
    const int pieces = ng * (G / 8);
    for (int m = warp; m < a.M; m += kWsWarps) {
      const uint16_t* row = static_cast<const uint16_t*>(a.x) + m * a.ldx + int64_t(g0) * G;
      uint4 v[8];
      auto load = [&](int p0) {
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int p = p0 + 32 * u + lane;
          v[u] = make_uint4(0, 0, 0, 0);
          if (p < pieces) {
            if (a.x_vec) {
              v[u] = __ldg(reinterpret_cast<const uint4*>(row + p * 8));
            } else {
              uint32_t e[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) e[j] = __ldg(row + p * 8 + 2 * j) | (uint32_t(__ldg(row + p * 8 + 2 * j + 1)) << 16);
              v[u] = make_uint4(e[0], e[1], e[2], e[3]);
            }
          }
        }
      };
      load(0);
      float inv = 1.0f, pow = 1.0f;
      if (!a.x_f16) {
        uint32_t top = 0;
        for (int p0 = 0;;) {
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            const uint32_t e[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) top = max(top, max(e[j] & 0x7FFFu, (e[j] >> 16) & 0x7FFFu));
          }
          if ((p0 += 256) >= pieces) break;
          load(p0);
        }
        if (pieces > 256) load(0);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        // (an infinity or NaN stays one at any power: its row takes the largest, at which
        // the finite values beside it stay finite)
        const int ex = min(max(static_cast<int>(top >> 7), 1), 253);
        inv = __uint_as_float(static_cast<uint32_t>(254 - ex) << 23);
        pow = __uint_as_float(static_cast<uint32_t>(ex) << 23);
      }
      if (lane == 0) x_pow[m] = pow;
      for (int p0 = 0;;) {
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int p = p0 + 32 * u + lane;
          if (p < pieces) {
            uint32_t e[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
            if (!a.x_f16) {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                e[j] = pack_f16x2(__uint_as_float(e[j] << 16) * inv, __uint_as_float(e[j] & 0xFFFF0000u) * inv);
            }
            const int grp = p / (G / 8), r = p % (G / 8);
            const int at = (grp * LW + r % LW) * 4 + r / LW;  // [group][word][quarter]
            // values 0 4 1 5 2 6 3 7
            *reinterpret_cast<uint4*>(xsm + m * pitch + at * 16) =
                make_uint4(__byte_perm(e[0], e[2], 0x5410), __byte_perm(e[0], e[2], 0x7632),
                           __byte_perm(e[1], e[3], 0x5410), __byte_perm(e[1], e[3], 0x7632));
          }
        }
        if ((p0 += 256) >= pieces) break;
        load(p0);
      }
    }
  }
  __syncthreads();

  const uint8_t* xs[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j)  // columns past M read row M - 1; their results are not used
    xs[j] = xsm + min(8 * j + g, a.M - 1) * pitch + t * 16;
  const int swz = rev3(g & 7);

  int slot = 0;
  for (int tile = tile0; tile < tiles; tile += tile_step) {
    float acc[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][i] = 0.0f;
    for (int st = 0; st < spt; ++st) {
      cp_async_wait<kWsStages - 2>();
      __syncwarp();  // the stage has landed for every lane, and the slot read last is free
      issue();
      __syncwarp();  // this stage's scales are in place
      const uint8_t* buf = ring + slot * 2048;
      const float2* szs = sz + slot * (GS * 16);
      slot = slot == kWsStages - 1 ? 0 : slot + 1;
#pragma unroll
      for (int q = 0; q < GS; ++q) {
        const int gl = st * GS + q;
        if (gl >= ng) break;
        uint32_t wa[LW], wb[LW];
        w4_words<LW>(buf, g, t, q, swz, wa);
        w4_words<LW>(buf + 1024, g, t, q, swz, wb);
        const float2 sa = szs[q * 16 + g], sb = szs[q * 16 + g + 8];
        const uint32_t za = __float_as_uint(sa.y), zb = __float_as_uint(sb.y);
        const uint32_t za0 = __byte_perm(za, 0, 0x1010), za1 = __byte_perm(za, 0, 0x3232);
        const uint32_t zb0 = __byte_perm(zb, 0, 0x1010), zb1 = __byte_perm(zb, 0, 0x3232);
        float sum[NT][4];
#pragma unroll
        for (int wi = 0; wi < LW; ++wi) {
          uint32_t pa[4], pb[4];
          w4_decode(wa[wi], za0, za1, pa);
          w4_decode(wb[wi], zb0, zb1, pb);
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const uint4 xv = *reinterpret_cast<const uint4*>(xs[j] + (gl * LW + wi) * 64);
            if (wi == 0) mma_f16_start(sum[j], pa[0], pb[0], pa[1], pb[1], xv.x, xv.y);
            else mma_f16(sum[j], pa[0], pb[0], pa[1], pb[1], xv.x, xv.y);
            mma_f16(sum[j], pa[2], pb[2], pa[3], pb[3], xv.z, xv.w);
          }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          acc[j][0] = fmaf(sa.x, sum[j][0], acc[j][0]);
          acc[j][1] = fmaf(sa.x, sum[j][1], acc[j][1]);
          acc[j][2] = fmaf(sb.x, sum[j][2], acc[j][2]);
          acc[j][3] = fmaf(sb.x, sum[j][3], acc[j][3]);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int n = tile * 16 + g + 8 * (i >> 1), m = 8 * j + 2 * t + (i & 1);
        if (n < a.N && m < a.M) {
          const float v = acc[j][i] * x_pow[m];
          if (a.part) a.part[(static_cast<int64_t>(slice) * a.M + m) * a.N + n] = v;
          else store_out(ep, m, n, epi_scaled(v, 1.0f, 1.0f, 1.0f, ep, n));
        }
      }
  }
}

// Adds the slices of each output (fp32 [slices][M][ld]) in order and runs the epilogue;
// grid M * chunks of 256 columns.
__global__ void __launch_bounds__(256)
    w4_join_kernel(const float* __restrict__ part, int slices, int64_t ld, int chunks, const EpiArgs ep) {
  griddep_wait();
  griddep_launch_dependents();
  const int m = blockIdx.x / chunks, n = (blockIdx.x - m * chunks) * 256 + threadIdx.x;
  if (n >= ep.N) return;
  const int64_t total = ep.M * ld, i = m * ld + n;
  float v = 0.0f;
#pragma unroll 8
  for (int s = 0; s < slices; ++s) v += part[s * total + i];
  store_out(ep, m, n, epi_scaled(v, 1.0f, 1.0f, 1.0f, ep, n));
}

// ---------------------------------------------------------------- few tokens, integer
// One to a few tokens, whose time is the weight stream: the instructions per weight
// are what has to be few, so the products run on the integer tensor path, where a
// nibble is an operand after one AND.
//
// x is split, group by group, into three int8 digits: with 2^E above the group's
// largest |x|, x 2^-E 64 = p0 + p1 / 128 + p2 / 128^2, within 2^-21 of 2^E.  Then
//   sum_k x_k (c_k - z) = 2^E / 64 sum_p 128^-p (sum_k p_k c_k - z sum_k p_k)
// with exact integer sums (|.| <= 128 * 15 * 64 < 2^17).  MMA m16n8k32: 16 weight
// rows x the 3 M digit columns; a word's 8 codes are two operand registers, w &
// 0x0F0F0F0F and (w >> 4) & 0x0F0F0F0F, with the digits staged in that order.  The
// accumulators start at the bits of 1.5 * 2^23, so one subtraction gives the fp32
// value.  A group holding inf or NaN gets a NaN scale.
//
// One CTA per SM makes the digits once for its teams of 8 warps; a team is persistent
// over 16-row tiles and its warps split K.  Each warp streams its rows' bytes through
// a ring of its own (cp.async, 128 bytes per row and stage, 16-byte chunks
// XOR-swizzled by the row so that the fragment reads have no bank conflicts); the ring
// runs on across tiles, so the loads of the next tile are in flight while one is
// summed.  A stage's scales and zero points travel with it: loaded to registers when
// its bytes are asked for, converted and put into the stage's slot just before it is read
// (waiting for them at the start of each tile cost more than the tile).  A tile's sums
// are double-buffered: one barrier per tile, and a different warp each time adds and
// stores them while the others go on.
//
// Bound: x's digits and the first loads for small weights, issue for large ones.  1 token,
// K = N = 5120, G 128: 6.4 us (2.1 TB/s of codes, 0.32 of the floor); K 5120, N 13824, G 64
// with zero points and GELU: 14.0 us (2.5 TB/s, 0.42).  fp16 MMAs took 23 us for the latter.
constexpr int kWdStages = 3;  // issue() relies on three
// Most teams per CTA, by the digit columns' register need.
constexpr int wd_teams(int nc) { return nc == 3 ? 2 : 3; }

struct W4DigitArgs {
  const void* x;
  int64_t ldx;
  const uint8_t* w;
  int64_t ldw;
  const void* scales;  // of x's type
  const uint8_t* zeros;
  int M, N, K;
  int x_vec;
  int tiles;  // ceil(N / 16)
};

__device__ __forceinline__ void mma_u8s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same with the accumulators starting at the bits of 1.5 * 2^23.
__device__ __forceinline__ void mma_u8s8_start(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
  const int z = 0x4B400000;
  asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(z));
}

// Shared memory: rings, digits [3M][pitch], {2^E / (64 * 128^p), digit sum}
// [groups][8 NC], {scale, -zero} [warp][stage][groups of a stage][16], warp sums.
__host__ __device__ __forceinline__ int wd_pitch(int K) { return K + ((K & 127) == 64 ? 0 : (64 + 128 - (K & 127)) & 127); }
struct WdLayout {
  int digits, table, sz, red, total;  // byte offsets
};
__host__ __device__ __forceinline__ WdLayout wd_layout(int M, int K, int G, int nc, int teams) {
  WdLayout l;
  const int KG = K / G;
  l.digits = teams * kW4Warps * kWdStages * 2048;
  l.table = l.digits + 3 * M * wd_pitch(K);
  l.sz = l.table + KG * 8 * nc * 8;
  l.red = l.sz + teams * kW4Warps * kWdStages * (256 / G) * 16 * 8;
  l.total = l.red + 2 * teams * kW4Warps * 16 * 8 * nc * 4;
  return l;
}

template <typename T, int LW, int NC>
__global__ void __launch_bounds__(NC == 3 ? 512 : 768) w4_digit_kernel(const W4DigitArgs a, const EpiArgs ep) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int G = 32 * LW;
  constexpr int GS = 8 / LW;           // groups per stage (128 bytes of a row)
  constexpr int LG = LW == 1 ? 4 : 8;  // lanes per group while making digits
  constexpr int EL = G / LG;           // values per lane there
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int KG = a.K / G;
  const int teams = blockDim.x / (kW4Warps * 32);
  const WdLayout L = wd_layout(a.M, a.K, G, NC, teams);
  const int pitch = wd_pitch(a.K);
  const int team = warp / kW4Warps, tw = warp % kW4Warps;
  const int g0 = static_cast<int>(int64_t(KG) * tw / kW4Warps);
  const int ng = static_cast<int>(int64_t(KG) * (tw + 1) / kW4Warps) - g0;
  const int spt = (ng + GS - 1) / GS;  // stages per tile
  uint8_t* ring = smem + warp * (kWdStages * 2048);
  const uint32_t ring_u = smem_u32(ring);
  float2* sz = reinterpret_cast<float2*>(smem + L.sz) + warp * (kWdStages * GS * 16);
  float* red = reinterpret_cast<float*>(smem + L.red) + team * (2 * kW4Warps * 16 * 8 * NC);
  const int tile0 = blockIdx.x * teams + team, tile_step = gridDim.x * teams;

  griddep_wait();
  griddep_launch_dependents();

  // ---- the ring: lane copies chunk lane % 8 of rows lane / 8 + 4 j, and loads entries
  // lane + 32 k = (group e / 16, row e % 16) of the stage's scales
  constexpr int SL = GS / 2;
  int it_tile = tile0, it_stage = 0, it_slot = 0;
  const int cp_row = lane >> 3, cp_ch = lane & 7;
  uint32_t s_next[2][SL], z_next[2][SL];  // of the last stage asked for, and the one before
#pragma unroll
  for (int k = 0; k < SL; ++k) s_next[0][k] = z_next[0][k] = s_next[1][k] = z_next[1][k] = 0;
  const uint8_t* src[4];   // this lane's rows of the tile being fetched
  uint32_t s_at = 0;
  auto aim = [&]() {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      src[j] = a.w + static_cast<int64_t>(min(it_tile * 16 + cp_row + 4 * j, a.N - 1)) * a.ldw + g0 * (LW * 16) + cp_ch * 16;
    s_at = static_cast<uint32_t>(min(it_tile * 16 + (lane & 15), a.N - 1)) * KG + g0;
  };
  if (spt == 0) it_tile = a.tiles;  // fewer groups than warps: nothing to fetch
  aim();
  const uint32_t dst0 = ring_u + cp_row * 128;
  uint32_t dst[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) dst[j] = dst0 + 512 * j + ((cp_ch ^ rev3((cp_row + 4 * j) & 7)) << 4);
  auto issue = [&]() {
    {  // the scales asked for two steps ago have arrived by now: the stage read next
      float2* to = sz + (it_slot == kWdStages - 1 ? 0 : it_slot + 1) * (GS * 16) + lane;
#pragma unroll
      for (int k = 0; k < SL; ++k) {
        const uint16_t bits = static_cast<uint16_t>(s_next[1][k]);
        to[32 * k] = make_float2(to_float<T>(*reinterpret_cast<const T*>(&bits)),
                                 __int_as_float(-static_cast<int>(z_next[1][k] & 15u)));
        s_next[1][k] = s_next[0][k];
        z_next[1][k] = z_next[0][k];
      }
    }
    if (it_tile < a.tiles) {
      if (it_stage * 8 + cp_ch < ng * LW) {
#pragma unroll
        for (int j = 0; j < 4; ++j) cp_async16(dst[j] + it_slot * 2048, src[j] + it_stage * 128);
      }
#pragma unroll
      for (int k = 0; k < SL; ++k) {
        const uint32_t at = s_at + min(it_stage * GS + 2 * k + (lane >> 4), ng - 1);
        s_next[0][k] = __ldg(static_cast<const uint16_t*>(a.scales) + at);
        z_next[0][k] = a.zeros ? __ldg(a.zeros + at) : 8;
      }
      if (++it_stage == spt) {
        it_stage = 0;
        it_tile += tile_step;
        aim();
      }
    }
    it_slot = it_slot == kWdStages - 1 ? 0 : it_slot + 1;
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kWdStages - 1; ++i) issue();

  // ---- digits of x, one (token, group) per LG lanes
  {
    const int unit0 = warp * (32 / LG) + lane / LG, li = lane % LG;
    for (int u = unit0; u < a.M * KG + unit0 % (32 / LG); u += teams * kW4Warps * (32 / LG)) {
      // (the whole warp runs the same iterations: the shuffles need every lane)
      const bool live = u < a.M * KG;
      const int m = live ? u / KG : 0, gi = live ? u - m * KG : 0;
      const uint16_t* src = static_cast<const uint16_t*>(a.x) + m * a.ldx + gi * G + li * EL;
      uint32_t raw[EL / 2];
      if (a.x_vec) {
#pragma unroll
        for (int j = 0; j < EL / 8; ++j) {
          const uint4 v = __ldg(reinterpret_cast<const uint4*>(src) + j);
          raw[4 * j] = v.x; raw[4 * j + 1] = v.y; raw[4 * j + 2] = v.z; raw[4 * j + 3] = v.w;
        }
      } else {
#pragma unroll
        for (int j = 0; j < EL / 2; ++j) raw[j] = __ldg(src + 2 * j) | (uint32_t(__ldg(src + 2 * j + 1)) << 16);
      }
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < EL / 2; ++j) top = max(top, max(raw[j] & 0x7FFFu, (raw[j] >> 16) & 0x7FFFu));
#pragma unroll
      for (int o = LG / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      float down, up;
      digit_scale(top, std::is_same<T, __half>::value, &down, &up);
      int sum[3] = {0, 0, 0};
#pragma unroll
      for (int wv = 0; wv < EL / 8; ++wv) {  // one 8-code word: digits of codes 0 2 4 6 | 1 3 5 7
        uint32_t p[3][8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint16_t e = static_cast<uint16_t>(raw[4 * wv + (i >> 1)] >> (16 * (i & 1)));
          digits3(to_float<T>(*reinterpret_cast<const T*>(&e)) * down, p[0][i], p[1][i], p[2][i]);
        }
        const int word = LW == 4 ? (li & 1) * 2 + wv : LW == 2 ? (li & 1) : 0;
        const int q = LW == 1 ? li : li >> 1;
        const int at = LW == 1 ? (gi * 4 + q) * 8
                     : LW == 2 ? (gi * 4 + q) * 16 + word * 8
                               : ((gi * 2 + word / 2) * 4 + q) * 16 + (word & 1) * 8;
#pragma unroll
        for (int d = 0; d < 3; ++d) {
          const uint32_t lo = low_bytes(p[d][0], p[d][2], p[d][4], p[d][6]);
          const uint32_t hi = low_bytes(p[d][1], p[d][3], p[d][5], p[d][7]);
          sum[d] = __dp4a(static_cast<int>(lo), 0x01010101, sum[d]);
          sum[d] = __dp4a(static_cast<int>(hi), 0x01010101, sum[d]);
          if (live)
            *reinterpret_cast<uint2*>(smem + L.digits + (3 * m + d) * pitch + at) = make_uint2(lo, hi);
        }
      }
#pragma unroll
      for (int d = 0; d < 3; ++d) {
#pragma unroll
        for (int o = LG / 2; o > 0; o >>= 1) sum[d] += __shfl_xor_sync(0xffffffffu, sum[d], o);
        if (live && li == d) {
          const float f = d == 0 ? up : d == 1 ? up * 0.0078125f : up * 0.00006103515625f;
          reinterpret_cast<float2*>(smem + L.table)[gi * 8 * NC + 3 * m + d] =
              make_float2(f, __int_as_float(sum[d]));
        }
      }
    }
  }
  __syncthreads();

  const uint8_t* xs[NC];
#pragma unroll
  for (int j = 0; j < NC; ++j)  // columns past 3 M read the last one; their results are not used
    xs[j] = smem + L.digits + min(8 * j + g, 3 * a.M - 1) * pitch + t * (LW == 1 ? 8 : 16);
  const float4* table = reinterpret_cast<const float4*>(smem + L.table);
  const int swz = rev3(g & 7);

  int slot = 0, turn = 0;
  for (int tile = tile0; tile < a.tiles; tile += tile_step) {
    float acc[NC][4];
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][i] = 0.0f;
    for (int st = 0; st < spt; ++st) {
      cp_async_wait<kWdStages - 2>();
      __syncwarp();  // the stage has landed for every lane, and the slot read last is free
      issue();
      __syncwarp();  // this stage's scales are in place
      const uint8_t* buf = ring + slot * 2048;
      const float2* szs = sz + slot * (GS * 16);
      slot = slot == kWdStages - 1 ? 0 : slot + 1;
#pragma unroll
      for (int q = 0; q < GS; ++q) {
        const int gl = st * GS + q;
        if (gl >= ng) break;
        uint32_t wa[LW], wb[LW];
        w4_words<LW>(buf, g, t, q, swz, wa);
        w4_words<LW>(buf + 1024, g, t, q, swz, wb);
        int d[NC][4];
#pragma unroll
        for (int wi = 0; wi < LW; wi += 2) {
          const uint32_t a0 = wa[wi] & 0x0F0F0F0Fu, a2 = (wa[wi] >> 4) & 0x0F0F0F0Fu;
          const uint32_t a1 = wb[wi] & 0x0F0F0F0Fu, a3 = (wb[wi] >> 4) & 0x0F0F0F0Fu;
          if constexpr (LW > 1) {
            const uint32_t e0 = wa[wi + 1] & 0x0F0F0F0Fu, e2 = (wa[wi + 1] >> 4) & 0x0F0F0F0Fu;
            const uint32_t e1 = wb[wi + 1] & 0x0F0F0F0Fu, e3 = (wb[wi + 1] >> 4) & 0x0F0F0F0Fu;
#pragma unroll
            for (int j = 0; j < NC; ++j) {
              const uint4 b = *reinterpret_cast<const uint4*>(xs[j] + ((g0 + gl) * (LW / 2) + wi / 2) * 64);
              if (wi == 0) mma_u8s8_start(d[j], a0, a1, a2, a3, b.x, b.y);
              else mma_u8s8(d[j], a0, a1, a2, a3, b.x, b.y);
              mma_u8s8(d[j], e0, e1, e2, e3, b.z, b.w);
            }
          } else {
#pragma unroll
            for (int j = 0; j < NC; ++j) {
              const uint2 b = *reinterpret_cast<const uint2*>(xs[j] + (g0 + gl) * 32);
              mma_u8s8_start(d[j], a0, a1, a2, a3, b.x, b.y);
            }
          }
        }
        const float2 sa = szs[q * 16 + g], sb = szs[q * 16 + g + 8];
#pragma unroll
        for (int j = 0; j < NC; ++j) {
          const float4 tb = table[(g0 + gl) * 4 * NC + 4 * j + t];  // columns 2t, 2t + 1
          const int za = __float_as_int(sa.y), zb = __float_as_int(sb.y);
          const int s0 = __float_as_int(tb.y), s1 = __float_as_int(tb.w);
          // f, a power of two, meets the scale first: f times the sum leaves fp32's range for
          // |x| from 2^110 on, f s only where the output does.  Sum and f s are exact
          const float i0 = __int_as_float(d[j][0] + za * s0) - 12582912.0f, i1 = __int_as_float(d[j][1] + za * s1) - 12582912.0f;
          const float i2 = __int_as_float(d[j][2] + zb * s0) - 12582912.0f, i3 = __int_as_float(d[j][3] + zb * s1) - 12582912.0f;
          acc[j][0] = fmaf(i0, tb.x * sa.x, acc[j][0]);
          acc[j][1] = fmaf(i1, tb.z * sa.x, acc[j][1]);
          acc[j][2] = fmaf(i2, tb.x * sb.x, acc[j][2]);
          acc[j][3] = fmaf(i3, tb.z * sb.x, acc[j][3]);
        }
      }
    }
    // ---- join the warps' K ranges and the digits, in a fixed order
    float* sums = red + (turn & 1) * (kW4Warps * 16 * 8 * NC);
    float* mine = sums + tw * (16 * 8 * NC);
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      mine[(8 * j + 2 * t) * 16 + g] = acc[j][0];
      mine[(8 * j + 2 * t + 1) * 16 + g] = acc[j][1];
      mine[(8 * j + 2 * t) * 16 + g + 8] = acc[j][2];
      mine[(8 * j + 2 * t + 1) * 16 + g + 8] = acc[j][3];
    }
    named_bar_sync(1 + team, kW4Warps * 32);
    if (tw == turn % kW4Warps) {
      for (int e = lane; e < 16 * a.M; e += 32) {
        const int m = e >> 4, row = e & 15, n = tile * 16 + row;
        float v = 0.0f;
#pragma unroll
        for (int k = 0; k < kW4Warps; ++k)
#pragma unroll
          for (int p = 2; p >= 0; --p) v += sums[k * (16 * 8 * NC) + (3 * m + p) * 16 + row];
        if (n < a.N) store_out(ep, m, n, epi_scaled(v, 1.0f, 1.0f, 1.0f, ep, n));
      }
    }
    ++turn;
  }
}

// ---------------------------------------------------------------- many tokens
// Operands of the tile GEMM, one warp per row.
//
// Weight rows: fp16 values s * (c - z) * 2^-e with 2^e the power of two of the row's
// largest |s| (at most 15 * 2 in magnitude, so fp16's range holds whatever the scales
// are); 2^e goes to w_pow[n] for the GEMM's column scale.  c - z is exact, its product
// with s is rounded once, to fp16's 11 bits: an eighth of a bf16 output's own rounding.
//
// bf16 token rows: x * 2^-e, 2^e the power of two of the row's largest |x|, to
// x_pow[m] for the GEMM's row scale.  Exact down to 2^-17 of the row's maximum, within
// 2^-25 of it below.  The GEMM multiplies by the row's power before the column's: 2^-22 of
// the former is kept for the scalar that comes last, so that sums of up to 2^23 times rows
// near fp32's largest value pass through finite numbers (and rows below 2^-105 lose bits of
// outputs near 2^-128).
//
// Bound: memory (half a byte read and two written per weight): 46 us for 13824 x 5120 and
// 2047 tokens, 4.4 TB/s; the product then takes 190 us, 0.93 of the measured GEMM rate.
struct W4PrepareArgs {
  const uint8_t* w;
  int64_t ldw;
  const void* scales;
  int scale_dtype;
  const uint8_t* zeros;
  int N, K, log_g;
  __half* w16;
  float* w_pow;
  const __nv_bfloat16* x;  // null: x is used as it is
  int64_t ldx;
  int M, x_vec;
  __half* x16;
  float* x_pow;
  float* last;  // 2^22
};

__global__ void __launch_bounds__(256) w4_prepare_kernel(const W4PrepareArgs a) {
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (item < a.N) {
    const int KG = a.K >> a.log_g;
    const int64_t s0 = item * KG;
    float m = 0.0f;
    for (int i = lane; i < KG; i += 32) m = fmaxf(m, fabsf(load_scale(a.scales, a.scale_dtype, s0 + i)));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    // exponent field of the maximum, kept where 2^e and 2^-e are both normal
    const int ex = min(max(static_cast<int>(__float_as_uint(m) >> 23), 1), 253);
    const float inv = __uint_as_float(static_cast<uint32_t>(254 - ex) << 23);
    if (lane == 0) a.w_pow[item] = __uint_as_float(static_cast<uint32_t>(ex) << 23);
    const uint32_t* src = reinterpret_cast<const uint32_t*>(a.w + item * a.ldw);
    uint4* dst = reinterpret_cast<uint4*>(a.w16 + item * a.K);
    const int words = a.K >> 3;
    for (int i0 = lane; i0 < words; i0 += 128) {
      uint32_t word[4];
      float s[4];
      uint32_t z[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + 32 * u;
        if (i < words) {
          word[u] = __ldg(src + i);
          const int64_t gi = s0 + ((i << 3) >> a.log_g);
          s[u] = load_scale(a.scales, a.scale_dtype, gi);
          z[u] = a.zeros ? __ldg(a.zeros + gi) & 15u : 8u;
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + 32 * u;
        if (i < words) {
          const uint32_t zz = w4_zero(z[u]);
          uint32_t p[4];
          w4_decode(word[u], __byte_perm(zz, 0, 0x1010), __byte_perm(zz, 0, 0x3232), p);
          const float f = s[u] * inv;
          float2 v[4];  // codes (0, 4), (1, 5), (2, 6), (3, 7)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            v[j] = __half22float2(*reinterpret_cast<const __half2*>(&p[j]));
            v[j].x *= f;
            v[j].y *= f;
          }
          dst[i] = make_uint4(pack_f16x2(v[0].x, v[1].x), pack_f16x2(v[2].x, v[3].x), pack_f16x2(v[0].y, v[1].y),
                              pack_f16x2(v[2].y, v[3].y));
        }
      }
    }
    return;
  }
  const int64_t m = item - (static_cast<int64_t>(a.N) + 7) / 8 * 8;  // (the weight's blocks end on a block)
  if (!a.x || m < 0 || m >= a.M) return;
  const uint16_t* row = reinterpret_cast<const uint16_t*>(a.x + m * a.ldx);
  const int pieces = a.K >> 3;
  auto piece = [&](int p) {
    if (a.x_vec) return __ldg(reinterpret_cast<const uint4*>(row + p * 8));
    uint32_t e[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) e[j] = __ldg(row + p * 8 + 2 * j) | (uint32_t(__ldg(row + p * 8 + 2 * j + 1)) << 16);
    return make_uint4(e[0], e[1], e[2], e[3]);
  };
  uint32_t top = 0;  // largest |x| as bits; infinities and NaN sort above
#pragma unroll 4
  for (int p = lane; p < pieces; p += 32) {
    const uint4 v = piece(p);
    const uint32_t e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) top = max(top, max(e[j] & 0x7FFFu, (e[j] >> 16) & 0x7FFFu));
  }
  top = __reduce_max_sync(0xffffffffu, top);
  // infinities and NaN carry through the product; finite values beside them stay finite
  const int ex = min(max(static_cast<int>(top >> 7), 1), 253);
  const float inv = __uint_as_float(static_cast<uint32_t>(254 - ex) << 23);
  if (lane == 0) a.x_pow[m] = __uint_as_float(static_cast<uint32_t>(ex) << 23) * 0x1p-22f;  // 2^-148 and up
  if (lane == 0 && m == 0) *a.last = 0x1p22f;
  uint4* dst = reinterpret_cast<uint4*>(a.x16 + m * a.K);
#pragma unroll 4
  for (int p = lane; p < pieces; p += 32) {
    const uint4 v = piece(p);
    const uint32_t e[4] = {v.x, v.y, v.z, v.w};
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      o[j] = pack_f16x2(__uint_as_float(e[j] << 16) * inv, __uint_as_float(e[j] & 0xFFFF0000u) * inv);
    dst[p] = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

}  // namespace b200q
