// 4-bit weight-only linear with group scales, few tokens:
//   out[m,n] = act( sum_k x[m,k] * s[n,k/G] * (c[n,k] - z[n,k/G]) + b[n] )
// c: unsigned 4-bit codes, two per byte along K (even k in the low nibble);
// s: one scale per row and group of G codes; z: one zero point (0..15) per row
// and group, 8 when absent.
//
// Mathematics.  Inside a group the scale is a constant, so the group's sum is
// taken over the exact integers c - z, and one fp32 multiply-add per group
// joins it to the row's accumulator:  acc += s * sum_{k in group} x_k (c_k - z).
// c - z is exact in bf16 and fp16: OR-ing a nibble into the mantissa of 128
// (bf16) or 1024 (fp16) gives 128 + c / 1024 + c, and subtracting 128 + z /
// 1024 + z is exact.  Products and sums run on warp MMAs (m16n8k16, fp32
// accumulation) with 16 weight rows as the MMA's rows and 8 tokens as its
// columns; nothing is rounded before the output.
//
// Layout.  The order of k inside a group is free as long as both operands
// agree.  Lane (g, t) = (lane / 4, lane % 4) reads the G/4 codes of its quarter t
// of the group for rows g and g + 8 as they are stored (one 16-byte load each at
// G = 128); pair i of an 8-code word w is (w >> 4i) & 0x000F000F = codes i and
// i + 4.  x is staged once per CTA in shared memory in that order (8 values as
// 0 4 1 5 2 6 3 7; quarter-major), so one 16-byte shared load feeds two MMAs,
// and the row pitch is 64 modulo 128 bytes, which makes those loads free of
// bank conflicts.
#pragma once

#include "numerics.cuh"
#include "ptx.cuh"

namespace b200q {

constexpr int kW4Warps = 8;

struct W4Args {
  const void* x;         // [M, K] bf16 / fp16
  int64_t ldx;           // elements
  const uint8_t* w;      // [N, K / 2]
  int64_t ldw;           // bytes
  const void* scales;    // [N, K / G]
  int scale_dtype;       // kBiasBF16 / kBiasF16 / kBiasF32
  const uint8_t* zeros;  // [N, K / G] or null (8)
  int M, N, K, G;
  int x_vec;             // rows of x are 16-byte aligned
  int wr;                // warps along the rows: the CTA's tile is 16 * wr rows
  int splits;            // cluster size: CTAs that share a row tile's K
};

__device__ __forceinline__ float load_scale(const void* p, int dtype, int64_t i) {
  if (dtype == kBiasBF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  if (dtype == kBiasF16) return __half2float(static_cast<const __half*>(p)[i]);
  return static_cast<const float*>(p)[i];
}

template <typename T>
struct W4Num;
template <>
struct W4Num<__nv_bfloat16> {
  static constexpr uint32_t kMagic = 0x43004300u;  // 128, 128
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                     *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                             uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};
template <>
struct W4Num<__half> {
  static constexpr uint32_t kMagic = 0x64006400u;  // 1024, 1024
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a),
                              *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                             uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

// The four exact pairs (c_i - z, c_{i+4} - z) of one 8-code word; zp = magic | z.
template <typename T>
__device__ __forceinline__ void w4_decode(uint32_t w, uint32_t zp, uint32_t (&p)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    p[i] = W4Num<T>::sub(((w >> (4 * i)) & 0x000F000Fu) | W4Num<T>::kMagic, zp);
}

// Shared bytes per token row for a slice of `k` codes.
__host__ __device__ __forceinline__ int w4_pitch(int k) {
  const int b = 2 * k;
  return b + ((b & 127) == 64 ? 0 : 64);
}
// Dynamic shared memory: x slice, warp partials, CTA partials.
__host__ __device__ __forceinline__ int w4_smem_bytes(int M, int k_slice, int cols, int wr) {
  return M * w4_pitch(k_slice) + (kW4Warps * 16 + 16 * wr) * cols * 4;
}

template <int LW>
__device__ __forceinline__ void w4_load(uint32_t (&r)[LW], const uint8_t* p) {
  if constexpr (LW == 4) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
    r[0] = v.x; r[1] = v.y; r[2] = v.z; r[3] = v.w;
  } else if constexpr (LW == 2) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
    r[0] = v.x; r[1] = v.y;
  } else {
    r[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
  }
}

// LW = G / 32 words per lane, row and group; NT = 8-token columns of the MMA.
template <typename T, int LW, int NT>
__global__ void __launch_bounds__(kW4Warps * 32)
    w4a16_kernel(const W4Args a, const EpiArgs ep) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int G = 32 * LW;
  constexpr int U = LW == 4 ? 2 : LW == 2 ? 4 : 8;  // groups per load batch
  constexpr int kCols = 8 * NT;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int rank = a.splits > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int tile = blockIdx.x / a.splits;
  const int KG = a.K / G;
  const int wk_n = kW4Warps / a.wr;
  const int wr_i = warp % a.wr, wk_i = warp / a.wr;
  // this CTA's groups, then this warp's
  const int cg0 = static_cast<int>(int64_t(KG) * rank / a.splits);
  const int cg1 = static_cast<int>(int64_t(KG) * (rank + 1) / a.splits);
  const int g0 = cg0 + (cg1 - cg0) * wk_i / wk_n;
  const int g1 = cg0 + (cg1 - cg0) * (wk_i + 1) / wk_n;
  const int max_slice = (KG + a.splits - 1) / a.splits * G;
  const int pitch = w4_pitch(max_slice);
  float* red = reinterpret_cast<float*>(smem + a.M * pitch);  // [warp][col][16]
  float* part = red + kW4Warps * 16 * kCols;                  // [col][16 * wr]

  griddep_wait();
  griddep_launch_dependents();

  // ---- stage x[:, cg0*G .. cg1*G) in fragment order
  {
    const int pieces = (cg1 - cg0) * (G / 8);
    for (int i = tid; i < pieces * a.M; i += kW4Warps * 32) {
      const int m = i / pieces, p = i - m * pieces;
      const T* src = static_cast<const T*>(a.x) + m * a.ldx + int64_t(cg0) * G + p * 8;
      uint16_t e[8];
      if (a.x_vec) {
        *reinterpret_cast<uint4*>(e) = __ldg(reinterpret_cast<const uint4*>(src));
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = __ldg(reinterpret_cast<const uint16_t*>(src) + j);
      }
      const int grp = p / (G / 8), r = p - grp * (G / 8);
      const int at = (grp * LW + r % LW) * 4 + r / LW;  // [group][word][quarter]
      uint4 v;
      v.x = e[0] | (uint32_t(e[4]) << 16);
      v.y = e[1] | (uint32_t(e[5]) << 16);
      v.z = e[2] | (uint32_t(e[6]) << 16);
      v.w = e[3] | (uint32_t(e[7]) << 16);
      *reinterpret_cast<uint4*>(smem + m * pitch + at * 16) = v;
    }
  }
  __syncthreads();

  // ---- this warp's 16 rows x its groups
  const int n0 = (tile * a.wr + wr_i) * 16;
  const int rA = min(n0 + g, a.N - 1), rB = min(n0 + g + 8, a.N - 1);
  const uint8_t* wA = a.w + int64_t(rA) * a.ldw + t * (4 * LW);
  const uint8_t* wB = a.w + int64_t(rB) * a.ldw + t * (4 * LW);
  const int64_t sA = int64_t(rA) * KG, sB = int64_t(rB) * KG;
  const uint8_t* xs[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j)  // columns past M read row M - 1; their results are not used
    xs[j] = smem + min(8 * j + g, a.M - 1) * pitch + t * 16;

  float acc[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[j][i] = 0.0f;

  uint32_t ca[U][LW], cb[U][LW];
  float fa[U], fb[U];
  uint32_t za[U], zb[U];
  auto load = [&](int gi) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int q = min(gi + u, g1 - 1);
      w4_load<LW>(ca[u], wA + int64_t(q) * (G / 2));
      w4_load<LW>(cb[u], wB + int64_t(q) * (G / 2));
      fa[u] = load_scale(a.scales, a.scale_dtype, sA + q);
      fb[u] = load_scale(a.scales, a.scale_dtype, sB + q);
      za[u] = a.zeros ? a.zeros[sA + q] & 15u : 8u;
      zb[u] = a.zeros ? a.zeros[sB + q] & 15u : 8u;
    }
  };
  for (int gi = g0; gi < g1; gi += U) {
    load(gi);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (gi + u >= g1) break;
      float part_[NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) part_[j][i] = 0.0f;
      const uint32_t zpa = W4Num<T>::kMagic | za[u] * 0x00010001u;
      const uint32_t zpb = W4Num<T>::kMagic | zb[u] * 0x00010001u;
      const int xo = (gi + u - cg0) * LW * 64;
#pragma unroll
      for (int wi = 0; wi < LW; ++wi) {
        uint32_t pa[4], pb[4];
        w4_decode<T>(ca[u][wi], zpa, pa);
        w4_decode<T>(cb[u][wi], zpb, pb);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const uint4 xv = *reinterpret_cast<const uint4*>(xs[j] + xo + wi * 64);
          W4Num<T>::mma(part_[j], pa[0], pb[0], pa[1], pb[1], xv.x, xv.y);
          W4Num<T>::mma(part_[j], pa[2], pb[2], pa[3], pb[3], xv.z, xv.w);
        }
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        acc[j][0] = fmaf(fa[u], part_[j][0], acc[j][0]);
        acc[j][1] = fmaf(fa[u], part_[j][1], acc[j][1]);
        acc[j][2] = fmaf(fb[u], part_[j][2], acc[j][2]);
        acc[j][3] = fmaf(fb[u], part_[j][3], acc[j][3]);
      }
    }
  }

  // ---- join the warps' K ranges, then the cluster's, in a fixed order
  float* mine = red + warp * 16 * kCols;
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    mine[(8 * j + 2 * t) * 16 + g] = acc[j][0];
    mine[(8 * j + 2 * t + 1) * 16 + g] = acc[j][1];
    mine[(8 * j + 2 * t) * 16 + g + 8] = acc[j][2];
    mine[(8 * j + 2 * t + 1) * 16 + g + 8] = acc[j][3];
  }
  __syncthreads();
  const int rows = 16 * a.wr;
  for (int e = tid; e < rows * a.M; e += kW4Warps * 32) {
    const int col = e / rows, row = e - col * rows;
    float v = 0.0f;
    for (int k = 0; k < wk_n; ++k)
      v += red[((k * a.wr + row / 16) * kCols + col) * 16 + (row & 15)];
    part[col * rows + row] = v;
  }
  if (a.splits > 1) cluster_sync(); else __syncthreads();
  const float xs_scale = 1.0f;
  for (int e = tid + kW4Warps * 32 * rank; e < rows * a.M; e += kW4Warps * 32 * a.splits) {
    const int col = e / rows, row = e - col * rows;
    const int n = tile * rows + row;
    float v = 0.0f;
    if (a.splits > 1) {
      const uint32_t at = smem_u32(part + col * rows + row);
      for (int r = 0; r < a.splits; ++r) {
        float f;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f) : "r"(mapa_shared(at, r)) : "memory");
        v += f;
      }
    } else {
      v = part[col * rows + row];
    }
    if (n < a.N) store_out(ep, col, n, epi_scaled(v, 1.0f, 1.0f, xs_scale, ep, n));
  }
  if (a.splits > 1) cluster_sync();  // the other CTAs may still be reading this one's partials
}

// ---------------------------------------------------------------- many tokens
// Decodes the weight to fp16 for the tile GEMM.  A row's values are
// s * (c - z) * 2^-e with 2^e the power of two of the row's largest |s| (at most
// 15 * 2 in magnitude, so fp16's range holds whatever the scales are), and 2^e
// goes to row_pow[n] for the GEMM's column scale.  One rounding to fp16's 11
// bits; an eighth of a bf16 output's own rounding.
__global__ void __launch_bounds__(256)
    w4_decode_rows_kernel(const uint8_t* __restrict__ w, int64_t ldw, const void* scales,
                          int scale_dtype, const uint8_t* __restrict__ zeros, int N, int K, int G,
                          __half* __restrict__ out, float* __restrict__ row_pow) {
  __shared__ float wmax[8];
  griddep_wait();
  griddep_launch_dependents();
  const int n = blockIdx.x, tid = threadIdx.x;
  const int KG = K / G;
  float m = 0.0f;
  for (int i = tid; i < KG; i += 256) m = fmaxf(m, fabsf(load_scale(scales, scale_dtype, int64_t(n) * KG + i)));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((tid & 31) == 0) wmax[tid >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, wmax[i]);
  // exponent field of the maximum, kept where 2^e and 2^-e are both normal
  int ex = static_cast<int>(__float_as_uint(m) >> 23);
  ex = min(max(ex, 1), 253);
  const float inv = __uint_as_float(static_cast<uint32_t>(254 - ex) << 23);
  if (tid == 0) row_pow[n] = __uint_as_float(static_cast<uint32_t>(ex) << 23);
  const uint8_t* src = w + int64_t(n) * ldw;
  for (int i = tid; i < K / 32; i += 256) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(src + int64_t(i) * 16));
    const int64_t gi = int64_t(n) * KG + i * 32 / G;
    const float s = load_scale(scales, scale_dtype, gi) * inv;
    const int z = zeros ? zeros[gi] & 15 : 8;
    const uint32_t wv[4] = {v.x, v.y, v.z, v.w};
    uint4* dst = reinterpret_cast<uint4*>(out + int64_t(n) * K + int64_t(i) * 32);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int lo = static_cast<int>((wv[q] >> (8 * j)) & 15u) - z;
        const int hi = static_cast<int>((wv[q] >> (8 * j + 4)) & 15u) - z;
        o[j] = pack_f16x2(s * static_cast<float>(lo), s * static_cast<float>(hi));
      }
      dst[q] = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

// A token row of bf16 as fp16: x * 2^-e, 2^e the power of two of the row's
// largest |x|, to row_pow[m] for the GEMM's row scale.  Exact down to 2^-17 of
// the row's maximum, within 2^-25 of it below.
__global__ void __launch_bounds__(256)
    w4_x_f16_kernel(const __nv_bfloat16* __restrict__ x, int64_t ldx, int K, int x_vec,
                    __half* __restrict__ out, float* __restrict__ row_pow) {
  __shared__ uint32_t wmax[8];
  griddep_wait();
  griddep_launch_dependents();
  const int64_t m = blockIdx.x;
  const int tid = threadIdx.x;
  const uint16_t* src = reinterpret_cast<const uint16_t*>(x + m * ldx);
  auto piece = [&](int i, uint16_t (&e)[8]) {
    if (x_vec) {
      *reinterpret_cast<uint4*>(e) = __ldg(reinterpret_cast<const uint4*>(src + i * 8));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = __ldg(src + i * 8 + j);
    }
  };
  uint32_t top = 0;  // largest |x| as bits; infinities and NaN sort above
  for (int i = tid; i < K / 8; i += 256) {
    uint16_t e[8];
    piece(i, e);
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, uint32_t(e[j] & 0x7FFFu));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((tid & 31) == 0) wmax[tid >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, wmax[i]);
  // a row holding inf or NaN keeps its values: they carry through the product
  int ex = static_cast<int>(top >> 7);
  ex = ex == 255 ? 127 : min(max(ex, 1), 253);
  const float inv = __uint_as_float(static_cast<uint32_t>(254 - ex) << 23);
  if (tid == 0) row_pow[m] = __uint_as_float(static_cast<uint32_t>(ex) << 23);
  for (int i = tid; i < K / 8; i += 256) {
    uint16_t e[8];
    piece(i, e);
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      o[j] = pack_f16x2(__uint_as_float(uint32_t(e[2 * j]) << 16) * inv,
                        __uint_as_float(uint32_t(e[2 * j + 1]) << 16) * inv);
    *reinterpret_cast<uint4*>(out + m * K + i * 8) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

}  // namespace b200q
