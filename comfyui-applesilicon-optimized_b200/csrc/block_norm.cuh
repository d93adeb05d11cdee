// The norms before and after a transformer block, with the block's gate, the
// residual scale and the next block's modulation, one pass over the rows:
//   after:   h   = a * residual + gate[b] * (norm_post(y) * w_post)
//   before:  out = norm(h) * w * (1 + scale[b]) + shift[b]
// norm is RMS (v * rsqrt(mean v^2 + eps)), layer ((v - mean) * rsqrt(var + eps))
// or none; b = row / rows_per_mod.  `out` is 16-bit, or INT8 codes with one
// scale per row: s = max|out| / 127, q = rint(out / s).
//
// A row stays in fp32 registers from its one load to its one store: the second
// norm and the quantization take the unrounded h and out, so each stored value
// is rounded once.  The variance is centred (a second pass over registers, not
// sum(v^2) - mean^2, which cancels for rows with a large mean): each warp centres its
// values on its own mean, and the warps' means and squares are joined by
//   D var = sum_w [ M2_w + n_w (mean_w - mean)^2 ],
// so one barrier per norm is enough.
//
// Bound: HBM.  Wan-shaped rows (65,520 x 5,120 bf16, 2.68 GB with h and out written: 459
// us in a captured graph, 0.89 of the measured copy, 476 among eager calls; h alone 321 us,
// 0.96; a norm alone 293 us, 0.70) run persistent CTAs: a CTA's rows share their modulation,
// which is folded once into three fp32 vectors in shared memory (gate * post_w, w * (1 +
// scale), shift) instead of being read again from L2 for every row, and the next row's loads
// are in flight while one is reduced.  Norms to INT8 are bound by a row's two dependent
// reductions and three CTAs an SM (15 warps, 102 registers): 4101 x 5120 34 us, 0.28; 65,520
// rows 446 us, 0.34, with the residual 492 us, 0.73.
#pragma once

#include <type_traits>

#include "digits.cuh"
#include "numerics.cuh"
#include "ptx.cuh"

namespace b200q {

enum NormKind : int { kNormNone = 0, kNormRms = 1, kNormLayer = 2 };

struct NormArgs {
  const void* x;  // residual stream (after) or the norm's input (before)
  int64_t ldx;
  const void* y;  // the block's output, or null (before only)
  int64_t ldy;
  const void* post_w;  // [D] or null
  int post_w_dtype;
  const void* w;  // [D] or null
  int w_dtype;
  const void *gate, *scale, *shift;  // [mods, D] or null
  int64_t ld_gate, ld_scale, ld_shift;
  int mod_dtype;
  float res_scale, eps;
  int post_kind, pre_kind;
  void* h;  // [rows, D] or null
  int64_t ldh;
  void* out;  // [rows, D] or null
  int64_t ldo;
  int8_t* q;  // [rows, D] or null
  int64_t ldq;
  float* q_scale;
  int rows, D, rows_per_mod;
};

// Sum (or maximum) over the block; every thread gets the result.  `buf` is one
// of two 32-word buffers used in turn, so one barrier per call is enough.
template <bool MAX>
__device__ __forceinline__ float block_all(float v, float* buf) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float u = __shfl_xor_sync(0xffffffffu, v, o);
    v = MAX ? fmaxf(v, u) : v + u;
  }
  const int warps = blockDim.x >> 5;
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  v = buf[0];
  for (int i = 1; i < warps; ++i) v = MAX ? fmaxf(v, buf[i]) : v + buf[i];
  return v;
}

// 8 consecutive values of a bf16 / fp16 / fp32 array (BiasDtype codes), or one.
template <int VEC>
__device__ __forceinline__ void load_vals(const void* p, int dtype, int64_t i, float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    if (dtype == kBiasF32) v[0] = static_cast<const float*>(p)[i];
    else if (dtype == kBiasBF16) v[0] = __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    else v[0] = __half2float(static_cast<const __half*>(p)[i]);
  } else {
    if (dtype == kBiasF32) {
      const float4* s = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
      const float4 a = s[0], b = s[1];
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
      const uint32_t uv[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (dtype == kBiasBF16) {
          v[2 * j] = __uint_as_float(uv[j] << 16);
          v[2 * j + 1] = __uint_as_float(uv[j] & 0xFFFF0000u);
        } else {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&uv[j]));
          v[2 * j] = f.x;
          v[2 * j + 1] = f.y;
        }
      }
    }
  }
}

template <int VEC>
__device__ __forceinline__ void store_vals16(void* p, int dtype, int64_t i, const float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    if (dtype == kBiasBF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v[0]);
    else static_cast<__half*>(p)[i] = __float2half_rn(v[0]);
  } else {
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      o[j] = dtype == kBiasBF16 ? pack_bf16x2(v[2 * j], v[2 * j + 1]) : pack_f16x2(v[2 * j], v[2 * j + 1]);
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// One CTA per row; thread i holds values i, i + threads, ...  The form for any D,
// stride and alignment, used where a row is too long for the other two.  Bound: single
// values, one row per CTA: 4096 x 12288 339 us for a norm, 694 after + before (0.09 of the
// copy rate).
template <int DTYPE, int NPT>
__global__ void __launch_bounds__(1024) block_norm_kernel(const NormArgs a) {
  __shared__ float bufs[2][32];
  int turn = 0;
  griddep_wait();
  griddep_launch_dependents();
  const int64_t row = blockIdx.x;
  const int mod = static_cast<int>(row / a.rows_per_mod);
  const float inv_d = 1.0f / static_cast<float>(a.D);
  float v[NPT][1];

  auto each = [&](auto f) {
#pragma unroll
    for (int k = 0; k < NPT; ++k) {
      const int i = threadIdx.x + k * blockDim.x;
      if (i < a.D) f(k, i);
    }
  };
  // norm of the row in v (zeros past its end)
  auto normalise = [&](int kind) {
    if (kind == kNormNone) return;
    if (kind == kNormLayer) {
      float s = 0.0f;
      each([&](int k, int) { s += v[k][0]; });
      const float mean = block_all<false>(s, bufs[turn ^= 1]) * inv_d;
      each([&](int k, int) { v[k][0] -= mean; });
    }
    float s = 0.0f;
    each([&](int k, int) { s = fmaf(v[k][0], v[k][0], s); });
    const float r = rsqrtf(block_all<false>(s, bufs[turn ^= 1]) * inv_d + a.eps);
    each([&](int k, int) { v[k][0] *= r; });
  };

  if (a.y) {
    each([&](int k, int c) { load_vals<1>(a.y, DTYPE, row * a.ldy + c, v[k]); });
    normalise(a.post_kind);
    each([&](int k, int c) {
      float u[1];
      if (a.post_w) {
        load_vals<1>(a.post_w, a.post_w_dtype, c, u);
        v[k][0] *= u[0];
      }
      if (a.gate) {
        load_vals<1>(a.gate, a.mod_dtype, mod * a.ld_gate + c, u);
        v[k][0] *= u[0];
      }
      load_vals<1>(a.x, DTYPE, row * a.ldx + c, u);
      v[k][0] = fmaf(a.res_scale, u[0], v[k][0]);
      if (a.h) store_vals16<1>(a.h, DTYPE, row * a.ldh + c, v[k]);
    });
  } else {
    each([&](int k, int c) { load_vals<1>(a.x, DTYPE, row * a.ldx + c, v[k]); });
  }
  if (!a.out && !a.q) return;
  normalise(a.pre_kind);
  float top = 0.0f;
  each([&](int k, int c) {
    float u[1];
    if (a.w) {
      load_vals<1>(a.w, a.w_dtype, c, u);
      v[k][0] *= u[0];
    }
    if (a.scale) {
      load_vals<1>(a.scale, a.mod_dtype, mod * a.ld_scale + c, u);
      v[k][0] *= 1.0f + u[0];
    }
    if (a.shift) {
      load_vals<1>(a.shift, a.mod_dtype, mod * a.ld_shift + c, u);
      v[k][0] += u[0];
    }
    if (a.out) store_vals16<1>(a.out, DTYPE, row * a.ldo + c, v[k]);
    // NaN must reach the maximum (fmaxf drops it): compare the bits
    top = __uint_as_float(max(__float_as_uint(top), __float_as_uint(v[k][0]) & 0x7FFFFFFFu));
  });
  if (!a.q) return;
  // a NaN anywhere in the row makes its scale NaN: block_all's fmaxf would drop it
  const bool bad = __syncthreads_or(!(top <= 3.402823466e38f));
  top = block_all<true>(top, bufs[turn ^= 1]);
  const float s = bad ? __uint_as_float(0x7FC00000u) : __fdiv_rn(top, 127.0f);
  if (threadIdx.x == 0) a.q_scale[row] = s;
  each([&](int k, int c) {
    const float f = s > 0.0f ? rintf(__fdiv_rn(v[k][0], s)) : 0.0f;
    a.q[row * a.ldq + c] = static_cast<int8_t>(fminf(fmaxf(f, -127.0f), 127.0f));
  });
}

// ---------------------------------------------------------------- aligned rows
// Rows of 8-value vectors, NPT per thread (16-byte aligned operands): thread i holds
// vectors i, i + threads, ...; absent ones are zeros.  inv_n_w: 1 / this warp's values, n_l:
// those of warp `lane`; buf: one pair of 32 words per norm in flight.
template <int NPT, bool FULL, int VEC = 8>
__device__ __forceinline__ void row_norm(float (&v)[NPT][VEC], int kind, const bool (&on)[NPT], float inv_n_w, float n_l,
                                         float inv_n_l, float inv_d, float eps, float (*buf)[32]) {
  if (kind == kNormNone) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const bool layer = kind == kNormLayer;
  float mean_w = 0.0f, s = 0.0f;
  if (layer) {
#pragma unroll
    for (int k = 0; k < NPT; ++k)
#pragma unroll
      for (int j = 0; j < VEC; ++j) s += v[k][j];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    mean_w = s * inv_n_w;
  }
  float q = 0.0f;
#pragma unroll
  for (int k = 0; k < NPT; ++k)
    if (FULL || on[k]) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) q = fmaf(v[k][j] - mean_w, v[k][j] - mean_w, q);
    }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
  if (lane == 0) {
    buf[0][warp] = s;
    buf[1][warp] = q;
  }
  __syncthreads();
  // every warp joins all warps: lane w has warp w's sums
  float mean = 0.0f, sq = lane < warps ? buf[1][lane] : 0.0f;
  if (layer) {
    const float sw = lane < warps ? buf[0][lane] : 0.0f;
    mean = sw;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mean += __shfl_xor_sync(0xffffffffu, mean, o);
    mean *= inv_d;
    const float d = fmaf(sw, inv_n_l, -mean);
    if (lane < warps) sq = fmaf(n_l * d, d, sq);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
  const float r = rsqrtf(fmaf(sq, inv_d, eps));
#pragma unroll
  for (int k = 0; k < NPT; ++k)
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[k][j] = (v[k][j] - mean) * r;
}

template <int DTYPE>
__device__ __forceinline__ void unpack8(const uint4& u, float (&v)[8]) {
  const uint32_t uv[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (DTYPE == kBiasBF16) {
      v[2 * j] = __uint_as_float(uv[j] << 16);
      v[2 * j + 1] = __uint_as_float(uv[j] & 0xFFFF0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&uv[j]));
      v[2 * j] = f.x;
      v[2 * j + 1] = f.y;
    }
  }
}
// The three vectors of 8 columns at c for modulation row `mod`: gate * post_w, w *
// (1 + scale), shift.
__device__ __forceinline__ void fold_mods(const NormArgs& a, int64_t mod, int c, float (&g)[8], float (&w)[8], float (&b)[8]) {
  float u[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    g[j] = w[j] = 1.0f;
    b[j] = 0.0f;
  }
  if (a.post_w) load_vals<8>(a.post_w, a.post_w_dtype, c, g);
  if (a.gate) {
    load_vals<8>(a.gate, a.mod_dtype, mod * a.ld_gate + c, u);
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] *= u[j];
  }
  if (a.w) load_vals<8>(a.w, a.w_dtype, c, w);
  if (a.scale) {
    load_vals<8>(a.scale, a.mod_dtype, mod * a.ld_scale + c, u);
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] *= 1.0f + u[j];
  }
  if (a.shift) load_vals<8>(a.shift, a.mod_dtype, mod * a.ld_shift + c, b);
}

// A row's INT8 codes: the nearest integers of the rounded quotients v / s (16-bit rows meet
// exact ties often, half of the row's largest value among them).  The quotient is the product
// with 1 / s and one correction by its remainder; the nearest integer is the low byte of its
// sum with 1.5 * 2^23.  `lift` brings a row whose scale is below 2^-100, where the remainder
// and the reciprocal leave fp32's range, up by 2^64 (and holds it to 127 of a scale that was
// rounded to a few bits).
struct RowCodes {
  float s, inv;
  __device__ __forceinline__ explicit RowCodes(float scale) {
    s = scale < 0x1p-100f ? scale * 0x1p64f : scale;
    inv = scale > 0.0f ? __fdiv_rn(1.0f, s) : 0.0f;
    if (!(scale > 0.0f)) s = 0.0f;  // of zeros, or NaN: codes of 0
  }
  template <int NPT, int VEC>
  __device__ __forceinline__ static void lift(float scale, float (&v)[NPT][VEC]) {
    if (!(scale > 0.0f && scale < 0x1p-100f)) return;
    const float most = 127.0f * (scale * 0x1p64f);
#pragma unroll
    for (int k = 0; k < NPT; ++k)
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[k][j] = fminf(fmaxf(v[k][j] * 0x1p64f, -most), most);
  }
  __device__ __forceinline__ uint32_t operator()(float v) const {
    const float y = v * inv;
    return __float_as_uint(fmaf(fmaf(-y, s, v), inv, y) + 12582912.0f);
  }
};

// PERSIST: CTAs loop over contiguous rows, the folded vectors in shared memory (AFTER 3,
// else 2; a thread writes and reads its own columns; the first four values of all
// vectors, then the other four, so that neighbouring threads read neighbouring words).  Otherwise one row per CTA, one
// vector per thread, every load in flight at once.  FULL: no thread has an absent
// vector.
template <int DTYPE, bool PERSIST, int NPT, bool FULL, bool QUANT, bool AFTER>
__global__ void __launch_bounds__(PERSIST ? 512 : 1024) block_norm_rows_kernel(const NormArgs a) {
  extern __shared__ float4 folded[];
  // by row parity: with one barrier per norm a fast warp may already be writing the next
  // row's sums while a slow one reads this row's
  __shared__ float bufs[2][3][2][32];
  griddep_wait();
  griddep_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const float inv_d = 1.0f / static_cast<float>(a.D);
  const int nv = a.D >> 3;
  int col[NPT];
  bool on[NPT];
  int nw = 0, nl = 0;
#pragma unroll
  for (int k = 0; k < NPT; ++k) {
    col[k] = (threadIdx.x + k * blockDim.x) * 8;
    on[k] = col[k] < a.D;
    nw += min(max(a.D - static_cast<int>(k * blockDim.x + warp * 32) * 8, 0), 256);
    nl += min(max(a.D - static_cast<int>(k * blockDim.x + lane * 32) * 8, 0), 256);
  }
  const float n_l = static_cast<float>(max(nl, 1)), inv_n_l = 1.0f / n_l, inv_n_w = 1.0f / static_cast<float>(max(nw, 1));
  const int64_t r0 = PERSIST ? static_cast<int64_t>(a.rows) * blockIdx.x / gridDim.x : blockIdx.x;
  const int64_t r1 = PERSIST ? static_cast<int64_t>(a.rows) * (blockIdx.x + 1) / gridDim.x : r0 + 1;
  uint4 xn[NPT], yn[NPT];  // the row after this one
  const uint16_t* xp = static_cast<const uint16_t*>(a.x) + r0 * a.ldx;
  const uint16_t* yp = static_cast<const uint16_t*>(a.y) + r0 * a.ldy;
  auto fetch = [&]() {
#pragma unroll
    for (int k = 0; k < NPT; ++k) {
      xn[k] = yn[k] = make_uint4(0, 0, 0, 0);
      if (FULL || on[k]) {
        xn[k] = __ldg(reinterpret_cast<const uint4*>(xp + col[k]));
        if (AFTER) yn[k] = __ldg(reinterpret_cast<const uint4*>(yp + col[k]));
      }
    }
    xp += a.ldx;
    yp += a.ldy;
  };
  if (r0 < r1) fetch();
  int64_t mod_end = r0;  // the first row that needs other vectors
  float g[8], w[8], b[8];  // (not PERSIST) the folded vectors
  char* hp = static_cast<char*>(a.h) + r0 * a.ldh * 2;
  char* op = static_cast<char*>(a.out) + r0 * a.ldo * 2;
  for (int64_t row = r0; row < r1; ++row, hp += a.ldh * 2, op += a.ldo * 2) {
    uint4 x0[NPT], y0[NPT];
#pragma unroll
    for (int k = 0; k < NPT; ++k) {
      x0[k] = xn[k];
      y0[k] = yn[k];
    }
    if (row + 1 < r1) fetch();
    if (row >= mod_end) {
      const int64_t mod = row / a.rows_per_mod;
      mod_end = (mod + 1) * a.rows_per_mod;
#pragma unroll
      for (int k = 0; k < NPT; ++k)
        if (FULL || on[k]) {
          fold_mods(a, mod, col[k], g, w, b);
          if (PERSIST) {
            float4* f = folded + (col[k] >> 3);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              f[j * nv] = make_float4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
              f[(2 + j) * nv] = make_float4(b[4 * j], b[4 * j + 1], b[4 * j + 2], b[4 * j + 3]);
              if (AFTER) f[(4 + j) * nv] = make_float4(g[4 * j], g[4 * j + 1], g[4 * j + 2], g[4 * j + 3]);
            }
          }
        }
    }
    auto vec = [&](int which, int c, float (&u)[8]) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float4 f = folded[(2 * which + j) * nv + (c >> 3)];
        u[4 * j] = f.x; u[4 * j + 1] = f.y; u[4 * j + 2] = f.z; u[4 * j + 3] = f.w;
      }
    };
    float v[NPT][8];
    if (AFTER) {
#pragma unroll
      for (int k = 0; k < NPT; ++k) unpack8<DTYPE>(y0[k], v[k]);
      row_norm<NPT, FULL>(v, a.post_kind, on, inv_n_w, n_l, inv_n_l, inv_d, a.eps, bufs[row & 1][0]);
#pragma unroll
      for (int k = 0; k < NPT; ++k) {
        if (FULL || on[k]) {
          float u[8];
          unpack8<DTYPE>(x0[k], u);
          if (PERSIST) vec(2, col[k], g);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[k][j] = fmaf(a.res_scale, u[j], v[k][j] * g[j]);
          if (a.h) store_vals16<8>(hp, DTYPE, col[k], v[k]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[k][j] = 0.0f;
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < NPT; ++k) unpack8<DTYPE>(x0[k], v[k]);
    }
    if (!QUANT && !a.out) continue;
    row_norm<NPT, FULL>(v, a.pre_kind, on, inv_n_w, n_l, inv_n_l, inv_d, a.eps, bufs[row & 1][1]);
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < NPT; ++k)
      if (FULL || on[k]) {
        if (PERSIST) {
          vec(0, col[k], w);
          vec(1, col[k], b);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[k][j] = fmaf(v[k][j], w[j], b[j]);
          if (QUANT) top = max(top, __float_as_uint(v[k][j]) & 0x7FFFFFFFu);  // as bits: NaN sorts above
        }
        if (!QUANT) store_vals16<8>(op, DTYPE, col[k], v[k]);
      }
    if (!QUANT) continue;
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) bufs[row & 1][2][0][warp] = __uint_as_float(top);
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, lane < warps ? __float_as_uint(bufs[row & 1][2][0][lane]) : 0u);
    // a row holding inf or NaN gets a NaN scale
    const float t = __uint_as_float(top);
    const float s = top >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : __fdiv_rn(t, 127.0f);
    if (threadIdx.x == 0) a.q_scale[row] = s;
    const RowCodes code(s);
    RowCodes::lift(s, v);
#pragma unroll
    for (int k = 0; k < NPT; ++k)
      if (FULL || on[k]) {
        uint32_t o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = code(v[k][j]);
        *reinterpret_cast<uint2*>(a.q + row * a.ldq + col[k]) =
            make_uint2(low_bytes(o[0], o[1], o[2], o[3]), low_bytes(o[4], o[5], o[6], o[7]));
      }
  }
}

// ---------------------------------------------------------------- other rows
// The same for rows that 16-byte vectors do not fit (odd D, strides, views): VW = 2 values
// per access when every row starts on a pair, else one.  A warp has 512 columns, lane i those
// at (32 s + i) * VW in step s: its accesses are contiguous and their offsets from the row's
// pointers constants (with steps of the CTA's width the addresses were half of the
// instructions: 75 us for the first size below).  Persistent CTAs, the folded vectors in shared
// memory and the next row's loads in flight, as above.  Bound: the instructions per value.
// After + before, fp32 modulation: 13824 x 1486 54 us, 0.46 of the copy rate (190 us with
// one CTA per row); 6558 x 2020 37 us (135); 159 x 783 8 us.
constexpr int kLooseValues = 16;  // per thread
template <int DTYPE, int VW, bool QUANT, bool AFTER>
__global__ void __launch_bounds__(512) block_norm_loose_kernel(const NormArgs a) {
  constexpr int S = kLooseValues / VW;
  using Raw = typename std::conditional<VW == 2, uint32_t, uint16_t>::type;
  extern __shared__ float4 folded[];
  float* const fold = reinterpret_cast<float*>(folded);  // w * (1 + scale), shift, gate * post_w
  __shared__ float bufs[2][3][2][32];                    // by row parity, as above
  griddep_wait();
  griddep_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const float inv_d = 1.0f / static_cast<float>(a.D);
  const int c0 = warp * (32 * kLooseValues) + lane * VW;  // the thread's first column
  constexpr int kStep = 32 * VW;
  bool on[S];
#pragma unroll
  for (int s = 0; s < S; ++s) on[s] = c0 + s * kStep < a.D;
  const int nw = min(max(a.D - warp * (32 * kLooseValues), 0), 32 * kLooseValues);
  const int nl = min(max(a.D - lane * (32 * kLooseValues), 0), 32 * kLooseValues);
  const float n_l = static_cast<float>(max(nl, 1)), inv_n_l = 1.0f / n_l, inv_n_w = 1.0f / static_cast<float>(max(nw, 1));
  const int64_t r0 = static_cast<int64_t>(a.rows) * blockIdx.x / gridDim.x;
  const int64_t r1 = static_cast<int64_t>(a.rows) * (blockIdx.x + 1) / gridDim.x;
  Raw xn[S], yn[S];  // the row after this one
  const uint16_t* xp = static_cast<const uint16_t*>(a.x) + r0 * a.ldx + c0;
  const uint16_t* yp = static_cast<const uint16_t*>(a.y) + r0 * a.ldy + c0;
  auto fetch = [&]() {
#pragma unroll
    for (int s = 0; s < S; ++s) {
      xn[s] = yn[s] = 0;
      if (on[s]) {
        xn[s] = __ldg(reinterpret_cast<const Raw*>(xp + s * kStep));
        if (AFTER) yn[s] = __ldg(reinterpret_cast<const Raw*>(yp + s * kStep));
      }
    }
    xp += a.ldx;
    yp += a.ldy;
  };
  auto unpack = [](Raw u, float (&v)[VW]) {
#pragma unroll
    for (int j = 0; j < VW; ++j) {
      const uint16_t e = static_cast<uint16_t>(u >> (16 * j));
      v[j] = DTYPE == kBiasBF16 ? __uint_as_float(static_cast<uint32_t>(e) << 16) : __half2float(__ushort_as_half(e));
    }
  };
  auto store = [&](uint16_t* p, const float (&v)[VW]) {
    if constexpr (VW == 2)
      *reinterpret_cast<uint32_t*>(p) = DTYPE == kBiasBF16 ? pack_bf16x2(v[0], v[1]) : pack_f16x2(v[0], v[1]);
    else
      store_vals16<1>(p, DTYPE, 0, v);
  };
  if (r0 < r1) fetch();
  int64_t mod_end = r0;  // the first row that needs other vectors
  for (int64_t row = r0; row < r1; ++row) {
    Raw x0[S], y0[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      x0[s] = xn[s];
      y0[s] = yn[s];
    }
    if (row + 1 < r1) fetch();
    if (row >= mod_end) {  // a thread writes and reads its own columns
      const int64_t mod = row / a.rows_per_mod;
      mod_end = (mod + 1) * a.rows_per_mod;
      float u[S][VW], t[S][VW];
      auto read = [&](const void* p, int dtype, int64_t at, float none, float (&to)[S][VW]) {
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
          for (int j = 0; j < VW; ++j) {
            float one[1] = {none};
            if (p && on[s]) load_vals<1>(p, dtype, at + c0 + s * kStep + j, one);
            to[s][j] = one[0];
          }
      };
      auto keep = [&](int which) {
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
          for (int j = 0; j < VW; ++j)
            if (on[s]) fold[which * a.D + c0 + s * kStep + j] = u[s][j];
      };
      auto times = [&](float plus) {
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
          for (int j = 0; j < VW; ++j) u[s][j] *= plus + t[s][j];
      };
      read(a.w, a.w_dtype, 0, 1.0f, u);
      read(a.scale, a.mod_dtype, mod * a.ld_scale, 0.0f, t);
      times(1.0f);
      keep(0);
      read(a.shift, a.mod_dtype, mod * a.ld_shift, 0.0f, u);
      keep(1);
      if (AFTER) {
        read(a.post_w, a.post_w_dtype, 0, 1.0f, u);
        read(a.gate, a.mod_dtype, mod * a.ld_gate, 1.0f, t);
        times(0.0f);
        keep(2);
      }
    }
    auto folded_at = [&](int which, int s, float (&to)[VW]) {
      const float* f = fold + which * a.D + c0 + s * kStep;
      if constexpr (VW == 2) {
        const float2 e = *reinterpret_cast<const float2*>(f);
        to[0] = e.x;
        to[1] = e.y;
      } else {
        to[0] = *f;
      }
    };
    float v[S][VW];
    if (AFTER) {
#pragma unroll
      for (int s = 0; s < S; ++s) unpack(y0[s], v[s]);
      row_norm<S, false, VW>(v, a.post_kind, on, inv_n_w, n_l, inv_n_l, inv_d, a.eps, bufs[row & 1][0]);
      uint16_t* hp = static_cast<uint16_t*>(a.h) + row * a.ldh + c0;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        float u[VW], g[VW];
        unpack(x0[s], u);
        if (on[s]) folded_at(2, s, g);
#pragma unroll
        for (int j = 0; j < VW; ++j) v[s][j] = on[s] ? fmaf(a.res_scale, u[j], v[s][j] * g[j]) : 0.0f;
        if (a.h && on[s]) store(hp + s * kStep, v[s]);
      }
    } else {
#pragma unroll
      for (int s = 0; s < S; ++s) unpack(x0[s], v[s]);
    }
    if (!QUANT && !a.out) continue;
    row_norm<S, false, VW>(v, a.pre_kind, on, inv_n_w, n_l, inv_n_l, inv_d, a.eps, bufs[row & 1][1]);
    uint16_t* op = static_cast<uint16_t*>(a.out) + row * a.ldo + c0;
    uint32_t top = 0;
#pragma unroll
    for (int s = 0; s < S; ++s)
      if (on[s]) {
        float w[VW], b[VW];
        folded_at(0, s, w);
        folded_at(1, s, b);
#pragma unroll
        for (int j = 0; j < VW; ++j) {
          v[s][j] = fmaf(v[s][j], w[j], b[j]);
          if (QUANT) top = max(top, __float_as_uint(v[s][j]) & 0x7FFFFFFFu);  // as bits: NaN sorts above
        }
        if (!QUANT) store(op + s * kStep, v[s]);
      }
    if (!QUANT) continue;
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) bufs[row & 1][2][0][warp] = __uint_as_float(top);
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, lane < warps ? __float_as_uint(bufs[row & 1][2][0][lane]) : 0u);
    const float t = __uint_as_float(top);
    const float sc = top >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : __fdiv_rn(t, 127.0f);
    if (threadIdx.x == 0) a.q_scale[row] = sc;
    const RowCodes code(sc);
    RowCodes::lift(sc, v);
    int8_t* qp = a.q + row * a.ldq + c0;
#pragma unroll
    for (int s = 0; s < S; ++s)
      if (on[s]) {
        uint32_t o[VW];
#pragma unroll
        for (int j = 0; j < VW; ++j) o[j] = code(v[s][j]);
        if constexpr (VW == 2)
          *reinterpret_cast<uint16_t*>(qp + s * kStep) = static_cast<uint16_t>(__byte_perm(o[0], o[1], 0x0040));
        else
          qp[s * kStep] = static_cast<int8_t>(o[0]);
      }
  }
}

}  // namespace b200q
