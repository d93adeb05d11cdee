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
// sum(v^2) - mean^2, which cancels for rows with a large mean).
#pragma once

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

// One CTA per row; thread i holds vectors i, i + threads, ... (NPT of VEC values).
template <int DTYPE, int VEC, int NPT>
__global__ void __launch_bounds__(1024) block_norm_kernel(const NormArgs a) {
  __shared__ float bufs[2][32];
  int turn = 0;
  griddep_wait();
  griddep_launch_dependents();
  const int64_t row = blockIdx.x;
  const int mod = static_cast<int>(row / a.rows_per_mod);
  const int nv = a.D / VEC;
  const float inv_d = 1.0f / static_cast<float>(a.D);
  float v[NPT][VEC];

  auto each = [&](auto f) {
#pragma unroll
    for (int k = 0; k < NPT; ++k) {
      const int i = threadIdx.x + k * blockDim.x;
      if (i < nv) f(k, i * VEC);
    }
  };
  // norm of the row in v (zeros past its end)
  auto normalise = [&](int kind) {
    if (kind == kNormNone) return;
    if (kind == kNormLayer) {
      float s = 0.0f;
      each([&](int k, int) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) s += v[k][j];
      });
      const float mean = block_all<false>(s, bufs[turn ^= 1]) * inv_d;
      each([&](int k, int) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[k][j] -= mean;
      });
    }
    float s = 0.0f;
    each([&](int k, int) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) s = fmaf(v[k][j], v[k][j], s);
    });
    const float r = rsqrtf(block_all<false>(s, bufs[turn ^= 1]) * inv_d + a.eps);
    each([&](int k, int) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[k][j] *= r;
    });
  };

  if (a.y) {
    each([&](int k, int c) { load_vals<VEC>(a.y, DTYPE, row * a.ldy + c, v[k]); });
    normalise(a.post_kind);
    each([&](int k, int c) {
      float u[VEC];
      if (a.post_w) {
        load_vals<VEC>(a.post_w, a.post_w_dtype, c, u);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[k][j] *= u[j];
      }
      if (a.gate) {
        load_vals<VEC>(a.gate, a.mod_dtype, mod * a.ld_gate + c, u);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[k][j] *= u[j];
      }
      load_vals<VEC>(a.x, DTYPE, row * a.ldx + c, u);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[k][j] = fmaf(a.res_scale, u[j], v[k][j]);
      if (a.h) store_vals16<VEC>(a.h, DTYPE, row * a.ldh + c, v[k]);
    });
  } else {
    each([&](int k, int c) { load_vals<VEC>(a.x, DTYPE, row * a.ldx + c, v[k]); });
  }
  if (!a.out && !a.q) return;
  normalise(a.pre_kind);
  float top = 0.0f;
  each([&](int k, int c) {
    float u[VEC];
    if (a.w) {
      load_vals<VEC>(a.w, a.w_dtype, c, u);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[k][j] *= u[j];
    }
    if (a.scale) {
      load_vals<VEC>(a.scale, a.mod_dtype, mod * a.ld_scale + c, u);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[k][j] *= 1.0f + u[j];
    }
    if (a.shift) {
      load_vals<VEC>(a.shift, a.mod_dtype, mod * a.ld_shift + c, u);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[k][j] += u[j];
    }
    if (a.out) store_vals16<VEC>(a.out, DTYPE, row * a.ldo + c, v[k]);
    // NaN must reach the maximum (fmaxf drops it): compare the bits
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      top = __uint_as_float(max(__float_as_uint(top), __float_as_uint(v[k][j]) & 0x7FFFFFFFu));
  });
  if (!a.q) return;
  // a NaN anywhere in the row makes its scale NaN: block_all's fmaxf would drop it
  const bool bad = __syncthreads_or(!(top <= 3.402823466e38f));
  top = block_all<true>(top, bufs[turn ^= 1]);
  const float s = bad ? __uint_as_float(0x7FC00000u) : __fdiv_rn(top, 127.0f);
  if (threadIdx.x == 0) a.q_scale[row] = s;
  each([&](int k, int c) {
    __align__(8) int8_t o[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float f = s > 0.0f ? rintf(__fdiv_rn(v[k][j], s)) : 0.0f;
      o[j] = static_cast<int8_t>(fminf(fmaxf(f, -127.0f), 127.0f));
    }
    if constexpr (VEC == 8)
      *reinterpret_cast<uint2*>(a.q + row * a.ldq + c) = *reinterpret_cast<const uint2*>(o);
    else
      a.q[row * a.ldq + c] = o[0];
  });
}

}  // namespace b200q
