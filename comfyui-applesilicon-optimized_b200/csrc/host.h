// Host-side helpers shared by the library's translation units (defined in
// capi.cu): the device gate, launch accounting, the programmatic-launch switch
// and the 16-bit tile GEMM.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "numerics.cuh"

namespace b200q {
namespace host {

// SM count of the current device, or 0 if it cannot run sm_100a code.
int device_sms();
// Checks the launch just made, counts it, and returns a B200Q_* status.
int finish_launch();
// B200Q_PDL (read per call): launch kernels as programmatic dependents.
bool pdl_on();
// Tensor map of a row-major [rows, cols] byte matrix with box box_cols x box_rows.
bool tmap_u8(CUtensorMap* map, const void* base, uint64_t cols, uint64_t rows, uint64_t ld_bytes,
             uint32_t box_cols, uint32_t box_rows, CUtensorMapSwizzle swizzle);
// The status word of lowbit.cu's kernels on the current device (read, and
// cleared when `reset`); b200q_get_device_status merges it with capi.cu's.
int lowbit_device_status(unsigned int* status, bool reset);
// out = epilogue(a . w^T) with a [M, K] and w [N, K] fp16, on the CTA-pair / single-CTA
// kind::f16 tile kernels.  16-byte aligned operands and row strides, K % 8 == 0; `ep` as
// for the FP8 scaled epilogue.
int gemm_f16_scaled(const void* a, int64_t lda, const void* w, int64_t ldw, int64_t M, int64_t N,
                    int64_t K, const EpiArgs& ep, cudaStream_t st);

}  // namespace host
}  // namespace b200q
