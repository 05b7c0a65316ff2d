// Numbers of the 8-bit decoder operators (sm_100a): e4m3 codes with one fp32 scale per
// group, shared by the kernels that write them (fp8_rows.cu, the gate/up epilogue of
// fp8_gemm.cu) and the one that reads them.
//
// A group of 128 values x has amax = max(max |x|, 2^-100), scale = amax / 448 and codes
// e4m3(x * (448 / amax)): 448 is the largest e4m3 value, so nothing saturates beyond the
// last rounding, and the floor keeps 448 / amax finite for a group of zeros (its codes are
// 0). A NaN makes the scale NaN and an infinity makes it infinite: either way every
// product with the group is non-finite, as it would be with the values themselves.
#pragma once

#include <cuda_fp8.h>

#include "dkv_common.cuh"

namespace dkv {

constexpr int kFp8Group = 128;        // columns per scale (and weight rows per block)
constexpr float kFp8Max = 448.f;      // largest e4m3 value
constexpr float kFp8Floor = 0x1p-100f;

// max of |.| that keeps a NaN (fmaxf drops it).
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Two values to e4m3 codes (round to nearest even, saturating; a NaN stays NaN), lo in
// the low byte.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  return e4m3x2(a, b) | (e4m3x2(c, d) << 16);
}

// 16 bf16 (two 16-byte words) to fp32.
__device__ __forceinline__ void unpack16(uint4 a, uint4 b, float* x) {
  x[0] = bf16_lo(a.x); x[1] = bf16_hi(a.x);
  x[2] = bf16_lo(a.y); x[3] = bf16_hi(a.y);
  x[4] = bf16_lo(a.z); x[5] = bf16_hi(a.z);
  x[6] = bf16_lo(a.w); x[7] = bf16_hi(a.w);
  x[8] = bf16_lo(b.x); x[9] = bf16_hi(b.x);
  x[10] = bf16_lo(b.y); x[11] = bf16_hi(b.y);
  x[12] = bf16_lo(b.z); x[13] = bf16_hi(b.z);
  x[14] = bf16_lo(b.w); x[15] = bf16_hi(b.w);
}

__device__ __forceinline__ float amax16(const float* x) {
  float m = fabsf(x[0]);
#pragma unroll
  for (int j = 1; j < 16; ++j) m = max_nan(m, fabsf(x[j]));
  return m;
}

// 16 values times `inverse` as 16 e4m3 codes.
__device__ __forceinline__ uint4 codes16(const float* x, float inverse) {
  float v[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) v[j] = __fmul_rn(x[j], inverse);
  return make_uint4(e4m3x4(v[0], v[1], v[2], v[3]), e4m3x4(v[4], v[5], v[6], v[7]),
                    e4m3x4(v[8], v[9], v[10], v[11]), e4m3x4(v[12], v[13], v[14], v[15]));
}

}  // namespace dkv
