// Matrix-core products, exponential and cross-lane moves the kernels of libta_nn.so are written in (gfx950, wave64).
//
// Layouts of one wave, lane l, c = l & 15, g = l >> 4 (D[16 x 16] = C + A[16 x K] B[K x 16]):
//   fp32    K = 4   A[c][g], B[g][c]                                one value per lane and operand
//   16-bit  K = 32  A[c][8 g + i], B[8 g + i][c], i = 0..7          eight values per lane and operand
//   C, D            D[4 g + r][c], r = 0..3                         four fp32 per lane
// A contraction may visit its K indices in any order as long as both operands use the same one: that is what lets the D of
// one product be the B of the next without leaving its registers (see attention.h).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ta_nn {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned short u16x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4 mfma(float a, float b, f32x4 c) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
#else
    return c;                                             // hipcc's host pass only parses this function
#endif
}
__device__ __forceinline__ f32x4 mfma(half8 a, half8 b, f32x4 c) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
#else
    return c;
#endif
}
__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
#else
    return c;
#endif
}

// 2^x by the hardware instruction (about 1 ulp; results below 2^-126 become 0), log2 likewise
__device__ __forceinline__ float exp2_hw(float x) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_exp2f(x);
#else
    return x;
#endif
}

__device__ __forceinline__ float lane_xor(float v, int mask) { return __shfl_xor(v, mask, 64); }
__device__ __forceinline__ int lane_xor(int v, int mask) { return __shfl_xor(v, mask, 64); }
__device__ __forceinline__ double lane_xor(double v, int mask) { return __shfl_xor(v, mask, 64); }

}  // namespace ta_nn
