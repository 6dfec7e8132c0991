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
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
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

// Four rows of 16 16-bit elements of an LDS tile, transposed: lane c of each group of 16 gets element c of rows 0 .. 3.  Lane c
// passes the address of row c / 4, elements 4 (c % 4) .. + 3 of the group's four rows; groups are independent.
__device__ __forceinline__ u16x4 read_transposed(const unsigned short* p) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef short v4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(u16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4*)(p)));
#else
    return u16x4{0, 0, 0, 0};
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

// the same value, as far as the compiler is concerned another one: what was computed from it before is not kept for later
__device__ __forceinline__ void forget(u32x4& v) {
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("" : "+v"(v));
#endif
}

// loads and stores are not moved across
__device__ __forceinline__ void order_memory() {
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("" ::: "memory");
#endif
}

// a wave's own LDS writes are seen by its later reads: the hardware does them in order, the compiler has to as well
__device__ __forceinline__ void wave_lds_order() {
#if defined(__HIP_DEVICE_COMPILE__)
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#endif
}

// the larger one, NaN if either is one
__device__ __forceinline__ float max_nan(float a, float b) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_elementwise_maximum(a, b);
#else
    return a;
#endif
}

// ---- all 64 lanes reduced to one value every lane has, in a fixed order, without LDS: within 16 lanes by DPP moves (the
// neighbour, the other pair, then mirror images: what they meet is uniform by then), across by the row swaps of gfx950
template <int CTRL, class V> __device__ __forceinline__ V dpp(V v) {
#if defined(__HIP_DEVICE_COMPILE__)
    if constexpr (sizeof(V) == 4) {
        return __builtin_bit_cast(V, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
    } else {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const unsigned lo = static_cast<unsigned>(__builtin_amdgcn_mov_dpp(static_cast<int>(u), CTRL, 0xF, 0xF, true));
        const unsigned hi = static_cast<unsigned>(__builtin_amdgcn_mov_dpp(static_cast<int>(u >> 32), CTRL, 0xF, 0xF, true));
        return __builtin_bit_cast(V, static_cast<uint64_t>(hi) << 32 | lo);
    }
#else
    return v;
#endif
}
// op(v of this row of 16 -- or half of 32 -- and of its neighbour), the same for both: rows 0 and 1, 2 and 3 / halves 0 and 1
template <bool HALVES, class V, class Op> __device__ __forceinline__ V with_neighbour(V v, Op op) {
#if defined(__HIP_DEVICE_COMPILE__)
    auto swap = [](unsigned x, unsigned (&r)[2]) {
        const auto both = HALVES ? __builtin_amdgcn_permlane32_swap(x, x, false, false) : __builtin_amdgcn_permlane16_swap(x, x, false, false);
        r[0] = both[0];
        r[1] = both[1];
    };
    if constexpr (sizeof(V) == 4) {
        unsigned r[2];
        swap(__builtin_bit_cast(unsigned, v), r);
        return op(__builtin_bit_cast(V, r[0]), __builtin_bit_cast(V, r[1]));
    } else {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        unsigned lo[2], hi[2];
        swap(static_cast<unsigned>(u), lo);
        swap(static_cast<unsigned>(u >> 32), hi);
        return op(__builtin_bit_cast(V, static_cast<uint64_t>(hi[0]) << 32 | lo[0]), __builtin_bit_cast(V, static_cast<uint64_t>(hi[1]) << 32 | lo[1]));
    }
#else
    return v;
#endif
}
template <class V, class Op> __device__ __forceinline__ V reduce_rows(V v, Op op) {       // across the four rows of 16 lanes only
    return with_neighbour<true>(with_neighbour<false>(v, op), op);
}
template <class V, class Op> __device__ __forceinline__ V reduce_wave(V v, Op op) {
    v = op(v, dpp<0xB1>(v));
    v = op(v, dpp<0x4E>(v));
    v = op(v, dpp<0x141>(v));
    v = op(v, dpp<0x140>(v));
    return reduce_rows(v, op);
}

}  // namespace ta_nn
