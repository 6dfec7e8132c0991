// Shared by the kernels of libta_nn.so: errors at the C boundary, element types, reductions in a fixed order.
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include "../../../include/ta_nn.h"
#include "ta_nn_mma.h"

namespace ta_nn {

void set_error(const char* fmt, ...);
int check_launch(const char* what);

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// ---- element types: T is what memory holds, arithmetic is fp32 (or fp64)
struct bf16 { unsigned short bits; };
struct fp16 { unsigned short bits; };

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(bf16 x) { return __uint_as_float(static_cast<unsigned>(x.bits) << 16); }
__device__ __forceinline__ float to_float(fp16 x) { return static_cast<float>(__builtin_bit_cast(_Float16, x.bits)); }
template <class T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
// round to nearest even, NaN kept
template <> __device__ __forceinline__ bf16 from_float<bf16>(float x) { return bf16{__builtin_bit_cast(unsigned short, static_cast<__bf16>(x))}; }
template <> __device__ __forceinline__ fp16 from_float<fp16>(float x) { return fp16{__builtin_bit_cast(unsigned short, static_cast<_Float16>(x))}; }

template <class T> struct alignas(16) Vec {               // one 16-byte access
    static constexpr int N = 16 / sizeof(T);
    T v[N];
};
// an access of 16 bytes at any element boundary (global memory takes unaligned accesses; only the speed differs)
template <class T> __device__ __forceinline__ Vec<T> load_vec(const T* p) {
    Vec<T> r;
    __builtin_memcpy(&r, p, 16);
    return r;
}
template <class T> __device__ __forceinline__ void store_vec(T* p, const Vec<T>& r) { __builtin_memcpy(p, &r, 16); }

// a scalar of a runtime type: 0 fp32, 1 bf16, 2 fp16 (TA_NN_F32 ...)
__device__ __forceinline__ float load_as_float(const void* p, int64_t i, int dtype) {
    if (dtype == TA_NN_F32) return static_cast<const float*>(p)[i];
    if (dtype == TA_NN_BF16) return to_float(static_cast<const bf16*>(p)[i]);
    return to_float(static_cast<const fp16*>(p)[i]);
}

// ---- reductions: butterflies inside a wave, waves in index order; every lane ends with the result, always the same bits
template <class V> __device__ __forceinline__ V wave_sum(V v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += lane_xor(v, off);
    return v;
}
template <class V> __device__ __forceinline__ V wave_max(V v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const V o = lane_xor(v, off);
        v = (v > o || v != v) ? v : o;                    // NaN wins
    }
    return v;
}
// `lds`: one V per wave; the barriers make it free for the next call
template <int WAVES, class V> __device__ __forceinline__ V block_sum(V v, V* lds) {
    v = wave_sum(v);
    if (WAVES == 1) return v;
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    V t = lds[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) t += lds[w];
    __syncthreads();
    return t;
}
template <int WAVES, class V> __device__ __forceinline__ V block_max(V v, V* lds) {
    v = wave_max(v);
    if (WAVES == 1) return v;
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    V t = lds[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) t = (t > lds[w] || t != t) ? t : lds[w];
    __syncthreads();
    return t;
}

constexpr float kLog2e = 1.4426950408889634f;

}  // namespace ta_nn

#define TA_NN_REQUIRE(cond, ...)              \
    do {                                      \
        if (!(cond)) {                        \
            ta_nn::set_error(__VA_ARGS__);    \
            return TA_NN_EINVAL;              \
        }                                     \
    } while (0)
