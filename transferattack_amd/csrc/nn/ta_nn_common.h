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

// One 16-byte access.  16-bit elements stay packed, two to a register, and are unpacked where they are used: as an array of
// elements each would take a register of its own.
template <class T> struct alignas(16) Vec {
    static constexpr int N = 16 / sizeof(T);
    u32x4 raw;
};
__device__ __forceinline__ float get(const Vec<float>& v, int i) { return __uint_as_float(v.raw[i]); }
__device__ __forceinline__ float get(const Vec<bf16>& v, int i) {
    return __uint_as_float(i & 1 ? v.raw[i >> 1] & 0xFFFF0000u : v.raw[i >> 1] << 16);
}
__device__ __forceinline__ float get(const Vec<fp16>& v, int i) {
    return to_float(fp16{static_cast<unsigned short>(i & 1 ? v.raw[i >> 1] >> 16 : v.raw[i >> 1])});
}
template <class T> __device__ __forceinline__ void set_bits(Vec<T>& v, int i, unsigned bits) {      // of one element
    if constexpr (sizeof(T) == 4) v.raw[i] = bits;
    else v.raw[i >> 1] = i & 1 ? (v.raw[i >> 1] & 0xFFFFu) | bits << 16 : (v.raw[i >> 1] & 0xFFFF0000u) | bits;
}
// the same for an index known at run time only: no memory, no unrolled copies of what is done rarely
template <class T> __device__ __forceinline__ unsigned word_at(const Vec<T>& v, int w) {
    return w < 2 ? (w == 0 ? v.raw[0] : v.raw[1]) : (w == 2 ? v.raw[2] : v.raw[3]);
}
__device__ __forceinline__ float get_at(const Vec<float>& v, int i) { return __uint_as_float(word_at(v, i)); }
__device__ __forceinline__ float get_at(const Vec<bf16>& v, int i) {
    return __uint_as_float(i & 1 ? word_at(v, i >> 1) & 0xFFFF0000u : word_at(v, i >> 1) << 16);
}
__device__ __forceinline__ float get_at(const Vec<fp16>& v, int i) {
    return to_float(fp16{static_cast<unsigned short>(word_at(v, i >> 1) >> (i & 1) * 16)});
}
template <class T> __device__ __forceinline__ void set_bits_at(Vec<T>& v, int i, unsigned bits) {
    const int w = sizeof(T) == 4 ? i : i >> 1, by = sizeof(T) == 4 ? 0 : (i & 1) * 16;
    const unsigned keep = sizeof(T) == 4 ? 0u : 0xFFFF0000u >> by;
#pragma unroll
    for (int x = 0; x < 4; ++x) v.raw[x] = x == w ? (v.raw[x] & keep) | bits << by : v.raw[x];
}
__device__ __forceinline__ unsigned bits_of(float x) { return __float_as_uint(x); }
__device__ __forceinline__ unsigned bits_of(bf16 x) { return x.bits; }
__device__ __forceinline__ unsigned bits_of(fp16 x) { return x.bits; }
template <class T> __device__ __forceinline__ void set(Vec<T>& v, int i, T x) { set_bits(v, i, bits_of(x)); }
template <class T> __device__ __forceinline__ unsigned lowest_bits();      // -inf
template <> __device__ __forceinline__ unsigned lowest_bits<float>() { return 0xFF800000u; }
template <> __device__ __forceinline__ unsigned lowest_bits<bf16>() { return 0xFF80u; }
template <> __device__ __forceinline__ unsigned lowest_bits<fp16>() { return 0xFC00u; }
__device__ __forceinline__ Vec<float> pack(const float (&f)[4]) {
    return Vec<float>{u32x4{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])}};
}
template <class T> __device__ __forceinline__ Vec<T> pack(const float (&f)[8]) {
    Vec<T> v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v.raw[i] = bits_of(from_float<T>(f[2 * i])) | bits_of(from_float<T>(f[2 * i + 1])) << 16;
    return v;
}
template <class T> __device__ __forceinline__ Vec<T> pack(const float (&f)[4]) { return pack(f); }
// an access of 16 bytes at any element boundary (global memory takes unaligned accesses; only the speed differs)
template <class T> __device__ __forceinline__ Vec<T> load_vec(const T* p) {
    Vec<T> r;
    __builtin_memcpy(&r.raw, p, 16);
    return r;
}
// the same at a byte offset from an address the whole workgroup shares: one 32-bit register to a lane
template <class T> __device__ __forceinline__ Vec<T> load_at(const T* base, unsigned offset) {
    Vec<T> r;
    __builtin_memcpy(&r.raw, reinterpret_cast<const char*>(base) + offset, 16);
    return r;
}
template <class T> __device__ __forceinline__ void store_vec(T* p, const Vec<T>& r) { __builtin_memcpy(p, &r.raw, 16); }
template <class T> __device__ __forceinline__ T element(const Vec<T>& v, int i) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(v.raw[i]);
    else return T{static_cast<unsigned short>(i & 1 ? v.raw[i >> 1] >> 16 : v.raw[i >> 1])};
}
// a scalar of a runtime type: 0 fp32, 1 bf16, 2 fp16 (TA_NN_F32 ...)
__device__ __forceinline__ float load_as_float(const void* p, int64_t i, int dtype) {
    if (dtype == TA_NN_F32) return static_cast<const float*>(p)[i];
    if (dtype == TA_NN_BF16) return to_float(static_cast<const bf16*>(p)[i]);
    return to_float(static_cast<const fp16*>(p)[i]);
}

// ---- reductions: inside a wave as reduce_wave says, waves in index order; every lane ends with the result, always the same bits
struct Sum {
    template <class V> __device__ __forceinline__ V operator()(V a, V b) const { return a + b; }
};
struct Max {                                             // NaN wins
    __device__ __forceinline__ float operator()(float a, float b) const { return max_nan(a, b); }
    __device__ __forceinline__ double operator()(double a, double b) const { return (a > b || a != a) ? a : b; }
};
__device__ __forceinline__ bool wave_any(bool v) { return __ballot(v) != 0; }
template <class V> __device__ __forceinline__ V wave_sum(V v) { return reduce_wave(v, Sum{}); }
template <class V> __device__ __forceinline__ V wave_max(V v) { return reduce_wave(v, Max{}); }
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
    for (int w = 1; w < WAVES; ++w) t = Max{}(t, lds[w]);
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
