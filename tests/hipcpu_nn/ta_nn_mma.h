// TEST INFRASTRUCTURE -- takes the place of csrc/nn/ta_nn_mma.h when the kernels of libta_nn.so are compiled for the host
// (build.py): the matrix instructions' arithmetic and layouts in plain C++, lane by lane, on tests/hipcpu's stand-in.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

static inline int __popcll(unsigned long long v) { return __builtin_popcountll(v); }
static inline int atomicAdd(int* p, int v) { const int old = *p; *p = old + v; return old; }
static inline unsigned atomicOr(unsigned* p, unsigned v) { const unsigned old = *p; *p = old | v; return old; }

namespace ta_nn_host {
// one slot per lane of a workgroup; a workgroup runs on one OS thread
inline thread_local unsigned char slots[16][64][64];
char* lds();                                             // the workgroup's dynamic LDS (160 KB)
inline void wave_sync() { (void)hipcpu::shfl_xor(0.0f, 0, 64); }
template <class V> inline void put(const V& v, int at = 0) {
    memcpy(&slots[threadIdx.x >> 6][threadIdx.x & 63][at], &v, sizeof(V));
}
template <class V> inline V get(int lane, int at = 0) {
    V v;
    memcpy(&v, &slots[threadIdx.x >> 6][lane][at], sizeof(V));
    return v;
}
}  // namespace ta_nn_host

static inline unsigned long long __ballot(int pred) {
    ta_nn_host::put(pred);
    ta_nn_host::wave_sync();
    unsigned long long r = 0;
    for (int l = 0; l < 64; ++l) r |= static_cast<unsigned long long>(ta_nn_host::get<int>(l) != 0) << l;
    ta_nn_host::wave_sync();
    return r;
}

namespace ta_nn {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned short u16x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

template <class V> inline V lane_exchange(V v, int mask) {
    ta_nn_host::put(v);
    ta_nn_host::wave_sync();
    const V r = ta_nn_host::get<V>((threadIdx.x & 63) ^ mask);
    ta_nn_host::wave_sync();
    return r;
}
template <class V, class Op> inline V reduce_rows(V v, Op op) {
    v = op(v, lane_exchange(v, 16));
    return op(v, lane_exchange(v, 32));
}
template <class V, class Op> inline V reduce_wave(V v, Op op) {
    for (int mask = 1; mask < 16; mask <<= 1) v = op(v, lane_exchange(v, mask));
    return reduce_rows(v, op);
}
inline void forget(u32x4&) {}
inline void order_memory() {}
inline void wave_lds_order() { ta_nn_host::wave_sync(); }
inline float max_nan(float a, float b) { return a != a || b != b ? NAN : a > b ? a : b; }
inline float exp2_hw(float x) { return x < -126.0f ? 0.0f : exp2f(x); }

template <class Row, int PER> inline f32x4 mfma_any(Row a, Row b, f32x4 acc) {
    ta_nn_host::put(a, 0);
    ta_nn_host::put(b, 32);
    ta_nn_host::wave_sync();
    const int lane = threadIdx.x & 63, col = lane & 15, first = 4 * (lane >> 4);
    for (int r = 0; r < 4; ++r) {
        double sum = acc[r];
        for (int k = 0; k < 4; ++k) {
            const Row x = ta_nn_host::get<Row>(16 * k + first + r, 0), y = ta_nn_host::get<Row>(16 * k + col, 32);
            if constexpr (PER == 1) sum += static_cast<double>(x) * static_cast<double>(y);
            else for (int i = 0; i < PER; ++i) sum += static_cast<double>(static_cast<float>(x[i])) * static_cast<double>(static_cast<float>(y[i]));
        }
        acc[r] = static_cast<float>(sum);
    }
    ta_nn_host::wave_sync();
    return acc;
}
inline u16x4 read_transposed(const unsigned short* p) {
    ta_nn_host::put(p);
    ta_nn_host::wave_sync();
    const int lane = threadIdx.x & 63, group = lane & 48, c = lane & 15;
    u16x4 r;
    for (int i = 0; i < 4; ++i) r[i] = ta_nn_host::get<const unsigned short*>(group + 4 * i + c / 4)[c % 4];
    ta_nn_host::wave_sync();
    return r;
}
inline f32x4 mfma(float a, float b, f32x4 c) { return mfma_any<float, 1>(a, b, c); }
inline f32x4 mfma(half8 a, half8 b, f32x4 c) { return mfma_any<half8, 8>(a, b, c); }
inline f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) { return mfma_any<bf16x8, 8>(a, b, c); }

}  // namespace ta_nn
