// What the attention kernels share: arguments, staging of a tile through LDS, fragments, the bias and the mask of a score.
//
//     s_ij = scale q_i . k_j + table[bucket(i, j)][head] + mask_ij          over the keys j that query i sees
//     p_ij = exp(s_ij - max_j s_ij) / sum_j exp(...)                        o_i = sum_j p_ij v_j
//
// Every kernel keeps one side -- the "columns", 16 to a wave -- in registers and streams the other -- the "rows", 64 to a
// tile -- through LDS.  It computes D = rows x columns, so a lane holds four consecutive rows of ONE column: maxima, sums and
// rescaling are per lane, and D is by itself the B operand of the next product, which contracts over the rows
// (O^T = V^T P^T and its like): probabilities never leave the registers.  For that product fp32 visits rows 4 g + r in step
// r; 16-bit types visit rows 4 g + i and 16 + 4 g + i of 32 in one step.
#pragma once
#include "ta_nn_common.h"

namespace ta_nn {

struct AttentionArgs : ta_nn_attention_args {
    int bias_in_lds;                                     // the bias values of a block's heads are staged in LDS
    float* delta;                                        // [batch][heads][m]: sum_d out grad
    float* partial;                                      // sums of score gradients, per batch chunk
    int chunks;
};

template <class T> struct Frag;
template <> struct Frag<float> {
    static constexpr int D = 16;                         // dims of a row fragment
    static constexpr int K = 16;                         // rows of a transposed fragment
    static constexpr int VE = 4;
    typedef f32x4 Row;
};
template <> struct Frag<bf16> {
    static constexpr int D = 32, K = 32, VE = 8;
    typedef bf16x8 Row;
};
template <> struct Frag<fp16> {
    static constexpr int D = 32, K = 32, VE = 8;
    typedef half8 Row;
};

__device__ __forceinline__ f32x4 mma_row(f32x4 a, f32x4 b, f32x4 c) {      // 16 dims in four steps; dim 4 g + i in step i
    c = mfma(a.x, b.x, c);
    c = mfma(a.y, b.y, c);
    c = mfma(a.z, b.z, c);
    return mfma(a.w, b.w, c);
}
__device__ __forceinline__ f32x4 mma_row(bf16x8 a, bf16x8 b, f32x4 c) { return mfma(a, b, c); }
__device__ __forceinline__ f32x4 mma_row(half8 a, half8 b, f32x4 c) { return mfma(a, b, c); }

// LDS tile: ROWS rows of DP elements, rows 16 bytes longer than they need to be so that the 16 rows of a fragment start in
// different banks
template <class T, int DP> struct Tile {
    static constexpr int LD = DP + 16 / static_cast<int>(sizeof(T));
    static constexpr int LOADS(int rows, int threads) { return (rows * DP / Frag<T>::VE + threads - 1) / threads; }
};

// ROWS x DP elements from memory into registers (zero past `rows` and `dim`); `put` moves them to LDS one barrier later.
// row_at(r): the pointer to row r (called for r < rows only)
template <class T, int DP, int ROWS, int THREADS> struct Staged {
    static constexpr int VE = Frag<T>::VE, PER_ROW = DP / VE, COUNT = (ROWS * PER_ROW + THREADS - 1) / THREADS;
    Vec<T> v[COUNT];
    template <class RowAt> __device__ __forceinline__ void load(RowAt row_at, int rows, int dim) {
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            const int e = static_cast<int>(threadIdx.x) + i * THREADS, r = e / PER_ROW, d = e % PER_ROW * VE;
            if ((ROWS * PER_ROW) % THREADS != 0 && e >= ROWS * PER_ROW) continue;
            v[i].raw = u32x4{0, 0, 0, 0};
            if (r < rows && d < dim) v[i] = load_part(row_at(r) + d, dim - d, 0u);
        }
    }
    __device__ __forceinline__ void put(T* lds) const {
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            const int e = static_cast<int>(threadIdx.x) + i * THREADS, r = e / PER_ROW, d = e % PER_ROW * VE;
            if ((ROWS * PER_ROW) % THREADS != 0 && e >= ROWS * PER_ROW) continue;
            *reinterpret_cast<Vec<T>*>(lds + r * Tile<T, DP>::LD + d) = v[i];
        }
    }
};

// row fragment `dc` of row `row` (= first row + lane & 15) of an LDS tile
template <class T, int DP> __device__ __forceinline__ typename Frag<T>::Row row_frag(const T* lds, int row, int dc, int g) {
    return *reinterpret_cast<const typename Frag<T>::Row*>(lds + row * Tile<T, DP>::LD + dc * Frag<T>::D + g * Frag<T>::VE);
}

// the same of a row in memory, for the side that stays in registers
template <class T> __device__ __forceinline__ typename Frag<T>::Row row_frag_global(const T* p, int dim, int dc, int g, bool valid) {
    const int d = dc * Frag<T>::D + g * Frag<T>::VE;
    Vec<T> v;
    v.raw = u32x4{0, 0, 0, 0};
    if (valid && d < dim) v = load_part(p + d, dim - d, 0u);
    return __builtin_bit_cast(typename Frag<T>::Row, v);
}

__device__ __forceinline__ bf16x8 pack8(f32x4 a, f32x4 b, bf16) {
    return bf16x8{static_cast<__bf16>(a.x), static_cast<__bf16>(a.y), static_cast<__bf16>(a.z), static_cast<__bf16>(a.w),
                  static_cast<__bf16>(b.x), static_cast<__bf16>(b.y), static_cast<__bf16>(b.z), static_cast<__bf16>(b.w)};
}
__device__ __forceinline__ half8 pack8(f32x4 a, f32x4 b, fp16) {
    return half8{static_cast<_Float16>(a.x), static_cast<_Float16>(a.y), static_cast<_Float16>(a.z), static_cast<_Float16>(a.w),
                 static_cast<_Float16>(b.x), static_cast<_Float16>(b.y), static_cast<_Float16>(b.z), static_cast<_Float16>(b.w)};
}
// acc[q][dt] += (tile^T)[dim 16 dt + ..][row] * w[q][row][column], over the 64 rows; w: the D registers of the score tiles.
// 16-bit: the weights are rounded to the tensors' type, as the matrix instruction takes them (an error of half a step per
// weight, independent from weight to weight, where the result itself is rounded by as much).
template <int DP, int NQ, int SUBS, class T>
__device__ __forceinline__ void mma_transposed(const T* lds, const f32x4 (&w)[NQ][SUBS], f32x4 (&acc)[NQ][DP / 16], int c, int g) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int t = 0; t < SUBS; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float* p = lds + (16 * t + 4 * g + r) * Tile<T, DP>::LD + c;
#pragma unroll
                for (int dt = 0; dt < DP / 16; ++dt) {
                    const float a = p[16 * dt];
#pragma unroll
                    for (int q = 0; q < NQ; ++q) acc[q][dt] = mfma(a, w[q][t][r], acc[q][dt]);
                }
            }
    } else {
#pragma unroll
        for (int s = 0; s < SUBS / 2; ++s) {
            typename Frag<T>::Row b[NQ];
#pragma unroll
            for (int q = 0; q < NQ; ++q) b[q] = pack8(w[q][2 * s], w[q][2 * s + 1], T{});
#pragma unroll
            for (int dt = 0; dt < DP / 16; ++dt) {
                u16x8 a;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    a[i] = lds[(32 * s + (i & 4) * 4 + 4 * g + (i & 3)) * Tile<T, DP>::LD + 16 * dt + c].bits;
#pragma unroll
                for (int q = 0; q < NQ; ++q) acc[q][dt] = mfma(__builtin_bit_cast(typename Frag<T>::Row, a), b[q], acc[q][dt]);
            }
        }
    }
}

// ---- bias and mask of a score
// Values of the table for the heads [h0, h0 + count) in LDS: by bucket (pairs) or by distance.
__device__ __forceinline__ int bias_entries(const AttentionArgs& a) { return a.distances ? a.distances : a.buckets; }

__device__ __forceinline__ void stage_bias(const AttentionArgs& a, float* lds, int h0, int count, int threads) {
    const int entries = bias_entries(a);
    for (int e = threadIdx.x; e < entries * count; e += threads) {
        const int h = e / entries, i = e % entries;
        const int bucket = a.distances ? static_cast<const int*>(a.index)[i] : i;
        lds[e] = load_as_float(a.table, static_cast<int64_t>(bucket) * a.heads + h0 + h, a.table_dtype);
    }
}

// the table's values for one head, staged or in memory
struct Bias {
    const AttentionArgs& a;
    const float* lds;
    int head;
    __device__ __forceinline__ float value(int entry) const {
        if (lds) return lds[entry];
        const int bucket = a.distances ? static_cast<const int*>(a.index)[entry] : entry;
        return load_as_float(a.table, static_cast<int64_t>(bucket) * a.heads + head, a.table_dtype);
    }
    __device__ __forceinline__ float clamped(int entry) const {
        return value(entry < 0 ? 0 : entry >= a.distances ? a.distances - 1 : entry);
    }
};

// positions may lie anywhere: clamped to where adding a token's number (below 2^30) can neither overflow nor change the answer
__device__ __forceinline__ int clamp_entry(int64_t e) {
    return static_cast<int>(max(-(static_cast<int64_t>(1) << 30), min(e, static_cast<int64_t>(0x7FFFFFFF))));
}
__device__ __forceinline__ int clamp_token(int64_t t) {
    return static_cast<int>(max(static_cast<int64_t>(-1), min(t, static_cast<int64_t>(1) << 30)));
}

// a mask entry as what is added to the score.  The lowest finite values are raised to -1e38: nothing changes (a score vanishes
// beside either), and neither it nor its product with log2 e overflows.  -inf stays.
__device__ __forceinline__ float mask_value(const AttentionArgs& a, int64_t at) {
    if (a.mask_kind == TA_NN_MASK_BOOL) return static_cast<const unsigned char*>(a.mask)[at] ? 0.0f : -INFINITY;
    const float f = load_as_float(a.mask, at, a.mask_kind - TA_NN_MASK_F32);
    return f < -1e38f && f != -INFINITY ? -1e38f : f;
}
__device__ __forceinline__ float masked(float s, float add) { return add == -INFINITY ? -INFINITY : s + add; }   // whatever s is


// scale, bias and mask of the scores of one column (a query) against keys j0 + 16 t + 4 g + r
__device__ __forceinline__ void score_column(const AttentionArgs& a, const Bias& bias, int64_t b, int query, int start, int j0, int keys,
                                             int g, f32x4 (&s)[4]) {
    const int64_t position = static_cast<int64_t>(start) + query;
    const int from = clamp_entry(-position - a.first);
    const int last = a.causal ? min(clamp_token(position), keys - 1) : keys - 1;
    const int64_t mask_row = a.mask_kind ? b % a.mask_period * a.mask_sb + bias.head * a.mask_sh + query * a.mask_sm : 0;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int j = j0 + 16 * t + 4 * g;
        u16x4 bucket{0, 0, 0, 0};
        if (a.distances == 0 && j < a.n)
            bucket = *reinterpret_cast<const u16x4*>(static_cast<const unsigned short*>(a.index) + query * a.index_stride + j);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float f = -INFINITY;
            if (j + r <= last) {
                f = s[t][r] * a.scale + (a.distances ? bias.clamped(j + r + from) : bias.value(bucket[r]));
                if (a.mask_kind) f = masked(f, mask_value(a, mask_row + (j + r) * a.mask_sn));
            }
            s[t][r] = f;
        }
    }
}

// the same for one column that is a key (one in use) against queries i0 + 16 t + 4 g + r
__device__ __forceinline__ void score_row(const AttentionArgs& a, const Bias& bias, int64_t b, int key, int start, int i0, bool used, int g,
                                          f32x4 (&s)[4]) {
    const int64_t lead = static_cast<int64_t>(key) - start;
    const int from = clamp_entry(lead - a.first);
    const int first = a.causal ? clamp_token(lead) : 0;
    const int64_t mask_at = a.mask_kind ? b % a.mask_period * a.mask_sb + bias.head * a.mask_sh + key * a.mask_sn : 0;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int i = i0 + 16 * t + 4 * g;
        u16x4 bucket{0, 0, 0, 0};
        if (a.distances == 0 && i < a.m && used)
            bucket = *reinterpret_cast<const u16x4*>(static_cast<const unsigned short*>(a.index_t) + key * a.index_t_stride + i);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float f = -INFINITY;
            if (used && i + r < a.m && i + r >= first) {
                f = s[t][r] * a.scale + (a.distances ? bias.clamped(from - i - r) : bias.value(bucket[r]));
                if (a.mask_kind) f = masked(f, mask_value(a, mask_at + (i + r) * a.mask_sm));
            }
            s[t][r] = f;
        }
    }
}

// dims 16 t + 4 g .. + 3 of a column, times f
template <class T, int DP> __device__ __forceinline__ void store_column(T* p, const f32x4 (&o)[DP / 16], float f, int dim, int g) {
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) {
        const int d = 16 * t + 4 * g;
        T v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = from_float<T>(o[t][r] * f);
        if (d + 4 <= dim) {
            __builtin_memcpy(p + d, v, sizeof(v));
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (d + r < dim) p[d + r] = v[r];
        }
    }
}

// LDS for the bias values of the heads that `columns` consecutive columns can span; 0, and the kernels read the table from
// memory, where that is more than 24 KB
inline size_t bias_lds_bytes(AttentionArgs& a, int64_t columns) {
    const int64_t group = a.heads / a.kv_heads;
    int64_t spans = (columns - 1) / a.m + 2;
    if (spans > group) spans = group;
    const int64_t bytes = spans * (a.distances ? a.distances : a.buckets) * 4;
    a.bias_in_lds = bytes <= 24 * 1024;
    return a.bias_in_lds ? static_cast<size_t>(bytes) : 0;
}

int check_attention(const ta_nn_attention_args* args, AttentionArgs& a);
int64_t workspace_floats(const ta_nn_attention_args& a, bool backward);

}  // namespace ta_nn

#define TA_NN_DIMS(call)                                                  \
    if (ta_nn_dim <= 32) { constexpr int DP = 32; return call; }          \
    if (ta_nn_dim <= 64) { constexpr int DP = 64; return call; }          \
    if (ta_nn_dim <= 96) { constexpr int DP = 96; return call; }          \
    constexpr int DP = 128;                                               \
    return call

#define TA_NN_BY_TYPE_AND_DIM(dtype, dim_, call)                          \
    const int ta_nn_dim = dim_;                                           \
    if (dtype == TA_NN_F32) { using T = float; TA_NN_DIMS(call); }        \
    if (dtype == TA_NN_BF16) { using T = ta_nn::bf16; TA_NN_DIMS(call); } \
    using T = ta_nn::fp16;                                                \
    TA_NN_DIMS(call)
