// What the attention kernels share: arguments, staging of a tile through LDS, fragments, the bias and the mask of a score.
//
//     s_ij = scale q_i . k_j + table[bucket(i, j)][head] + mask_ij          over the keys j that query i sees
//     p_ij = exp(s_ij - max_j s_ij) / sum_j exp(...)                        o_i = sum_j p_ij v_j
//
// Every kernel keeps one side -- the "columns", 16 or 32 to a wave -- in registers and streams the other -- the "rows", 64 or
// 32 to a tile -- through LDS.  It computes D = rows x columns, so a lane holds four consecutive rows of ONE column: maxima, sums and
// rescaling are per lane, and D is by itself the B operand of the next product, which contracts over the rows
// (O^T = V^T P^T and its like): probabilities never leave the registers.  For that product fp32 visits rows 4 g + r in step
// r; 16-bit types visit rows 4 g + i and 16 + 4 g + i of 32 in one step.
#pragma once
#include "ta_nn_common.h"

namespace ta_nn {

struct AttentionArgs : ta_nn_attention_args {
    int bias_in_lds;                                     // the bias values of a block's heads are staged in LDS
    float* delta;                                        // [batch][heads][m]: sum_j p dp
    float* partial;                                      // sums of score gradients, per batch chunk
    float* far;                                          // distances: [batch][heads][64 queries][2] sums past either end
    float* by_distance;                                  // distances: [heads][64 (tile difference)][128] sums of the near tiles
    int chunks;
};

template <class T> struct Frag;
template <> struct Frag<float> {
    static constexpr int D = 16;                         // dims of a row fragment
    static constexpr int K = 16;                         // rows of a transposed fragment
    static constexpr int VE = 4;
    static constexpr bool NARROW = false;
    typedef f32x4 Row;
};
template <> struct Frag<bf16> {
    static constexpr int D = 32, K = 32, VE = 8;
    static constexpr bool NARROW = false;
    typedef bf16x8 Row;
};
template <> struct Frag<fp16> {
    static constexpr int D = 32, K = 32, VE = 8;
    static constexpr bool NARROW = true;                 // the range of fp32 does not fit
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

// rows of a tile over 16: as many as leave the accumulators their registers
template <int DP> constexpr int kSubs = DP <= 64 ? 4 : 2;

// Elements between rows of an LDS tile: 16-bit rows start 8 of the 64 banks further on than a multiple of them, so that what reads
// a tile transposed -- 16 lanes four rows of 32 bytes -- meets no bank twice; what reads it by rows (16 lanes a row each, 16 bytes)
// meets each twice.  With 4 banks instead, the other way round: 8191 keys in fp16 507 us (455 with 8), 1023 padded tokens in bf16
// forward 64, backward 81 + 105 us (59, 71 + 91 with 8).
template <class T, int DP> struct Tile {
    static constexpr int LD = DP + (sizeof(T) == 2 ? 16 : 4);
};

// ROWS x DP elements from memory into registers (zero past `rows` and `dim`, a multiple of a vector); `put` moves them to LDS one
// barrier later.  `base`: row 0, the same for the workgroup; a row is less than 2^23 elements behind the last
template <class T, int DP, int ROWS, int THREADS> struct Staged {
    static constexpr int VE = Frag<T>::VE, PER_ROW = DP / VE, COUNT = (ROWS * PER_ROW + THREADS - 1) / THREADS;
    __device__ __forceinline__ static bool mine(int e) { return (ROWS * PER_ROW) % THREADS == 0 || e < ROWS * PER_ROW; }
    Vec<T> v[COUNT];
    __device__ __forceinline__ void load(const T* base, int64_t stride, int rows, int dim) {
        const unsigned step = static_cast<unsigned>(stride);
        const bool whole = rows >= ROWS && dim == DP;
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            const int e = static_cast<int>(threadIdx.x) + i * THREADS, r = e / PER_ROW, d = e % PER_ROW * VE;
            const unsigned offset = (r * step + d) * static_cast<unsigned>(sizeof(T));
            if (whole) {
                if (mine(e)) v[i] = load_at(base, offset);
            } else {
                v[i].raw = u32x4{0, 0, 0, 0};
                if (mine(e) && r < rows && d < dim) v[i] = load_at(base, offset);
            }
        }
    }
    __device__ __forceinline__ void put(T* lds) const {
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            const int e = static_cast<int>(threadIdx.x) + i * THREADS, r = e / PER_ROW, d = e % PER_ROW * VE;
            if (mine(e)) *reinterpret_cast<Vec<T>*>(lds + r * Tile<T, DP>::LD + d) = v[i];
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
    if (valid && d < dim) v = load_vec(p + d);
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
// ---- fp16's range: 11 bits from 2^-14 up to 65504.  Probabilities are multiplied by 2^kLift before they are rounded (so down to 2^-26
// of 1 keep their bits, and even scores that the passes make 2.7 apart do not overflow), score gradients, which may have any size, by a
// power of two for each column that brings the largest so far to 2^11 .. 2^15.  All exact, and taken out of the sums again.  It costs
// the queries' and the keys' kernel some 10 % each (8 x 12 x 1023 padded tokens of 64, step in fp16 320 us; bf16 281).
template <class T> constexpr bool kNarrow = Frag<T>::NARROW;
template <class T> constexpr int kLift = kNarrow<T> ? 12 : 0;
template <int SUBS> __device__ __forceinline__ float peak_of(const f32x4 (&w)[SUBS]) {      // of a column, over its four lanes (NaN aside)
    float peak = 0.0f;
#pragma unroll
    for (int t = 0; t < SUBS; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) peak = fmaxf(peak, fabsf(w[t][r]));
    return reduce_rows(peak, [](float u, float v) { return fmaxf(u, v); });
}
__device__ __forceinline__ float lift_of(float peak) {   // 2^x with peak 2^x in [2^11, 2^12); 2^127 for the smallest
    return __uint_as_float(static_cast<unsigned>(min(265 - static_cast<int>(__float_as_uint(peak) >> 23), 254)) << 23);
}
// w, a column's score gradients of one tile, times `up`; where that leaves the range, first `up` and the sums so far are made smaller
template <int SUBS, int DT> __device__ __forceinline__ void into_range(f32x4 (&w)[SUBS], f32x4 (&sums)[DT], float& up) {
    const float peak = peak_of(w);
    const bool leaves = peak * up > 32768.0f;
    if (wave_any(leaves)) {
        const float to = leaves ? lift_of(peak) : up, by = to / up;
        up = to;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) sums[dt] *= by;
    }
#pragma unroll
    for (int t = 0; t < SUBS; ++t) w[t] *= up;
}
constexpr float kMostLift = 0x1p127f;                    // `up` before the first tile: any number that is not 0 leaves the range

// ---- products that contract over a tile's rows
// The weights of one column for 16 SUBS rows, as the matrix instructions take them: fp32 as they are; for 16-bit tensors
// rounded to their type (an error of half a step per weight, independent from weight to weight, where the result itself is
// rounded by as much: results are 1.2 to 1.5 times as far off as their own rounding), or in two parts, which leaves nothing of that.
// Two parts where they cost little or few terms average little out: single tokens (148 us either way), windows (forward 90 us either
// way, backward 163 -> 202 us at 32 dims, 150 -> 166 at 64), backward of short rows.  One in the tiles of long rows, whose second
// products would cost: 8191 tokens of 128 in fp16 428 -> 530 us, and the backward's as attention_bwd.hip says.
template <class T, int SUBS> struct Weights {
    typename Frag<T>::Row v[SUBS / 2];                   // step s: rows 32 s + 4 g + i and 32 s + 16 + 4 g + i
    __device__ __forceinline__ void from_tiles(const f32x4 (&w)[SUBS]) {
#pragma unroll
        for (int s = 0; s < SUBS / 2; ++s) v[s] = pack8(w[2 * s], w[2 * s + 1], T{});
    }
    // what `rounded` lacks of w
    __device__ __forceinline__ void rest_of(const f32x4 (&w)[SUBS], const Weights& rounded) {
#pragma unroll
        for (int s = 0; s < SUBS / 2; ++s) {
            f32x4 lo = w[2 * s], hi = w[2 * s + 1];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                lo[i] -= static_cast<float>(rounded.v[s][i]);
                hi[i] -= static_cast<float>(rounded.v[s][4 + i]);
            }
            v[s] = pack8(lo, hi, T{});
        }
    }
};
template <int SUBS> struct Weights<float, SUBS> {
    f32x4 v[SUBS];
    __device__ __forceinline__ void from_tiles(const f32x4 (&w)[SUBS]) {
#pragma unroll
        for (int t = 0; t < SUBS; ++t) v[t] = w[t];
    }
};

// acc[q][dt] += (tile^T)[dim 16 dt + ..][row] * w[q][row][column], over the rows
template <int DP, int NQ, int SUBS, class T>
__device__ __forceinline__ void mma_transposed(const T* lds, const Weights<T, SUBS> (&w)[NQ], f32x4 (&acc)[NQ][DP / 16], int c, int g) {
    // operands of one group of products are read while the last group's are multiplied
    if constexpr (sizeof(T) == 4) {
        float a[2][4][DP / 16];
        auto read = [&](int t) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int dt = 0; dt < DP / 16; ++dt) a[t & 1][r][dt] = lds[(16 * t + 4 * g + r) * Tile<T, DP>::LD + c + 16 * dt];
        };
        read(0);
#pragma unroll
        for (int t = 0; t < SUBS; ++t) {
            if (t + 1 < SUBS) read(t + 1);
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int dt = 0; dt < DP / 16; ++dt)
#pragma unroll
                    for (int q = 0; q < NQ; ++q) acc[q][dt] = mfma(a[t & 1][r][dt], w[q].v[t][r], acc[q][dt]);
        }
    } else {
#pragma unroll
        for (int s = 0; s < SUBS / 2; ++s)
#pragma unroll
            for (int dt = 0; dt < DP / 16; ++dt) {
                const unsigned short* p = reinterpret_cast<const unsigned short*>(lds) + (32 * s + 4 * g + (c >> 2)) * Tile<T, DP>::LD
                                          + 16 * dt + 4 * (c & 3);
                const u16x4 lo = read_transposed(p), hi = read_transposed(p + 16 * Tile<T, DP>::LD);
                const u16x8 a = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                for (int q = 0; q < NQ; ++q) acc[q][dt] = mfma(__builtin_bit_cast(typename Frag<T>::Row, a), w[q].v[s], acc[q][dt]);
            }
    }
}
// the same, the first SPLIT of the weights in two 16-bit parts
template <int DP, int NQ, int SUBS, int SPLIT = 0, class T>
__device__ __forceinline__ void mma_transposed(const T* lds, const f32x4 (&w)[NQ][SUBS], f32x4 (&acc)[NQ][DP / 16], int c, int g) {
    Weights<T, SUBS> packed[NQ];
#pragma unroll
    for (int q = 0; q < NQ; ++q) packed[q].from_tiles(w[q]);
    if constexpr (SPLIT == 0 || sizeof(T) == 4) {
        mma_transposed<DP, NQ, SUBS, T>(lds, packed, acc, c, g);
    } else {
        Weights<T, SUBS> rest[SPLIT];
#pragma unroll
        for (int q = 0; q < SPLIT; ++q) rest[q].rest_of(w[q], packed[q]);
#pragma unroll
        for (int s = 0; s < SUBS / 2; ++s)
#pragma unroll
            for (int dt = 0; dt < DP / 16; ++dt) {
                const unsigned short* p = reinterpret_cast<const unsigned short*>(lds) + (32 * s + 4 * g + (c >> 2)) * Tile<T, DP>::LD
                                          + 16 * dt + 4 * (c & 3);
                const u16x4 lo = read_transposed(p), hi = read_transposed(p + 16 * Tile<T, DP>::LD);
                const u16x8 a = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                for (int q = 0; q < NQ; ++q) {
                    acc[q][dt] = mfma(__builtin_bit_cast(typename Frag<T>::Row, a), packed[q].v[s], acc[q][dt]);
                    if (q < SPLIT) acc[q][dt] = mfma(__builtin_bit_cast(typename Frag<T>::Row, a), rest[q].v[s], acc[q][dt]);
                }
            }
    }
}

// ---- bias and mask of a score
// Scores are kept times log2 e, so that the exponential is one instruction: s' = (scale log2 e) q.k + (table log2 e) + mask log2 e.
// The table's values for a block's heads stand in LDS, multiplied already, by bucket (pairs) or by distance; the latter with
// its ends repeated kPad times, so that a tile that touches the range at all needs no clamping.
constexpr int kPad = 192;                                // > 64 rows + 128 columns
__host__ __device__ inline int bias_entries(const AttentionArgs& a, int pad = kPad) { return a.distances ? a.distances + 2 * pad : a.buckets; }

__device__ __forceinline__ float table_value(const AttentionArgs& a, int entry, int head) {
    const int bucket = a.distances ? static_cast<const int*>(a.index)[entry] : entry;
    return load_as_float(a.table, static_cast<int64_t>(bucket) * a.heads + head, a.table_dtype) * kLog2e;
}
__device__ __forceinline__ int clamp_distance(const AttentionArgs& a, int e) { return e < 0 ? 0 : e >= a.distances ? a.distances - 1 : e; }

__device__ __forceinline__ void stage_bias(const AttentionArgs& a, float* lds, int h0, int count, int threads, int pad = kPad) {
    const int entries = bias_entries(a, pad);
    for (int e = threadIdx.x; e < entries * count; e += threads) {
        const int h = e / entries, i = e % entries;
        lds[e] = table_value(a, a.distances ? clamp_distance(a, i - pad) : i, h0 + h);
    }
}

// Positions may lie anywhere: clamped to where adding (a query's column, rows count up) or subtracting (a key's, they count down) a
// token's number, below 2^30 and a tile, can neither overflow nor change the answer; there are fewer than 2^29 distances.
__device__ __forceinline__ int clamp_query_entry(int64_t e) {
    return static_cast<int>(max(-(static_cast<int64_t>(1) << 30) - 64, min(e, static_cast<int64_t>(1) << 29)));
}
__device__ __forceinline__ int clamp_key_entry(int64_t e) {
    return static_cast<int>(max(-(static_cast<int64_t>(1) << 29), min(e, static_cast<int64_t>(0x7FFFFFFF))));
}
__device__ __forceinline__ int clamp_token(int64_t t) {
    return static_cast<int>(max(static_cast<int64_t>(-1), min(t, static_cast<int64_t>(1) << 30)));
}

// a mask entry as what is added to s'.  The lowest finite values are raised to -1e38: nothing changes (a score vanishes
// beside either), and neither it nor its product with log2 e overflows.  -inf stays.
__device__ __forceinline__ float mask_value(const AttentionArgs& a, int64_t at) {
    if (a.mask_kind == TA_NN_MASK_BOOL) return static_cast<const unsigned char*>(a.mask)[at] ? 0.0f : -INFINITY;
    const float f = load_as_float(a.mask, at, a.mask_kind - TA_NN_MASK_F32);
    return (f < -1e38f && f != -INFINITY ? -1e38f : f) * kLog2e;
}
__device__ __forceinline__ float masked(float s, float add) { return add == -INFINITY ? -INFINITY : s + add; }   // whatever s is

// What one lane knows of its column: a query against a tile of keys, or a key against a tile of queries.
struct Column {
    const float* bias;                                   // its head's values in LDS, or null: the table is read in memory
    int head;
    int from;                                            // distances: entry of row 0; rows count up (keys) or down (queries)
    int bound;                                           // rows seen: <= bound (keys), >= bound (queries)
    const unsigned short* pairs;                         // pairs: the column's row of the index
    int64_t mask;                                        // offset of row 0
};
__device__ __forceinline__ Column query_column(const AttentionArgs& a, const float* bias, int64_t b, int head, int query, int start,
                                               int keys) {
    const int64_t position = static_cast<int64_t>(start) + query;
    return Column{bias, head, clamp_query_entry(-position - a.first), a.causal ? min(clamp_token(position), keys - 1) : keys - 1,
                  a.distances ? nullptr : static_cast<const unsigned short*>(a.index) + query * a.index_stride,
                  a.mask_kind ? b % a.mask_period * a.mask_sb + head * a.mask_sh + query * a.mask_sm : 0};
}
__device__ __forceinline__ Column key_column(const AttentionArgs& a, const float* bias, int64_t b, int head, int key, int start) {
    const int64_t lead = static_cast<int64_t>(key) - start;
    return Column{bias, head, clamp_key_entry(lead - a.first), a.causal ? clamp_token(lead) : 0,
                  a.distances ? nullptr : static_cast<const unsigned short*>(a.index_t) + key * a.index_t_stride,
                  a.mask_kind ? b % a.mask_period * a.mask_sb + head * a.mask_sh + key * a.mask_sn : 0};
}

// How the scores of a tile are made.  A kernel is compiled for one of three Biases, so that none carries the registers of the
// others; within it every tile has one Kind, the same for the workgroup, and the loop's body is compiled for each, without branches.
enum Biases {
    kByDistance,                                         // distances in LDS, no mask
    kByPair,                                             // pairs, the table in LDS, no mask
    kAny                                                 // anything: masks, tables too large for LDS
};
enum Kind {
    kConstant,                                           // every pair is seen and lies past the same end of the distances
    kNear,                                               // every pair is seen; distances from LDS without clamping
    kSeen,                                               // every pair is seen; buckets from the index
    kEdge                                                // whatever there is
};

// Whether all distances of a tile of 64 keys lie past the same end (and which: -1 the first, 1 the last entry): the table's
// gradient then needs but the sum of the tile.  `low`, `high`: the lowest and the highest entry.
__host__ __device__ inline int far_end(const AttentionArgs& a, int64_t low, int64_t high) { return high <= 0 ? -1 : low >= a.distances - 1 ? 1 : 0; }
// the key tiles that are not so for queries i0 .. i0 + 63 (all sequences begin at the same position): the first, and how many at most
__host__ __device__ inline int near_tiles(const AttentionArgs& a) {
    const int tiles = (a.n + 63) / 64, most = (a.distances + 125) / 64 + 1;
    return tiles < most ? tiles : most;
}
__device__ __forceinline__ int first_near_tile(const AttentionArgs& a, int i0) {
    const int64_t after = static_cast<int64_t>(a.start) + i0 + a.first - 63;       // tile t is past the first entry if 64 t > after
    const int64_t t = after < 0 ? 0 : after / 64 + 1, last = (a.n + 63) / 64 - near_tiles(a);
    return static_cast<int>(t < last ? t : last);
}

// `low`, `high`: the lowest and the highest entry of the distances in the tile
template <int BIASES> __device__ __forceinline__ Kind tile_kind(const AttentionArgs& a, bool all_seen, bool one_head, int64_t low, int64_t high) {
    if (BIASES == kAny || !all_seen) return kEdge;
    if (BIASES == kByPair) return kSeen;
    if (high <= 0 || low >= a.distances - 1) return kConstant;
    return one_head ? kNear : kEdge;
}

template <int K> struct KindTag { static constexpr int kind = K; };
// body(KindTag<..>) for the tile's kind
template <int BIASES, class Body> __device__ __forceinline__ void by_kind(Kind kind, Body&& body) {
    if constexpr (BIASES == kByDistance) {
        if (kind == kConstant) return body(KindTag<kConstant>{});
        if (kind == kNear) return body(KindTag<kNear>{});
    }
    if constexpr (BIASES == kByPair) {
        if (kind == kSeen) return body(KindTag<kSeen>{});
    }
    body(KindTag<kEdge>{});
}

// s (q.k of rows row0 + 16 t + 4 g + r) -> s'; DOWN: rows are queries, whose distance falls as they rise
template <int BIASES, int KIND, bool DOWN, int PAD = kPad, int SUBS>
__device__ __forceinline__ void score_tile(const AttentionArgs& a, const Column& col, int row0, int g, f32x4 (&s)[SUBS]) {
    const float c = a.scale * kLog2e;
    if constexpr (KIND == kConstant) {
        const int at = DOWN ? col.from - row0 : col.from + row0;       // all on the same side of the range
        const float add = col.bias[PAD + (at < a.distances / 2 ? 0 : a.distances - 1)];
#pragma unroll
        for (int t = 0; t < SUBS; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[t][r] = fmaf(s[t][r], c, add);
    } else if constexpr (KIND == kNear) {
        const float* p = col.bias + PAD + (DOWN ? col.from - row0 - 4 * g : col.from + row0 + 4 * g);
#pragma unroll
        for (int t = 0; t < SUBS; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[t][r] = fmaf(s[t][r], c, p[DOWN ? -(16 * t + r) : 16 * t + r]);
    } else if constexpr (KIND == kSeen) {
#pragma unroll
        for (int t = 0; t < SUBS; ++t) {
            const u16x4 bucket = *reinterpret_cast<const u16x4*>(col.pairs + row0 + 16 * t + 4 * g);
#pragma unroll
            for (int r = 0; r < 4; ++r) s[t][r] = fmaf(s[t][r], c, col.bias[bucket[r]]);
        }
    } else {
        const int rows = DOWN ? a.m : a.n;
        const int64_t step = DOWN ? a.mask_sm : a.mask_sn;
        const bool distances = BIASES == kByDistance || (BIASES == kAny && a.distances != 0);
#pragma unroll
        for (int t = 0; t < SUBS; ++t) {
            if (BIASES == kAny) order_memory();          // not the loads of all at once: that takes their addresses' registers
            const int row = row0 + 16 * t + 4 * g;
            u16x4 bucket{0, 0, 0, 0};
            if (!distances && row < rows) bucket = *reinterpret_cast<const u16x4*>(col.pairs + row);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const bool seen = DOWN ? row + r < rows && row + r >= col.bound : row + r <= col.bound;
                int e = bucket[r];
                if (distances) e = clamp_distance(a, DOWN ? col.from - row - r : col.from + row + r);
                if constexpr (BIASES != kAny) {
                    const float f = fmaf(s[t][r], c, col.bias[distances ? e + PAD : e]);
                    s[t][r] = seen ? f : -INFINITY;
                } else {
                    float f = -INFINITY;
                    if (seen) {
                        f = fmaf(s[t][r], c, col.bias ? col.bias[distances ? e + PAD : e] : table_value(a, e, col.head));
                        if (a.mask_kind) f = masked(f, mask_value(a, col.mask + (row + r) * step));
                    }
                    s[t][r] = f;
                }
            }
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
        if (d < dim) __builtin_memcpy(p + d, v, sizeof(v));
    }
}

// The 127 diagonals of the workgroup's 64 x 64 tile of sums (column 16 wave + c: a query): number d + 63 is distance key - query
// = d.  `tile`: 64 x 65 floats of LDS that nobody uses any more; number 127 is 0.
__device__ __forceinline__ void store_diagonals(float* tile, const f32x4 (&sum)[4], int wave, int c, int g, float* out) {
    __syncthreads();
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) tile[(16 * t + 4 * g + r) * 65 + 16 * wave + c] = sum[t][r];
    __syncthreads();
    const int tid = threadIdx.x;
    if (tid < 128) {
        const int diagonal = tid - 63;
        float total = 0.0f;
        if (tid < 127)
            for (int i = max(0, -diagonal); i < 64 - max(0, diagonal); ++i) total += tile[(i + diagonal) * 65 + i];
        out[tid] = total;
    }
}

// LDS for the bias values of the heads that `columns` consecutive columns can span; 0, and the kernels read the table from
// memory, where that is more than 24 KB
inline size_t bias_lds_bytes(AttentionArgs& a, int64_t columns, int pad = kPad) {
    const int64_t group = a.heads / a.kv_heads;
    int64_t spans = (columns - 1) / a.m + 2;
    if (spans > group) spans = group;
    const int64_t bytes = spans * bias_entries(a, pad) * 4;
    a.bias_in_lds = bytes <= 24 * 1024;
    return a.bias_in_lds ? static_cast<size_t>(bytes) : 0;
}

inline int biases_of(const AttentionArgs& a) { return a.mask_kind || !a.bias_in_lds ? kAny : a.distances ? kByDistance : kByPair; }

// Many short sequences whose pairs are the same in all of them (or in every mask_period-th): attention_window.hip.
__host__ __device__ inline bool is_window(const ta_nn_attention_args& a) {
    return a.m <= 64 && a.n <= 64 && a.dim <= 64 && a.heads == a.kv_heads && !a.key_lengths && !a.query_start;
}
inline int window_periods(const ta_nn_attention_args& a) { return a.mask_kind ? a.mask_period : 1; }
// Parts to divide `count` sequences into, each a workgroup of `classes` kinds: what takes the fewest rounds of sequences when `slots`
// workgroups run at once (a part costs half a sequence by itself).
inline int balanced_parts(int64_t classes, int64_t count, int64_t slots) {
    int64_t best = 1, least = INT64_MAX;
    for (int64_t p = 1; p <= count && (p - 1) * classes < 4 * slots; ++p) {
        const int64_t cost = ceil_div(classes * p, slots) * (2 * ceil_div(count, p) + 1);
        if (cost < least) least = cost, best = p;
    }
    return static_cast<int>(best);
}
// Parts that the sequences of one head and mask are divided into, a workgroup each.
inline int window_parts(const ta_nn_attention_args& a, bool backward) {
    return balanced_parts(static_cast<int64_t>(window_periods(a)) * a.heads, ceil_div(a.batch, window_periods(a)),
                          backward ? 512 : 768);         // two and three to a CU, by the registers they take
}
int launch_window(AttentionArgs a, bool backward, hipStream_t st);

// Few queries against many keys -- the next token of every sequence: attention_few.hip.
inline bool is_few(const ta_nn_attention_args& a) { return static_cast<int64_t>(a.heads / a.kv_heads) * a.m <= 16 && !is_window(a); }
// Keys of a workgroup.  At least 512, four times what its waves take at once, and no split at all below 1024 keys: joining costs a
// launch.  Otherwise as many as make some 2048 workgroups, so that sequences of unequal length even out.
inline int few_chunk(const ta_nn_attention_args& a) {
    if (a.n <= 1024) return (a.n + 127) / 128 * 128;
    const int64_t splits = ceil_div(2048, static_cast<int64_t>(a.batch) * a.kv_heads);
    const int64_t chunk = ceil_div(ceil_div(a.n, splits), 128) * 128;
    return static_cast<int>(chunk < 512 ? 512 : chunk);
}
inline int few_splits(const ta_nn_attention_args& a) { return static_cast<int>(ceil_div(a.n, few_chunk(a))); }
int launch_few(AttentionArgs a, hipStream_t st);

int check_attention(const ta_nn_attention_args* args, AttentionArgs& a);
int64_t workspace_floats(const ta_nn_attention_args& a, bool backward);

}  // namespace ta_nn

// launch<.., BIASES>(...) for the call's biases
#define TA_NN_BY_BIASES(a, call)                                          \
    switch (ta_nn::biases_of(a)) {                                        \
        case ta_nn::kByDistance: { constexpr int BIASES = ta_nn::kByDistance; call; break; } \
        case ta_nn::kByPair: { constexpr int BIASES = ta_nn::kByPair; call; break; }         \
        default: { constexpr int BIASES = ta_nn::kAny; call; break; }     \
    }

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
