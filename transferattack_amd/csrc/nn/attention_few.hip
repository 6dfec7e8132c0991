// Attention of a few queries -- up to 16 columns: the queries of all heads that share a key head -- against many keys, as when
// the next token of every sequence meets its cache.  Bound by reading keys and values once, so nothing is shared between waves:
// each takes 32 keys (wide fp32 heads: 16) at a time for itself, keys straight from memory into the matrix instruction's layout, values through
// as many rows of LDS of its own, with its own maximum and sum; the next ones are on their way while it works.  A workgroup's four
// waves are joined in LDS, the workgroups of a long sequence by a second kernel.  Measured: 32 sequences of up to 16384 keys, 4 key
// heads of 128 in bf16, 142 us (4.7 TB/s; a large copy reaches 5.0) and 7 us for the join; 1 x 12 heads x 511 keys of 64, 8 us, of
// which the launch is most.  With waves sharing tiles through LDS and a barrier for each the first took 1880 us.
#include "attention.h"

namespace ta_nn {

// 16 keys a wave and step over: 32, or for wide fp32 heads 16 (twice their keys would not fit its registers)
template <class T, int DP> constexpr int few_subs = sizeof(T) == 4 && DP > 64 ? 1 : 2;

template <class T, int DP, int BIASES>
__global__ __launch_bounds__(256, 2) void attention_few(AttentionArgs a, int chunk, int splits) {
    constexpr int DC = DP / Frag<T>::D, DT = DP / 16, VE = Frag<T>::VE, PER_ROW = DP / VE;
    constexpr int SUBS = few_subs<T, DP>, ROWS = 16 * SUBS, TILE = ROWS * Tile<T, DP>::LD;
    constexpr int LOADS = ROWS * PER_ROW / 64, OLD = DP + 4;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ float wave_m[4][16], wave_l[4][16], total_l[16];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, c = tid & 15, g = (tid >> 4) & 3;
    T* vs = reinterpret_cast<T*>(smem) + wave * TILE;
    float* joined = reinterpret_cast<float*>(smem);      // [4][16][OLD], once the values are done with
    constexpr size_t VALUES = 4 * TILE * sizeof(T), JOIN = 4 * 16 * OLD * 4;
    float* bias_lds = reinterpret_cast<float*>(smem + (VALUES > JOIN ? VALUES : JOIN));
    const int group = a.heads / a.kv_heads, columns = group * a.m;
    const int64_t block = blockIdx.x;
    const int split = static_cast<int>(block % splits), hk = static_cast<int>(block / splits % a.kv_heads);
    const int64_t b = block / splits / a.kv_heads;
    const int start = a.query_start ? a.query_start[b] : a.start;
    int keys = a.key_lengths ? max(0, min(a.key_lengths[b], a.n)) : a.n;
    if (a.causal) keys = min(keys, clamp_token(static_cast<int64_t>(start) + a.m - 1) + 1);
    const int begin = split * chunk, end = min(keys, begin + chunk);
    if (begin >= end && split > 0) return;               // (the first one writes, also where no key is seen)

    const bool valid = c < columns;
    const int own = valid ? c : columns - 1, head = hk * group + own / a.m, query = own % a.m;
    const T* k_base = static_cast<const T*>(a.k) + b * a.k_sb + hk * a.k_sh;
    const T* v_base = static_cast<const T*>(a.v) + b * a.v_sb + hk * a.v_sh;
    const unsigned k_step = static_cast<unsigned>(a.k_sn), v_step = static_cast<unsigned>(a.v_sn);
    constexpr unsigned ES = sizeof(T);
    typename Frag<T>::Row k[SUBS][DC];
    Vec<T> v[LOADS];
    auto fetch = [&](int j0) {
        if (j0 >= end) return;
        const T* kp = k_base + static_cast<int64_t>(j0) * a.k_sn;
        const T* vp = v_base + static_cast<int64_t>(j0) * a.v_sn;
        if (j0 + ROWS <= end && a.dim == DP) {
#pragma unroll
            for (int t = 0; t < SUBS; ++t)
#pragma unroll
                for (int dc = 0; dc < DC; ++dc)
                    k[t][dc] = __builtin_bit_cast(typename Frag<T>::Row, load_at(kp, ((16 * t + c) * k_step + dc * Frag<T>::D + g * VE) * ES));
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int e = lane + 64 * i;
                v[i] = load_at(vp, (e / PER_ROW * v_step + e % PER_ROW * VE) * ES);
            }
        } else {
#pragma unroll
            for (int t = 0; t < SUBS; ++t)
#pragma unroll
                for (int dc = 0; dc < DC; ++dc)
                    k[t][dc] = row_frag_global<T>(kp + (16 * t + c) * k_step, a.dim, dc, g, j0 + 16 * t + c < end);
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int e = lane + 64 * i, r = e / PER_ROW, d = e % PER_ROW * VE;
                v[i].raw = u32x4{0, 0, 0, 0};
                if (j0 + r < end && d < a.dim) v[i] = load_at(vp, (r * v_step + d) * ES);
            }
        }
    };
    fetch(begin + ROWS * wave);
    if (a.bias_in_lds) stage_bias(a, bias_lds, hk * group, group, 256, 0);
    const Column col = query_column(a, a.bias_in_lds ? bias_lds + (head - hk * group) * bias_entries(a, 0) : nullptr, b, head, query, start, keys);
    typename Frag<T>::Row q[DC];
    {
        const T* p = static_cast<const T*>(a.q) + b * a.q_sb + head * a.q_sh + query * a.q_sm;
#pragma unroll
        for (int dc = 0; dc < DC; ++dc) q[dc] = row_frag_global<T>(p, a.dim, dc, g, valid);
    }
    const int64_t pos0 = start, pos1 = static_cast<int64_t>(start) + a.m - 1;
    f32x4 o[1][DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[0][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m_run = -INFINITY, l = 0.0f;
    __syncthreads();
    for (int j0 = begin + ROWS * wave; j0 < end; j0 += 4 * ROWS) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int e = lane + 64 * i;
            *reinterpret_cast<Vec<T>*>(vs + e / PER_ROW * Tile<T, DP>::LD + e % PER_ROW * VE) = v[i];
        }
        f32x4 s[1][SUBS];
#pragma unroll
        for (int t = 0; t < SUBS; ++t) {
            s[0][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int dc = 0; dc < DC; ++dc) s[0][t] = mma_row(k[t][dc], q[dc], s[0][t]);
        }
        fetch(j0 + 4 * ROWS);
        Kind kind = tile_kind<BIASES>(a, j0 + ROWS <= keys && (!a.causal || j0 + ROWS - 1 <= pos0), false,
                                      j0 - pos1 - a.first, j0 + ROWS - 1 - pos0 - a.first);
        by_kind<BIASES>(kind, [&](auto tag) { score_tile<BIASES, decltype(tag)::kind, false, 0>(a, col, j0, g, s[0]); });
        float top = s[0][0][0];
#pragma unroll
        for (int t = 0; t < SUBS; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) top = fmaxf(top, s[0][t][r]);
        top = reduce_rows(top, [](float x, float y) { return fmaxf(x, y); }) - kLift<T>;      // (the reference: below the largest)
        const float m_new = fmaxf(m_run, top), m_ref = m_new == -INFINITY ? 0.0f : m_new;
        const float shrink = exp2_hw(m_run - m_ref);
        m_run = m_new;
        float sum = 0.0f;
#pragma unroll
        for (int t = 0; t < SUBS; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[0][t][r] = exp2_hw(s[0][t][r] - m_ref);
                sum += s[0][t][r];
            }
        l = l * shrink + sum;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[0][dt] *= shrink;
        wave_lds_order();                                // (the wave's own rows: its LDS operations are done in order)
        mma_transposed<DP, 1, SUBS, 1>(vs, s, o, c, g);
        wave_lds_order();
    }
    l = reduce_rows(l, Sum{});
    if (g == 0) {
        wave_m[wave][c] = m_run;
        wave_l[wave][c] = l;
    }
    __syncthreads();
    float m_all = wave_m[0][c], l_all = 0.0f;
#pragma unroll
    for (int w = 1; w < 4; ++w) m_all = fmaxf(m_all, wave_m[w][c]);
    const float m_ref = m_all == -INFINITY ? 0.0f : m_all;
#pragma unroll
    for (int w = 0; w < 4; ++w) l_all += wave_l[w][c] * exp2_hw(wave_m[w][c] - m_ref);
    const float mine = exp2_hw(m_run - m_ref);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4*>(joined + (wave * 16 + c) * OLD + 16 * dt + 4 * g) = o[0][dt] * mine;
    if (wave == 0 && g == 0) total_l[c] = l_all;
    __syncthreads();
    const float inv_all = l_all == 0.0f ? 0.0f : 1.0f / l_all;
    if (splits > 1 && tid < 16 && tid < columns) {
        float* ml = a.workspace + ((b * a.kv_heads + hk) * splits + split) * 32 + 2 * tid;
        ml[0] = m_all;
        ml[1] = l_all;
    }
    if (splits == 1 && a.stats && tid < 16 && tid < columns) {
        float* st = a.stats + 2 * ((b * a.heads + head) * a.m + query);
        st[0] = m_ref;
        st[1] = inv_all;
    }
    float* partial = a.workspace + static_cast<int64_t>(a.batch) * a.kv_heads * splits * 32 + ((b * a.kv_heads + hk) * splits + split) * 16 * a.dim;
    for (int e = tid; e < columns * DP; e += 256) {
        const int x = e / DP, d = e % DP;
        if (d >= a.dim) continue;
        float f = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) f += joined[(w * 16 + x) * OLD + d];
        if (splits > 1) {
            partial[x * a.dim + d] = f;
        } else {
            const float sum = total_l[x];
            f *= sum == 0.0f ? 0.0f : 1.0f / sum;
            const int h = hk * group + x / a.m, i = x % a.m;
            static_cast<T*>(a.out)[b * a.o_sb + h * a.o_sh + i * a.o_sm + d] = from_float<T>(f);
        }
    }
}

// one wave to a column: the workgroups' parts of a sequence, in order
template <class T> __global__ __launch_bounds__(64) void attention_join(AttentionArgs a, int chunk, int splits) {
    const int group = a.heads / a.kv_heads, columns = group * a.m, lane = threadIdx.x;
    const int64_t block = blockIdx.x;
    const int x = static_cast<int>(block % columns), hk = static_cast<int>(block / columns % a.kv_heads);
    const int64_t b = block / columns / a.kv_heads;
    const int start = a.query_start ? a.query_start[b] : a.start;
    int keys = a.key_lengths ? max(0, min(a.key_lengths[b], a.n)) : a.n;
    if (a.causal) keys = min(keys, clamp_token(static_cast<int64_t>(start) + a.m - 1) + 1);
    const int parts = max(1, (keys + chunk - 1) / chunk);
    const float* ml = a.workspace + (b * a.kv_heads + hk) * splits * 32 + 2 * x;
    const float* partial = a.workspace + static_cast<int64_t>(a.batch) * a.kv_heads * splits * 32 + (b * a.kv_heads + hk) * splits * 16 * a.dim + x * a.dim;
    __shared__ float weight[64];
    float top = -INFINITY;
    for (int s = lane; s < parts; s += 64) top = max_nan(top, ml[32 * s]);
    top = wave_max(top);
    const float m_ref = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f, f0 = 0.0f, f1 = 0.0f;
    const int d0 = min(lane, a.dim - 1), d1 = min(lane + 64, a.dim - 1);
    for (int first = 0; first < parts; first += 64) {
        const int count = min(64, parts - first);
        wave_lds_order();
        if (lane < count) {
            weight[lane] = exp2_hw(ml[32 * (first + lane)] - m_ref);
            sum += ml[32 * (first + lane) + 1] * weight[lane];
        }
        wave_lds_order();
        const float* p = partial + static_cast<int64_t>(first) * 16 * a.dim;
#pragma unroll 8
        for (int s = 0; s < count; ++s) {
            f0 += p[s * 16 * a.dim + d0] * weight[s];
            f1 += p[s * 16 * a.dim + d1] * weight[s];
        }
    }
    sum = wave_sum(sum);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const int head = hk * group + x / a.m, query = x % a.m;
    T* out = static_cast<T*>(a.out) + b * a.o_sb + head * a.o_sh + query * a.o_sm;
    const int64_t row = (b * a.heads + head) * a.m + query;
    if (lane < a.dim) out[d0] = from_float<T>(f0 * inv);
    if (lane + 64 < a.dim) out[d1] = from_float<T>(f1 * inv);
    if (a.stats && lane == 0) {
        a.stats[2 * row] = m_ref;
        a.stats[2 * row + 1] = inv;
    }
}

template <class T, int DP> int launch_few_by(AttentionArgs a, hipStream_t st) {
    const int chunk = few_chunk(a), splits = few_splits(a);
    const int64_t blocks = static_cast<int64_t>(a.batch) * a.kv_heads * splits, columns = static_cast<int64_t>(a.heads / a.kv_heads) * a.m;
    TA_NN_REQUIRE(blocks <= 0x7FFFFFFF && static_cast<int64_t>(a.batch) * a.heads * a.m <= 0x7FFFFFFF, "too many sequences for one launch");
    TA_NN_REQUIRE(splits == 1 || a.workspace, "null pointer");
    const size_t values = 4 * 16 * few_subs<T, DP> * Tile<T, DP>::LD * sizeof(T), join = 4 * 16 * (DP + 4) * 4;
    const size_t lds = (values > join ? values : join) + bias_lds_bytes(a, 16 * static_cast<int64_t>(a.m), 0);      // (all heads of the group)
    TA_NN_BY_BIASES(a, hipLaunchKernelGGL((attention_few<T, DP, BIASES>), dim3(static_cast<unsigned>(blocks)), dim3(256), lds, st, a, chunk, splits));
    if (splits > 1)
        hipLaunchKernelGGL((attention_join<T>), dim3(static_cast<unsigned>(a.batch * a.kv_heads * columns)), dim3(64), 0, st, a, chunk, splits);
    return check_launch("ta_nn_attention");
}

int launch_few(AttentionArgs a, hipStream_t st) {
    TA_NN_BY_TYPE_AND_DIM(a.dtype, a.dim, (launch_few_by<T, DP>(a, st)));
}

}  // namespace ta_nn
