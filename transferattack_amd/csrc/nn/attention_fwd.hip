// Attention with a learned relative position bias, forward (see attention.h for the formulas and the layout).
#include "attention.h"

namespace ta_nn {

constexpr float kSlack = 8.0f;
template <class T> constexpr float kBelow = kNarrow<T> ? 15.0f - kSlack : 0.0f;      // how far below the largest score the reference is

// One workgroup: 64 NQ columns (queries; those of all heads that share a key head in one row, so that shared heads share the
// tiles) against every key they see, a tile at a time.  Two tiles in LDS: while one is worked on, the next arrives in registers
// and is put into the other's place, with one barrier a tile.  Bound by LDS reads and by issue (16 columns to a wave: a byte of LDS
// for every 16 operations; one exponential and a few fp32 operations a score), not by memory: 16 x 8191 causal tokens of 128 in
// fp16, 4 key heads, 430 us = 640 Tflop/s of the 1310 a large matrix product reaches; 8 x 12 x 1023 padded tokens of 64 in bf16 52 us.
// Three waves to a SIMD for 16-bit types although wide heads then spill a few registers outside the loop: 507 against 511 us.
template <class T, int DP, int NQ, int BIASES>
__global__ __launch_bounds__(256, sizeof(T) == 2 && NQ == 1 ? 3 : 2) void attention_fwd(AttentionArgs a) {
    constexpr int DC = DP / Frag<T>::D, DT = DP / 16, SUBS = kSubs<DP>, ROWS = 16 * SUBS, TILE = ROWS * Tile<T, DP>::LD;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    T* tiles = reinterpret_cast<T*>(smem);               // [2][keys, values][ROWS][LD]
    float* bias_lds = reinterpret_cast<float*>(tiles + 4 * TILE);
    const int tid = threadIdx.x, wave = tid >> 6, c = tid & 15, g = (tid >> 4) & 3;
    const int group = a.heads / a.kv_heads;
    // Columns: the group's queries head by head; a tile of them never spans heads where one has as many (tiles that span heads, whose
    // queries stand far apart, take the slow kind of tile throughout)
    const int64_t columns = static_cast<int64_t>(group) * a.m;
    const bool by_head = a.m >= 64 * NQ;
    const int per_head = (a.m + 64 * NQ - 1) / (64 * NQ);
    // workgroups go to the XCDs in turn: with sequence and head as the fastest index an XCD's L2 holds few heads' keys and values
    const int64_t block = blockIdx.x, lanes = static_cast<int64_t>(a.kv_heads) * a.batch;
    const int hk = static_cast<int>(block % lanes % a.kv_heads);
    const int64_t b = block % lanes / a.kv_heads;
    const int tile = static_cast<int>(block / lanes);
    int64_t col0, col1;
    if (by_head) {                                       // causal: the longest begin, the last queries of every head
        const int h = tile % group, i0 = (a.causal ? per_head - 1 - tile / group : tile / group) * 64 * NQ;
        col0 = static_cast<int64_t>(h) * a.m + i0;
        col1 = static_cast<int64_t>(h) * a.m + min(i0 + 64 * NQ, a.m) - 1;
    } else {
        col0 = static_cast<int64_t>(tile) * 64 * NQ;
        col1 = min(col0 + 64 * NQ, columns) - 1;
    }
    const int h0 = static_cast<int>(col0 / a.m), h1 = static_cast<int>(col1 / a.m);
    const int start = a.query_start ? a.query_start[b] : a.start;
    // positions of the block's first and last query (of any, where it spans heads)
    const int64_t pos0 = static_cast<int64_t>(start) + (h0 == h1 ? col0 - static_cast<int64_t>(h0) * a.m : 0);
    const int64_t pos1 = static_cast<int64_t>(start) + (h0 == h1 ? col1 - static_cast<int64_t>(h1) * a.m : a.m - 1);
    int keys = a.key_lengths ? max(0, min(a.key_lengths[b], a.n)) : a.n;
    if (a.causal) keys = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(keys), pos1 + 1)));

    const T* k_base = static_cast<const T*>(a.k) + b * a.k_sb + hk * a.k_sh;
    const T* v_base = static_cast<const T*>(a.v) + b * a.v_sb + hk * a.v_sh;
    Staged<T, DP, ROWS, 256> kr, vr;
    auto fetch = [&](int j0) {
        if (j0 >= keys) return;
        kr.load(k_base + static_cast<int64_t>(j0) * a.k_sn, a.k_sn, keys - j0, a.dim);
        vr.load(v_base + static_cast<int64_t>(j0) * a.v_sn, a.v_sn, keys - j0, a.dim);
    };
    fetch(0);
    if (a.bias_in_lds) stage_bias(a, bias_lds, hk * group + h0, h1 - h0 + 1, 256);

    int query[NQ];
    bool valid[NQ];
    Column col[NQ];
    typename Frag<T>::Row q[NQ][DC];
    f32x4 o[NQ][DT];
    float m_run[NQ], l[NQ];
#pragma unroll
    for (int x = 0; x < NQ; ++x) {
        const int64_t at = col0 + (wave * NQ + x) * 16 + c;
        valid[x] = at <= col1;
        const int64_t own = valid[x] ? at : col1;
        const int h = static_cast<int>(own / a.m);
        query[x] = static_cast<int>(own - static_cast<int64_t>(h) * a.m);
        const int head = hk * group + h;
        col[x] = query_column(a, a.bias_in_lds ? bias_lds + (h - h0) * bias_entries(a) : nullptr, b, head, query[x], start, keys);
        const T* p = static_cast<const T*>(a.q) + b * a.q_sb + head * a.q_sh + query[x] * a.q_sm;
#pragma unroll
        for (int dc = 0; dc < DC; ++dc) q[x][dc] = row_frag_global<T>(p, a.dim, dc, g, valid[x]);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[x][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        m_run[x] = -INFINITY;
        l[x] = 0.0f;
    }
    const bool busy = wave_any(valid[0]);                // (a wave behind the last query only stages tiles)
    if (keys > 0) {
        kr.put(tiles);
        vr.put(tiles + TILE);
        fetch(ROWS);
    }
    __syncthreads();
    auto kind_at = [&](int j0) {
        return tile_kind<BIASES>(a, j0 + ROWS <= keys && (!a.causal || j0 + ROWS - 1 <= pos0), h0 == h1, j0 - pos1 - a.first,
                                 j0 + ROWS - 1 - pos0 - a.first);
    };
    int j0 = 0, turn = 0;
    while (j0 < keys) {
        // a loop of its own for a run of tiles of one kind: the accumulators stay where they are from tile to tile
        by_kind<BIASES>(kind_at(j0), [&](auto tag) {
          do {
            const T* ks = tiles + turn * 2 * TILE;
            const T* vs = ks + TILE;
            if (busy) {
                f32x4 s[NQ][SUBS];
#pragma unroll
                for (int t = 0; t < SUBS; ++t) {
#pragma unroll
                    for (int x = 0; x < NQ; ++x) s[x][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                    if (decltype(tag)::kind == kEdge && 16 * t >= keys - j0) continue;
#pragma unroll
                    for (int dc = 0; dc < DC; ++dc) {
                        const typename Frag<T>::Row kf = row_frag<T, DP>(ks, 16 * t + c, dc, g);
#pragma unroll
                        for (int x = 0; x < NQ; ++x) s[x][t] = mma_row(kf, q[x][dc], s[x][t]);
                    }
                }
                bool more = false;
                float top[NQ];
#pragma unroll
                for (int x = 0; x < NQ; ++x) {
                    score_tile<BIASES, decltype(tag)::kind, false>(a, col[x], j0, g, s[x]);
                    top[x] = s[x][0][0];
#pragma unroll
                    for (int t = 0; t < SUBS; ++t)
#pragma unroll
                        for (int r = 0; r < 4; ++r) top[x] = fmaxf(top[x], s[x][t][r]);
                    top[x] = reduce_rows(top[x], [](float u, float v) { return fmaxf(u, v); }) - kBelow<T>;
                    more = more || top[x] > m_run[x] + kSlack;
                }
                // The reference is the largest score up to 2^kSlack (fp16: and 2^7 below it, so that the many small probabilities of a
                // long row keep their bits): sums and outputs are rescaled only where one exceeds it by more, which after a few tiles is
                // hardly ever.  (Probabilities up to 2^kSlack cost no precision; they stay below 2^15.)
                if (__ballot(more) != 0) {
#pragma unroll
                    for (int x = 0; x < NQ; ++x) {
                        const float m_new = fmaxf(m_run[x], top[x]);
                        const float shrink = m_new == -INFINITY ? 1.0f : exp2_hw(m_run[x] - m_new);
                        m_run[x] = m_new;
                        l[x] *= shrink;
#pragma unroll
                        for (int dt = 0; dt < DT; ++dt) o[x][dt] *= shrink;
                    }
                }
#pragma unroll
                for (int x = 0; x < NQ; ++x) {
                    const float m_ref = m_run[x] == -INFINITY ? 0.0f : m_run[x];
                    float sum = 0.0f;
#pragma unroll
                    for (int t = 0; t < SUBS; ++t)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            s[x][t][r] = exp2_hw(s[x][t][r] - m_ref);
                            sum += s[x][t][r];
                        }
                    l[x] += sum;
                }
                mma_transposed<DP, NQ, SUBS>(vs, s, o, c, g);
            }
            if (j0 + ROWS < keys) {
                T* next = tiles + (turn ^ 1) * 2 * TILE; // (everyone has left it: the barrier of the last turn)
                kr.put(next);
                vr.put(next + TILE);
                fetch(j0 + 2 * ROWS);
            }
            __syncthreads();
            j0 += ROWS;
            turn ^= 1;
          } while (j0 < keys && kind_at(j0) == decltype(tag)::kind);
        });
    }
#pragma unroll
    for (int x = 0; x < NQ; ++x) {
        const float sum = reduce_rows(l[x], Sum{});
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        if (!valid[x]) continue;
        T* p = static_cast<T*>(a.out) + b * a.o_sb + col[x].head * a.o_sh + query[x] * a.o_sm;
        store_column<T, DP>(p, o[x], inv, a.dim, g);
        const int64_t row = (b * a.heads + col[x].head) * a.m + query[x];
        if (a.stats && g == 0) {
            float* st = a.stats + 2 * row;
            st[0] = m_run[x] == -INFINITY ? 0.0f : m_run[x];
            st[1] = inv;
        }
    }
}

template <class T, int DP, int NQ> int launch_forward_by(AttentionArgs a, hipStream_t st) {
    const int64_t columns = static_cast<int64_t>(a.heads / a.kv_heads) * a.m;
    const int64_t tiles = a.m >= 64 * NQ ? ceil_div(a.m, 64 * NQ) * (a.heads / a.kv_heads) : ceil_div(columns, 64 * NQ);
    const int64_t blocks = tiles * a.kv_heads * a.batch;
    TA_NN_REQUIRE(blocks <= 0x7FFFFFFF, "too many queries: %lld workgroups", static_cast<long long>(blocks));
    const size_t lds = 4 * 16 * kSubs<DP> * Tile<T, DP>::LD * sizeof(T) + bias_lds_bytes(a, 64 * NQ);
    if constexpr (NQ == 2) {                             // pairs only: no instance for distances
        if (biases_of(a) == kByPair) hipLaunchKernelGGL((attention_fwd<T, DP, NQ, kByPair>), dim3(static_cast<unsigned>(blocks)), dim3(256), lds, st, a);
        else hipLaunchKernelGGL((attention_fwd<T, DP, NQ, kAny>), dim3(static_cast<unsigned>(blocks)), dim3(256), lds, st, a);
    } else {
        TA_NN_BY_BIASES(a, hipLaunchKernelGGL((attention_fwd<T, DP, NQ, BIASES>), dim3(static_cast<unsigned>(blocks)), dim3(256), lds, st, a));
    }
    return check_launch("ta_nn_attention");
}

template <class T, int DP> int launch_forward(AttentionArgs a, hipStream_t st) {
    const int64_t columns = static_cast<int64_t>(a.heads / a.kv_heads) * a.m;
    // 32 columns to a wave halve the LDS reads per product, but leave room for two waves to a SIMD instead of three: 48 against 53 us
    // for pairs (64 x 12 heads, 196 tokens of 64, bf16), 63 against 57 us for distances (8 x 12 heads, 1023 tokens of 64), whose
    // scores are ready sooner.  Not where it leaves CUs idle, nor for wide heads, whose accumulators leave no room.
    constexpr int WIDE = sizeof(T) == 2 && DP <= 64 ? 2 : 1;
    if (WIDE == 2 && a.distances == 0 && ceil_div(columns, 128) * a.kv_heads * a.batch >= 512) return launch_forward_by<T, DP, WIDE>(a, st);
    return launch_forward_by<T, DP, 1>(a, st);
}

}  // namespace ta_nn

extern "C" int64_t ta_nn_attention_workspace(const ta_nn_attention_args* args, int backward) {
    if (args == nullptr) return 0;
    return ta_nn::workspace_floats(*args, backward != 0);
}

extern "C" int ta_nn_attention(const ta_nn_attention_args* args, void* stream) {
    ta_nn::AttentionArgs a{};
    if (int rc = ta_nn::check_attention(args, a)) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (ta_nn::is_window(a)) return ta_nn::launch_window(a, false, st);
    if (ta_nn::is_few(a)) return ta_nn::launch_few(a, st);
    TA_NN_BY_TYPE_AND_DIM(a.dtype, a.dim, (ta_nn::launch_forward<T, DP>(a, st)));
}
