// Backward of attention with a learned relative position bias.  With p from the forward pass's maximum and sum:
//     dp_ij = grad_i . v_j      ds_ij = p_ij (dp_ij - delta_i)      delta_i = sum_j p_ij dp_ij (= out_i . grad_i)
//     dq_i = scale sum_j ds_ij k_j     dk_j = scale sum_i ds_ij q_i     dv_j = sum_i p_ij grad_i
//     dtable[u][h] = sum of ds over sequences and over the pairs of bucket u
// Three kernels in the forward's form, each recomputing the scores: queries stay (dq, and delta for the others), keys stay
// (dk, dv), and a tile of pairs stays while the batch streams past it (the table).  No sum crosses workgroups except the
// table's, whose partial sums a last kernel adds in a fixed order.
// p and ds are rounded to 16 bits where they enter a 16-bit matrix instruction: half a step of each term (in fp16 brought into its
// range before, see attention.h), which makes gradients about sqrt(2) of the rounding of their results off.  Over few terms -- calls of
// up to 64 keys, or of 64 queries times the heads that share a key head -- it is up to 1.9 of it, and there both enter in two parts (1.0).
// Over many that would cost 251 instead of 233 us (64 x 12 x 196 tokens, all gradients and the forward pass) and 313 instead of 280
// (8 x 12 x 1023).
// Together 9 products of m n dim, the forward's two aside, where 5 are needed (16-bit types: 10, with dq's correction): scores and dp
// are computed once for each kernel, since dq and dk, dv sum over different sides of the same scores.  Bound like the forward by LDS
// reads and issue.  Measured, bf16, heads of 64: 8 x 12 x 1023 padded tokens, queries 80 us (74 without the correction), keys 87,
// table 42 + 20 (near tiles only: what is past an end of the distances is summed by the queries' kernel, which meets those pairs
// anyway); 64 x 12 x 196 tokens in pairs, 52, 57, 60 + 15 us.  64-row tiles (two waves to a SIMD) instead of 32: 81 and 105 us for the
// first two, against 71 and 91 at the time.
#include "attention.h"

namespace ta_nn {

constexpr int kFewTerms = 64;                            // of a sum over keys, or over queries and the heads that share a key head

template <class T, int DP, int BIASES, int FEW>
__global__ __launch_bounds__(256, sizeof(T) == 2 && DP <= 64 ? 3 : 2) void attention_bwd_q(AttentionArgs a) {
    constexpr int DC = DP / Frag<T>::D, DT = DP / 16, SUBS = sizeof(T) == 2 ? 2 : kSubs<DP>, ROWS = 16 * SUBS;
    constexpr int SUMS = sizeof(T) == 2 ? 2 : 1;         // of ds k, and of p k for the correction below
    extern __shared__ __attribute__((aligned(16))) char smem[];
    T* ks = reinterpret_cast<T*>(smem);
    T* vs = ks + ROWS * Tile<T, DP>::LD;
    float* bias_lds = reinterpret_cast<float*>(vs + ROWS * Tile<T, DP>::LD);
    const int tid = threadIdx.x, wave = tid >> 6, c = tid & 15, g = (tid >> 4) & 3;
    const int group = a.heads / a.kv_heads;
    const int tiles = (a.m + 63) / 64;
    const int64_t block = blockIdx.x, lanes = static_cast<int64_t>(a.heads) * a.batch;     // as in attention_fwd
    const int head = static_cast<int>(block % lanes % a.heads);
    const int64_t b = block % lanes / a.heads;
    const int i0 = (a.causal ? tiles - 1 - static_cast<int>(block / lanes) : static_cast<int>(block / lanes)) * 64;
    const int hk = head / group;
    const int start = a.query_start ? a.query_start[b] : a.start;
    int keys = a.key_lengths ? max(0, min(a.key_lengths[b], a.n)) : a.n;
    if (a.causal) {
        const int64_t last = static_cast<int64_t>(start) + min(i0 + 64, a.m) - 1;
        keys = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(keys), last + 1)));
    }
    if (a.bias_in_lds) stage_bias(a, bias_lds, head, 1, 256);

    const bool valid = i0 + 16 * wave + c < a.m;
    const bool busy = wave_any(valid);                   // (a wave behind the last query only stages tiles)
    const int query = min(i0 + 16 * wave + c, a.m - 1);
    const T* qp = static_cast<const T*>(a.q) + b * a.q_sb + head * a.q_sh + query * a.q_sm;
    const T* gp = static_cast<const T*>(a.grad) + b * a.g_sb + head * a.g_sh + query * a.g_sm;
    const T* op = static_cast<const T*>(a.out) + b * a.o_sb + head * a.o_sh + query * a.o_sm;
    const int64_t at = (b * a.heads + head) * a.m + query;
    typename Frag<T>::Row q[DC], go[DC];
    float delta = 0.0f;
#pragma unroll
    for (int dc = 0; dc < DC; ++dc) {
        q[dc] = row_frag_global<T>(qp, a.dim, dc, g, valid);
        go[dc] = row_frag_global<T>(gp, a.dim, dc, g, valid);
        const Vec<T> gv = __builtin_bit_cast(Vec<T>, go[dc]);
        const Vec<T> o = __builtin_bit_cast(Vec<T>, row_frag_global<T>(op, a.dim, dc, g, valid));
#pragma unroll
        for (int i = 0; i < Frag<T>::VE; ++i) delta += get(o, i) * get(gv, i);
    }
    delta = reduce_rows(delta, Sum{});
    const float top = a.stats[2 * at], inv = a.stats[2 * at + 1];
    const Column col = query_column(a, a.bias_in_lds ? bias_lds : nullptr, b, head, query, start, keys);
    const int64_t pos0 = static_cast<int64_t>(start) + i0, pos1 = static_cast<int64_t>(start) + min(i0 + 64, a.m) - 1;

    // delta while the keys pass is out . grad.  For 16-bit tensors out is rounded, and so were the probabilities it was made with; the
    // exact one, sum_j p_ij dp_ij, is known at the end of the row (or at once, where the row is a single tile).  It is written for the
    // other kernels, and what dq lacks is put right:  dq = sum ds k + (out . grad - delta) sum p k.  The second sum takes its operands
    // from the fragments that the first has read.  Without it dq of bf16 rows whose mass lies on a few of 200 keys is 5 times as far
    // off as its rounding.
    float exact = 0.0f;
    float up = kNarrow<T> ? kMostLift : 1.0f;
    constexpr float LIFT = 1 << kLift<T>;
    // sums past either end of the distances, for the table: of p and of p dp, since delta is not known yet
    float far_p[2] = {0.0f, 0.0f}, far_dp[2] = {0.0f, 0.0f};
    const bool wants_far = BIASES != kByPair && a.far != nullptr;
    f32x4 dq[SUMS][DT];
#pragma unroll
    for (int x = 0; x < SUMS; ++x)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) dq[x][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const T* k_base = static_cast<const T*>(a.k) + b * a.k_sb + hk * a.k_sh;
    const T* v_base = static_cast<const T*>(a.v) + b * a.v_sb + hk * a.v_sh;
    Staged<T, DP, ROWS, 256> kr, vr;
    auto fetch = [&](int j0) {
        kr.load(k_base + static_cast<int64_t>(j0) * a.k_sn, a.k_sn, keys - j0, a.dim);
        vr.load(v_base + static_cast<int64_t>(j0) * a.v_sn, a.v_sn, keys - j0, a.dim);
    };
    if (keys > 0) fetch(0);
    for (int j0 = 0; j0 < keys; j0 += ROWS) {
        __syncthreads();
        kr.put(ks);
        vr.put(vs);
        __syncthreads();
        if (j0 + ROWS < keys) fetch(j0 + ROWS);
        const Kind kind = tile_kind<BIASES>(a, j0 + ROWS <= keys && (!a.causal || j0 + ROWS - 1 <= pos0), true, j0 - pos1 - a.first,
                                            j0 + ROWS - 1 - pos0 - a.first);
        if (busy) by_kind<BIASES>(kind, [&](auto tag) {
        f32x4 s[SUBS], ds[SUMS][SUBS];
#pragma unroll
        for (int t = 0; t < SUBS; ++t) {
            s[t] = ds[0][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if (decltype(tag)::kind == kEdge && 16 * t >= keys - j0) continue;
#pragma unroll
            for (int dc = 0; dc < DC; ++dc) {
                s[t] = mma_row(row_frag<T, DP>(ks, 16 * t + c, dc, g), q[dc], s[t]);
                ds[0][t] = mma_row(row_frag<T, DP>(vs, 16 * t + c, dc, g), go[dc], ds[0][t]);
            }
        }
        score_tile<BIASES, decltype(tag)::kind, false>(a, col, j0, g, s);
        float exact_tile = 0.0f;
#pragma unroll
        for (int t = 0; t < SUBS; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[t][r] = exp2_hw(s[t][r] - top) * inv;
                exact_tile += s[t][r] * ds[0][t][r];
            }
        if (keys <= ROWS) delta = reduce_rows(exact_tile, Sum{});
#pragma unroll
        for (int t = 0; t < SUBS; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                ds[0][t][r] = s[t][r] * (ds[0][t][r] - delta);
                if constexpr (SUMS == 2) ds[1][t][r] = s[t][r] * LIFT;
            }
        if constexpr (kNarrow<T>) into_range(ds[0], dq[0], up);
        exact += exact_tile;
        if constexpr (BIASES != kByPair && decltype(tag)::kind != kNear) {
            const int64_t j64 = j0 & ~63;
            const int end = wants_far ? far_end(a, j64 - pos1 - a.first, j64 + 63 - pos0 - a.first) : 0;
            if (end != 0) {
                float sum = 0.0f;
#pragma unroll
                for (int t = 0; t < SUBS; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) sum += s[t][r];
                far_p[0] += end < 0 ? sum : 0.0f;
                far_p[1] += end > 0 ? sum : 0.0f;
                far_dp[0] += end < 0 ? exact_tile : 0.0f;
                far_dp[1] += end > 0 ? exact_tile : 0.0f;
            }
        }
        mma_transposed<DP, SUMS, SUBS, FEW>(ks, ds, dq, c, g);
        });
    }
    exact = reduce_rows(exact, Sum{});
    if constexpr (SUMS == 2) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) dq[0][dt] = dq[0][dt] * (1.0f / up) + dq[1][dt] * ((delta - exact) / LIFT);
    }
    if (valid && g == 0) a.delta[at] = exact;
    if (BIASES != kByPair && wants_far) {
        __shared__ float far_lds[4][2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float sum = wave_sum(valid ? far_dp[e] - exact * far_p[e] : 0.0f);
            if ((tid & 63) == 0) far_lds[wave][e] = sum;
        }
        __syncthreads();
        if (tid < 2)
            a.far[((b * a.heads + head) * tiles + i0 / 64) * 2 + tid] = far_lds[0][tid] + far_lds[1][tid] + far_lds[2][tid] + far_lds[3][tid];
    }
    if (valid) store_column<T, DP>(static_cast<T*>(a.dq) + b * a.dq_sb + head * a.dq_sh + query * a.dq_sm, dq[0], a.scale, a.dim, g);
}

template <class T, int DP, int BIASES, int FEW>
__global__ __launch_bounds__(256, sizeof(T) == 2 && DP <= 64 ? 3 : 2) void attention_bwd_kv(AttentionArgs a) {
    constexpr int DC = DP / Frag<T>::D, DT = DP / 16, SUBS = sizeof(T) == 2 ? 2 : kSubs<DP>, ROWS = 16 * SUBS;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    T* qs = reinterpret_cast<T*>(smem);
    T* gs = qs + ROWS * Tile<T, DP>::LD;
    float* row_top = reinterpret_cast<float*>(gs + ROWS * Tile<T, DP>::LD);
    float* row_inv = row_top + 64;
    float* row_delta = row_inv + 64;
    float* bias_lds = row_delta + 64;
    const int tid = threadIdx.x, wave = tid >> 6, c = tid & 15, g = (tid >> 4) & 3;
    const int group = a.heads / a.kv_heads;
    const int64_t block = blockIdx.x, lanes = static_cast<int64_t>(a.kv_heads) * a.batch;  // as in attention_fwd
    const int hk = static_cast<int>(block % lanes % a.kv_heads);
    const int64_t b = block % lanes / a.kv_heads;
    const int j0 = static_cast<int>(block / lanes) * 64;
    const int start = a.query_start ? a.query_start[b] : a.start;
    const int keys = a.key_lengths ? max(0, min(a.key_lengths[b], a.n)) : a.n;
    const bool valid = j0 + 16 * wave + c < a.n;
    const int key = min(j0 + 16 * wave + c, a.n - 1);
    const bool used = valid && key < keys;
    const bool busy = wave_any(used);

    typename Frag<T>::Row k[DC], v[DC];
    const T* kp = static_cast<const T*>(a.k) + b * a.k_sb + hk * a.k_sh + static_cast<int64_t>(key) * a.k_sn;
    const T* vp = static_cast<const T*>(a.v) + b * a.v_sb + hk * a.v_sh + static_cast<int64_t>(key) * a.v_sn;
#pragma unroll
    for (int dc = 0; dc < DC; ++dc) {
        k[dc] = row_frag_global<T>(kp, a.dim, dc, g, used);
        v[dc] = row_frag_global<T>(vp, a.dim, dc, g, used);
    }
    f32x4 dk[1][DT], dv[1][DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) dk[0][dt] = dv[0][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    float up = kNarrow<T> ? kMostLift : 1.0f;
    constexpr float LIFT = 1 << kLift<T>;

    // the first query that sees any key of the block
    const int i_first = a.causal ? max(0, clamp_token(static_cast<int64_t>(j0) - start)) / ROWS * ROWS : 0;
    const int rows = j0 < keys ? max(0, a.m - i_first) : 0;
    const int steps = (rows + ROWS - 1) / ROWS;                  // per head of the group
    Staged<T, DP, ROWS, 256> qr, gr;
    float st_top = 0.0f, st_inv = 0.0f, st_delta = 0.0f;
    auto fetch = [&](int step) {
        const int head = hk * group + step / steps, i0 = i_first + step % steps * ROWS;
        const T* q_base = static_cast<const T*>(a.q) + b * a.q_sb + head * a.q_sh;
        const T* g_base = static_cast<const T*>(a.grad) + b * a.g_sb + head * a.g_sh;
        qr.load(q_base + static_cast<int64_t>(i0) * a.q_sm, a.q_sm, a.m - i0, a.dim);
        gr.load(g_base + static_cast<int64_t>(i0) * a.g_sm, a.g_sm, a.m - i0, a.dim);
        if (tid < ROWS) {
            const bool in = i0 + tid < a.m;
            const int64_t at = (b * a.heads + head) * a.m + min(i0 + tid, a.m - 1);
            st_top = in ? a.stats[2 * at] : 0.0f;
            st_inv = in ? a.stats[2 * at + 1] : 0.0f;
            st_delta = in ? a.delta[at] : 0.0f;
        }
    };
    if (steps > 0) fetch(0);
    for (int step = 0; step < steps * group; ++step) {
        const int head = hk * group + step / steps, i0 = i_first + step % steps * ROWS;
        __syncthreads();
        qr.put(qs);
        gr.put(gs);
        if (tid < ROWS) {
            row_top[tid] = st_top;
            row_inv[tid] = st_inv;
            row_delta[tid] = st_delta;
        }
        if (a.bias_in_lds && step % steps == 0) stage_bias(a, bias_lds, head, 1, 256);
        __syncthreads();
        if (step + 1 < steps * group) fetch(step + 1);
        const Column col = key_column(a, a.bias_in_lds ? bias_lds : nullptr, b, head, key, start);
        // (a key out of use gets no gradient whatever its column holds: zeros are stored for it)
        const int64_t lead0 = static_cast<int64_t>(j0) - start, lead1 = static_cast<int64_t>(min(j0 + 64, a.n)) - 1 - start;
        const Kind kind = tile_kind<BIASES>(a, i0 + ROWS <= a.m && (!a.causal || i0 >= lead1), true, lead0 - i0 - ROWS + 1 - a.first,
                                            lead1 - i0 - a.first);
        if (busy) by_kind<BIASES>(kind, [&](auto tag) {
        f32x4 p[1][SUBS], ds[1][SUBS];
#pragma unroll
        for (int t = 0; t < SUBS; ++t) {
            p[0][t] = ds[0][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if (decltype(tag)::kind == kEdge && 16 * t >= a.m - i0) continue;
#pragma unroll
            for (int dc = 0; dc < DC; ++dc) {
                p[0][t] = mma_row(row_frag<T, DP>(qs, 16 * t + c, dc, g), k[dc], p[0][t]);
                ds[0][t] = mma_row(row_frag<T, DP>(gs, 16 * t + c, dc, g), v[dc], ds[0][t]);
            }
        }
        score_tile<BIASES, decltype(tag)::kind, true>(a, col, i0, g, p[0]);
#pragma unroll
        for (int t = 0; t < SUBS; ++t) {
            const f32x4 top = *reinterpret_cast<const f32x4*>(row_top + 16 * t + 4 * g);
            const f32x4 inv = *reinterpret_cast<const f32x4*>(row_inv + 16 * t + 4 * g);
            const f32x4 delta = *reinterpret_cast<const f32x4*>(row_delta + 16 * t + 4 * g);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float w = exp2_hw(p[0][t][r] - top[r]) * inv[r];
                p[0][t][r] = w * LIFT;
                ds[0][t][r] = w * (ds[0][t][r] - delta[r]);
            }
        }
        if constexpr (kNarrow<T>) into_range(ds[0], dk[0], up);
        mma_transposed<DP, 1, SUBS, FEW>(gs, p, dv, c, g);
        mma_transposed<DP, 1, SUBS, FEW>(qs, ds, dk, c, g);
        });
    }
    if (!used) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) dk[0][dt] = dv[0][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    if (valid) {
        store_column<T, DP>(static_cast<T*>(a.dk) + b * a.dk_sb + hk * a.dk_sh + static_cast<int64_t>(key) * a.dk_sn, dk[0], a.scale * (1.0f / up), a.dim, g);
        store_column<T, DP>(static_cast<T*>(a.dv) + b * a.dv_sb + hk * a.dv_sh + static_cast<int64_t>(key) * a.dv_sn, dv[0], 1.0f / LIFT, a.dim, g);
    }
}

// ds of one tile of 64 queries x 64 keys of a head, summed over the sequences of a chunk.  Pairs: the tile as it is; distances:
// its 127 diagonals (the distance is the same along each), and only tiles that are not past an end altogether.
template <class T, int DP, int BIASES>
__global__ __launch_bounds__(256, sizeof(T) == 2 && DP <= 64 ? 3 : 2) void attention_bwd_table(AttentionArgs a) {
    constexpr int DC = DP / Frag<T>::D;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    T* ks = reinterpret_cast<T*>(smem);
    T* vs = ks + 64 * Tile<T, DP>::LD;
    float* bias_lds = reinterpret_cast<float*>(vs + 64 * Tile<T, DP>::LD);
    const int tid = threadIdx.x, wave = tid >> 6, c = tid & 15, g = (tid >> 4) & 3;
    const int group = a.heads / a.kv_heads;
    const int q_tiles = (a.m + 63) / 64, k_tiles = a.distances ? near_tiles(a) : (a.n + 63) / 64;
    // as in attention_fwd: the tiles of one head and chunk meet in one XCD's L2 (tile by tile over all of them: 67 us, so: 52)
    const int64_t block = blockIdx.x, lanes = static_cast<int64_t>(a.heads) * a.chunks;
    const int head = static_cast<int>(block % lanes % a.heads), chunk = static_cast<int>(block % lanes / a.heads);
    const int k_tile = static_cast<int>(block / lanes % k_tiles), q_tile = static_cast<int>(block / lanes / k_tiles);
    const int i0 = q_tile * 64, j0 = (a.distances ? first_near_tile(a, i0) + k_tile : k_tile) * 64, hk = head / group;
    const bool valid = i0 + 16 * wave + c < a.m;
    const bool busy = wave_any(valid);
    const int query = min(i0 + 16 * wave + c, a.m - 1);
    if (a.bias_in_lds) stage_bias(a, bias_lds, head, 1, 256);
    f32x4 sum[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) sum[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const int b0 = static_cast<int>(static_cast<int64_t>(a.batch) * chunk / a.chunks);
    const int b1 = static_cast<int>(static_cast<int64_t>(a.batch) * (chunk + 1) / a.chunks);
    // the keys that sequence b's queries of this tile see, and the first sequence from b on whose sum this tile takes part in (the same
    // for the whole workgroup): it has keys in use, and is not past an end of the distances (then it is in attention_bwd_q's sums)
    auto seen_keys = [&](int64_t b) {
        const int keys = a.key_lengths ? max(0, min(a.key_lengths[b], a.n)) : a.n;
        if (!a.causal) return keys;
        const int64_t last = static_cast<int64_t>(a.query_start ? a.query_start[b] : a.start) + min(i0 + 64, a.m) - 1;
        return static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(keys), last + 1)));
    };
    auto from = [&](int64_t b) {
        for (; b < b1; ++b) {
            const int64_t start = a.query_start ? a.query_start[b] : a.start;
            if (j0 < seen_keys(b) && (a.distances == 0 || far_end(a, j0 - (start + min(i0 + 64, a.m) - 1) - a.first,
                                                                  j0 + 63 - (start + i0) - a.first) == 0)) break;
        }
        return b;
    };
    Staged<T, DP, 64, 256> kr, vr;
    typename Frag<T>::Row next_q[DC], next_go[DC];
    float next_top = 0.0f, next_inv = 0.0f, next_delta = 0.0f;
    auto fetch = [&](int64_t b, int keys) {
        const T* k_base = static_cast<const T*>(a.k) + b * a.k_sb + hk * a.k_sh;
        const T* v_base = static_cast<const T*>(a.v) + b * a.v_sb + hk * a.v_sh;
        kr.load(k_base + static_cast<int64_t>(j0) * a.k_sn, a.k_sn, keys - j0, a.dim);
        vr.load(v_base + static_cast<int64_t>(j0) * a.v_sn, a.v_sn, keys - j0, a.dim);
        const T* qp = static_cast<const T*>(a.q) + b * a.q_sb + head * a.q_sh + query * a.q_sm;
        const T* gp = static_cast<const T*>(a.grad) + b * a.g_sb + head * a.g_sh + query * a.g_sm;
#pragma unroll
        for (int dc = 0; dc < DC; ++dc) {
            next_q[dc] = row_frag_global<T>(qp, a.dim, dc, g, valid);
            next_go[dc] = row_frag_global<T>(gp, a.dim, dc, g, valid);
        }
        const int64_t at = (b * a.heads + head) * a.m + query;
        next_top = a.stats[2 * at];
        next_inv = a.stats[2 * at + 1];
        next_delta = a.delta[at];
    };
    // the next sequence arrives while one is worked on, where registers hold both
    constexpr bool AHEAD = sizeof(T) == 2 && DP <= 64;
    int64_t next = from(b0);
    if (AHEAD && next < b1) fetch(next, seen_keys(next));
    while (next < b1) {
        const int64_t b = next;
        const int start = a.query_start ? a.query_start[b] : a.start, keys = seen_keys(b);
        if (!AHEAD) fetch(b, keys);
        __syncthreads();
        kr.put(ks);
        vr.put(vs);
        typename Frag<T>::Row q[DC], go[DC];
#pragma unroll
        for (int dc = 0; dc < DC; ++dc) {
            q[dc] = next_q[dc];
            go[dc] = next_go[dc];
        }
        const float top = next_top, inv = valid ? next_inv : 0.0f, delta = next_delta;
        __syncthreads();
        next = from(b + 1);
        if (AHEAD && next < b1) fetch(next, seen_keys(next));
        const Column col = query_column(a, a.bias_in_lds ? bias_lds : nullptr, b, head, query, start, keys);
        const int64_t pos0 = static_cast<int64_t>(start) + i0, pos1 = static_cast<int64_t>(start) + min(i0 + 64, a.m) - 1;
        const Kind kind = tile_kind<BIASES>(a, j0 + 64 <= keys && (!a.causal || j0 + 63 <= pos0), true, j0 - pos1 - a.first,
                                            j0 + 63 - pos0 - a.first);
        if (busy) by_kind<BIASES>(kind, [&](auto tag) {
        f32x4 s[4], dp[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            s[t] = dp[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if (decltype(tag)::kind == kEdge && 16 * t >= keys - j0) continue;
#pragma unroll
            for (int dc = 0; dc < DC; ++dc) {
                s[t] = mma_row(row_frag<T, DP>(ks, 16 * t + c, dc, g), q[dc], s[t]);
                dp[t] = mma_row(row_frag<T, DP>(vs, 16 * t + c, dc, g), go[dc], dp[t]);
            }
        }
        score_tile<BIASES, decltype(tag)::kind, false>(a, col, j0, g, s);
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float p = valid ? exp2_hw(s[t][r] - top) * inv : 0.0f;
                sum[t][r] += p * (dp[t][r] - delta);
            }
        });
    }
    if (a.distances == 0) {
        float* out = a.partial + ((static_cast<int64_t>(chunk) * a.heads + head) * a.m + query) * a.n;
        if (valid)
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (j0 + 16 * t + 4 * g + r < a.n) out[j0 + 16 * t + 4 * g + r] = sum[t][r];
        return;
    }
    store_diagonals(reinterpret_cast<float*>(smem), sum, wave, c, g,
                    a.partial + (((static_cast<int64_t>(chunk) * a.heads + head) * q_tiles + q_tile) * k_tiles + k_tile) * 128);
}

__device__ __forceinline__ void store_as(void* p, int64_t i, int dtype, float v) {
    if (dtype == TA_NN_F32) static_cast<float*>(p)[i] = v;
    else if (dtype == TA_NN_BF16) static_cast<bf16*>(p)[i] = from_float<bf16>(v);
    else static_cast<fp16*>(p)[i] = from_float<fp16>(v);
}

// Pairs, first: the chunks' sums of every pair, 64 pairs to a workgroup, its four waves a quarter of the chunks each; 64-bit sums,
// rounded to 32 bits over the first chunk's place.  (Reading them bucket by bucket instead touches a line for every value.)
__global__ __launch_bounds__(256) void attention_pair_sums(AttentionArgs a) {
    __shared__ double red[4][64];
    const int64_t pairs = static_cast<int64_t>(a.m) * a.n, tiles = (pairs + 63) / 64;
    const int head = static_cast<int>(blockIdx.x / tiles), wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t pair = blockIdx.x % tiles * 64 + lane;
    double sum = 0.0;
    if (pair < pairs) {
        const float* p = a.partial + head * pairs + pair;
        const int c0 = static_cast<int>(static_cast<int64_t>(a.chunks) * wave / 4), c1 = static_cast<int>(static_cast<int64_t>(a.chunks) * (wave + 1) / 4);
#pragma unroll 8
        for (int chunk = c0; chunk < c1; ++chunk) sum += p[static_cast<int64_t>(chunk) * a.heads * pairs];
    }
    red[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && pair < pairs)
        a.partial[head * pairs + pair] = static_cast<float>(red[0][lane] + red[1][lane] + red[2][lane] + red[3][lane]);
}

// Distances, first: the near tiles' diagonals by distance.  A workgroup has one head and one difference between the numbers of key
// and query tile; thread t adds diagonal t of all such tiles and chunks, in order, in 64 bits.
__global__ __launch_bounds__(128) void attention_distance_sums(AttentionArgs a) {
    const int q_tiles = (a.m + 63) / 64, k_tiles = (a.n + 63) / 64, near = near_tiles(a), offsets = q_tiles + k_tiles - 1;
    const int head = static_cast<int>(blockIdx.x) / offsets, offset = static_cast<int>(blockIdx.x) % offsets - (q_tiles - 1);
    double sum = 0.0;
    for (int q = max(0, -offset); q < q_tiles && q + offset < k_tiles; ++q) {
        const int at = is_window(a) ? 0 : q + offset - first_near_tile(a, 64 * q);
        if (at < 0 || at >= near) continue;
#pragma unroll 4
        for (int chunk = 0; chunk < a.chunks; ++chunk)
            sum += a.partial[(((static_cast<int64_t>(chunk) * a.heads + head) * q_tiles + q) * near + at) * 128 + threadIdx.x];
    }
    a.by_distance[static_cast<int64_t>(blockIdx.x) * 128 + threadIdx.x] = static_cast<float>(sum);
}

// one workgroup for each bucket and head: the sums of its pairs or distances in a fixed order, in 64 bits
__global__ __launch_bounds__(256) void attention_table_sums(AttentionArgs a) {
    __shared__ double red[4];
    const int bucket = static_cast<int>(blockIdx.x) / a.heads, head = static_cast<int>(blockIdx.x) % a.heads;
    double sum = 0.0;
    if (a.distances == 0) {
        const int64_t pairs = static_cast<int64_t>(a.m) * a.n;
        const int from = a.pair_starts[bucket], to = a.pair_starts[bucket + 1];
        for (int e = from + static_cast<int>(threadIdx.x); e < to; e += 256) sum += a.partial[head * pairs + a.pair_order[e]];
    } else {
        const int q_tiles = (a.m + 63) / 64, k_tiles = (a.n + 63) / 64, offsets = q_tiles + k_tiles - 1;
        const int* index = static_cast<const int*>(a.index);
        for (int e = threadIdx.x; e < offsets * 128; e += 256) {
            const int64_t d = static_cast<int64_t>(e / 128 - (q_tiles - 1)) * 64 + (e & 127) - 63 - a.start - a.first;
            const int at = d < 0 ? 0 : d >= a.distances ? a.distances - 1 : static_cast<int>(d);
            if (index[at] == bucket) sum += a.by_distance[static_cast<int64_t>(head) * offsets * 128 + e];
        }
        if (!is_window(a)) {
            const int64_t rows = static_cast<int64_t>(a.batch) * q_tiles;
            for (int end = 0; end < 2; ++end)
                if (index[end == 0 ? 0 : a.distances - 1] == bucket)
                    for (int64_t e = threadIdx.x; e < rows; e += 256)
                        sum += a.far[((e / q_tiles * a.heads + head) * q_tiles + e % q_tiles) * 2 + end];
        }
    }
    sum = block_sum<4>(sum, red);
    if (threadIdx.x == 0) store_as(a.dtable, static_cast<int64_t>(bucket) * a.heads + head, a.table_dtype, static_cast<float>(sum));
}

int launch_table_sums(const AttentionArgs& a, hipStream_t st) {
    if (a.distances == 0) {
        const int64_t blocks = ceil_div(static_cast<int64_t>(a.m) * a.n, 64) * a.heads;
        TA_NN_REQUIRE(blocks <= 0x7FFFFFFF, "%d x %d pairs", a.m, a.n);
        hipLaunchKernelGGL(attention_pair_sums, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st, a);
    } else {
        const int64_t blocks = (ceil_div(a.m, 64) + ceil_div(a.n, 64) - 1) * a.heads;
        TA_NN_REQUIRE(blocks * 128 <= 0x7FFFFFFF, "%d x %d tokens", a.m, a.n);
        hipLaunchKernelGGL(attention_distance_sums, dim3(static_cast<unsigned>(blocks)), dim3(128), 0, st, a);
    }
    hipLaunchKernelGGL(attention_table_sums, dim3(static_cast<unsigned>(a.buckets) * a.heads), dim3(256), 0, st, a);
    return check_launch("ta_nn_attention_backward");
}

template <class T, int DP> int launch_backward(AttentionArgs a, hipStream_t st) {
    const size_t tiles = 2 * 16 * kSubs<DP> * Tile<T, DP>::LD * sizeof(T), table_tiles = 2 * 64 * Tile<T, DP>::LD * sizeof(T);
    const size_t bias = bias_lds_bytes(a, 1);
    const int64_t q_blocks = ceil_div(a.m, 64) * a.heads * a.batch, k_blocks = ceil_div(a.n, 64) * a.kv_heads * a.batch;
    const int64_t t_blocks = ceil_div(a.m, 64) * (a.distances ? near_tiles(a) : ceil_div(a.n, 64)) * a.heads * a.chunks;
    TA_NN_REQUIRE(q_blocks <= 0x7FFFFFFF && k_blocks <= 0x7FFFFFFF && t_blocks <= 0x7FFFFFFF, "too many tokens for one launch");
    // (short calls have one instance, the one that takes any bias)
    if (sizeof(T) == 2 && a.n <= kFewTerms) {
        hipLaunchKernelGGL((attention_bwd_q<T, DP, kAny, sizeof(T) == 2>), dim3(static_cast<unsigned>(q_blocks)), dim3(256), tiles + bias, st, a);
    } else {
        TA_NN_BY_BIASES(a, hipLaunchKernelGGL((attention_bwd_q<T, DP, BIASES, 0>), dim3(static_cast<unsigned>(q_blocks)), dim3(256), tiles + bias, st, a));
    }
    const size_t kv_lds = tiles + 3 * 64 * 4 + bias;
    if (sizeof(T) == 2 && static_cast<int64_t>(a.m) * (a.heads / a.kv_heads) <= kFewTerms) {
        hipLaunchKernelGGL((attention_bwd_kv<T, DP, kAny, sizeof(T) == 2>), dim3(static_cast<unsigned>(k_blocks)), dim3(256), kv_lds, st, a);
    } else {
        TA_NN_BY_BIASES(a, hipLaunchKernelGGL((attention_bwd_kv<T, DP, BIASES, 0>), dim3(static_cast<unsigned>(k_blocks)), dim3(256), kv_lds, st, a));
    }
    if (a.dtable) {
        const size_t diagonals = 64 * 65 * 4;
        const size_t lds = table_tiles + bias > diagonals ? table_tiles + bias : diagonals;
        TA_NN_BY_BIASES(a, hipLaunchKernelGGL((attention_bwd_table<T, DP, BIASES>), dim3(static_cast<unsigned>(t_blocks)), dim3(256), lds, st, a));
        return launch_table_sums(a, st);
    }
    return check_launch("ta_nn_attention_backward");
}

}  // namespace ta_nn

extern "C" int ta_nn_attention_backward(const ta_nn_attention_args* args, void* stream) {
    ta_nn::AttentionArgs a{};
    if (int rc = ta_nn::check_attention(args, a)) return rc;
    TA_NN_REQUIRE(a.grad && a.stats && a.dq && a.dk && a.dv && a.workspace, "null pointer");
    if (a.distances == 0) {
        TA_NN_REQUIRE(a.index_t && a.index_t_stride >= a.m && a.index_t_stride % 4 == 0 && reinterpret_cast<uintptr_t>(a.index_t) % 8 == 0,
                      "transposed index stride %lld of %d queries", static_cast<long long>(a.index_t_stride), a.m);
        TA_NN_REQUIRE(!a.dtable || (a.pair_order && a.pair_starts), "null pointer");
        TA_NN_REQUIRE(!a.dtable || static_cast<int64_t>(a.m) * a.n < 0x7FFFFFFF, "%d x %d pairs", a.m, a.n);
    }
    TA_NN_REQUIRE(!(a.dtable && a.query_start && a.distances), "the table's gradient needs one position of query 0 for all sequences");
    TA_NN_REQUIRE(static_cast<int64_t>(a.buckets) * a.heads <= 0x7FFFFFFF, "%d buckets, %d heads", a.buckets, a.heads);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (ta_nn::is_window(a)) {
        if (int rc = ta_nn::launch_window(a, true, st)) return rc;
        return a.dtable ? ta_nn::launch_table_sums(a, st) : 0;
    }
    TA_NN_BY_TYPE_AND_DIM(a.dtype, a.dim, (ta_nn::launch_backward<T, DP>(a, st)));
}
