// Attention over many short sequences -- the windows of an image, up to 64 tokens -- whose pairs have the same bias, mask and
// visibility in every sequence, or in every mask_period-th.  A workgroup keeps what is added to its 64 x 64 scores in
// registers (16 to a lane), and streams sequences of its head past them: the next arrives in registers while one is worked on.
// Backward computes everything of a sequence at once, scores once instead of once per gradient: probabilities and score
// gradients are transposed through LDS for dk and dv, and score gradients add up in registers over the workgroup's sequences
// for the table.  What bounds it: fp32 products (7 of 64 x 64 x dim a sequence, a tenth of the 16-bit rate, 49 of 64 rows and
// columns in use) and memory alike: 8000 windows x 3 heads of 49 x 32 in fp32 with a mask for each of 64 windows, forward 147 us
// (3.3 TB/s), backward 375 us (2.1 TB/s of q, k, v, gradients and output; matrix units half busy); 32 x 24 without mask, 12.5 us.
#include "attention.h"

namespace ta_nn {

// the workgroup's share: sequences `cls`, + period, ...: numbers [first, last) of that series
struct Share {
    int head, cls, period, first, last, part;
    __device__ __forceinline__ Share(const AttentionArgs& a, int parts) {
        period = a.mask_kind ? a.mask_period : 1;
        const int64_t block = blockIdx.x;
        head = static_cast<int>(block % a.heads);
        cls = static_cast<int>(block / a.heads % period);
        const int p = static_cast<int>(block / a.heads / period);
        part = p * period + cls;
        const int count = (a.batch - cls + period - 1) / period;
        first = static_cast<int>(static_cast<int64_t>(count) * p / parts);
        last = static_cast<int>(static_cast<int64_t>(count) * (p + 1) / parts);
    }
    __device__ __forceinline__ int64_t sequence(int i) const { return cls + static_cast<int64_t>(i) * period; }
};

// what is added to the scores of query 16 wave + c and keys 16 t + 4 g + r, times log2 e; -inf: not seen
__device__ __forceinline__ void window_bias(const AttentionArgs& a, const Share& share, int query, int g, f32x4 (&add)[4]) {
    const Column col = query_column(a, nullptr, share.cls, share.head, min(query, a.m - 1), a.start, a.n);
    u16x4 bucket[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        bucket[t] = u16x4{0, 0, 0, 0};
        if (a.distances == 0 && 16 * t + 4 * g < a.n) bucket[t] = *reinterpret_cast<const u16x4*>(col.pairs + 16 * t + 4 * g);
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int key = 16 * t + 4 * g + r;
            const bool seen = query < a.m && key <= col.bound;
            add[t][r] = seen ? table_value(a, a.distances ? clamp_distance(a, col.from + key) : bucket[t][r], share.head) : -INFINITY;
        }
    if (a.mask_kind) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int key = 16 * t + 4 * g + r;
                if (add[t][r] != -INFINITY) add[t][r] = masked(add[t][r], mask_value(a, col.mask + key * a.mask_sn));
            }
    }
}

template <class T, int DP>
__global__ __launch_bounds__(256, 2) void window_fwd(AttentionArgs a, int parts) {
    constexpr int DC = DP / Frag<T>::D, DT = DP / 16, TILE = 64 * Tile<T, DP>::LD;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    T* tiles = reinterpret_cast<T*>(smem);               // [2][keys, values][64][LD]
    const int tid = threadIdx.x, wave = tid >> 6, c = tid & 15, g = (tid >> 4) & 3;
    const Share share(a, parts);
    if (share.first >= share.last) return;
    const int query = 16 * wave + c;
    const bool valid = query < a.m, active = 16 * wave < a.m;
    Staged<T, DP, 64, 256> kr, vr;
    typename Frag<T>::Row q[DC], q_next[DC];
    auto fetch = [&](int i) {
        if (i >= share.last) return;
        const int64_t b = share.sequence(i);
        kr.load(static_cast<const T*>(a.k) + b * a.k_sb + share.head * a.k_sh, a.k_sn, a.n, a.dim);
        vr.load(static_cast<const T*>(a.v) + b * a.v_sb + share.head * a.v_sh, a.v_sn, a.n, a.dim);
        const T* p = static_cast<const T*>(a.q) + b * a.q_sb + share.head * a.q_sh + (valid ? query : 0) * a.q_sm;
#pragma unroll
        for (int dc = 0; dc < DC; ++dc) q_next[dc] = row_frag_global<T>(p, a.dim, dc, g, valid);
    };
    fetch(share.first);
    f32x4 add[4];
    window_bias(a, share, query, g, add);
    const float scale = a.scale * kLog2e;
    for (int i = share.first, turn = 0; i < share.last; ++i, turn ^= 1) {
        T* ks = tiles + turn * 2 * TILE;
        T* vs = ks + TILE;
        kr.put(ks);                                      // (everyone has left this half: the barrier of the last turn)
        vr.put(vs);
#pragma unroll
        for (int dc = 0; dc < DC; ++dc) q[dc] = q_next[dc];
        __syncthreads();
        fetch(i + 1);
        if (!active) continue;
        f32x4 s[1][4], o[1][DT];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            s[0][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int dc = 0; dc < DC; ++dc) s[0][t] = mma_row(row_frag<T, DP>(ks, 16 * t + c, dc, g), q[dc], s[0][t]);
        }
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[0][t][r] = fmaf(s[0][t][r], scale, add[t][r]);
                top = fmaxf(top, s[0][t][r]);
            }
        top = reduce_rows(top, [](float x, float y) { return fmaxf(x, y); });
        const float m_ref = top == -INFINITY ? 0.0f : top;
        float sum = 0.0f;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[0][t][r] = exp2_hw(s[0][t][r] - m_ref);
                sum += s[0][t][r];
            }
        sum = reduce_rows(sum, Sum{});
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[0][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        mma_transposed<DP, 1, 4, 1>(vs, s, o, c, g);
        if (valid) {
            const int64_t b = share.sequence(i);
            store_column<T, DP>(static_cast<T*>(a.out) + b * a.o_sb + share.head * a.o_sh + query * a.o_sm, o[0], inv, a.dim, g);
            if (a.stats && g == 0) {
                float* st = a.stats + 2 * ((b * a.heads + share.head) * a.m + query);
                st[0] = m_ref;
                st[1] = inv;
            }
        }
    }
}

template <class T, int DP>
__global__ __launch_bounds__(256, 2) void window_bwd(AttentionArgs a, int parts) {
    constexpr int DC = DP / Frag<T>::D, DT = DP / 16, TILE = 64 * Tile<T, DP>::LD;
    constexpr int WLD = 64 + 4;                          // rows of the transposed weights, [key][query], in 32 bits
    extern __shared__ __attribute__((aligned(16))) char smem[];
    T* ks = reinterpret_cast<T*>(smem);
    T* vs = ks + TILE;
    T* qs = vs + TILE;
    T* gs = qs + TILE;
    float* ps = reinterpret_cast<float*>(gs + TILE);
    float* dss = ps + 64 * WLD;
    constexpr float LIFT = 1 << kLift<T>;
    const int tid = threadIdx.x, wave = tid >> 6, c = tid & 15, g = (tid >> 4) & 3;
    const Share share(a, parts);
    const int own = 16 * wave + c;                       // this lane's query, and later its key
    f32x4 table_sum[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) table_sum[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    Staged<T, DP, 64, 256> kr, vr, qr, gr;
    float top_next = 0.0f, inv_next = 0.0f;
    auto fetch = [&](int i) {
        if (i >= share.last) return;
        const int64_t b = share.sequence(i);
        kr.load(static_cast<const T*>(a.k) + b * a.k_sb + share.head * a.k_sh, a.k_sn, a.n, a.dim);
        vr.load(static_cast<const T*>(a.v) + b * a.v_sb + share.head * a.v_sh, a.v_sn, a.n, a.dim);
        qr.load(static_cast<const T*>(a.q) + b * a.q_sb + share.head * a.q_sh, a.q_sm, a.m, a.dim);
        gr.load(static_cast<const T*>(a.grad) + b * a.g_sb + share.head * a.g_sh, a.g_sm, a.m, a.dim);
        const int query = min(own, a.m - 1);
        const int64_t at = (b * a.heads + share.head) * a.m + query;
        top_next = a.stats[2 * at];
        inv_next = a.stats[2 * at + 1];
    };
    fetch(share.first);
    f32x4 add[4];
    window_bias(a, share, own, g, add);
    const float scale = a.scale * kLog2e;
    for (int i = share.first; i < share.last; ++i) {
        const int64_t b = share.sequence(i);
        kr.put(ks);
        vr.put(vs);
        qr.put(qs);
        gr.put(gs);
        const float top = top_next, inv = inv_next;
        __syncthreads();
        fetch(i + 1);
        f32x4 p[4], ds[1][4];
        {
            typename Frag<T>::Row q[DC], go[DC];
#pragma unroll
            for (int dc = 0; dc < DC; ++dc) {
                q[dc] = row_frag<T, DP>(qs, own, dc, g);
                go[dc] = row_frag<T, DP>(gs, own, dc, g);
            }
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                p[t] = ds[0][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int dc = 0; dc < DC; ++dc) {
                    p[t] = mma_row(row_frag<T, DP>(ks, 16 * t + c, dc, g), q[dc], p[t]);
                    ds[0][t] = mma_row(row_frag<T, DP>(vs, 16 * t + c, dc, g), go[dc], ds[0][t]);
                }
            }
            float delta = 0.0f;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    p[t][r] = exp2_hw(fmaf(p[t][r], scale, add[t][r]) - top) * inv;
                    delta += p[t][r] * ds[0][t][r];                               // sum_j p dp is out . grad, unrounded
                }
            delta = reduce_rows(delta, Sum{});
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float w = p[t][r];
                    ds[0][t][r] = w * (ds[0][t][r] - delta);
                    table_sum[t][r] += ds[0][t][r];
                    ps[(16 * t + 4 * g + r) * WLD + own] = w * LIFT;
                    dss[(16 * t + 4 * g + r) * WLD + own] = ds[0][t][r];
                }
        }
        {
            f32x4 dq[1][DT];
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) dq[0][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            float up = kNarrow<T> ? kMostLift : 1.0f;
            if constexpr (kNarrow<T>) into_range(ds[0], dq[0], up);
            mma_transposed<DP, 1, 4, 1>(ks, ds, dq, c, g);
            if (own < a.m)
                store_column<T, DP>(static_cast<T*>(a.dq) + b * a.dq_sb + share.head * a.dq_sh + own * a.dq_sm, dq[0], a.scale * (1.0f / up), a.dim, g);
        }
        __syncthreads();
        {
            f32x4 dk[1][DT], dv[1][DT];
            f32x4 w[1][4];
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) dk[0][dt] = dv[0][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int t = 0; t < 4; ++t) w[0][t] = *reinterpret_cast<const f32x4*>(ps + own * WLD + 16 * t + 4 * g);
            mma_transposed<DP, 1, 4, 1>(gs, w, dv, c, g);
#pragma unroll
            for (int t = 0; t < 4; ++t) w[0][t] = *reinterpret_cast<const f32x4*>(dss + own * WLD + 16 * t + 4 * g);
            float up = kNarrow<T> ? kMostLift : 1.0f;
            if constexpr (kNarrow<T>) into_range(w[0], dk[0], up);
            mma_transposed<DP, 1, 4, 1>(qs, w, dk, c, g);
            if (own < a.n) {
                store_column<T, DP>(static_cast<T*>(a.dk) + b * a.dk_sb + share.head * a.dk_sh + own * a.dk_sn, dk[0], a.scale * (1.0f / up), a.dim, g);
                store_column<T, DP>(static_cast<T*>(a.dv) + b * a.dv_sb + share.head * a.dv_sh + own * a.dv_sn, dv[0], 1.0f / LIFT, a.dim, g);
            }
        }
        __syncthreads();                                 // the tiles are free
    }
    if (a.dtable == nullptr) return;
    const int64_t part = static_cast<int64_t>(share.part) * a.heads + share.head;
    if (a.distances == 0) {
        float* out = a.partial + (part * a.m + own) * a.n;
        if (own < a.m)
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (16 * t + 4 * g + r < a.n) out[16 * t + 4 * g + r] = table_sum[t][r];
        return;
    }
    float* tile = reinterpret_cast<float*>(smem);
    store_diagonals(tile, table_sum, wave, c, g, a.partial + part * 128);
}

template <class T, int DP> int launch_window_by(AttentionArgs a, bool backward, hipStream_t st) {
    const int parts = window_parts(a, backward);
    const int64_t blocks = static_cast<int64_t>(a.heads) * window_periods(a) * parts;
    TA_NN_REQUIRE(blocks <= 0x7FFFFFFF, "too many windows for one launch");
    const size_t tile = 64 * Tile<T, DP>::LD * sizeof(T);
    if (!backward) {
        hipLaunchKernelGGL((window_fwd<T, DP>), dim3(static_cast<unsigned>(blocks)), dim3(256), 4 * tile, st, a, parts);
        return check_launch("ta_nn_attention");
    }
    const size_t lds = 4 * tile + 2 * 64 * (64 + 4) * 4, diagonals = 64 * 65 * 4;
    hipLaunchKernelGGL((window_bwd<T, DP>), dim3(static_cast<unsigned>(blocks)), dim3(256), lds > diagonals ? lds : diagonals, st, a, parts);
    return check_launch("ta_nn_attention_backward");
}

int launch_window(AttentionArgs a, bool backward, hipStream_t st) {
    if (a.dtype == TA_NN_F32) return a.dim <= 32 ? launch_window_by<float, 32>(a, backward, st) : launch_window_by<float, 64>(a, backward, st);
    if (a.dtype == TA_NN_BF16) return a.dim <= 32 ? launch_window_by<bf16, 32>(a, backward, st) : launch_window_by<bf16, 64>(a, backward, st);
    return a.dim <= 32 ? launch_window_by<fp16, 32>(a, backward, st) : launch_window_by<fp16, 64>(a, backward, st);
}

}  // namespace ta_nn
