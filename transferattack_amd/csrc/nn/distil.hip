// Distillation from a teacher's top logits: the teacher's side (ta_nn_top_logits) and the loss with its gradient.
//
// A teacher answers a row with K classes c_k, their logits t_k and, if it can, R = log sum exp(t / T) over all its other
// classes.  With x the student's logits, both at temperature T:
//     p_k = exp(t_k / T) / (sum_j exp(t_j / T) + exp(R))         p_R = exp(R) / (...)      (without R: p_R absent)
//     q_v = exp(x_v / T) / sum_u exp(x_u / T)                     q_R = sum of q_v over v not in {c_k}
//     loss = T^2 (sum_k p_k (log p_k - log q_{c_k}) + p_R (log p_R - log q_R))
//     d loss / d x_v = T (q_v - sum of p_k over c_k = v)          v among the classes answered
//                    = T (q_v - p_R q_v / q_R)                    any other v
// A row's other classes enter through their maximum m and s = sum exp((x_v - m) / T) alone, so one pass over the row gives
// both, and the gradient of every other class is exp((x_v - m) / T) * (q_R - p_R) / s: the difference that cancels is
// taken once per row, in 64 bits, as is everything that concerns the K classes answered (their differences of logarithms
// nearly cancel where the student is close to the teacher).  s is a sum of fp32 terms per thread, added up in 64 bits.
#include "ta_nn_common.h"

namespace ta_nn {

constexpr int kMaxTop = 1024;
constexpr int kMaxClasses = 458752;                      // the marks of the classes answered: one bit each, 56 of 64 KB LDS

struct DistilArgs {
    const void* x;
    int64_t x_stride;
    int classes;
    const float* top_values;
    const void* top_classes;
    int classes64;
    int k;
    const float* rest;
    const float* weight;
    double temperature;
    float factor;                                        // of every row's gradient; times *scale where that is given
    const float* scale;
    const float* upstream;                               // gradient of the loss: one value, or one for each row
    int upstream_per_row;
    float* row_loss;
    float* stats;                                        // [rows][kStats]
    void* grad;
    int64_t grad_stride;
};

constexpr int kStats = 5;                                // m, (q_R - p_R) / s, M = max over all, 1 / Z, whether a class repeats

__device__ __forceinline__ int class_at(const DistilArgs& a, int64_t row, int i) {
    const int64_t at = row * a.k + i;
    if (!a.classes64) return static_cast<const int*>(a.top_classes)[at];
    const int64_t c = static_cast<const int64_t*>(a.top_classes)[at];
    return c < -1 ? -2 : c >= a.classes ? a.classes : static_cast<int>(c);
}

__device__ __forceinline__ double exp_ratio(double x, double m) {      // exp(x - m), 0 where both are -inf
    return x == -INFINITY ? 0.0 : exp(x - m);
}

// ---- the row's elements, VPT 16-byte vectors of a thread kept in registers (VPT = 0: read again in every pass)
template <class T, int THREADS, int VPT> struct Row {
    static constexpr int N = Vec<T>::N;
    const T* p;
    int classes;
    Vec<T> kept[VPT > 0 ? VPT : 1];

    __device__ __forceinline__ int passes() const { return VPT > 0 ? VPT : (classes + THREADS * N - 1) / (THREADS * N); }
    __device__ __forceinline__ static int base(int j) { return (j * THREADS + static_cast<int>(threadIdx.x)) * N; }
    __device__ __forceinline__ Vec<T> fetch(int j) const {
        const int at = base(j);
        Vec<T> r;
        if (at + N <= classes) return load_vec(p + at);
#pragma unroll
        for (int i = 0; i < N; ++i) r.v[i] = at + i < classes ? p[at + i] : from_float<T>(-INFINITY);
        return r;
    }
    __device__ __forceinline__ void init(const T* row, int n) {
        p = row;
        classes = n;
        if (VPT > 0) {
#pragma unroll
            for (int j = 0; j < VPT; ++j) kept[j] = fetch(j);
        }
    }
    __device__ __forceinline__ Vec<T> get(int j) const { return VPT > 0 ? kept[j] : fetch(j); }
};

template <class T> __device__ __forceinline__ void store_part(T* row, int at, int classes, const Vec<T>& v) {
    constexpr int N = Vec<T>::N;
    if (at + N <= classes) {
        store_vec(row + at, v);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (at + i < classes) row[at + i] = v.v[i];
    }
}

template <class T, int THREADS> __device__ __forceinline__ void fill_row(T* row, int classes, float value) {
    Vec<T> v;
#pragma unroll
    for (int i = 0; i < Vec<T>::N; ++i) v.v[i] = from_float<T>(value);
    for (int at = static_cast<int>(threadIdx.x) * Vec<T>::N; at < classes; at += THREADS * Vec<T>::N) store_part(row, at, classes, v);
}

// what the first wave finds out about the classes answered; every lane of it returns the same
struct TopSide {
    double teacher_max, teacher_sum;                     // log p_k = t_k / T - teacher_max - log teacher_sum
    bool any;                                            // at least one bin (a class or the rest)
};

__device__ __forceinline__ TopSide teacher_side(const DistilArgs& a, int64_t row, const int* cls) {
    const int lane = threadIdx.x & 63;
    TopSide r;
    double top = -INFINITY;
    bool any = a.rest != nullptr;
    for (int i = lane; i < a.k; i += 64)
        if (cls[i] >= 0) {
            const double b = static_cast<double>(a.top_values[row * a.k + i]) / a.temperature;
            top = (b > top || b != b) ? b : top;
            any = true;
        }
    if (a.rest != nullptr) {
        const double b = a.rest[row];
        top = (b > top || b != b) ? b : top;
    }
    r.teacher_max = wave_max(top);
    double sum = 0.0;
    for (int i = lane; i < a.k; i += 64)
        if (cls[i] >= 0) sum += exp_ratio(static_cast<double>(a.top_values[row * a.k + i]) / a.temperature, r.teacher_max);
    if (a.rest != nullptr && lane == 0) sum += exp_ratio(a.rest[row], r.teacher_max);
    r.teacher_sum = wave_sum(sum);
    r.any = wave_max(any ? 1.0f : 0.0f) > 0.0f;
    return r;
}

// gradients of the classes answered, by the first wave, over what the pass over the row has written there
template <class T>
__device__ __forceinline__ void top_gradients(const DistilArgs& a, int64_t row, const int* cls, const T* x, T* grad, const TopSide& t,
                                              double m_all, double inv_z, bool repeats, double coef) {
    const int lane = threadIdx.x & 63;
    const double log_teacher = t.teacher_max + log(t.teacher_sum);
    for (int i = lane; i < a.k; i += 64) {
        const int c = cls[i];
        if (c < 0 || c >= a.classes) continue;
        double p = 0.0;
        bool first = true;
        if (!repeats) {
            p = exp_ratio(static_cast<double>(a.top_values[row * a.k + i]) / a.temperature, log_teacher);
        } else {
            for (int j = 0; j < a.k; ++j)
                if (cls[j] == c) {
                    first = first && j >= i;
                    p += exp_ratio(static_cast<double>(a.top_values[row * a.k + j]) / a.temperature, log_teacher);
                }
        }
        if (first) {
            const double q = exp_ratio(static_cast<double>(to_float(x[c])) / a.temperature, m_all / a.temperature) * inv_z;
            grad[c] = from_float<T>(static_cast<float>(coef * (q - p)));
        }
    }
}

// One workgroup a row: loss (times the row's weight) and either the row's statistics for a later gradient, or the gradient.
template <class T, int THREADS, int VPT, bool GRAD>
__global__ __launch_bounds__(THREADS) void distil_rows(DistilArgs a) {
    constexpr int WAVES = THREADS / 64, N = Vec<T>::N;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ float red_f[WAVES];
    __shared__ double red_d[WAVES];
    __shared__ int cls[kMaxTop];
    __shared__ int flags[2];                             // a class out of range, a class given twice
    __shared__ double found[2];                          // gradient's factor of the other classes
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    T* grad = GRAD ? static_cast<T*>(a.grad) + row * a.grad_stride : nullptr;
    const float w = a.weight ? a.weight[row] : 1.0f;
    float* stats = a.stats ? a.stats + row * kStats : nullptr;
    if (w == 0.0f) {                                     // a row that does not count: whatever it holds is not looked at
        if (GRAD) fill_row<T, THREADS>(grad, a.classes, 0.0f);
        if (tid == 0) a.row_loss[row] = 0.0f;
        if (stats && tid < kStats) stats[tid] = 0.0f;
        return;
    }
    unsigned* marks = reinterpret_cast<unsigned*>(smem);
    const int words = (a.classes + 31) / 32;
    Row<T, THREADS, VPT> r;
    r.init(x, a.classes);
    for (int i = tid; i < words; i += THREADS) marks[i] = 0;
    if (tid < 2) flags[tid] = 0;
    __syncthreads();
    for (int i = tid; i < a.k; i += THREADS) {
        const int c = class_at(a, row, i);
        cls[i] = c < -1 || c >= a.classes ? -2 : c;
        if (c < -1 || c >= a.classes) {
            flags[0] = 1;
        } else if (c >= 0) {
            if (atomicOr(&marks[c >> 5], 1u << (c & 31)) >> (c & 31) & 1u) flags[1] = 1;
        }
    }
    __syncthreads();
    const unsigned char* mark_bytes = reinterpret_cast<const unsigned char*>(smem);
    auto marked = [&](int at) -> unsigned {              // the N marks of the vector at `at`
        if (at >= a.classes) return 0u;
        const unsigned b = mark_bytes[at >> 3];
        return N == 8 ? b : (b >> (at & 4)) & 15u;
    };
    // maximum and sum of the other classes
    float m = -INFINITY;
    {
        const int passes = r.passes();
#pragma unroll VPT > 0 ? VPT : 1
        for (int j = 0; j < passes; ++j) {
            const Vec<T> v = r.get(j);
            const unsigned bits = marked(r.base(j));
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float f = (bits >> i & 1u) ? -INFINITY : to_float(v.v[i]);
                m = (f > m || f != f) ? f : m;
            }
        }
    }
    m = block_max<WAVES>(m, red_f);
    const float m_ref = m == -INFINITY ? 0.0f : m;
    const float c2 = static_cast<float>(1.4426950408889634 / a.temperature);
    float part = 0.0f;
    {
        const int passes = r.passes();
#pragma unroll VPT > 0 ? VPT : 1
        for (int j = 0; j < passes; ++j) {
            const Vec<T> v = r.get(j);
            const unsigned bits = marked(r.base(j));
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float e = exp2_hw((to_float(v.v[i]) - m_ref) * c2);
                part += (bits >> i & 1u) ? 0.0f : e;
            }
        }
    }
    const double s = block_sum<WAVES>(static_cast<double>(part), red_d);
    // the classes answered
    const bool bad = flags[0] != 0, repeats = flags[1] != 0;
    TopSide t{};
    double m_all = 0.0, inv_z = 0.0;
    if (tid < 64) {
        const int lane = tid;
        const double T_ = a.temperature;
        t = teacher_side(a, row, cls);
        float top = m;
        for (int i = lane; i < a.k; i += 64)
            if (cls[i] >= 0) {
                const float f = to_float(x[cls[i]]);
                top = (f > top || f != f) ? f : top;
            }
        m_all = wave_max(top);
        double z = 0.0;
        for (int i = lane; i < a.k; i += 64)
            if (cls[i] >= 0) {
                bool first = true;
                if (repeats)
                    for (int j = 0; j < i; ++j) first = first && cls[j] != cls[i];
                if (first) z += exp_ratio(static_cast<double>(to_float(x[cls[i]])) / T_, m_all / T_);
            }
        const double others = m == -INFINITY ? 0.0 : s * exp((static_cast<double>(m) - m_all) / T_);
        z = wave_sum(z) + others;
        if (m_all == -INFINITY) z = NAN;                 // no class has any weight: not a distribution
        const double log_z = log(z), log_teacher = t.teacher_max + log(t.teacher_sum);
        inv_z = 1.0 / z;
        double kl = 0.0;
        for (int i = lane; i < a.k; i += 64)
            if (cls[i] >= 0) {
                const double log_p = static_cast<double>(a.top_values[row * a.k + i]) / T_ - log_teacher;
                const double p = exp(log_p);
                if (p != 0.0) kl += p * (log_p - ((static_cast<double>(to_float(x[cls[i]])) - m_all) / T_ - log_z));
            }
        double p_rest = 0.0;
        if (a.rest != nullptr) {
            const double log_p = a.rest[row] - log_teacher;
            p_rest = exp(log_p);
            if (p_rest != 0.0 && lane == 0) kl += p_rest * (log_p - ((static_cast<double>(m) - m_all) / T_ + log(s) - log_z));
        }
        kl = wave_sum(kl);
        // (q_R - p_R) / s, the factor of exp((x_v - m) / T) in the other classes' gradients
        double kappa = s > 0.0 ? (others * inv_z - p_rest) / s : 0.0;
        if (z != z || m != m || m_all != m_all) kappa = NAN;
        if (!t.any) kl = 0.0, kappa = 0.0, inv_z = 0.0;
        if (bad) kl = NAN, kappa = NAN, inv_z = NAN;
        if (lane == 0) {
            a.row_loss[row] = static_cast<float>(kl * T_ * T_ * static_cast<double>(w));
            if (stats) {
                stats[0] = m_ref;
                stats[1] = static_cast<float>(kappa);
                stats[2] = static_cast<float>(m_all);
                stats[3] = static_cast<float>(inv_z);
                stats[4] = repeats ? 1.0f : 0.0f;
            }
            found[0] = kappa;
        }
    }
    if (!GRAD) return;
    __syncthreads();
    double coef = a.temperature * static_cast<double>(w) * static_cast<double>(a.factor);
    if (a.scale) coef *= static_cast<double>(*a.scale);
    const float each = static_cast<float>(found[0] * coef);
    {
        const int passes = r.passes();
#pragma unroll VPT > 0 ? VPT : 1
        for (int j = 0; j < passes; ++j) {
            const int at = r.base(j);
            if (at >= a.classes) continue;
            const Vec<T> v = r.get(j);
            Vec<T> o;
#pragma unroll
            for (int i = 0; i < N; ++i) o.v[i] = from_float<T>(exp2_hw((to_float(v.v[i]) - m_ref) * c2) * each);
            store_part(grad, at, a.classes, o);
        }
    }
    __syncthreads();                                     // the row's stores are done: the classes answered go over them
    if (tid < 64 && !bad) top_gradients(a, row, cls, x, grad, t, t.any ? m_all : 0.0, inv_z, repeats, t.any ? coef : 0.0);
}

// The gradient from the statistics of the forward pass: one read and one write of the row.
template <class T, int THREADS>
__global__ __launch_bounds__(THREADS) void distil_backward(DistilArgs a) {
    constexpr int N = Vec<T>::N;
    __shared__ int cls[kMaxTop];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    T* grad = static_cast<T*>(a.grad) + row * a.grad_stride;
    const float w = a.weight ? a.weight[row] : 1.0f;
    if (w == 0.0f) {
        fill_row<T, THREADS>(grad, a.classes, 0.0f);
        return;
    }
    const float* stats = a.stats + row * kStats;
    const float m_ref = stats[0], kappa = stats[1], m_all = stats[2], inv_z = stats[3];
    const bool repeats = stats[4] != 0.0f;
    double coef = a.temperature * static_cast<double>(w) * static_cast<double>(a.factor);
    if (a.scale) coef *= static_cast<double>(*a.scale);
    if (a.upstream) coef *= static_cast<double>(a.upstream[a.upstream_per_row ? row : 0]);
    const float each = static_cast<float>(static_cast<double>(kappa) * coef);
    const float c2 = static_cast<float>(1.4426950408889634 / a.temperature);
    for (int i = tid; i < a.k; i += THREADS) {
        const int c = class_at(a, row, i);
        cls[i] = c < -1 || c >= a.classes ? -2 : c;
    }
    for (int at = tid * N; at < a.classes; at += THREADS * N) {
        Vec<T> v, o;
        if (at + N <= a.classes) {
            v = load_vec(x + at);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v.v[i] = at + i < a.classes ? x[at + i] : from_float<T>(0.0f);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) o.v[i] = from_float<T>(exp2_hw((to_float(v.v[i]) - m_ref) * c2) * each);
        store_part(grad, at, a.classes, o);
    }
    __syncthreads();
    if (tid < 64 && inv_z == inv_z && kappa == kappa) {
        const TopSide t = teacher_side(a, row, cls);
        top_gradients(a, row, cls, x, grad, t, t.any ? m_all : 0.0, inv_z, repeats, t.any ? coef : 0.0);
    }
}

// loss = sum of the rows' losses (each times its weight) / total weight, in 64 bits and a fixed order; one workgroup
__global__ __launch_bounds__(1024) void distil_total(const float* row_loss, const float* weight, int64_t rows, int mean, float* loss,
                                                     float* scale) {
    __shared__ double red[16];
    double sum = 0.0, total = 0.0;
    for (int64_t i = threadIdx.x; i < rows; i += 1024) {
        if (row_loss) sum += row_loss[i];
        total += weight ? static_cast<double>(weight[i]) : 1.0;
    }
    sum = block_sum<16>(sum, red);
    total = block_sum<16>(total, red);
    if (threadIdx.x == 0) {
        const double by = !mean ? 1.0 : total != 0.0 ? 1.0 / total : 0.0;       // no row counts: loss and gradient are 0
        if (loss) *loss = total == 0.0 && mean ? 0.0f : static_cast<float>(sum * by);
        if (scale) *scale = static_cast<float>(by);
    }
}

// ---------------------------------------------------------------------------------------------------- the teacher's side
struct TopArgs {
    const void* x;
    int64_t x_stride;
    int classes, k;
    float temperature;
    float* values;
    int64_t* top_classes;
    float* rest;
};

constexpr int kCandidates = 2048;

__device__ __forceinline__ unsigned order_of(float f) {  // whole numbers in the order of the values, +0 = -0, NaN above all
    if (f != f) return 0xFFFFFFFFu;
    const unsigned b = __float_as_uint(f + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// The K largest of a row, equal values by the lowest class, and the log-sum-exp of the others.  A thread's largest element
// is one of the row's: the K-th largest of those maxima is at most the row's K-th largest value, so few elements besides
// the K reach it.  They are collected, each one's rank is the number of collected keys above it (keys are unique: value,
// then class), and nothing is ever sorted.  Rows where too many reach it (long runs of equal values) find the K-th key by
// bisection over its 64 bits instead.
template <class T, int THREADS, int VPT>
__global__ __launch_bounds__(THREADS) void top_logits(TopArgs a) {
    constexpr int WAVES = THREADS / 64, N = Vec<T>::N;
    __shared__ float red_f[WAVES];
    __shared__ double red_d[WAVES];
    __shared__ int red_i[WAVES];
    __shared__ unsigned maxima[THREADS];
    __shared__ uint64_t cand[kCandidates];
    __shared__ int count;
    __shared__ unsigned limit;
    __shared__ uint64_t kth;
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x;
    Row<T, THREADS, VPT> r;
    r.init(static_cast<const T*>(a.x) + row * a.x_stride, a.classes);
    const int passes = r.passes();
    auto key_of = [](float f, int at) { return static_cast<uint64_t>(order_of(f)) << 32 | (0xFFFFFFFFu - static_cast<unsigned>(at)); };
    unsigned top = 0;                                    // below every value's key
#pragma unroll VPT > 0 ? VPT : 1
    for (int j = 0; j < passes; ++j) {
        const Vec<T> v = r.get(j);
        const int at = r.base(j);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const unsigned o = order_of(to_float(v.v[i]));
            if (at + i < a.classes && o > top) top = o;
        }
    }
    maxima[tid] = top;
    if (tid == 0) count = 0;
    __syncthreads();
    if (tid < 64) {
        unsigned mine[WAVES];
#pragma unroll
        for (int w = 0; w < WAVES; ++w) mine[w] = maxima[64 * w + tid];
        unsigned found = 0;
        for (int bit = 31; bit >= 8; --bit) {            // the low bits only make the limit sharper than it needs to be
            const unsigned trial = found | 1u << bit;
            int n = 0;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) n += __popcll(__ballot(mine[w] >= trial));
            if (n >= a.k) found = trial;
        }
        if (tid == 0) limit = found == 0 ? 1u : found;
    }
    __syncthreads();
    const unsigned from = limit;
#pragma unroll VPT > 0 ? VPT : 1
    for (int j = 0; j < passes; ++j) {
        const Vec<T> v = r.get(j);
        const int at = r.base(j);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float f = to_float(v.v[i]);
            if (at + i < a.classes && order_of(f) >= from) {
                const int slot = atomicAdd(&count, 1);
                if (slot < kCandidates) cand[slot] = key_of(f, at + i);
            }
        }
    }
    __syncthreads();
    int have = count;
    if (have > kCandidates) {
        uint64_t found = 0;
        for (int bit = 63; bit >= 0; --bit) {
            const uint64_t trial = found | 1ull << bit;
            int n = 0;
            for (int j = 0; j < passes; ++j) {
                const Vec<T> v = r.fetch(j);
                const int at = r.base(j);
                for (int i = 0; i < N; ++i) n += at + i < a.classes && key_of(to_float(v.v[i]), at + i) >= trial ? 1 : 0;
            }
            if (block_sum<WAVES>(n, red_i) >= a.k) found = trial;
        }
        if (tid == 0) count = 0;
        __syncthreads();
        for (int j = 0; j < passes; ++j) {
            const Vec<T> v = r.fetch(j);
            const int at = r.base(j);
            for (int i = 0; i < N; ++i) {
                const uint64_t key = key_of(to_float(v.v[i]), at + i);
                if (at + i < a.classes && key >= found) {
                    const int slot = atomicAdd(&count, 1);
                    if (slot < kCandidates) cand[slot] = key;
                }
            }
        }
        __syncthreads();
        have = min(count, kCandidates);                  // exactly K: the keys are unique
    }
    for (int i = tid; i < have; i += THREADS) {
        const uint64_t key = cand[i];
        int rank = 0;
        for (int j = 0; j < have; ++j) rank += cand[j] > key ? 1 : 0;
        if (rank < a.k) {
            const int c = static_cast<int>(0xFFFFFFFFu - static_cast<unsigned>(key));
            a.values[row * a.k + rank] = to_float(r.p[c]);
            a.top_classes[row * a.k + rank] = c;
            if (rank == a.k - 1) kth = key;
        }
    }
    if (a.rest == nullptr) return;
    __syncthreads();
    const uint64_t last = kth;
    float m = -INFINITY;
#pragma unroll VPT > 0 ? VPT : 1
    for (int j = 0; j < passes; ++j) {
        const Vec<T> v = r.get(j);
        const int at = r.base(j);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float f = to_float(v.v[i]);
            if (at + i < a.classes && key_of(f, at + i) < last) m = (f > m || f != f) ? f : m;
        }
    }
    m = block_max<WAVES>(m, red_f);
    const float m_ref = m == -INFINITY ? 0.0f : m;
    const float c2 = static_cast<float>(1.4426950408889634 / static_cast<double>(a.temperature));
    float part = 0.0f;
#pragma unroll VPT > 0 ? VPT : 1
    for (int j = 0; j < passes; ++j) {
        const Vec<T> v = r.get(j);
        const int at = r.base(j);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float f = to_float(v.v[i]);
            const float e = exp2_hw((f - m_ref) * c2);
            part += at + i < a.classes && key_of(f, at + i) < last ? e : 0.0f;
        }
    }
    const double s = block_sum<WAVES>(static_cast<double>(part), red_d);
    if (tid == 0) a.rest[row] = static_cast<float>(static_cast<double>(m_ref) / static_cast<double>(a.temperature) + log(s));
}

// ------------------------------------------------------------------------------------------------------------- launches
template <class T, bool GRAD> int launch_rows(const DistilArgs& a, int64_t rows, hipStream_t st) {
    const int vectors = static_cast<int>(ceil_div(a.classes, Vec<T>::N));
    const size_t lds = static_cast<size_t>(ceil_div(a.classes, 32)) * 4;
    const dim3 grid(static_cast<unsigned>(rows));
    if (vectors <= 64 * 4) hipLaunchKernelGGL((distil_rows<T, 64, 4, GRAD>), grid, dim3(64), lds, st, a);
    else if (vectors <= 256 * 4) hipLaunchKernelGGL((distil_rows<T, 256, 4, GRAD>), grid, dim3(256), lds, st, a);
    else if (vectors <= 512 * 8) hipLaunchKernelGGL((distil_rows<T, 512, 8, GRAD>), grid, dim3(512), lds, st, a);
    else if (vectors <= 1024 * 8) hipLaunchKernelGGL((distil_rows<T, 1024, 8, GRAD>), grid, dim3(1024), lds, st, a);
    else hipLaunchKernelGGL((distil_rows<T, 1024, 0, GRAD>), grid, dim3(1024), lds, st, a);
    return check_launch("ta_nn_distil");
}

template <class T> int launch_backward(const DistilArgs& a, int64_t rows, hipStream_t st) {
    const dim3 grid(static_cast<unsigned>(rows));
    if (a.classes <= 64 * 32) hipLaunchKernelGGL((distil_backward<T, 64>), grid, dim3(64), 0, st, a);
    else if (a.classes <= 256 * 64) hipLaunchKernelGGL((distil_backward<T, 256>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((distil_backward<T, 1024>), grid, dim3(1024), 0, st, a);
    return check_launch("ta_nn_distil_backward");
}

template <class T> int launch_top(const TopArgs& a, int64_t rows, hipStream_t st) {
    const int vectors = static_cast<int>(ceil_div(a.classes, Vec<T>::N));
    const dim3 grid(static_cast<unsigned>(rows));
    if (vectors <= 64 * 4) hipLaunchKernelGGL((top_logits<T, 64, 4>), grid, dim3(64), 0, st, a);
    else if (vectors <= 256 * 4) hipLaunchKernelGGL((top_logits<T, 256, 4>), grid, dim3(256), 0, st, a);
    else if (vectors <= 512 * 8) hipLaunchKernelGGL((top_logits<T, 512, 8>), grid, dim3(512), 0, st, a);
    else if (vectors <= 1024 * 8) hipLaunchKernelGGL((top_logits<T, 1024, 8>), grid, dim3(1024), 0, st, a);
    else hipLaunchKernelGGL((top_logits<T, 1024, 0>), grid, dim3(1024), 0, st, a);
    return check_launch("ta_nn_top_logits");
}

static int check_rows(const DistilArgs& a, int64_t rows) {
    TA_NN_REQUIRE(a.x && a.top_values && a.top_classes, "null pointer");
    TA_NN_REQUIRE(rows >= 1 && rows <= 0x7FFFFFFF, "rows %lld", static_cast<long long>(rows));
    TA_NN_REQUIRE(a.classes >= 1 && a.classes <= kMaxClasses, "classes %d (1 .. %d)", a.classes, kMaxClasses);
    TA_NN_REQUIRE(a.k >= 1 && a.k <= kMaxTop, "top classes %d (1 .. %d)", a.k, kMaxTop);
    TA_NN_REQUIRE(a.x_stride >= a.classes, "row stride %lld of %d classes", static_cast<long long>(a.x_stride), a.classes);
    TA_NN_REQUIRE(a.temperature > 0.0 && a.temperature < INFINITY, "temperature %g", a.temperature);
    return 0;
}

}  // namespace ta_nn

#define TA_NN_BY_TYPE(dtype, call)                                        \
    switch (dtype) {                                                      \
        case TA_NN_F32: { using T = float; return call; }                 \
        case TA_NN_BF16: { using T = ta_nn::bf16; return call; }          \
        case TA_NN_F16: { using T = ta_nn::fp16; return call; }           \
    }                                                                     \
    ta_nn::set_error("element type %d", dtype);                           \
    return TA_NN_EINVAL

extern "C" int ta_nn_top_logits(const void* x, int dtype, int64_t x_stride, int64_t rows, int classes, int k, float temperature,
                                float* values, int64_t* top_classes, float* rest, void* stream) {
    TA_NN_REQUIRE(x && values && top_classes, "null pointer");
    TA_NN_REQUIRE(rows >= 1 && rows <= 0x7FFFFFFF, "rows %lld", static_cast<long long>(rows));
    TA_NN_REQUIRE(classes >= 1 && x_stride >= classes, "%d classes, row stride %lld", classes, static_cast<long long>(x_stride));
    TA_NN_REQUIRE(k >= 1 && k <= classes && k <= ta_nn::kMaxTop, "%d of %d classes (at most %d)", k, classes, ta_nn::kMaxTop);
    TA_NN_REQUIRE(temperature > 0.0f && temperature < INFINITY, "temperature %g", static_cast<double>(temperature));
    const ta_nn::TopArgs a{x, x_stride, classes, k, temperature, values, top_classes, rest};
    TA_NN_BY_TYPE(dtype, ta_nn::launch_top<T>(a, rows, static_cast<hipStream_t>(stream)));
}

extern "C" int ta_nn_distil(const void* x, int dtype, int64_t x_stride, int64_t rows, int classes, const float* top_values,
                            const void* top_classes, int classes64, int k, const float* rest, const float* weight, double temperature,
                            float factor, const float* scale, float* row_loss, float* stats, void* grad, int64_t grad_stride,
                            void* stream) {
    const ta_nn::DistilArgs a{x, x_stride, classes, top_values, top_classes, classes64, k, rest, weight, temperature, factor,
                              scale, nullptr, 0, row_loss, stats, grad, grad_stride};
    if (int rc = ta_nn::check_rows(a, rows)) return rc;
    TA_NN_REQUIRE(row_loss, "null pointer");
    TA_NN_REQUIRE(!grad || grad_stride >= classes, "gradient row stride %lld of %d classes", static_cast<long long>(grad_stride), classes);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (grad) {
        TA_NN_BY_TYPE(dtype, (ta_nn::launch_rows<T, true>(a, rows, st)));
    }
    TA_NN_BY_TYPE(dtype, (ta_nn::launch_rows<T, false>(a, rows, st)));
}

extern "C" int ta_nn_distil_backward(const void* x, int dtype, int64_t x_stride, int64_t rows, int classes, const float* top_values,
                                     const void* top_classes, int classes64, int k, const float* rest, const float* weight,
                                     double temperature, float factor, const float* scale, const float* upstream, int upstream_per_row,
                                     const float* stats, void* grad, int64_t grad_stride, void* stream) {
    const ta_nn::DistilArgs a{x, x_stride, classes, top_values, top_classes, classes64, k, rest, weight, temperature, factor,
                              scale, upstream, upstream_per_row, nullptr, const_cast<float*>(stats), grad, grad_stride};
    if (int rc = ta_nn::check_rows(a, rows)) return rc;
    TA_NN_REQUIRE(stats && grad && upstream, "null pointer");
    TA_NN_REQUIRE(grad_stride >= classes, "gradient row stride %lld of %d classes", static_cast<long long>(grad_stride), classes);
    TA_NN_BY_TYPE(dtype, (ta_nn::launch_backward<T>(a, rows, static_cast<hipStream_t>(stream))));
}

extern "C" int ta_nn_distil_total(const float* row_loss, const float* weight, int64_t rows, int mean, float* loss, float* scale,
                                  void* stream) {
    TA_NN_REQUIRE(rows >= 1, "rows %lld", static_cast<long long>(rows));
    TA_NN_REQUIRE((row_loss && loss) || scale, "null pointer");
    hipLaunchKernelGGL(ta_nn::distil_total, dim3(1), dim3(1024), 0, static_cast<hipStream_t>(stream), row_loss, weight, rows, mean,
                       row_loss ? loss : nullptr, scale);
    return ta_nn::check_launch("ta_nn_distil_total");
}
