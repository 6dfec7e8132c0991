// Distillation from a teacher's top logits: the teacher's side (ta_nn_top_logits) and the loss with its gradient.
//
// A teacher answers a row with K classes c_k, their logits t_k and, if it can, R = log sum exp(t / T) over all its other
// classes.  With x the student's logits, both at temperature T:
//     p_k = exp(t_k / T) / (sum_j exp(t_j / T) + exp(R))         p_R = exp(R) / (...)      (without R: p_R absent)
//     q_v = exp(x_v / T) / sum_u exp(x_u / T)                     q_R = sum of q_v over v not in {c_k}
//     loss = T^2 (sum_k p_k (log p_k - log q_{c_k}) + p_R (log p_R - log q_R))
//     d loss / d x_v = T (q_v - sum of p_k over c_k = v)          v among the classes answered
//                    = T (q_v - p_R q_v / q_R)                    any other v
// A row's other classes enter through s = sum exp((x_v - m) / T) alone, m near their maximum, so one pass over the row is all
// it takes, and the gradient of every other class is exp((x_v - m) / T) * (q_R - p_R) / s: the difference that cancels is
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

// m, (q_R - p_R) / s, M = max over all, 1 / Z in two parts (q - p of a class answered nearly cancels near the teacher), the first one
// negative where a class repeats
constexpr int kStats = 5;

__device__ __forceinline__ int class_at(const DistilArgs& a, int64_t row, int i) {
    const int64_t at = row * a.k + i;
    if (!a.classes64) return static_cast<const int*>(a.top_classes)[at];
    const int64_t c = static_cast<const int64_t*>(a.top_classes)[at];
    return c < -1 ? -2 : c >= a.classes ? a.classes : static_cast<int>(c);
}

__device__ __forceinline__ double exp_ratio(double x, double m) {      // exp(x - m), 0 where both are -inf
    return x == -INFINITY ? 0.0 : exp(x - m);
}

// ---- a row: whole 16-byte vectors, VPT of a thread kept in registers (VPT = 0: read again in every pass), and the up to seven
// elements behind them, one to a thread.  What a thread has no element for is -inf.  Loads past the row read its last whole
// vector instead and are replaced afterwards, so that none waits on a branch.
template <class T, int THREADS, int VPT> struct Row {
    static constexpr int N = Vec<T>::N;
    const T* p;
    int classes, full;
    Vec<T> kept[VPT > 0 ? VPT : 1];
    float tail;                                          // element full + thread

    __device__ __forceinline__ int passes() const { return VPT > 0 ? VPT : (full + THREADS * N - 1) / (THREADS * N); }
    __device__ __forceinline__ static int base(int j) { return (j * THREADS + static_cast<int>(threadIdx.x)) * N; }
    __device__ __forceinline__ int tail_class() const { return full + static_cast<int>(threadIdx.x); }
    __device__ __forceinline__ bool has_tail() const { return tail_class() < classes; }
    __device__ __forceinline__ Vec<T> fetch(int j) const {
        const unsigned fill = sizeof(T) == 4 ? lowest_bits<T>() : lowest_bits<T>() * 0x10001u;
        Vec<T> r{u32x4{fill, fill, fill, fill}};
        if (full > 0) {                                  // (the same for the whole grid)
            const int at = base(j);
            const Vec<T> v = load_vec(p + min(at, full - N));
#pragma unroll
            for (int i = 0; i < 4; ++i) r.raw[i] = at < full ? v.raw[i] : fill;
        }
        return r;
    }
    __device__ __forceinline__ void init(const T* row, int n) {
        p = row;
        classes = n;
        full = n / N * N;
        if (VPT > 0) {
#pragma unroll
            for (int j = 0; j < VPT; ++j) kept[j] = fetch(j);
        }
        tail = has_tail() ? to_float(p[tail_class()]) : -INFINITY;
    }
    __device__ __forceinline__ Vec<T> get(int j) const { return VPT > 0 ? kept[j] : fetch(j); }
    // between passes: unpacked elements of the last one are not carried to the next (they would take twice the registers)
    __device__ __forceinline__ void forget_unpacked() {
        if (VPT > 0) {
#pragma unroll
            for (int j = 0; j < VPT; ++j) forget(kept[j].raw);
        }
    }
};

template <class T, int THREADS> __device__ __forceinline__ void fill_row(T* row, int classes, float value) {
    constexpr int N = Vec<T>::N;
    float f[N];
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = value;
    const Vec<T> v = pack<T>(f);
    const int full = classes / N * N;
    for (int at = static_cast<int>(threadIdx.x) * N; at < full; at += THREADS * N) store_vec(row + at, v);
    if (full + static_cast<int>(threadIdx.x) < classes) row[full + threadIdx.x] = from_float<T>(value);
}

// What concerns the classes answered: the first wave's work, in 64 bits; every lane returns the same.
struct TopSide {
    double log_teacher;                                  // log p_k = t_k / T - log_teacher, log p_R = R - log_teacher
    double p_rest, log_p_rest;
    double mass;                                         // sum of p_k
    double x_max, x_sum;                                 // over the student's logits there: maximum, sum exp((x - x_max) / T)
    double cross;                                        // sum_k p_k (log p_k - (x_k - x_max) / T)
    bool any;                                            // at least one bin (a class or the rest)
};

template <class T>
__device__ __forceinline__ TopSide top_side(const DistilArgs& a, int64_t row, const int* cls, const T* x, bool repeats) {
    const int lane = threadIdx.x & 63;
    const double per_t = 1.0 / a.temperature;
    const float* values = a.top_values + row * a.k;
    TopSide r;
    double top = -INFINITY, x_top = -INFINITY;
    bool any = false;
    for (int i = lane; i < a.k; i += 64)
        if (cls[i] >= 0) {
            const double b = static_cast<double>(values[i]) * per_t, f = to_float(x[cls[i]]);
            top = (b > top || b != b) ? b : top;
            x_top = (f > x_top || f != f) ? f : x_top;
            any = true;
        }
    const double rest = a.rest ? static_cast<double>(a.rest[row]) : -INFINITY;
    top = (rest > top || rest != rest) ? rest : top;
    top = wave_max(top);
    r.x_max = wave_max(x_top);
    r.any = a.rest != nullptr || __ballot(any) != 0;
    double sum = 0.0, x_sum = 0.0;
    for (int i = lane; i < a.k; i += 64)
        if (cls[i] >= 0) {
            sum += exp_ratio(static_cast<double>(values[i]) * per_t, top);
            bool first = true;
            if (repeats)
                for (int j = 0; j < i; ++j) first = first && cls[j] != cls[i];
            if (first) x_sum += exp_ratio(static_cast<double>(to_float(x[cls[i]])) * per_t, r.x_max * per_t);
        }
    if (lane == 0) sum += exp_ratio(rest, top);
    r.x_sum = wave_sum(x_sum);
    r.log_teacher = top + log(wave_sum(sum));
    double mass = 0.0, cross = 0.0;
    for (int i = lane; i < a.k; i += 64)
        if (cls[i] >= 0) {
            const double log_p = static_cast<double>(values[i]) * per_t - r.log_teacher, p = exp(log_p);
            mass += p;
            if (p != 0.0) cross += p * (log_p - (static_cast<double>(to_float(x[cls[i]])) - r.x_max) * per_t);
        }
    r.mass = wave_sum(mass);
    r.cross = wave_sum(cross);
    if (r.x_max == -INFINITY && r.any) r.cross = r.mass > 0.0 ? INFINITY : 0.0;      // the student rules all of them out
    r.log_p_rest = rest - r.log_teacher;
    r.p_rest = a.rest ? exp(r.log_p_rest) : 0.0;
    return r;
}

// gradients of the classes answered, by the first wave, over what the pass over the row has written there
template <class T>
__device__ __forceinline__ void top_gradients(const DistilArgs& a, int64_t row, const int* cls, const T* x, T* grad, double log_teacher,
                                              double m_all, double inv_z, bool repeats, double coef) {
    const int lane = threadIdx.x & 63;
    const double per_t = 1.0 / a.temperature;
    const float* values = a.top_values + row * a.k;
    for (int i = lane; i < a.k; i += 64) {
        const int c = cls[i];
        if (c < 0) continue;
        double p = 0.0;
        bool first = true;
        if (!repeats) {
            p = exp_ratio(static_cast<double>(values[i]) * per_t, log_teacher);
        } else {
            for (int j = 0; j < a.k; ++j)
                if (cls[j] == c) {
                    first = first && j >= i;
                    p += exp_ratio(static_cast<double>(values[j]) * per_t, log_teacher);
                }
        }
        if (first) {
            const double q = exp_ratio(static_cast<double>(to_float(x[c])) * per_t, m_all * per_t) * inv_z;
            grad[c] = from_float<T>(static_cast<float>(coef * (q - p)));
        }
    }
}

// One workgroup a row: loss (times the row's weight) and either the row's statistics for a later gradient, or the gradient.
// The vector units are what limits this: with 32 000 classes there is time for some 25 operations an element at the memory's
// rate, an exponential being four.  So the classes answered are set to -inf where the row lies in registers, once, instead of
// being asked for in every pass; the exponentials take their place there (as far as there is room) and the gradient is a product.
// Measured: loss and gradient of 8192 x 32768 bf16 against 32 classes, 243 us (4.4 TB/s; a large copy reaches 5.0); statistics of
// 4095 x 21841 fp32 against 17, 123 us (2.9 TB/s).
template <class T, int THREADS, int VPT, bool GRAD>
__global__ __launch_bounds__(THREADS, 4) void distil_rows(DistilArgs a) {
    constexpr int WAVES = THREADS / 64, N = Vec<T>::N;
    constexpr bool KEEP = GRAD && VPT > 0 && VPT <= 8;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ float red_f[WAVES];
    __shared__ double red_d[WAVES];
    __shared__ int cls[kMaxTop];
    __shared__ int flags[2];                             // a class out of range, a class given twice
    __shared__ float other_factor;
    __shared__ TopSide side;                             // (in registers it would stand beside the row)
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
    const bool bad = flags[0] != 0, repeats = flags[1] != 0;
    if (tid < 64) {
        const TopSide t = top_side(a, row, cls, x, repeats);
        if (tid == 0) side = t;
        wave_lds_order();                                // only this wave reads it, in workgroups of one wave without a barrier between
    }
    const unsigned char* mark_bytes = reinterpret_cast<const unsigned char*>(smem);
    auto unmarked = [&](int j, Vec<T> v) -> Vec<T> {     // the classes answered are not among the others
        const int at = r.base(j);
        if (at < r.full) {
            const unsigned b = mark_bytes[at >> 3];
            const unsigned bits = N == 8 ? b : (b >> (at & 4)) & 15u;
            if (bits != 0) {
#pragma unroll
                for (int i = 0; i < N; ++i) set_bits(v, i, bits >> i & 1u ? lowest_bits<T>() : bits_of(element(v, i)));
            }
        }
        return v;
    };
    // maximum and sum of the other classes.  A NaN is passed over by the maximum and found by the sum.
    const int passes = r.passes();
    if (r.has_tail() && (marks[r.tail_class() >> 5] >> (r.tail_class() & 31) & 1u)) r.tail = -INFINITY;
    float m = r.tail;
#pragma unroll VPT > 0 ? VPT : 1
    for (int j = 0; j < passes; ++j) {
        const Vec<T> v = unmarked(j, r.get(j));
        if constexpr (VPT > 0) r.kept[j] = v;
#pragma unroll
        for (int i = 0; i < N; ++i) m = fmaxf(m, get(v, i));
    }
    r.forget_unpacked();
    m = block_max<WAVES>(m, red_f);
    // exponentials are taken as 2^((x - m) c), the difference first: 2^(x c - m c) would be one product-sum, but the rounding of m c
    // is as large as the exponent itself where every other class holds a masking constant (-1e10 and below)
    const float c2 = static_cast<float>(1.4426950408889634 / a.temperature);
    const float ref = m == -INFINITY ? 0.0f : m;
    r.tail = exp2_hw((r.tail - ref) * c2);
    float part = r.tail;
    float kept[KEEP ? VPT : 1][N];
#pragma unroll VPT > 0 ? VPT : 1
    for (int j = 0; j < passes; ++j) {
        const Vec<T> v = VPT > 0 ? r.get(j) : unmarked(j, r.get(j));
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float e = exp2_hw((get(v, i) - ref) * c2);
            sum += e;
            if constexpr (KEEP) kept[j][i] = e;
        }
        part += sum;
    }
    r.forget_unpacked();
    const double s = block_sum<WAVES>(static_cast<double>(part), red_d);
    double m_all = 0.0, inv_z = 0.0;
    double coef = 0.0;
    if (GRAD) {
        coef = a.temperature * static_cast<double>(w) * static_cast<double>(a.factor);
        if (a.scale) coef *= static_cast<double>(*a.scale);
    }
    if (tid < 64) {
        const TopSide t = side;
        const double per_t = 1.0 / a.temperature;
        m_all = (m > t.x_max || t.x_max != t.x_max) ? static_cast<double>(m) : t.x_max;
        if (t.x_max != t.x_max) m_all = t.x_max;
        // s is relative to exp(m / T): to exp(m_all / T) instead
        const double shift = m == -INFINITY ? -INFINITY : (static_cast<double>(m) - m_all) * per_t;
        const double others = s == 0.0 ? 0.0 : s * exp(shift);
        double z = others + (t.x_sum == 0.0 ? 0.0 : t.x_sum * exp((t.x_max - m_all) * per_t));
        if (m_all == -INFINITY) z = NAN;                 // no class has any weight: not a distribution
        const double log_z = log(z);
        inv_z = 1.0 / z;
        double kl = t.cross == INFINITY ? INFINITY : t.cross + (t.mass == 0.0 ? 0.0 : t.mass * ((m_all - t.x_max) * per_t + log_z));
        if (t.p_rest != 0.0) kl += t.p_rest * (t.log_p_rest - (shift + log(s) - log_z));
        // (q_R - p_R) / s, the factor of the exponentials in the other classes' gradients
        double kappa = s == 0.0 ? 0.0 : (others * inv_z - t.p_rest) / s;
        if (z != z) kl = NAN, kappa = NAN;
        if (!t.any) kl = 0.0, kappa = 0.0, inv_z = 0.0;
        if (bad) kl = NAN, kappa = NAN, inv_z = NAN;
        if (tid == 0) {
            a.row_loss[row] = static_cast<float>(kl * a.temperature * a.temperature * static_cast<double>(w));
            if (stats) {
                stats[0] = ref;
                stats[1] = static_cast<float>(kappa);
                stats[2] = static_cast<float>(m_all);
                const float high = static_cast<float>(inv_z);
                stats[3] = repeats ? -high : high;
                stats[4] = static_cast<float>(inv_z - static_cast<double>(high));
            }
            other_factor = static_cast<float>(kappa * coef);
        }
    }
    if constexpr (GRAD) {
        __syncthreads();
        const float each = other_factor;
#pragma unroll VPT > 0 ? VPT : 1
        for (int j = 0; j < passes; ++j) {
            const int at = r.base(j);
            if (at >= r.full) continue;
            float o[N];
            const Vec<T> v = KEEP ? Vec<T>{} : r.get(j);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float e;
                if constexpr (KEEP) e = kept[j][i];
                else e = exp2_hw((get(v, i) - ref) * c2);
                o[i] = e * each;
            }
            store_vec(grad + at, pack<T>(o));
        }
        if (r.has_tail()) grad[r.tail_class()] = from_float<T>(r.tail * each);
        __syncthreads();                                 // the row's stores are done: the classes answered go over them
        if (tid < 64 && !bad) top_gradients(a, row, cls, x, grad, side.log_teacher, side.any ? m_all : 0.0, inv_z, repeats, side.any ? coef : 0.0);
    }
}

// The gradient from the statistics of the forward pass: one read and one write of the row.  4095 x 21841 fp32, 110 us (6.5 TB/s, part
// of the row still in the cache that the forward pass left).
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
    const float ref = stats[0], kappa = stats[1], m_all = stats[2];
    const bool repeats = stats[3] < 0.0f;
    const double inv_z = static_cast<double>(fabsf(stats[3])) + static_cast<double>(stats[4]);
    double coef = a.temperature * static_cast<double>(w) * static_cast<double>(a.factor);
    if (a.scale) coef *= static_cast<double>(*a.scale);
    if (a.upstream) coef *= static_cast<double>(a.upstream[a.upstream_per_row ? row : 0]);
    const float each = static_cast<float>(static_cast<double>(kappa) * coef);
    const float c2 = static_cast<float>(1.4426950408889634 / a.temperature);
    for (int i = tid; i < a.k; i += THREADS) {
        const int c = class_at(a, row, i);
        cls[i] = c < -1 || c >= a.classes ? -2 : c;
    }
    const int full = a.classes / N * N;
#pragma unroll 4
    for (int at = tid * N; at < full; at += THREADS * N) {
        const Vec<T> v = load_vec(x + at);
        float o[N];
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = exp2_hw((get(v, i) - ref) * c2) * each;
        store_vec(grad + at, pack<T>(o));
    }
    if (full + tid < a.classes) grad[full + tid] = from_float<T>(exp2_hw((to_float(x[full + tid]) - ref) * c2) * each);
    __syncthreads();
    if (tid < 64 && inv_z == inv_z && kappa == kappa) {
        const TopSide t = top_side(a, row, cls, x, repeats);
        top_gradients(a, row, cls, x, grad, t.log_teacher, t.any ? m_all : 0.0, inv_z, repeats, t.any ? coef : 0.0);
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

constexpr int kCandidates = 1280, kHits = 384;         // at least kMaxTop of the former

__device__ __forceinline__ unsigned order_of(float f) {  // whole numbers in the order of the values, +0 = -0, NaN above all
    if (f != f) return 0xFFFFFFFFu;
    const unsigned b = __float_as_uint(f + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ uint64_t key_of(float f, int at) {          // unique: value, then the lowest class
    return static_cast<uint64_t>(order_of(f)) << 32 | (0xFFFFFFFFu - static_cast<unsigned>(at));
}

__device__ __forceinline__ float value_of_order(unsigned o) {          // the inverse, for numbers no NaN has
    if (o < 0x00800000u) return -INFINITY;
    return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}

// The K largest of a row, equal values by the lowest class, and the log-sum-exp of the others.  A thread's largest element
// is one of the row's: the K-th largest of those maxima is at most the row's K-th largest value, so few elements besides
// the K reach it.  They are collected, each one's rank is the number of collected keys above it (keys are unique), and
// nothing is ever sorted.  Rows where too many reach it (long runs of equal values) and rows with a NaN find the K-th key by
// bisection over its 64 bits, reading the row again for each.
// In the common case an element is looked at twice in registers: for its vector's maximum and for its exponential.  Vectors that
// reach the limit, one or two for each of the K, are copied to LDS and leave the row; their elements get a thread each.
// Measured: 64 of 65536 bf16, 4096 rows, 174 us (3.1 TB/s: vector units and the first wave's ranking, several rows to a CU at
// different stages); 5 of 1000 fp32, 32 rows, 5.6 us, most of it the launch and one row's chain of dependent steps.
template <class T, int THREADS, int VPT>
__global__ __launch_bounds__(THREADS, 4) void top_logits(TopArgs a) {
    constexpr int WAVES = THREADS / 64, N = Vec<T>::N, KEPT = VPT > 0 ? VPT : 1;
    __shared__ float red_f[WAVES];
    __shared__ double red_d[WAVES];
    __shared__ int red_i[WAVES];
    __shared__ float maxima[THREADS];
    __shared__ uint64_t cand[kCandidates];
    __shared__ u32x4 hit[kHits];                         // vectors that reach the limit, and where they begin
    __shared__ int hit_at[kHits];
    __shared__ int count, hits;
    __shared__ unsigned limit;
    __shared__ uint64_t kth;
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x;
    Row<T, THREADS, VPT> r;
    r.init(static_cast<const T*>(a.x) + row * a.x_stride, a.classes);
    const int passes = r.passes();
    float best[KEPT];                                    // of each vector
    float top = r.tail;
    if constexpr (VPT > 0) {
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            float b = get(r.kept[j], 0);
#pragma unroll
            for (int i = 1; i < N; ++i) b = max_nan(b, get(r.kept[j], i));
            best[j] = b;
            top = max_nan(top, b);
        }
    } else {
        for (int j = 0; j < passes; ++j) {
            const Vec<T> v = r.fetch(j);
#pragma unroll
            for (int i = 0; i < N; ++i) top = max_nan(top, get(v, i));
        }
    }
    r.forget_unpacked();
    maxima[tid] = top;
    if (tid == 0) count = hits = 0;
    __syncthreads();
    if (tid < 64) {
        unsigned mine[WAVES];
        bool nan = false;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float f = maxima[64 * w + tid];
            nan = nan || f != f;
            mine[w] = (64 * w + tid) * N >= r.full && 64 * w + tid >= a.classes - r.full ? 0u : order_of(f);   // a thread without an element
        }
        unsigned found = 0;
        constexpr int kLow = sizeof(T) == 2 ? 16 : 8;    // lower bits are the same for all, or only make the limit sharper than it
        for (int bit = 31; bit >= kLow; --bit) {         // needs to be
            const unsigned trial = found | 1u << bit;
            int n = 0;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) n += __popcll(__ballot(mine[w] >= trial));
            if (n >= a.k) found = trial;
        }
        const bool any_nan = __ballot(nan) != 0;
        if (tid == 0) limit = any_nan ? 0xFFFFFFFFu : found;
    }
    __syncthreads();
    const unsigned from = limit;
    const bool nan = from == 0xFFFFFFFFu;
    const float at_least = value_of_order(from);
    auto collect = [&](float f, int at) {
        const int slot = atomicAdd(&count, 1);
        if (slot < kCandidates) cand[slot] = key_of(f, at);
    };
    const bool few = VPT > 0 && !nan;                    // the vectors that matter are copied to LDS and leave the row
    if (!nan && r.has_tail() && r.tail >= at_least) collect(r.tail, r.tail_class());
    if constexpr (VPT > 0) {
        if (few) {
#pragma unroll
            for (int j = 0; j < VPT; ++j)
                if (best[j] >= at_least && r.base(j) < r.full) {
                    const int slot = atomicAdd(&hits, 1);
                    if (slot < kHits) {
                        hit[slot] = r.kept[j].raw;
                        hit_at[slot] = r.base(j);
                    }
                    const unsigned lowest = sizeof(T) == 4 ? lowest_bits<T>() : lowest_bits<T>() * 0x10001u;
                    r.kept[j].raw = u32x4{lowest, lowest, lowest, lowest};
                    best[j] = -INFINITY;
                }
        }
    } else if (!nan) {
        for (int j = 0; j < passes; ++j) {
            const Vec<T> v = r.fetch(j);
            const int at = r.base(j);
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (get(v, i) >= at_least && at < r.full) collect(get(v, i), at + i);
        }
    }
    __syncthreads();
    const int pairs = few ? min(hits, kHits) * N : 0;    // elements of those vectors, one to a thread
    auto element_of = [&](int e) -> float {
        const Vec<T> v{hit[e / N]};
        return get_at(v, e % N);
    };
    if (few) {
        for (int e = tid; e < pairs; e += THREADS) {
            const float f = element_of(e);
            if (f >= at_least) collect(f, hit_at[e / N] + e % N);
        }
        __syncthreads();
    }
    int have = count;
    const bool general = nan || have > kCandidates || hits > kHits;
    if (general) {
        __syncthreads();                                 // everyone has read the counts
        const int again = (r.full + THREADS * N - 1) / (THREADS * N);
        uint64_t found = 0;
#pragma unroll 1
        for (int bit = 63; bit >= 0; --bit) {
            const uint64_t trial = found | 1ull << bit;
            int n = r.has_tail() && key_of(r.tail, r.tail_class()) >= trial ? 1 : 0;
#pragma unroll 1
            for (int j = 0; j < again; ++j) {
                const Vec<T> v = r.fetch(j);
                const int at = r.base(j);
                for (int i = 0; i < N; ++i) n += at < r.full && key_of(get(v, i), at + i) >= trial ? 1 : 0;
            }
            if (block_sum<WAVES>(n, red_i) >= a.k) found = trial;
        }
        if (tid == 0) count = 0;
        __syncthreads();
#pragma unroll 1
        for (int j = 0; j < again; ++j) {
            const Vec<T> v = r.fetch(j);
            const int at = r.base(j);
            for (int i = 0; i < N; ++i) {
                const uint64_t key = key_of(get(v, i), at + i);
                if (at < r.full && key >= found) {
                    const int slot = atomicAdd(&count, 1);
                    if (slot < kCandidates) cand[slot] = key;
                }
            }
        }
        if (r.has_tail() && key_of(r.tail, r.tail_class()) >= found) {
            const int slot = atomicAdd(&count, 1);
            if (slot < kCandidates) cand[slot] = key_of(r.tail, r.tail_class());
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
    // the others: all but what was answered
    auto left = [&](int j) -> Vec<T> {
        Vec<T> v = r.fetch(j);
        const int at = r.base(j);
#pragma unroll 1
        for (int i = 0; i < N; ++i)
            if (key_of(get_at(v, i), at + i) >= last) set_bits_at(v, i, lowest_bits<T>());
        return v;
    };
    const bool kept = VPT > 0 && !general;
    const int all = (r.full + THREADS * N - 1) / (THREADS * N);
    if (r.has_tail() && key_of(r.tail, r.tail_class()) >= last) r.tail = -INFINITY;
    float m = r.tail;
    if (kept) {
#pragma unroll
        for (int j = 0; j < KEPT; ++j) m = max_nan(m, best[j]);
        for (int e = tid; e < pairs; e += THREADS) {
            const float f = element_of(e);
            if (key_of(f, hit_at[e / N] + e % N) < last) m = max_nan(m, f);
        }
    } else {
#pragma unroll 1
        for (int j = 0; j < all; ++j) {
            const Vec<T> v = left(j);
#pragma unroll
            for (int i = 0; i < N; ++i) m = max_nan(m, get(v, i));
        }
    }
    r.forget_unpacked();
    m = block_max<WAVES>(m, red_f);
    const float c2 = static_cast<float>(1.4426950408889634 / static_cast<double>(a.temperature));
    const float ref = m == -INFINITY ? 0.0f : m;         // as in distil_rows
    float part = exp2_hw((r.tail - ref) * c2);
    auto add = [&](const Vec<T>& v) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) sum += exp2_hw((get(v, i) - ref) * c2);
        part += sum;
    };
    // The copied elements come in the order the atomics gave out their places, another one in every run.  Their exponentials, at most 1,
    // are rounded to multiples of 2^-40 (beside a sum of at least 1, the largest element's), so that the sum of all of them is
    // exact in 64 bits and no order changes it.
    double copied = 0.0;
    static_assert(kHits * N <= 4096, "2^12 of them in multiples of 2^-40 are 52 bits");
    if (kept) {
#pragma unroll
        for (int j = 0; j < KEPT; ++j) add(r.kept[j]);
        for (int e = tid; e < pairs; e += THREADS) {
            const float f = element_of(e);
            if (key_of(f, hit_at[e / N] + e % N) < last) copied += (static_cast<double>(exp2_hw((f - ref) * c2)) + 4096.0) - 4096.0;
        }
        copied = block_sum<WAVES>(copied, red_d);
    } else {
#pragma unroll 1
        for (int j = 0; j < all; ++j) add(left(j));
    }
    const double s = block_sum<WAVES>(static_cast<double>(part), red_d) + copied;
    if (tid == 0) {
        const double value = static_cast<double>(m) / static_cast<double>(a.temperature) + log(s);
        a.rest[row] = m == -INFINITY || m == INFINITY ? m : static_cast<float>(value);
    }
}

// ------------------------------------------------------------------------------------------------------------- launches
// Rows in registers: as many 16-byte vectors to a thread as leave room for four waves to a SIMD (16: half of its registers),
// so that several rows are at different stages on each CU; short rows spread over more threads for the sake of latency.
template <class T, bool GRAD> int launch_rows(const DistilArgs& a, int64_t rows, hipStream_t st) {
    const int vectors = a.classes / Vec<T>::N;
    const size_t lds = static_cast<size_t>(ceil_div(a.classes, 32)) * 4;
    const dim3 grid(static_cast<unsigned>(rows));
    if (vectors <= 64 * 4) hipLaunchKernelGGL((distil_rows<T, 64, 4, GRAD>), grid, dim3(64), lds, st, a);
    else if (vectors <= 256 * 4) hipLaunchKernelGGL((distil_rows<T, 256, 4, GRAD>), grid, dim3(256), lds, st, a);
    else if (vectors <= 256 * 16) hipLaunchKernelGGL((distil_rows<T, 256, 16, GRAD>), grid, dim3(256), lds, st, a);
    else if (vectors <= 512 * 12) hipLaunchKernelGGL((distil_rows<T, 512, 12, GRAD>), grid, dim3(512), lds, st, a);     // 21841 fp32: 123 us (16: 135)
    else if (vectors <= 512 * 16) hipLaunchKernelGGL((distil_rows<T, 512, 16, GRAD>), grid, dim3(512), lds, st, a);
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
    const int vectors = a.classes / Vec<T>::N;
    const dim3 grid(static_cast<unsigned>(rows));
    if (vectors <= 64 * 4) hipLaunchKernelGGL((top_logits<T, 64, 4>), grid, dim3(64), 0, st, a);
    else if (vectors <= 256 * 4) hipLaunchKernelGGL((top_logits<T, 256, 4>), grid, dim3(256), 0, st, a);
    else if (vectors <= 256 * 16) hipLaunchKernelGGL((top_logits<T, 256, 16>), grid, dim3(256), 0, st, a);
    else if (vectors <= 512 * 16) hipLaunchKernelGGL((top_logits<T, 512, 16>), grid, dim3(512), 0, st, a);
    else hipLaunchKernelGGL((top_logits<T, 1024, 0>), grid, dim3(1024), 0, st, a);
    return check_launch("ta_nn_top_logits");
}

// log2 e / T is an ordinary number of 32 bits, so that it times a difference of 0 or -inf is what it should be
static bool temperature_in_range(double t) { return t >= 0x1p-126 && t <= 0x1p126; }

static int check_rows(const DistilArgs& a, int64_t rows) {
    TA_NN_REQUIRE(a.x && a.top_values && a.top_classes, "null pointer");
    TA_NN_REQUIRE(rows >= 1 && rows <= 0x7FFFFFFF, "rows %lld", static_cast<long long>(rows));
    TA_NN_REQUIRE(a.classes >= 1 && a.classes <= kMaxClasses, "classes %d (1 .. %d)", a.classes, kMaxClasses);
    TA_NN_REQUIRE(a.k >= 1 && a.k <= kMaxTop, "top classes %d (1 .. %d)", a.k, kMaxTop);
    TA_NN_REQUIRE(a.x_stride >= a.classes, "row stride %lld of %d classes", static_cast<long long>(a.x_stride), a.classes);
    TA_NN_REQUIRE(temperature_in_range(a.temperature), "temperature %g (2^-126 .. 2^126)", a.temperature);
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
    // (a thread's place in its last pass lies up to 8192 elements behind the row)
    TA_NN_REQUIRE(classes >= 1 && classes <= (1 << 30) && x_stride >= classes, "%d classes (1 .. 2^30), row stride %lld", classes,
                  static_cast<long long>(x_stride));
    TA_NN_REQUIRE(k >= 1 && k <= classes && k <= ta_nn::kMaxTop, "%d of %d classes (at most %d)", k, classes, ta_nn::kMaxTop);
    TA_NN_REQUIRE(ta_nn::temperature_in_range(temperature), "temperature %g (2^-126 .. 2^126)", static_cast<double>(temperature));
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
