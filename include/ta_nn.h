/*
 * ta_nn.h -- C ABI of libta_nn.so: operators of transformer surrogates and of learning from a victim's answers, as MI355X
 * (gfx950) kernels.
 *   ta_nn_attention*   attention whose scores carry a learned relative position bias (a table of buckets x heads), forward,
 *                      backward (queries, keys, values, table) and for single tokens against a cache
 *   ta_nn_top_logits   a teacher's K largest logits per row, in order, and the log-sum-exp of the others
 *   ta_nn_distil*      distillation from such answers: loss and gradient
 * The transformer these serve: the reference's victims and surrogates of transferattack/utils.py:16-17 (the window
 * transformer's attention adds relative_position_bias_table to its scores).
 *
 * Conventions
 *   - every pointer is a DEVICE pointer; `stream` is a hipStream_t passed as void*; calls are asynchronous on it, never
 *     synchronise, never allocate, keep nothing -> safe inside hipGraph capture; workspaces are the caller's;
 *   - element types: TA_NN_F32 / _BF16 / _F16; strides count elements; the innermost dimension is contiguous;
 *   - sums, maxima, softmax statistics and gradients are accumulated in fp32 or fp64 whatever the tensors' type;
 *   - return value: 0, a hipError_t (> 0) or TA_NN_EINVAL (-1); ta_nn_last_error() has the calling thread's last message;
 *   - results are deterministic: no floating-point atomics, every reduction has a fixed order or is exact.
 */
#ifndef TA_NN_H
#define TA_NN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define TA_NN_ABI_VERSION 1
#define TA_NN_EINVAL (-1)

#define TA_NN_F32 0
#define TA_NN_BF16 1
#define TA_NN_F16 2

#define TA_NN_MASK_NONE 0
#define TA_NN_MASK_BOOL 1     /* one byte: may be seen or not */
#define TA_NN_MASK_F32 2      /* added to the score; then TA_NN_MASK_F32 + element type */
#define TA_NN_MASK_BF16 3
#define TA_NN_MASK_F16 4

int ta_nn_abi_version(void);
const char* ta_nn_last_error(void);

/* ---- attention with a relative position bias --------------------------------------------------------------------------
 *   s_ij = scale q_i . k_j + table[bucket(i, j)][head] + mask_ij     p = softmax of s over the keys seen     o_i = sum p_ij v_j
 * A query that sees no key gives zeros, and zero gradients. */
typedef struct ta_nn_attention_args {
    int dtype;                                   /* of q, k, v, out, grad, dq, dk, dv */
    int batch, heads, kv_heads, m, n, dim;       /* m queries, n keys; heads a multiple of kv_heads; dim <= 128,
                                                    16 bytes or a multiple of that */
    const void *q, *k, *v;
    int64_t q_sb, q_sh, q_sm, k_sb, k_sh, k_sn, v_sb, v_sh, v_sn;      /* token strides (_sm, _sn): 0 .. 2^23 - 1 */
    float scale;
    int table_dtype, buckets;
    const void* table;                           /* [buckets][heads], contiguous */
    int distances, first;                        /* distances > 0: bucket of distance d = j - (start + i) is
                                                    index[clamp(d - first, 0, distances - 1)], index int32.
                                                    distances == 0: index is uint16 [m][index_stride], the bucket of the pair,
                                                    index_t uint16 [n][index_t_stride] its transpose; strides multiples of 4 */
    const void *index, *index_t;
    int64_t index_stride, index_t_stride;
    int mask_kind, mask_period;                  /* mask of sequence b is number b % mask_period */
    const void* mask;
    int64_t mask_sb, mask_sh, mask_sm, mask_sn;
    const int32_t* key_lengths;                  /* [batch] keys in use (what lies behind is not read), or NULL */
    const int32_t* query_start;                  /* [batch] position of query 0, or NULL: start */
    int start, causal;                           /* causal: key j is seen if j <= start + i */
    void* out;
    int64_t o_sb, o_sh, o_sm;
    float* stats;                                /* [batch][heads][m][2]: a score near the largest and 1 / sum of the exponentials
                                                    relative to it, for a backward pass; or NULL */
    float* workspace;                            /* ta_nn_attention_workspace() floats, or NULL where that is 0 */
    /* backward: */
    const void* grad;                            /* of out; out and stats are the forward pass's */
    int64_t g_sb, g_sh, g_sm;
    void *dq, *dk, *dv;
    int64_t dq_sb, dq_sh, dq_sm, dk_sb, dk_sh, dk_sn, dv_sb, dv_sh, dv_sn;
    void* dtable;                                /* [buckets][heads] of table_dtype, or NULL */
    const int32_t* pair_order;                   /* pairs: [m * n] pair numbers i * n + j sorted by bucket, */
    const int32_t* pair_starts;                  /*        [buckets + 1] where each bucket begins among them */
} ta_nn_attention_args;

/* floats of workspace the call needs (pointers of args need not be set yet, but dtable has to be NULL or not); 0: none, or
 * sizes that the call refuses */
int64_t ta_nn_attention_workspace(const ta_nn_attention_args* args, int backward);
int ta_nn_attention(const ta_nn_attention_args* args, void* stream);
int ta_nn_attention_backward(const ta_nn_attention_args* args, void* stream);

/* ---- a teacher's top logits -------------------------------------------------------------------------------------------
 * values / top_classes [rows][k]: the k largest of each row in falling order, equal ones by the lowest class (NaN above all);
 * rest [rows] (or NULL): log sum exp(x / temperature) over the other classes, -inf if there are none.  At most 2^30 classes. */
int ta_nn_top_logits(const void* x, int dtype, int64_t x_stride, int64_t rows, int classes, int k, float temperature, float* values,
                     int64_t* top_classes, float* rest, void* stream);

/* ---- distillation from top logits -------------------------------------------------------------------------------------
 *   loss_n = weight_n T^2 KL(teacher || student), both at temperature T; the teacher's distribution lies on its classes answered
 *   and, with `rest`, on one bin for all others.  A class of -1 is no answer; one that is out of range makes its row NaN; one given twice
 *   counts with both masses.  A row of weight 0 is not looked at: loss and gradient are 0.
 * ta_nn_distil           row_loss [rows]; and either stats [rows][5] for ta_nn_distil_backward, or -- grad given -- the gradient
 *                        (factor * *scale) * d loss_n / d x in the same pass over the row
 * ta_nn_distil_backward  grad = (factor * *scale * upstream) * d loss_n / d x from the statistics
 * ta_nn_distil_total     *loss = sum of row_loss (mean: / sum of weights), *scale = 1 / sum of weights (mean) or 1; NULL where not
 *                        wanted; weight NULL: ones.  If no row counts both are 0. */
int ta_nn_distil(const void* x, int dtype, int64_t x_stride, int64_t rows, int classes, const float* top_values,
                 const void* top_classes, int classes64, int k, const float* rest, const float* weight, double temperature,
                 float factor, const float* scale, float* row_loss, float* stats, void* grad, int64_t grad_stride, void* stream);
int ta_nn_distil_backward(const void* x, int dtype, int64_t x_stride, int64_t rows, int classes, const float* top_values,
                          const void* top_classes, int classes64, int k, const float* rest, const float* weight, double temperature,
                          float factor, const float* scale, const float* upstream, int upstream_per_row, const float* stats,
                          void* grad, int64_t grad_stride, void* stream);
int ta_nn_distil_total(const float* row_loss, const float* weight, int64_t rows, int mean, float* loss, float* scale, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* TA_NN_H */
