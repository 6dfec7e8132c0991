// Argument checks and workspace sizes of the attention entry points.
#include "attention.h"

namespace ta_nn {

// tiles of 64 queries x 64 keys whose score gradients the table's gradient needs one by one
static int64_t table_tiles(const AttentionArgs& a) { return ceil_div(a.m, 64) * (a.distances ? near_tiles(a) : ceil_div(a.n, 64)); }

static int table_chunks(const AttentionArgs& a) {
    if (is_window(a)) return window_parts(a, true) * window_periods(a);
    return balanced_parts(table_tiles(a) * a.heads, a.batch, 512);
}

// backward: delta, then the table's partial sums, then (distances) the sums past the ends and the sums by distance
static int64_t layout(AttentionArgs& a) {
    int64_t floats = static_cast<int64_t>(a.batch) * a.heads * a.m;
    a.delta = a.workspace;
    if (a.dtable == nullptr) return floats;
    a.chunks = table_chunks(a);
    const int64_t per_chunk = a.distances ? table_tiles(a) * 128 : static_cast<int64_t>(a.m) * a.n;
    a.partial = a.workspace + floats;
    floats += per_chunk * a.heads * a.chunks;
    if (a.distances) {
        a.far = a.workspace + floats;
        floats += static_cast<int64_t>(a.batch) * a.heads * ceil_div(a.m, 64) * 2;
        a.by_distance = a.workspace + floats;
        floats += a.heads * (ceil_div(a.m, 64) + ceil_div(a.n, 64) - 1) * 128;
    }
    return floats;
}

// what sizes and strides have to be; pointers may still be missing
static int check_sizes(const ta_nn_attention_args& a) {
    TA_NN_REQUIRE(a.dtype >= TA_NN_F32 && a.dtype <= TA_NN_F16, "element type %d", a.dtype);
    TA_NN_REQUIRE(a.table_dtype >= TA_NN_F32 && a.table_dtype <= TA_NN_F16, "element type %d of the table", a.table_dtype);
    TA_NN_REQUIRE(a.batch >= 1 && a.m >= 1 && a.n >= 1 && a.heads >= 1 && a.kv_heads >= 1, "batch %d, heads %d / %d, %d queries, %d keys",
                  a.batch, a.heads, a.kv_heads, a.m, a.n);
    TA_NN_REQUIRE(a.m < (1 << 30) && a.n < (1 << 30) && a.distances < (1 << 29), "more than 2^30 tokens");
    TA_NN_REQUIRE(a.heads % a.kv_heads == 0, "%d heads do not share %d key heads evenly", a.heads, a.kv_heads);
    TA_NN_REQUIRE(a.dim >= 1 && a.dim <= 128, "head dimension %d (1 .. 128)", a.dim);
    TA_NN_REQUIRE(a.dim % (a.dtype == TA_NN_F32 ? 4 : 8) == 0, "head dimension %d is not a multiple of 16 bytes", a.dim);
    TA_NN_REQUIRE(a.buckets >= 1 && a.buckets <= 65536, "%d buckets", a.buckets);
    TA_NN_REQUIRE(a.distances >= 0, "%d distances", a.distances);
    TA_NN_REQUIRE(a.mask_kind >= TA_NN_MASK_NONE && a.mask_kind <= TA_NN_MASK_F16, "mask kind %d", a.mask_kind);
    TA_NN_REQUIRE(a.mask_kind == TA_NN_MASK_NONE || a.mask_period >= 1, "mask period %d", a.mask_period);
    const int64_t steps[] = {a.q_sm, a.k_sn, a.v_sn, a.g_sm};
    for (int64_t step : steps)
        TA_NN_REQUIRE(step >= 0 && step < (1 << 23), "token stride %lld (below 2^23 elements)", static_cast<long long>(step));
    return 0;
}

int64_t workspace_floats(const ta_nn_attention_args& args, bool backward) {
    if (check_sizes(args)) return 0;                     // (the call itself says what is wrong with them)
    if (!backward) {
        const int splits = is_few(args) ? few_splits(args) : 1;
        return splits == 1 ? 0 : static_cast<int64_t>(args.batch) * args.kv_heads * splits * (32 + 16 * args.dim);
    }
    AttentionArgs a{};
    static_cast<ta_nn_attention_args&>(a) = args;
    return layout(a);
}

int check_attention(const ta_nn_attention_args* args, AttentionArgs& a) {
    TA_NN_REQUIRE(args, "null pointer");
    static_cast<ta_nn_attention_args&>(a) = *args;
    if (int rc = check_sizes(a)) return rc;
    TA_NN_REQUIRE(a.q && a.k && a.v && a.table && a.index && a.out, "null pointer");
    if (a.distances == 0) {
        TA_NN_REQUIRE(a.index_stride >= a.n && a.index_stride % 4 == 0 && reinterpret_cast<uintptr_t>(a.index) % 8 == 0,
                      "index stride %lld of %d keys", static_cast<long long>(a.index_stride), a.n);
    }
    TA_NN_REQUIRE(a.mask_kind == TA_NN_MASK_NONE || a.mask, "null pointer");
    layout(a);
    return 0;
}

}  // namespace ta_nn
