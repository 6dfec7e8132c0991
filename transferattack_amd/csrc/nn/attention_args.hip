// Argument checks and workspace sizes of the attention entry points.
#include "attention.h"

namespace ta_nn {

// batch chunks of the table's gradient: enough workgroups to fill 256 CUs a few times over, a chunk never without a sequence
static int table_chunks(const ta_nn_attention_args& a) {
    if (is_window(a)) return window_parts(a, true) * window_periods(a);
    const int64_t tiles = ceil_div(a.m, 64) * ceil_div(a.n, 64) * a.heads;
    const int64_t wanted = ceil_div(2048, tiles);
    return static_cast<int>(wanted < a.batch ? wanted : a.batch);
}

int64_t workspace_floats(const ta_nn_attention_args& a, bool backward) {
    if (!backward) {
        const int splits = is_few(a) ? few_splits(a) : 1;
        return splits == 1 ? 0 : static_cast<int64_t>(a.batch) * a.kv_heads * splits * (32 + 16 * a.dim);
    }
    int64_t floats = static_cast<int64_t>(a.batch) * a.heads * a.m;
    if (a.dtable) {
        const int64_t per_chunk = a.distances ? ceil_div(a.m, 64) * ceil_div(a.n, 64) * 128 : static_cast<int64_t>(a.m) * a.n;
        floats += per_chunk * a.heads * table_chunks(a);
    }
    return floats;
}

int check_attention(const ta_nn_attention_args* args, AttentionArgs& a) {
    TA_NN_REQUIRE(args, "null pointer");
    static_cast<ta_nn_attention_args&>(a) = *args;
    TA_NN_REQUIRE(a.dtype >= TA_NN_F32 && a.dtype <= TA_NN_F16, "element type %d", a.dtype);
    TA_NN_REQUIRE(a.table_dtype >= TA_NN_F32 && a.table_dtype <= TA_NN_F16, "element type %d of the table", a.table_dtype);
    TA_NN_REQUIRE(a.batch >= 1 && a.m >= 1 && a.n >= 1 && a.heads >= 1 && a.kv_heads >= 1, "batch %d, heads %d / %d, %d queries, %d keys",
                  a.batch, a.heads, a.kv_heads, a.m, a.n);
    TA_NN_REQUIRE(a.m < (1 << 30) && a.n < (1 << 30) && a.distances < (1 << 29), "more than 2^30 tokens");
    TA_NN_REQUIRE(a.heads % a.kv_heads == 0, "%d heads do not share %d key heads evenly", a.heads, a.kv_heads);
    TA_NN_REQUIRE(a.dim >= 1 && a.dim <= 128, "head dimension %d (1 .. 128)", a.dim);
    TA_NN_REQUIRE(a.q && a.k && a.v && a.table && a.index && a.out, "null pointer");
    TA_NN_REQUIRE(a.buckets >= 1 && a.buckets <= 65536, "%d buckets", a.buckets);
    TA_NN_REQUIRE(a.distances >= 0, "%d distances", a.distances);
    if (a.distances == 0) {
        TA_NN_REQUIRE(a.index_stride >= a.n && a.index_stride % 4 == 0 && reinterpret_cast<uintptr_t>(a.index) % 8 == 0,
                      "index stride %lld of %d keys", static_cast<long long>(a.index_stride), a.n);
    }
    TA_NN_REQUIRE(a.mask_kind >= TA_NN_MASK_NONE && a.mask_kind <= TA_NN_MASK_F16, "mask kind %d", a.mask_kind);
    TA_NN_REQUIRE(a.mask_kind == TA_NN_MASK_NONE || (a.mask && a.mask_period >= 1), "mask period %d", a.mask_period);
    const int64_t steps[] = {a.q_sm, a.k_sn, a.v_sn, a.g_sm};
    for (int64_t step : steps)
        TA_NN_REQUIRE(step > -(1 << 24) && step < (1 << 24), "token stride %lld (below 2^24 elements)", static_cast<long long>(step));
    a.chunks = table_chunks(a);
    return 0;
}

}  // namespace ta_nn
