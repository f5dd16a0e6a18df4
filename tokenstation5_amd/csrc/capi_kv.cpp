// The entry points of include/ts5hip.h around a KV cache beyond decode, verify and prompt
// attention: trees of drafts, accumulated key weights and eviction, block-sparse
// attention. Host checks here, the context's last (so that arguments can be checked without a
// GPU); kernels through kernels.h. And around caches in pages and drafts judged by probabilities.
#include <algorithm>

#include "common_host.h"
#include "kernels.h"
#include "runtime.h"

using namespace ts5hip;

namespace {

// The context's device made current for a call that may come from a thread with another
// one, and that one again afterwards.
struct OnDevice {
    int before = -1;
    explicit OnDevice(int device) {
        if (hipGetDevice(&before) != hipSuccess || before == device || hipSetDevice(device) != hipSuccess) before = -1;
    }
    ~OnDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

bool aligned(const void *p, size_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

// A cache as the kernels of attn_rows.h read it; with `values` its V half too.
int check_cache(ts5hip_ctx *ctx, int B, int n_head_kv, int head_dim, int kv_type, const void *k, const void *ks,
                const void *v, const void *vs, int n_ctx, bool values) {
    if (kv_type != KV_Q8 && kv_type != KV_F16) return fail(ctx, TS5HIP_ERR_UNSUPPORTED, "cache type %d", kv_type);
    const bool q8 = kv_type == KV_Q8;
    if (!k || (values && !v) || (q8 && (!ks || (values && !vs)))) return fail(ctx, TS5HIP_ERR_ARG, "null argument");
    if (head_dim != 64 && head_dim != 128 && head_dim != 256)
        return fail(ctx, TS5HIP_ERR_UNSUPPORTED, "head dimension %d (64, 128 or 256)", head_dim);
    if (B < 1 || B > 4096 || n_head_kv < 1 || n_head_kv > 512 || n_ctx < 1)
        return fail(ctx, TS5HIP_ERR_ARG, "%d caches of %d KV heads, %d slots", B, n_head_kv, n_ctx);
    // A KV head's rows are one buffer with 32-bit offsets.
    if ((int64_t)n_ctx * head_dim * (q8 ? 1 : 2) > INT32_MAX)
        return fail(ctx, TS5HIP_ERR_UNSUPPORTED, "%d slots of %d values", n_ctx, head_dim);
    if (!aligned(k, 16) || !aligned(v, 16) || !aligned(ks, 4) || !aligned(vs, 4))
        return fail(ctx, TS5HIP_ERR_ARG, "cache rows need 16-byte, scales 4-byte alignment");
    return TS5HIP_OK;
}

int check_heads(ts5hip_ctx *ctx, int n_head, int n_head_kv, int head_dim) {
    if (!attn_rows_supported(n_head, n_head_kv, head_dim))
        return fail(ctx, TS5HIP_ERR_UNSUPPORTED, "attention for %d/%d heads of %d", n_head, n_head_kv, head_dim);
    return TS5HIP_OK;
}

KvLayer layer(const void *k, const void *ks, const void *v, const void *vs) {
    return KvLayer{(int8_t *)k, (uint16_t *)ks, (int8_t *)v, (uint16_t *)vs};
}

struct Range {
    const void *p;
    size_t bytes;
};
bool overlap(const Range &a, const Range &b) {
    const uintptr_t x = (uintptr_t)a.p, y = (uintptr_t)b.p;
    return a.p && b.p && a.bytes && b.bytes && x < y + b.bytes && y < x + a.bytes;
}

// No output lies over an input or over another output.
template <int N_OUT, int N_IN>
int check_apart(ts5hip_ctx *ctx, const Range (&out)[N_OUT], const Range (&in)[N_IN]) {
    for (int o = 0; o < N_OUT; o++)
        for (int i = 0; i < N_IN + o; i++)
            if (overlap(out[o], i < N_IN ? in[i] : out[i - N_IN]))
                return fail(ctx, TS5HIP_ERR_ARG, "outputs lie over inputs or each other");
    return TS5HIP_OK;
}

// A pool of pages and the tables of n_seq sequences.
int check_pool(ts5hip_ctx *ctx, int n_head_kv, int head_dim, int kv_type, const void *k, const void *ks, const void *v,
               const void *vs, int n_pages, int page, const int32_t *table_dev, int n_seq, int n_table) {
    if (!table_dev) return fail(ctx, TS5HIP_ERR_ARG, "null argument");
    if (page != 16 && page != 32 && page != 64 && page != 128 && page != 256)
        return fail(ctx, TS5HIP_ERR_UNSUPPORTED, "pages of %d slots (16, 32, 64, 128 or 256)", page);
    if (int rc = check_cache(ctx, 1, n_head_kv, head_dim, kv_type, k, ks, v, vs, page, true)) return rc;
    if (n_pages < 1 || n_seq < 1 || n_table < 1 || (int64_t)n_table * page > 1 << 30)
        return fail(ctx, TS5HIP_ERR_ARG, "%d pages, tables of %d pages of %d sequences", n_pages, n_table, n_seq);
    return TS5HIP_OK;
}
// Bytes of a pool's values (K or V) and of their scales.
size_t pool_values(int n_pages, int page, int n_head_kv, int head_dim, int kv_type) {
    return (size_t)n_pages * page * n_head_kv * head_dim * (kv_type == KV_Q8 ? 1 : 2);
}
size_t pool_scales(int n_pages, int page, int n_head_kv, int head_dim) {
    return (size_t)n_pages * page * n_head_kv * (head_dim / 32) * 2;
}

// The sums of key weights, [B][n_head_kv][n_ctx], before and after.
int check_sums(ts5hip_ctx *ctx, int B, int n_head_kv, int n_ctx, const float *acc, const float *acc_out) {
    const size_t bytes = (size_t)B * n_head_kv * n_ctx * 4;
    if (acc != acc_out && overlap({acc, bytes}, {acc_out, bytes}))
        return fail(ctx, TS5HIP_ERR_ARG, "acc_out is acc or does not overlap it");
    return TS5HIP_OK;
}

}  // namespace

extern "C" {

int ts5hip_rope_kv_append_at(ts5hip_ctx *ctx, const float *qkv, int ntok, const int32_t *pos_dev,
                             const int32_t *slot0_dev, int n_head, int n_head_kv, int head_dim, int n_rot, int neox,
                             const float *rope_cs, int n_pos, int n_ctx, int kv_type, const float *bias,
                             const float *q_norm, const float *k_norm, float eps, float *q_out, void *k, void *ks,
                             void *v, void *vs) {
    if (!qkv || !pos_dev || !slot0_dev || !rope_cs || !q_out) return fail(ctx, TS5HIP_ERR_ARG, "null argument");
    if (int rc = check_cache(ctx, 1, n_head_kv, head_dim, kv_type, k, ks, v, vs, n_ctx, true)) return rc;
    if (n_head < 1 || n_head % n_head_kv || n_head > 65535 - 2 * n_head_kv || n_rot < 0 || n_rot > head_dim || n_rot % 2)
        return fail(ctx, TS5HIP_ERR_UNSUPPORTED, "rope/kv for %d/%d heads of %d (n_rot %d)", n_head, n_head_kv,
                    head_dim, n_rot);
    if (ntok < 1 || ntok > 4096 || n_pos < 1) return fail(ctx, TS5HIP_ERR_ARG, "%d tokens, %d positions", ntok, n_pos);
    if (!ctx) return fail(nullptr, TS5HIP_ERR_ARG, "ctx is null");
    const OnDevice on(ctx->device);
    TS5_HIP(ctx, launch_rope_kv_at(qkv, (int64_t)(n_head + 2 * n_head_kv) * head_dim, bias, q_norm, k_norm, eps, rope_cs,
                                   n_pos, n_rot, neox, pos_dev, slot0_dev, n_head, n_head_kv, head_dim, n_ctx, ntok,
                                   q_out, layer(k, ks, v, vs), kv_type == KV_F16, ctx->stream));
    return TS5HIP_OK;
}

int ts5hip_attn_tree(ts5hip_ctx *ctx, const float *q, int B, int n_tree, int n_head, int n_head_kv, int head_dim,
                     int kv_type, const void *k, const void *ks, const void *v, const void *vs, int n_ctx,
                     const int32_t *n_past_dev, const uint64_t *mask_dev, float scale, float *out) {
    if (!q || !n_past_dev || !mask_dev || !out) return fail(ctx, TS5HIP_ERR_ARG, "null argument");
    if (int rc = check_heads(ctx, n_head, n_head_kv, head_dim)) return rc;
    if (int rc = check_cache(ctx, B, n_head_kv, head_dim, kv_type, k, ks, v, vs, n_ctx, true)) return rc;
    if (n_tree < 1 || n_tree > 64 || n_tree > n_ctx)
        return fail(ctx, TS5HIP_ERR_ARG, "a tree of %d tokens (1..64) in a cache of %d", n_tree, n_ctx);
    if (!aligned(q, 16) || !aligned(out, 16) || !aligned(mask_dev, 8))
        return fail(ctx, TS5HIP_ERR_ARG, "q and out need 16-byte, masks 8-byte alignment");
    if (!ctx) return fail(nullptr, TS5HIP_ERR_ARG, "ctx is null");
    const OnDevice on(ctx->device);
    if (int rc = ensure_scratch(ctx, attn_tree_scratch_bytes(B, n_tree, n_head, n_head_kv, head_dim, kv_type == KV_F16, n_ctx,
                                                              ctx->n_cu)))
        return rc;
    TS5_HIP(ctx, launch_attn_tree(q, B, n_tree, n_head, n_head_kv, head_dim, layer(k, ks, v, vs), kv_type == KV_F16,
                                  n_ctx, n_past_dev, mask_dev, scale, (float *)ctx->scratch, out, ctx->n_cu,
                                  ctx->stream));
    return TS5HIP_OK;
}

int ts5hip_kv_path(ts5hip_ctx *ctx, int B, int n_head_kv, int head_dim, int kv_type, void *k, void *ks, void *v, void *vs,
                   int n_ctx, const int32_t *slots_dev, int n, const int32_t *slot0_dev) {
    if (!slots_dev || !slot0_dev) return fail(ctx, TS5HIP_ERR_ARG, "null argument");
    if (int rc = check_cache(ctx, B, n_head_kv, head_dim, kv_type, k, ks, v, vs, n_ctx, true)) return rc;
    if (n < 1 || n > KV_PATH_MAX) return fail(ctx, TS5HIP_ERR_ARG, "a path of %d rows (1..%d)", n, KV_PATH_MAX);
    if (!ctx) return fail(nullptr, TS5HIP_ERR_ARG, "ctx is null");
    const OnDevice on(ctx->device);
    TS5_HIP(ctx, launch_kv_path(B, n_head_kv, head_dim, layer(k, ks, v, vs), kv_type == KV_F16, n_ctx, slots_dev, n,
                                slot0_dev, ctx->stream));
    return TS5HIP_OK;
}

int ts5hip_attn_decode_weights(ts5hip_ctx *ctx, const float *q, int B, int n_head, int n_head_kv, int head_dim,
                               int kv_type, const void *k, const void *ks, const void *v, const void *vs, int n_ctx,
                               const int32_t *n_keys_dev, float scale, float *out, const float *acc, float *acc_out) {
    if (!q || !n_keys_dev || !out || !acc || !acc_out) return fail(ctx, TS5HIP_ERR_ARG, "null argument");
    if (int rc = check_heads(ctx, n_head, n_head_kv, head_dim)) return rc;
    if (int rc = check_cache(ctx, B, n_head_kv, head_dim, kv_type, k, ks, v, vs, n_ctx, true)) return rc;
    if (!aligned(q, 16) || !aligned(out, 16)) return fail(ctx, TS5HIP_ERR_ARG, "q and out need 16-byte alignment");
    if (int rc = check_sums(ctx, B, n_head_kv, n_ctx, acc, acc_out)) return rc;
    if (!ctx) return fail(nullptr, TS5HIP_ERR_ARG, "ctx is null");
    const OnDevice on(ctx->device);
    if (int rc = ensure_scratch(ctx, attn_one_weights_scratch_bytes(B, n_head, n_head_kv, head_dim, n_ctx, ctx->n_cu)))
        return rc;
    TS5_HIP(ctx, launch_attn_one_weights(q, B, n_head, n_head_kv, head_dim, layer(k, ks, v, vs), kv_type == KV_F16,
                                         n_ctx, n_keys_dev, scale, ctx->scratch, out, acc, acc_out, ctx->n_cu,
                                         ctx->stream));
    return TS5HIP_OK;
}

int ts5hip_attn_prompt_weights(ts5hip_ctx *ctx, const float *q, int nq, int n_head, int n_head_kv, int head_dim,
                               int kv_type, const void *k, const void *ks, const void *v, const void *vs, int n_ctx,
                               int pos0, float scale, float *out, const float *acc, float *acc_out) {
    if (!q || !out || !acc || !acc_out) return fail(ctx, TS5HIP_ERR_ARG, "null argument");
    if (int rc = check_heads(ctx, n_head, n_head_kv, head_dim)) return rc;
    if (int rc = check_cache(ctx, 1, n_head_kv, head_dim, kv_type, k, ks, v, vs, n_ctx, true)) return rc;
    if (nq < 1 || nq > 4096 || pos0 < 0 || (int64_t)pos0 + nq > n_ctx)
        return fail(ctx, TS5HIP_ERR_ARG, "%d queries (1..4096) at %d in a cache of %d", nq, pos0, n_ctx);
    if ((int64_t)n_head * nq > 960000)  // (blocks of 16 rows or more along the grid's y)
        return fail(ctx, TS5HIP_ERR_UNSUPPORTED, "%d queries of %d heads (960000 in all)", nq, n_head);
    if (!aligned(q, 16) || !aligned(out, 16)) return fail(ctx, TS5HIP_ERR_ARG, "q and out need 16-byte alignment");
    if (int rc = check_sums(ctx, 1, n_head_kv, n_ctx, acc, acc_out)) return rc;
    if (!ctx) return fail(nullptr, TS5HIP_ERR_ARG, "ctx is null");
    const OnDevice on(ctx->device);
    if (int rc = ensure_scratch(ctx, attn_prompt_weights_scratch_bytes(nq, n_head, n_head_kv, head_dim, kv_type == KV_F16,
                                                                       pos0 + nq, ctx->n_cu)))
        return rc;
    TS5_HIP(ctx, launch_attn_prompt_weights(q, nq, n_head, n_head_kv, head_dim, layer(k, ks, v, vs), kv_type == KV_F16,
                                            n_ctx, pos0, scale, ctx->scratch, out, acc, acc_out, ctx->n_cu,
                                            ctx->stream));
    return TS5HIP_OK;
}

int ts5hip_kv_evict(ts5hip_ctx *ctx, int B, int n_head_kv, int head_dim, int kv_type, const void *k, const void *ks,
                    const void *v, const void *vs, int n_ctx, const int32_t *n_keys_dev, const float *acc, int n_keep,
                    int n_first, int n_last, int n_ctx_out, void *k_out, void *ks_out, void *v_out, void *vs_out,
                    float *acc_out, int32_t *kept_dev, int32_t *n_out_dev) {
    if (!n_keys_dev || !acc || !acc_out || !kept_dev) return fail(ctx, TS5HIP_ERR_ARG, "null argument");
    if (int rc = check_cache(ctx, B, n_head_kv, head_dim, kv_type, k, ks, v, vs, n_ctx, true)) return rc;
    if (int rc = check_cache(ctx, B, n_head_kv, head_dim, kv_type, k_out, ks_out, v_out, vs_out, n_ctx_out, true))
        return rc;
    if (n_keep < 1 || n_keep > n_ctx_out || n_first < 0 || n_last < 0 || (int64_t)n_first + n_last > n_keep)
        return fail(ctx, TS5HIP_ERR_ARG, "keeping %d keys (the first %d, the last %d) in a cache of %d", n_keep, n_first,
                    n_last, n_ctx_out);
    const size_t heads = (size_t)B * n_head_kv, rows = heads * n_ctx, rows_out = heads * n_ctx_out;
    const size_t row = head_dim * (kv_type == KV_Q8 ? 1 : 2), sc = kv_type == KV_Q8 ? head_dim / 32 * 2 : 0;  // bytes (f16: no scales)
    const Range in[] = {{k, rows * row}, {v, rows * row}, {ks, rows * sc}, {vs, rows * sc}, {acc, rows * 4}, {n_keys_dev, (size_t)B * 4}};
    const Range out[] = {{k_out, rows_out * row}, {v_out, rows_out * row}, {ks_out, rows_out * sc}, {vs_out, rows_out * sc},
                         {acc_out, rows_out * 4}, {n_out_dev, (size_t)B * 4}, {kept_dev, heads * n_keep * 4}};
    constexpr int N_IN = sizeof in / sizeof *in, N_OUT = sizeof out / sizeof *out;
    for (int o = 0; o < N_OUT; o++) {
        // kept_dev last, and only for a call that has a context: without one its address may be any.
        if (o == N_OUT - 1 && !ctx) break;
        for (int i = 0; i < N_IN + o; i++)
            if (overlap(out[o], i < N_IN ? in[i] : out[i - N_IN]))
                return fail(ctx, TS5HIP_ERR_ARG, "an eviction's outputs lie over its inputs or each other");
    }
    if (!ctx) return fail(nullptr, TS5HIP_ERR_ARG, "ctx is null");
    const OnDevice on(ctx->device);
    TS5_HIP(ctx, launch_kv_evict(B, n_head_kv, head_dim, layer(k, ks, v, vs), kv_type == KV_F16, n_ctx, n_keys_dev, acc,
                                 n_keep, n_first, n_last, n_ctx_out, layer(k_out, ks_out, v_out, vs_out), acc_out,
                                 kept_dev, n_out_dev, ctx->stream));
    return TS5HIP_OK;
}

static bool block_ok(int block) { return block == 16 || block == 32 || block == 64 || block == 128; }

int64_t ts5hip_kv_bounds_bytes(int B, int n_head_kv, int head_dim, int n_ctx, int block) {
    if (B < 1 || n_head_kv < 1 || head_dim < 1 || n_ctx < 1 || !block_ok(block)) return -1;
    return (int64_t)B * n_head_kv * (((int64_t)n_ctx + block - 1) / block) * head_dim * 4;
}

int ts5hip_kv_block_bounds(ts5hip_ctx *ctx, int B, int n_head_kv, int head_dim, int kv_type, const void *k,
                           const void *ks, int n_ctx, const int32_t *n_keys_dev, int n_new, int block, void *bounds) {
    if (!n_keys_dev || !bounds) return fail(ctx, TS5HIP_ERR_ARG, "null argument");
    if (int rc = check_cache(ctx, B, n_head_kv, head_dim, kv_type, k, ks, nullptr, nullptr, n_ctx, false)) return rc;
    if (!block_ok(block)) return fail(ctx, TS5HIP_ERR_UNSUPPORTED, "blocks of %d keys (16, 32, 64 or 128)", block);
    if (n_new < 1) return fail(ctx, TS5HIP_ERR_ARG, "%d new keys", n_new);
    if (!aligned(bounds, 16)) return fail(ctx, TS5HIP_ERR_ARG, "bounds need 16-byte alignment");
    if (!ctx) return fail(nullptr, TS5HIP_ERR_ARG, "ctx is null");
    const OnDevice on(ctx->device);
    TS5_HIP(ctx, launch_block_bounds(B, n_head_kv, head_dim, layer(k, ks, nullptr, nullptr), kv_type == KV_F16, n_ctx,
                                     n_keys_dev, std::min(n_new, n_ctx), block, bounds, ctx->stream));
    return TS5HIP_OK;
}

int ts5hip_attn_sparse(ts5hip_ctx *ctx, const float *q, int B, int n_head, int n_head_kv, int head_dim, int kv_type,
                       const void *k, const void *ks, const void *v, const void *vs, int n_ctx,
                       const int32_t *n_keys_dev, int kv_per_batch, const void *bounds, int block, int n_pick,
                       float scale, float *out, int32_t *picked_dev) {
    if (!q || !n_keys_dev || !bounds || !out) return fail(ctx, TS5HIP_ERR_ARG, "null argument");
    if (int rc = check_heads(ctx, n_head, n_head_kv, head_dim)) return rc;
    if (int rc = check_cache(ctx, B, n_head_kv, head_dim, kv_type, k, ks, v, vs, n_ctx, true)) return rc;
    if (!block_ok(block)) return fail(ctx, TS5HIP_ERR_UNSUPPORTED, "blocks of %d keys (16, 32, 64 or 128)", block);
    if (B * n_head_kv > 4096)  // the joins' counters
        return fail(ctx, TS5HIP_ERR_ARG, "batch of %d x %d KV heads", B, n_head_kv);
    if (n_pick < 1 || n_pick > (1 << 20) || !(scale > 0.f))
        return fail(ctx, TS5HIP_ERR_ARG, "%d blocks picked at scale %g (scores rank by a positive scale)", n_pick, scale);
    if (!aligned(q, 16) || !aligned(out, 16) || !aligned(bounds, 16))
        return fail(ctx, TS5HIP_ERR_ARG, "q, bounds and out need 16-byte alignment");
    if (!ctx) return fail(nullptr, TS5HIP_ERR_ARG, "ctx is null");
    const OnDevice on(ctx->device);
    if (int rc = ensure_scratch(ctx, attn_sparse_scratch_bytes(B, n_head, n_head_kv, head_dim, n_ctx, block, n_pick,
                                                               ctx->n_cu)))
        return rc;
    TS5_HIP(ctx, launch_attn_sparse(q, B, n_head, n_head_kv, head_dim, layer(k, ks, v, vs), kv_type == KV_F16, n_ctx,
                                    n_keys_dev, kv_per_batch != 0, bounds, block, n_pick, scale, ctx->scratch,
                                    ctx->counters, out, picked_dev, ctx->n_cu, ctx->stream));
    return TS5HIP_OK;
}

int ts5hip_rope_kv_append_paged(ts5hip_ctx *ctx, const float *qkv, int ntok, const int32_t *seq_dev, const int32_t *pos_dev,
                                int n_head, int n_head_kv, int head_dim, int n_rot, int neox, const float *rope_cs,
                                int n_pos, const float *bias, const float *q_norm, const float *k_norm, float eps,
                                float *q_out, int kv_type, void *k, void *ks, void *v, void *vs, int n_pages, int page,
                                const int32_t *table_dev, int n_seq, int n_table) {
    if (!qkv || !seq_dev || !pos_dev || !rope_cs || !q_out) return fail(ctx, TS5HIP_ERR_ARG, "null argument");
    if (int rc = check_pool(ctx, n_head_kv, head_dim, kv_type, k, ks, v, vs, n_pages, page, table_dev, n_seq, n_table))
        return rc;
    if (n_head < 1 || n_head % n_head_kv || n_head > 65535 - 2 * n_head_kv || n_rot < 0 || n_rot > head_dim || n_rot % 2)
        return fail(ctx, TS5HIP_ERR_UNSUPPORTED, "rope/kv for %d/%d heads of %d (n_rot %d)", n_head, n_head_kv,
                    head_dim, n_rot);
    if (ntok < 1 || ntok > 65535 || n_pos < 1) return fail(ctx, TS5HIP_ERR_ARG, "%d tokens, %d positions", ntok, n_pos);
    if (!aligned(qkv, 16) || !aligned(q_out, 16) || !aligned(bias, 16) || !aligned(q_norm, 16) || !aligned(k_norm, 16) ||
        !aligned(rope_cs, 16))
        return fail(ctx, TS5HIP_ERR_ARG, "q, k, v, biases, norms and angles need 16-byte alignment");
    const size_t heads = (size_t)ntok * head_dim * 4;
    const size_t pool = pool_values(n_pages, page, n_head_kv, head_dim, kv_type);
    const size_t scales = kv_type == KV_Q8 ? pool_scales(n_pages, page, n_head_kv, head_dim) : 0;
    const Range table{table_dev, (size_t)n_seq * n_table * 4}, rows{qkv, heads * (n_head + 2 * n_head_kv)};
    const size_t row = (size_t)(n_head + 2 * n_head_kv) * head_dim * 4, norm = (size_t)head_dim * 4;
    if (int rc = check_apart(ctx, {{k, pool}, {v, pool}, {ks, scales}, {vs, scales}}, {rows, table})) return rc;
    if (int rc = check_apart(ctx, {{q_out, heads * n_head}},
                             {rows, {k, pool}, {v, pool}, {ks, scales}, {vs, scales}, table, {seq_dev, (size_t)ntok * 4},
                              {pos_dev, (size_t)ntok * 4}, {bias, row}, {q_norm, norm}, {k_norm, norm},
                              {rope_cs, (size_t)n_pos * n_rot * 4}}))
        return rc;
    if (!ctx) return fail(nullptr, TS5HIP_ERR_ARG, "ctx is null");
    const OnDevice on(ctx->device);
    TS5_HIP(ctx, launch_append_paged(qkv, ntok, seq_dev, pos_dev, n_head, n_head_kv, head_dim, bias, q_norm, k_norm, eps,
                                     rope_cs, n_pos, n_rot, neox, q_out, layer(k, ks, v, vs), kv_type == KV_F16, n_pages,
                                     page, table_dev, n_seq, n_table, ctx->stream));
    return TS5HIP_OK;
}

int ts5hip_kv_read_paged(ts5hip_ctx *ctx, int ntok, const int32_t *seq_dev, const int32_t *pos_dev, int n_head_kv,
                         int head_dim, int kv_type, const void *k, const void *ks, const void *v, const void *vs,
                         int n_pages, int page, const int32_t *table_dev, int n_seq, int n_table, int out_type,
                         void *k_out, void *v_out) {
    if (!seq_dev || !pos_dev || !k_out || !v_out) return fail(ctx, TS5HIP_ERR_ARG, "null argument");
    if (int rc = check_pool(ctx, n_head_kv, head_dim, kv_type, k, ks, v, vs, n_pages, page, table_dev, n_seq, n_table))
        return rc;
    if (ntok < 1 || ntok > 1 << 24) return fail(ctx, TS5HIP_ERR_ARG, "%d tokens (1..2^24)", ntok);
    if (out_type != TS5HIP_F32 && out_type != TS5HIP_F16)
        return fail(ctx, TS5HIP_ERR_UNSUPPORTED, "rows of type %d (f32 or f16)", out_type);
    if (!aligned(k_out, 16) || !aligned(v_out, 16)) return fail(ctx, TS5HIP_ERR_ARG, "rows need 16-byte alignment");
    const size_t rows = (size_t)ntok * n_head_kv * head_dim * (out_type == TS5HIP_F32 ? 4 : 2);
    const size_t pool = pool_values(n_pages, page, n_head_kv, head_dim, kv_type);
    const size_t scales = kv_type == KV_Q8 ? pool_scales(n_pages, page, n_head_kv, head_dim) : 0;
    if (int rc = check_apart(ctx, {{k_out, rows}, {v_out, rows}}, {{k, pool}, {v, pool}, {ks, scales}, {vs, scales},
                                                                  {table_dev, (size_t)n_seq * n_table * 4},
                                                                  {seq_dev, (size_t)ntok * 4}, {pos_dev, (size_t)ntok * 4}}))
        return rc;
    if (!ctx) return fail(nullptr, TS5HIP_ERR_ARG, "ctx is null");
    const OnDevice on(ctx->device);
    TS5_HIP(ctx, launch_read_paged(ntok, seq_dev, pos_dev, n_head_kv, head_dim, layer(k, ks, v, vs), kv_type == KV_F16,
                                   n_pages, page, table_dev, n_seq, n_table, out_type == TS5HIP_F16, k_out, v_out,
                                   ctx->stream));
    return TS5HIP_OK;
}

int ts5hip_attn_paged(ts5hip_ctx *ctx, const float *q, int B, int n_new, int n_head, int n_head_kv, int head_dim,
                      int kv_type, const void *k, const void *ks, const void *v, const void *vs, int n_pages, int page,
                      const int32_t *table_dev, int n_table, const int32_t *n_keys_dev, int window, float scale,
                      float *out) {
    if (!q || !n_keys_dev || !out) return fail(ctx, TS5HIP_ERR_ARG, "null argument");
    if (int rc = check_heads(ctx, n_head, n_head_kv, head_dim)) return rc;
    if (int rc = check_pool(ctx, n_head_kv, head_dim, kv_type, k, ks, v, vs, n_pages, page, table_dev, B, n_table)) return rc;
    if (B > 4096 || (int64_t)B * n_table * page > (int64_t)1 << 34)
        return fail(ctx, TS5HIP_ERR_ARG, "%d sequences of up to %lld keys", B, (long long)n_table * page);
    if (n_new < 1 || n_new > ATTN_MAX_NEW || window < 0)
        return fail(ctx, TS5HIP_ERR_ARG, "%d new tokens (1..%d), window %d", n_new, ATTN_MAX_NEW, window);
    if (!aligned(q, 16) || !aligned(out, 16)) return fail(ctx, TS5HIP_ERR_ARG, "q and out need 16-byte alignment");
    const size_t rows = (size_t)B * n_new * n_head * head_dim * 4;
    const size_t pool = pool_values(n_pages, page, n_head_kv, head_dim, kv_type);
    const size_t scales = kv_type == KV_Q8 ? pool_scales(n_pages, page, n_head_kv, head_dim) : 0;
    if (int rc = check_apart(ctx, {{out, rows}}, {{q, rows}, {k, pool}, {v, pool}, {ks, scales}, {vs, scales},
                                                  {table_dev, (size_t)B * n_table * 4}, {n_keys_dev, (size_t)B * 4}}))
        return rc;
    if (!ctx) return fail(nullptr, TS5HIP_ERR_ARG, "ctx is null");
    const OnDevice on(ctx->device);
    if (int rc = ensure_scratch(ctx, attn_paged_scratch_bytes(B, n_new, n_head, n_head_kv, head_dim, ctx->n_cu))) return rc;
    TS5_HIP(ctx, launch_attn_paged(q, B, n_new, n_head, n_head_kv, head_dim, layer(k, ks, v, vs), kv_type == KV_F16,
                                   n_pages, page, table_dev, n_table, n_keys_dev, window, scale, ctx->scratch,
                                   ctx->counters, out, ctx->n_cu, ctx->stream));
    return TS5HIP_OK;
}

int ts5hip_verify_drafts(ts5hip_ctx *ctx, const float *logits, int64_t ld, const float *draft_logits, int64_t ld_draft,
                         int n_vocab, int B, int n_draft, const int32_t *drafts_dev, const int32_t *n_draft_dev,
                         const float *temperature_dev, const float *uniform_dev, int32_t *tokens_dev,
                         int32_t *n_tokens_dev, float *logp_dev) {
    if (!logits || !temperature_dev || !uniform_dev || !tokens_dev || !n_tokens_dev || (n_draft > 0 && !drafts_dev))
        return fail(ctx, TS5HIP_ERR_ARG, "null argument");
    if (n_vocab < 1 || n_vocab > verify_max_vocab() || ld < n_vocab || (draft_logits && ld_draft < n_vocab))
        return fail(ctx, TS5HIP_ERR_ARG, "%d entries (1..%d) of rows of %lld and %lld", n_vocab, verify_max_vocab(),
                    (long long)ld, (long long)ld_draft);
    if (B < 1 || B > 4096 || n_draft < 0 || n_draft > verify_max_drafts())
        return fail(ctx, TS5HIP_ERR_ARG, "%d sequences of %d drafts (0..%d)", B, n_draft, verify_max_drafts());
    const size_t rows = (size_t)B * (n_draft + 1), drafts = (size_t)B * n_draft;
    if (ld > (int64_t)1 << 40 || (draft_logits && ld_draft > (int64_t)1 << 40))
        return fail(ctx, TS5HIP_ERR_ARG, "rows of %lld and %lld entries", (long long)ld, (long long)ld_draft);
    if (int rc = check_apart(ctx, {{tokens_dev, rows * 4}, {n_tokens_dev, (size_t)B * 4}, {logp_dev, rows * 4}},
                             {{logits, rows * (size_t)ld * 4}, {draft_logits, drafts * (size_t)ld_draft * 4}, {drafts_dev, drafts * 4},
                              {n_draft_dev, (size_t)B * 4}, {temperature_dev, (size_t)B * 4}, {uniform_dev, rows * 4}}))
        return rc;
    if (!ctx) return fail(nullptr, TS5HIP_ERR_ARG, "ctx is null");
    const OnDevice on(ctx->device);
    if (int rc = ensure_scratch(ctx, verify_scratch_bytes(n_vocab, B, n_draft))) return rc;
    TS5_HIP(ctx, launch_verify(logits, ld, n_draft ? draft_logits : nullptr, ld_draft, n_vocab, B, n_draft, drafts_dev,
                               n_draft_dev, temperature_dev, uniform_dev, ctx->scratch, ctx->counters, tokens_dev,
                               n_tokens_dev, logp_dev, ctx->stream));
    return TS5HIP_OK;
}

}  // extern "C"
