// ovk_attention_kv4: checks, launch plan and dispatch (the kernel: attention_kv4.cuh).
#include "attention_kv4.cuh"

namespace {

struct Plan {
    int tiles;    // 8-row column tiles of a CTA: 1 or 2
    int unit;     // tokens that a CTA takes at a time
    size_t slot;  // floats of a partial result
};

template <int D, int NT, int PARTS> Plan plan_of()
{
    using S = kv4::Shape<D, NT, PARTS>;
    return {NT, S::UNIT, size_t(S::SLOT)};
}
template <int D> Plan plan_for(int tiles, bool f32)
{
    if (f32)
        return tiles == 1 ? plan_of<D, 1, 2>() : plan_of<D, 2, 2>();
    return tiles == 1 ? plan_of<D, 1, 1>() : plan_of<D, 2, 1>();
}
Plan plan_for(int64_t head_dim, int tiles, bool f32)
{
    return head_dim == 64 ? plan_for<64>(tiles, f32) : head_dim == 128 ? plan_for<128>(tiles, f32) : plan_for<256>(tiles, f32);
}
// One tile of eight rows where a sequence's new tokens and a group's heads fit in it, two otherwise: the
// second tile's products ride on the same unpacked codes.
int tiles_for(int64_t max_tokens, int64_t group) { return max_tokens * group <= 8 ? 1 : 2; }

constexpr size_t COUNTERS = 4096;  // bytes: a counter per CTA
static_assert(COUNTERS == OVK_KV4_COUNTERS * sizeof(unsigned int), "the context's counters");

size_t bytes_for(const Plan &p, int64_t ctas) { return COUNTERS + size_t(ctas) * 2 * p.slot * sizeof(float); }

int32_t check(ovk_ctx *ctx, const char *op, const ovk_kv4_cache *cache, int64_t q_heads, int64_t max_tokens, int32_t dtype)
{
    int32_t rc = ovk_check_kv4(ctx, op, cache);
    if (rc != OVK_OK)
        return rc;
    OVK_REFUSE(ctx, !ovk_is_activation(dtype), "%s: dtype %d (f32 or f16)", op, dtype);
    OVK_REQUIRE(ctx, q_heads >= 1 && q_heads <= OVK_MAX_HEADS && q_heads % cache->kv_heads == 0,
                "%s: %lld query heads for %lld key heads", op, (long long)q_heads, (long long)cache->kv_heads);
    OVK_REQUIRE(ctx, max_tokens >= 1 && max_tokens < (int64_t(1) << 31), "%s: max_tokens %lld", op, (long long)max_tokens);
    return OVK_OK;
}

}  // namespace

extern "C" int32_t ovk_attention_kv4_workspace(ovk_ctx *ctx, const ovk_kv4_cache *cache, int64_t q_heads, int64_t max_tokens,
                                               int32_t dtype, size_t *bytes)
{
    const char *op = "AttentionKV4";
    int32_t rc = check(ctx, op, cache, q_heads, max_tokens, dtype);
    if (rc != OVK_OK)
        return rc;
    OVK_REQUIRE(ctx, bytes, "%s: bytes is null", op);
    OVK_REQUIRE(ctx, ctx, "%s: null context", op);
    *bytes = 0;
    for (int tiles = 1; tiles <= tiles_for(max_tokens, q_heads / cache->kv_heads); tiles++) {
        const Plan p = plan_for(cache->head_dim, tiles, dtype == OVK_FLOAT);
        *bytes = std::max(*bytes, bytes_for(p, std::min(ctx->sm_count, OVK_KV4_COUNTERS)));
    }
    return OVK_OK;
}

extern "C" int32_t ovk_attention_kv4(ovk_ctx *ctx, const ovk_kv4_cache *cache, const ovk_kv4_batch *batch, const ovk_heads *q,
                                     const ovk_heads *out, int32_t dtype, int64_t max_tokens, float scale, int64_t window,
                                     void *workspace, size_t workspace_bytes)
{
    const char *op = "AttentionKV4";
    int32_t rc = ovk_check_kv4_batch(ctx, op, batch);
    if (rc != OVK_OK)
        return rc;
    OVK_REQUIRE(ctx, cache && q && out, "%s: null argument", op);
    rc = check(ctx, op, cache, q->heads, max_tokens, dtype);
    if (rc != OVK_OK)
        return rc;
    const size_t elem = ovk_elem_bytes(dtype);
    rc = ovk_check_heads(ctx, op, "q", q, batch->tokens, cache->head_dim, elem, false);
    if (rc == OVK_OK)
        rc = ovk_check_heads(ctx, op, "out", out, batch->tokens, cache->head_dim, elem, true);
    if (rc != OVK_OK)
        return rc;
    OVK_REQUIRE(ctx, out->heads == q->heads, "%s: %lld query heads, %lld in the output", op, (long long)q->heads, (long long)out->heads);
    OVK_REQUIRE(ctx, batch->tokens == 0 || (ovk_rows_aligned(q, elem) && ovk_rows_aligned(out, elem)),
                "%s: rows of q and out must be 16-byte aligned", op);
    OVK_REQUIRE(ctx, batch->tokens * q->heads < (int64_t(1) << 31) - 64, "%s: %lld tokens of %lld heads are too many for one call", op,
                (long long)batch->tokens, (long long)q->heads);
    OVK_REQUIRE(ctx, window >= 0, "%s: window %lld", op, (long long)window);
    const float factor = ovk_scale_log2e(scale);
    OVK_REQUIRE(ctx, factor - factor == 0.0f, "%s: scale %g is not finite, or not in powers of two", op, double(scale));
    OVK_REQUIRE(ctx, ctx, "%s: null context", op);
    if (batch->tokens == 0 || batch->batch == 0)
        return OVK_OK;
    DeviceGuard guard(ctx->device);

    Kv4Args a = {};
    // a cache without pages may come without data: copies of no bytes still name an address
    auto data = [&](const void *p) { return static_cast<const uint8_t *>(cache->pages ? p : ctx->dev_status); };
    a.codes[0] = data(cache->k), a.codes[1] = data(cache->v), a.scales[0] = data(cache->k_scales), a.scales[1] = data(cache->v_scales);
    if (cache->k_zero_points)
        a.zero_points[0] = data(cache->k_zero_points), a.zero_points[1] = data(cache->v_zero_points);
    a.cu = batch->cu_tokens, a.lens = batch->lens, a.table = batch->block_table;
    a.q = q->data, a.out = out->data;
    a.q_token = q->token_stride, a.q_head = q->head_stride, a.o_token = out->token_stride, a.o_head = out->head_stride;
    a.max_pages = batch->max_pages, a.window = ovk_window(window);
    a.tokens = int(batch->tokens), a.batch = int(batch->batch), a.pages = int(cache->pages), a.kv_heads = int(cache->kv_heads);
    a.group = int(q->heads / cache->kv_heads), a.page_size = int(cache->page_size);
    a.page_shift = -1;
    for (int s = 0; s < 31; s++)
        if ((int64_t(1) << s) == cache->page_size)
            a.page_shift = s;
    a.blocks = int(cache->head_dim / cache->block_size);
    a.chunk_shift = cache->block_size == 32 ? 0 : cache->block_size == 64 ? 1 : 2;
    a.scale_log2e = factor;
    a.status = ctx->dev_status;

    const int tiles = tiles_for(max_tokens, a.group);
    const Plan p = plan_for(cache->head_dim, tiles, dtype == OVK_FLOAT);
    // no more CTAs than the longest sequences the block table has room for would fill
    const int64_t units = batch->max_pages * cache->page_size / p.unit + 2;
    const int64_t items = (batch->batch + ceil_div64(batch->tokens * a.group, 8 * tiles)) * cache->kv_heads;
    const int64_t full = std::min(ctx->sm_count, OVK_KV4_COUNTERS);
    const int64_t ctas = items >= full || units >= full ? full : std::min(full, units * items);
    const bool own = !workspace;
    if (workspace) {
        OVK_REQUIRE(ctx, aligned_to(workspace, 16) && workspace_bytes >= bytes_for(p, ctas),
                    "%s: a workspace of %zu bytes at %p, %zu are needed on a 16-byte boundary", op, workspace_bytes, workspace,
                    bytes_for(p, ctas));
    } else {
        // the context's workspace would be shared by every graph captured from it
        cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
        OVK_CUDA(ctx, cudaStreamIsCapturing(ctx->stream, &capture));
        OVK_REQUIRE(ctx, capture == cudaStreamCaptureStatusNone, "%s: a captured call needs a workspace of its own (%zu bytes)", op,
                    bytes_for(p, ctas));
        rc = ovk_scratch(ctx, bytes_for(p, ctas), &workspace);
        if (rc != OVK_OK)
            return rc;
    }
    a.counters = own ? ctx->kv4_counters : static_cast<unsigned int *>(workspace);
    a.partial = reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + COUNTERS);
    return cache->head_dim == 64    ? ovk_kv4_launch_64(ctx, a, dtype, tiles, int(ctas))
           : cache->head_dim == 128 ? ovk_kv4_launch_128(ctx, a, dtype, tiles, int(ctas))
                                    : ovk_kv4_launch_256(ctx, a, dtype, tiles, int(ctas));
}
