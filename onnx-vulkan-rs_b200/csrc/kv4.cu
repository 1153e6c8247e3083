// The 4-bit key / value cache: argument checks and the write of new tokens.
//
// Bytes ought to bound the write: 2 or 4 bytes are read per value and about 0.6
// stored.  What does is latency: 21784 tokens in f32, one head of 256, keys and values,
// 50 MB, take 17.3 us from memory (2.9 TB/s), 12.6 from L2, with 53 % of the issue slots
// and 32 % of the memory's rate in use: 1.2 of 6.7 warps a scheduler can issue, since a
// row is asked for behind three dependent reads (bounds, length, page).  (With eight
// values a thread issue did, 74 % of the slots at 19.6 us; asking for rows before the
// page gained nothing there and was not tried since.)
// A thread holds sixteen values of a row - two 32-bit words of codes - and the
// block_size / 16 threads of a block find its range with shuffles; keys and values
// of a row go through the same thread, so its place in the cache is found once.
//
// The quotients are rounded exactly without dividing.  x * (1 / s), the reciprocal
// good to two units of its last place, is within 2^-17 of x / s up to 32 (beyond, the
// code is 0 or 15 either way), so n = rint(x * (1 / s)) is right wherever the product
// lies farther than 2^-16 from a border - all sixteen of a
// thread but for one thread in some thousands, seven operations a value.  Elsewhere (and
// where a value is not finite): for an fp16 scale s and an integer n <= 16, n s has
// at most 16 significant bits, and the rest r = x - n s of a value within a step of n
// s is a whole number of units of its last place that fits 24 bits - so fma(-n, s, x)
// is r exactly, and n, off by at most one, is set right by comparing |r| with s / 2.
// The scale itself is one f64 quotient a block, keys' on the even lanes and values'
// on the odd.
#include "attention.cuh"

int32_t ovk_check_kv4(ovk_ctx *ctx, const char *op, const ovk_kv4_cache *c)
{
    OVK_REQUIRE(ctx, c, "%s: the cache is null", op);
    OVK_REFUSE(ctx, c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256, "%s: head_dim %lld (64, 128 or 256)", op,
               (long long)c->head_dim);
    OVK_REFUSE(ctx, c->block_size != 32 && c->block_size != 64 && c->block_size != 128, "%s: block_size %lld (32, 64 or 128)", op,
               (long long)c->block_size);
    OVK_REQUIRE(ctx, c->head_dim % c->block_size == 0, "%s: block_size %lld does not divide head_dim %lld", op,
                (long long)c->block_size, (long long)c->head_dim);
    OVK_REQUIRE(ctx, c->pages >= 0 && c->kv_heads >= 1 && c->kv_heads <= OVK_MAX_HEADS && c->page_size >= 1 &&
                         c->page_size < (int64_t(1) << 31) && c->pages < (int64_t(1) << 31) &&
                         (c->pages == 0 || c->kv_heads * c->page_size < (int64_t(1) << 31) / c->pages + 1) &&
                         c->pages * c->kv_heads * c->page_size < (int64_t(1) << 31),
                "%s: a cache of %lld pages of %lld heads x %lld places (fewer than 2^31 rows)", op, (long long)c->pages,
                (long long)c->kv_heads, (long long)c->page_size);
    OVK_REQUIRE(ctx, c->pages == 0 || (c->k && c->v && c->k_scales && c->v_scales), "%s: the cache has no data", op);
    OVK_REQUIRE(ctx, !c->k_zero_points == !c->v_zero_points, "%s: zero points for keys and values, or for neither", op);
    OVK_REQUIRE(ctx, aligned_to(c->k, 16) && aligned_to(c->v, 16) && aligned_to(c->k_scales, 16) && aligned_to(c->v_scales, 16) &&
                         aligned_to(c->k_zero_points, 16) && aligned_to(c->v_zero_points, 16),
                "%s: the cache's tensors must be 16-byte aligned", op);
    return OVK_OK;
}

int32_t ovk_check_kv4_batch(ovk_ctx *ctx, const char *op, const ovk_kv4_batch *b)
{
    OVK_REQUIRE(ctx, b, "%s: the batch is null", op);
    OVK_REQUIRE(ctx, b->tokens >= 0 && b->tokens < (int64_t(1) << 31) && b->batch >= 0 && b->batch < (1 << 24) && b->max_pages >= 0 &&
                         b->max_pages < (int64_t(1) << 31),
                "%s: %lld tokens of %lld sequences, %lld pages each", op, (long long)b->tokens, (long long)b->batch,
                (long long)b->max_pages);
    OVK_REQUIRE(ctx, b->batch == 0 || (b->cu_tokens && b->lens && (b->block_table || b->max_pages == 0)), "%s: null sequence arrays", op);
    OVK_REQUIRE(ctx, aligned_to(b->cu_tokens, 4) && aligned_to(b->lens, 4) && aligned_to(b->block_table, 4), "%s: misaligned sequence arrays", op);
    return OVK_OK;
}

namespace {

struct AppendArgs {
    const void *x[2];  // keys, values
    int64_t token_stride[2], head_stride[2];
    uint8_t *codes[2];
    __half *scales[2];
    uint8_t *zero_points[2];
    const int32_t *cu, *lens, *table;
    int tokens, batch, heads, page_size, pages;
    int pair_shift, lane_shift, block_shift;  // log2 of the pairs of words of a row and of a block, and the blocks of a row
    int page_shift;                           // log2 of page_size, or -1
    int64_t max_pages;
    int *status;
};

// x / s rounded to the nearest integer, ties to even, as a float; inv is about 1 / s, half is s / 2 (infinity where s is 0:
// then the quotient counts as 0).  Beyond +-2^22 the result is only large.
__device__ __forceinline__ float quotient(float x, float s, float inv, float half)
{
    const float magic = 12582912.0f;  // 1.5 * 2^23: the sum's last bits are the integer
    const float t = fmaf(x, inv, magic), n = t - magic, rest = fmaf(-n, s, x), off = fabsf(rest);
    const bool moves = off > half || (off == half && (__float_as_uint(t) & 1u));
    return moves ? n + copysignf(1.0f, rest) : n;
}

// x / N to its exact rounding: the rest of the rounded product with a rounded reciprocal corrects it (Markstein, "Computation of
// elementary functions on the IBM RISC System/6000 processor", 1990).  x is finite.
template <int N> __device__ __forceinline__ double divided(double x)
{
    constexpr double inverse = 1.0 / N;
    const double q = x * inverse;
    return fma(fma(-double(N), q, x), inverse, q);
}

// The larger of the two, NaN where one of them is.
__device__ __forceinline__ float max_or_nan(float a, float b)
{
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) kv4_append_kernel(const AppendArgs a)
{
    // a block's threads: the pairs of words (up to 16, a row lies inside a warp) of 256 / pairs tokens; its head is blockIdx.y
    const int pair = threadIdx.x & ((1 << a.pair_shift) - 1), head = blockIdx.y;
    const int64_t first = int64_t(blockIdx.x) << (8 - a.pair_shift);  // below 2^31 but for the last block's end
    const int token = int(min(first + (threadIdx.x >> a.pair_shift), int64_t(a.tokens)));
    OVK_PDL_LAUNCH_DEPENDENTS();
    OVK_PDL_WAIT();
    // bounds that leave the tensors: reported here for the whole batch, left out below
    if (head == 0 && blockIdx.x <= unsigned(a.batch - 1) / 256)  // few blocks of a large grid
        for (int64_t b = int64_t(blockIdx.x) * 256 + threadIdx.x; b < a.batch; b += int64_t(gridDim.x) * 256)
            if (a.cu[b] < 0 || a.cu[b + 1] < a.cu[b] || a.cu[b + 1] > a.tokens)
                atomicExch(a.status, OVK_DEV_BAD_SEQUENCE);
    int row = -1;  // rows of the cache are fewer than 2^31
    if (token < a.tokens) {
        const int b = sequence_of(a.cu, a.batch, token, a.tokens);
        if (b >= 0) {
            const int length = a.lens[b], first = a.cu[b], end = a.cu[b + 1], from_end = end - token;  // one way to memory
            const bool inside = first >= 0 && end <= a.tokens;
            const uint32_t position = uint32_t(length) - uint32_t(from_end);
            const uint32_t page = a.page_shift >= 0 ? position >> a.page_shift : position / uint32_t(a.page_size);
            const int where = inside && length >= from_end && page < a.max_pages ? a.table[b * a.max_pages + page] : -1;
            if (where >= 0 && where < a.pages)
                row = (where * a.heads + head) * a.page_size + int(position - page * a.page_size);
            else if (inside && pair == 0)
                atomicExch(a.status, OVK_DEV_BAD_PAGE);
        }
    }
    const int lanes = 1 << a.lane_shift, blocks = 1 << a.block_shift;
    const int block = pair >> a.lane_shift;
    float x[2][16];
#pragma unroll
    for (int j = 0; j < 2; j++) {
        if (row >= 0) {
            load_row<T, 16, VEC>(static_cast<const T *>(a.x[j]) + token * a.token_stride[j] + head * a.head_stride[j] + 16 * pair, x[j]);
        } else {
#pragma unroll
            for (int e = 0; e < 16; e++)
                x[j][e] = 0.0f;
        }
    }
    float lo[2] = {0.0f, 0.0f}, hi[2] = {0.0f, 0.0f};  // fminf and fmaxf drop a NaN
#pragma unroll
    for (int j = 0; j < 2; j++) {
#pragma unroll
        for (int e = 0; e < 16; e++)
            lo[j] = fminf(lo[j], x[j][e]), hi[j] = fmaxf(hi[j], x[j][e]);
        for (int o = 1; o < lanes; o <<= 1) {
            lo[j] = fminf(lo[j], __shfl_xor_sync(0xffffffffu, lo[j], o));
            hi[j] = fmaxf(hi[j], __shfl_xor_sync(0xffffffffu, hi[j], o));
        }
    }
    const int mine = threadIdx.x & 1;
    const float most = 3.4e38f;  // an infinity's scale is 65504, and this one's
    const double top = fminf(mine ? hi[1] : hi[0], most), low = fmaxf(mine ? lo[1] : lo[0], -most);
    const double step = a.zero_points[0] ? divided<15>(top - low) : fmax(divided<7>(top), -low * 0.125);
    const float my_scale = fminf(float(step), 65504.0f), other_scale = __shfl_xor_sync(0xffffffffu, my_scale, 1);
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const __half scale = __float2half_rn(mine == j ? my_scale : other_scale);
        const float s = __half2float(scale);
        const float inv = s > 0.0f ? __fdividef(1.0f, s) : 0.0f, half = s > 0.0f ? 0.5f * s : INFINITY;  // a scale is at least 2^-24: finite
        float zero_f = 8.0f;
        if (a.zero_points[j])
            zero_f = fminf(fmaxf(quotient(-lo[j], s, inv, half), 0.0f), 15.0f);
        const int zero = int(zero_f);
        // 1.5 * 2^23 + n has the integer in its last bits, and each word so shifted in leaves its leading ones behind
        const float magic = 12582912.0f, to_zero = magic + zero_f;
        constexpr uint32_t left_over = 0x4b400000u * 0x11111111u;
        uint32_t codes[2] = {0, 0};
        float off = 0.0f;
#pragma unroll
        for (int e = 15; e >= 0; e--) {
            const float t = fmaf(x[j][e], inv, to_zero);
            off = max_or_nan(off, fabsf(fmaf(x[j][e], inv, to_zero - t)));
            codes[e / 8] = (codes[e / 8] << 4) + __float_as_uint(fminf(fmaxf(t, magic), magic + 15.0f));
        }
        codes[0] -= left_over, codes[1] -= left_over;
        if (!(off < 0.5f - 0x1p-16f)) {
            codes[0] = codes[1] = 0;
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const float v = x[j][e] == x[j][e] ? x[j][e] : 0.0f;
                codes[e / 8] |= uint32_t(fminf(fmaxf(quotient(v, s, inv, half) + zero_f, 0.0f), 15.0f)) << (4 * (e % 8));
            }
        }
        // the block to the right shares this block's byte of zero points
        const int next = __shfl_down_sync(0xffffffffu, zero, lanes);
        if (row >= 0) {
            const int64_t at = row;
            reinterpret_cast<uint2 *>(a.codes[j])[(at << a.pair_shift) + pair] = make_uint2(codes[0], codes[1]);
            if ((pair & (lanes - 1)) == 0) {
                a.scales[j][(at << a.block_shift) + block] = scale;
                if (a.zero_points[j] && block % 2 == 0)
                    a.zero_points[j][(at << max(a.block_shift - 1, 0)) + block / 2] = uint8_t(zero | (block + 1 < blocks ? next << 4 : 0));
            }
        }
    }
}

}  // namespace

extern "C" int32_t ovk_kv4_append(ovk_ctx *ctx, const ovk_kv4_cache *cache, const ovk_kv4_batch *batch, const ovk_heads *k,
                                  const ovk_heads *v, int32_t dtype)
{
    const char *op = "KV4Append";
    int32_t rc = ovk_check_kv4(ctx, op, cache);
    if (rc == OVK_OK)
        rc = ovk_check_kv4_batch(ctx, op, batch);
    if (rc != OVK_OK)
        return rc;
    OVK_REFUSE(ctx, !ovk_is_activation(dtype), "%s: dtype %d (f32 or f16)", op, dtype);
    const size_t elem = ovk_elem_bytes(dtype);
    rc = ovk_check_heads(ctx, op, "k", k, batch->tokens, cache->head_dim, elem, false);
    if (rc == OVK_OK)
        rc = ovk_check_heads(ctx, op, "v", v, batch->tokens, cache->head_dim, elem, false);
    if (rc != OVK_OK)
        return rc;
    OVK_REQUIRE(ctx, k->heads == cache->kv_heads && v->heads == cache->kv_heads, "%s: %lld and %lld heads for a cache of %lld", op,
                (long long)k->heads, (long long)v->heads, (long long)cache->kv_heads);
    OVK_REQUIRE(ctx, ctx, "%s: null context", op);
    if (batch->tokens == 0 || batch->batch == 0)
        return OVK_OK;
    DeviceGuard guard(ctx->device);
    AppendArgs a = {};
    a.x[0] = k->data, a.x[1] = v->data;
    a.token_stride[0] = k->token_stride, a.token_stride[1] = v->token_stride;
    a.head_stride[0] = k->head_stride, a.head_stride[1] = v->head_stride;
    a.codes[0] = static_cast<uint8_t *>(cache->k), a.codes[1] = static_cast<uint8_t *>(cache->v);
    a.scales[0] = static_cast<__half *>(cache->k_scales), a.scales[1] = static_cast<__half *>(cache->v_scales);
    a.zero_points[0] = static_cast<uint8_t *>(cache->k_zero_points), a.zero_points[1] = static_cast<uint8_t *>(cache->v_zero_points);
    a.cu = batch->cu_tokens, a.lens = batch->lens, a.table = batch->block_table;
    a.tokens = int(batch->tokens);
    auto log2_of = [](int64_t n) {  // of a power of two, -1 of any other number
        int shift = 0;
        while (int64_t(1) << shift < n)
            shift++;
        return int64_t(1) << shift == n ? shift : -1;
    };
    a.pair_shift = log2_of(cache->head_dim / 16), a.lane_shift = log2_of(cache->block_size / 16);
    a.block_shift = log2_of(cache->head_dim / cache->block_size), a.page_shift = log2_of(cache->page_size);
    a.batch = int(batch->batch), a.heads = int(cache->kv_heads);
    a.page_size = int(cache->page_size), a.pages = int(cache->pages), a.max_pages = batch->max_pages;
    a.status = ctx->dev_status;
    const dim3 grid(unsigned(ceil_div64(batch->tokens, 256 >> a.pair_shift)), unsigned(cache->kv_heads));
    const bool vec = ovk_rows_aligned(k, elem) && ovk_rows_aligned(v, elem);
    void (*kernel)(AppendArgs) = dtype == OVK_FLOAT ? (vec ? kv4_append_kernel<float, true> : kv4_append_kernel<float, false>)
                                                    : (vec ? kv4_append_kernel<__half, true> : kv4_append_kernel<__half, false>);
    OVK_CUDA(ctx, ovk_launch_pdl(kernel, grid, dim3(256), 0, ctx->stream, a));
    OVK_LAUNCHED(ctx, vec ? "kv4_append" : "kv4_append_scalar");
    return OVK_OK;
}
