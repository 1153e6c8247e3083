// ovk_attention_prompt: checks and dispatch, and the kernel for f32 and for
// layouts the tensor-core kernel (attention_prompt_tc.cu) does not take.
//
//   x[i][j] = scale * q[i] . k[j],  out[i] = sum_j 2^(x log2 e - m) v[j] / sum_j 2^(x log2 e - m),
//
// one pass over the keys with the running maximum m and sum of each row.  A block
// holds 64 query rows of one head and walks 64 keys at a time; a thread computes 8
// (256-wide heads: 4) x 4 scores, then as many rows x head_dim / 16 columns of the
// result.  All of it is f32 arithmetic on the CUDA cores: with Q and K transposed in
// shared memory a step over d is three 16-byte loads for 32 multiply-adds, so the
// adders and not shared memory bound it.
#include "attention_prompt.cuh"

namespace {

constexpr int BM = 64, BN = 64, PITCH = BM + 4;

// rows of a thread: eight (128 threads) where the registers hold their results
template <int DMAX> constexpr int rows_of() { return DMAX == 256 ? 4 : 8; }
template <int DMAX> constexpr int threads_of() { return BM / rows_of<DMAX>() * 16; }

template <int DMAX> constexpr size_t simt_smem() { return size_t(2 * DMAX * PITCH + BN * DMAX + BN * PITCH) * 4; }

// rows of a [tokens, heads, d] tensor as columns of `t`: t[d][row], zeros outside
template <typename T, int DMAX>
__device__ __forceinline__ void load_transposed(float *t, const T *base, int64_t stride, int rows, int d, bool vec)
{
    constexpr int V = 16 / sizeof(T), PARTS = threads_of<DMAX>() / BM;  // threads of a row
    const int r = threadIdx.x / PARTS, part = threadIdx.x % PARTS;
    const T *src = base + int64_t(r) * stride;
#pragma unroll 4
    for (int e = part * V; e < DMAX; e += PARTS * V) {
        float v[V];
        if (r < rows && vec && e + V <= d) {
            load_row<T, V, true>(src + e, v);
        } else {
#pragma unroll
            for (int i = 0; i < V; i++)
                v[i] = r < rows && e + i < d ? to_f32<T>(src[e + i]) : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < V; i++)
            t[(e + i) * PITCH + r] = v[i];
    }
}

template <typename T, int DMAX>
__global__ void __launch_bounds__(threads_of<DMAX>()) attention_prompt_simt_kernel(const PromptArgs a)
{
    constexpr int RT = rows_of<DMAX>(), THREADS = threads_of<DMAX>();
    extern __shared__ __align__(16) float sm[];
    float *const qt = sm, *const kt = qt + DMAX * PITCH, *const vs = kt + DMAX * PITCH, *const pt = vs + BN * DMAX;
    __shared__ PromptTile where;
    const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
    if (tid < 32)
        find_prompt_tile<BM>(a, blockIdx.x, where);
    __syncthreads();
    const PromptTile w = where;
    if (w.b < 0)
        return;
    const int head = blockIdx.y, kv_head = head / a.group, D = a.head_dim;
    const int rows = min(BM, w.n_q - w.row0);
    const int64_t first = int64_t(w.n_k) - w.n_q + w.row0;  // position of the tile's first row
    const KeyRange range = key_range(a, w, rows);
    const T *q = static_cast<const T *>(a.q) + int64_t(w.first_q + w.row0) * a.q_token + int64_t(head) * a.q_head;
    const T *k = static_cast<const T *>(a.k) + int64_t(w.first_k) * a.k_token + int64_t(kv_head) * a.k_head;
    const T *v = static_cast<const T *>(a.v) + int64_t(w.first_k) * a.v_token + int64_t(kv_head) * a.v_head;
    load_transposed<T, DMAX>(qt, q, a.q_token, rows, D, a.vec);

    constexpr int OC = DMAX / 64;
    float o[RT][OC][4], m[RT], l[RT];
#pragma unroll
    for (int i = 0; i < RT; i++) {
        m[i] = -1e30f, l[i] = 0.0f;
#pragma unroll
        for (int c = 0; c < OC; c++)
            o[i][c][0] = o[i][c][1] = o[i][c][2] = o[i][c][3] = 0.0f;
    }
    for (int64_t j0 = range.begin; j0 < range.end; j0 += BN) {
        const int keys = int(min(int64_t(BN), range.end - j0));
        __syncthreads();
        load_transposed<T, DMAX>(kt, k + j0 * a.k_token, a.k_token, keys, D, a.vec);
        bool odd_value = false;  // an infinity or NaN among the values
        {
            constexpr int V = 16 / sizeof(T), PER = DMAX / V;
            for (int i = tid; i < BN * PER; i += THREADS) {
                const int r = i / PER, e = (i - r * PER) * V;
                const T *src = v + (j0 + r) * a.v_token + e;
                float x[V];
                if (r < keys && a.vec && e + V <= D) {
                    load_row<T, V, true>(src, x);
                } else {
#pragma unroll
                    for (int u = 0; u < V; u++)
                        x[u] = r < keys && e + u < D ? to_f32<T>(src[u]) : 0.0f;
                }
#pragma unroll
                for (int u = 0; u < V; u++) {
                    odd_value |= !(x[u] - x[u] == 0.0f);
                    vs[r * DMAX + e + u] = x[u];
                }
            }
        }
        odd_value = __syncthreads_or(odd_value);
        float s[RT][4];
#pragma unroll
        for (int i = 0; i < RT; i++)
            s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.0f;
#pragma unroll 8
        for (int d = 0; d < DMAX; d++) {
            float xs[RT];
#pragma unroll
            for (int i = 0; i < RT; i += 4) {
                const float4 x = *reinterpret_cast<const float4 *>(qt + d * PITCH + ty * RT + i);
                xs[i] = x.x, xs[i + 1] = x.y, xs[i + 2] = x.z, xs[i + 3] = x.w;
            }
            const float4 y = *reinterpret_cast<const float4 *>(kt + d * PITCH + tx * 4);
            const float ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int i = 0; i < RT; i++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    s[i][j] = fmaf(xs[i], ys[j], s[i][j]);
        }
        const bool masked = keys < BN || (a.causal && j0 + BN - 1 > first) || (a.window > 0 && j0 <= first + rows - 1 - a.window);
#pragma unroll
        for (int i = 0; i < RT; i++) {
            const int64_t p = first + ty * RT + i;
            float most = -1e30f;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int64_t key = j0 + tx * 4 + j;
                s[i][j] *= a.scale_log2e;
                if (masked && (key >= w.n_k || (a.causal && key > p) || (a.window > 0 && key <= p - a.window)))
                    s[i][j] = -INFINITY;
                most = fmaxf(most, s[i][j]);
            }
#pragma unroll
            for (int x = 1; x < 16; x <<= 1)
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, x));
            const float to = fmaxf(m[i], most), f = exp2_approx(m[i] - to);
            m[i] = to;
            l[i] *= f;
#pragma unroll
            for (int c = 0; c < OC; c++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    o[i][c][e] *= f;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                s[i][j] = exp2_approx(s[i][j] - to);
                l[i] += s[i][j];
            }
        }
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int i = 0; i < RT; i += 4)
                *reinterpret_cast<float4 *>(pt + (tx * 4 + j) * PITCH + ty * RT + i) = make_float4(s[i][j], s[i + 1][j], s[i + 2][j], s[i + 3][j]);
        __syncthreads();
        if (masked && odd_value) {
            // 0 times an infinity is NaN: rows that do not read a key skip it
            for (int n = 0; n < keys; n++)
#pragma unroll
                for (int i = 0; i < RT; i++) {
                    const float p = pt[n * PITCH + ty * RT + i];
                    const int64_t key = j0 + n, at = first + ty * RT + i;
                    if ((a.causal && key > at) || (a.window > 0 && key <= at - a.window))
                        continue;
#pragma unroll
                    for (int c = 0; c < OC; c++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            o[i][c][e] = fmaf(p, vs[n * DMAX + c * 64 + tx * 4 + e], o[i][c][e]);
                }
            continue;
        }
#pragma unroll 4
        for (int n = 0; n < BN; n++) {
            float xs[RT];
#pragma unroll
            for (int i = 0; i < RT; i += 4) {
                const float4 x = *reinterpret_cast<const float4 *>(pt + n * PITCH + ty * RT + i);
                xs[i] = x.x, xs[i + 1] = x.y, xs[i + 2] = x.z, xs[i + 3] = x.w;
            }
#pragma unroll
            for (int c = 0; c < OC; c++) {
                const float4 y = *reinterpret_cast<const float4 *>(vs + n * DMAX + c * 64 + tx * 4);
#pragma unroll
                for (int i = 0; i < RT; i++) {
                    o[i][c][0] = fmaf(xs[i], y.x, o[i][c][0]);
                    o[i][c][1] = fmaf(xs[i], y.y, o[i][c][1]);
                    o[i][c][2] = fmaf(xs[i], y.z, o[i][c][2]);
                    o[i][c][3] = fmaf(xs[i], y.w, o[i][c][3]);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < RT; i++) {
        const int r = ty * RT + i;
        float sum = l[i];
#pragma unroll
        for (int x = 1; x < 16; x <<= 1)
            sum += __shfl_xor_sync(0xffffffffu, sum, x);
        const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
        if (r >= rows)
            continue;
        T *dst = static_cast<T *>(a.out) + int64_t(w.first_q + w.row0 + r) * a.o_token + int64_t(head) * a.o_head;
#pragma unroll
        for (int c = 0; c < OC; c++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int d = c * 64 + tx * 4 + e;
                if (d < D)
                    dst[d] = from_f32<T>(o[i][c][e] * inverse);
            }
    }
}

template <typename T, int DMAX> int32_t launch_simt(ovk_ctx *ctx, const PromptArgs &a, unsigned tiles)
{
    constexpr size_t smem = simt_smem<DMAX>();
    OVK_CUDA(ctx, ovk_allow_smem(attention_prompt_simt_kernel<T, DMAX>, smem, ctx->device));
    attention_prompt_simt_kernel<T, DMAX><<<dim3(tiles, unsigned(a.heads)), threads_of<DMAX>(), smem, ctx->stream>>>(a);
    OVK_LAUNCHED(ctx, sizeof(T) == 4 ? "attention_prompt_f32" : "attention_prompt_simt");
    return OVK_OK;
}

}  // namespace

extern "C" int32_t ovk_attention_prompt(ovk_ctx *ctx, const ovk_prompt_params *p, const ovk_heads *q, const ovk_heads *k,
                                        const ovk_heads *v, const int32_t *cu_q, const int32_t *cu_k, const ovk_heads *out)
{
    const char *op = "AttentionPrompt";
    OVK_REQUIRE(ctx, p && q && k && v && out, "%s: null argument", op);
    OVK_REFUSE(ctx, !ovk_is_activation(p->dtype), "%s: dtype %d (f32 or f16)", op, p->dtype);
    OVK_REFUSE(ctx, p->head_dim < 1 || p->head_dim > 256, "%s: head_dim %lld (1 to 256)", op, (long long)p->head_dim);
    OVK_REQUIRE(ctx, p->q_tokens >= 0 && p->q_tokens < (int64_t(1) << 30) && p->k_tokens >= 0 && p->k_tokens < (int64_t(1) << 30) &&
                         p->batch >= 0 && p->batch < (1 << 24),
                "%s: %lld query and %lld key rows of %lld sequences", op, (long long)p->q_tokens, (long long)p->k_tokens, (long long)p->batch);
    OVK_REQUIRE(ctx, p->max_q >= 0, "%s: max_q %d", op, p->max_q);
    OVK_REQUIRE(ctx, p->window >= 0, "%s: window %lld", op, (long long)p->window);
    OVK_REQUIRE(ctx, p->scale - p->scale == 0.0f, "%s: scale is not finite", op);
    const size_t elem = ovk_elem_bytes(p->dtype);
    int32_t rc = ovk_check_heads(ctx, op, "q", q, p->q_tokens, p->head_dim, elem, false);
    if (rc == OVK_OK)
        rc = ovk_check_heads(ctx, op, "k", k, p->k_tokens, p->head_dim, elem, false);
    if (rc == OVK_OK)
        rc = ovk_check_heads(ctx, op, "v", v, p->k_tokens, p->head_dim, elem, false);
    if (rc == OVK_OK)
        rc = ovk_check_heads(ctx, op, "out", out, p->q_tokens, p->head_dim, elem, true);
    if (rc != OVK_OK)
        return rc;
    OVK_REQUIRE(ctx, k->heads == v->heads && q->heads == out->heads && q->heads % k->heads == 0,
                "%s: %lld query, %lld key, %lld value and %lld output heads", op, (long long)q->heads, (long long)k->heads,
                (long long)v->heads, (long long)out->heads);
    OVK_REQUIRE(ctx, p->batch == 0 || (cu_q && cu_k), "%s: null sequence bounds", op);
    OVK_REQUIRE(ctx, aligned_to(cu_q, 4) && aligned_to(cu_k, 4), "%s: misaligned sequence bounds", op);
    OVK_REQUIRE(ctx, ctx, "%s: null context", op);
    if (p->q_tokens == 0 || p->batch == 0)
        return OVK_OK;
    OVK_REQUIRE(ctx, q->heads <= 65535, "%s: %lld query heads", op, (long long)q->heads);
    DeviceGuard guard(ctx->device);
    PromptArgs a = {};
    a.q = q->data, a.k = k->data, a.v = v->data, a.out = out->data;
    a.q_token = q->token_stride, a.q_head = q->head_stride, a.k_token = k->token_stride, a.k_head = k->head_stride;
    a.v_token = v->token_stride, a.v_head = v->head_stride, a.o_token = out->token_stride, a.o_head = out->head_stride;
    a.cu_q = cu_q, a.cu_k = cu_k;
    a.q_tokens = int(p->q_tokens), a.k_tokens = int(p->k_tokens), a.batch = int(p->batch);
    a.heads = int(q->heads), a.group = int(q->heads / k->heads), a.head_dim = int(p->head_dim);
    a.causal = p->causal != 0, a.window = p->window, a.scale_log2e = p->scale * 1.4426950408889634f;
    a.max_q = p->max_q;
    a.vec = ovk_rows_aligned(q, elem) && ovk_rows_aligned(k, elem) && ovk_rows_aligned(v, elem);
    a.status = ctx->dev_status;
    const unsigned tiles = unsigned(prompt_tiles(a, BM));
    if (p->dtype == OVK_FLOAT)
        return p->head_dim <= 64    ? launch_simt<float, 64>(ctx, a, tiles)
               : p->head_dim <= 128 ? launch_simt<float, 128>(ctx, a, tiles)
                                    : launch_simt<float, 256>(ctx, a, tiles);
    bool taken = false;
    rc = ovk_prompt_tc(ctx, a, &taken);
    if (taken || rc != OVK_OK)
        return rc;
    return p->head_dim <= 64    ? launch_simt<__half, 64>(ctx, a, tiles)
           : p->head_dim <= 128 ? launch_simt<__half, 128>(ctx, a, tiles)
                                : launch_simt<__half, 256>(ctx, a, tiles);
}
