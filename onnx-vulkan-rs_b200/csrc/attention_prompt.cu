// ovk_attention_prompt: checks and dispatch, and the kernel for f32 and for
// layouts the tensor-core kernel (attention_prompt_tc.cu) does not take.
//
//   x[i][j] = scale * q[i] . k[j],  out[i] = sum_j 2^(x log2 e - m) v[j] / sum_j 2^(x log2 e - m),
//
// one pass over the keys with the running maximum m and sum of each row.  A block
// holds 64 query rows of one head and walks 64 or 32 keys at a time; a thread
// computes 8 (256-wide heads: 4) x 4 or 2 scores, then as many rows x head_dim / 16
// columns of the result.  All of it is f32 arithmetic on the CUDA cores: a step over
// four d is twelve 16-byte loads of shared memory for 128 multiply-adds, and both pipes
// are busy half of the time (adders 49 %, shared memory 50 %, issue 62 %, 2.2 warps a
// scheduler).  Four chunks of some 600 queries after 333 keys, f32, 8 heads of 64: 189 us,
// 20.8 TFLOP/s counted over the pairs that are read (29 % of the adders' 72): the diagonal's
// tiles are computed whole, and 376 blocks of unequal length are one uneven wave.
#include "attention_prompt.cuh"

namespace {

constexpr int BM = 64;

// Per padded head_dim: rows of a thread (eight where the registers hold their results) and keys of a tile (so that two
// blocks or more fit an SM).  Rows in shared memory are four floats apart beyond their length, which spreads the eight
// rows that a quarter of a warp reads at once over all banks.
template <int DMAX> struct Simt {
    static constexpr int RT = DMAX == 256 ? 4 : 8, THREADS = BM / RT * 16, BN = DMAX == 64 ? 64 : 32, CT = BN / 16;
    static constexpr int PITCH = DMAX + 4, P_PITCH = BM + 4, OC = DMAX / 64;
    static constexpr size_t SMEM = size_t(BM * PITCH + BN * PITCH + BN * DMAX + BN * P_PITCH) * 4;
};

// ROWS rows of a [tokens, heads, d] tensor into shared memory as f32, zeros outside.  f32 rows on 16-byte boundaries are
// copied asynchronously (wait_copies makes them visible to the thread that copied them).
template <typename T, int DMAX, int ROWS, int PITCH>
__device__ __forceinline__ void load_rows(float *dst, const T *base, int64_t stride, int rows, int d, bool vec)
{
    constexpr int V = 16 / sizeof(T), PER = DMAX / V;
#pragma unroll 4
    for (int i = threadIdx.x; i < ROWS * PER; i += Simt<DMAX>::THREADS) {
        const int r = i / PER, e = (i - r * PER) * V;
        const T *src = base + int64_t(r) * stride + e;
        float *to = dst + r * PITCH + e;
        if constexpr (sizeof(T) == 4) {
            if (vec && (e + V <= d || e >= d)) {
                const int bytes = r < rows && e < d ? 16 : 0;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(uint32_t(__cvta_generic_to_shared(to))),
                             "l"(bytes ? static_cast<const void *>(src) : static_cast<const void *>(base)), "r"(bytes)
                             : "memory");
                continue;
            }
        }
        float v[V];
        if (r < rows && vec && e + V <= d) {
            load_row<T, V, true>(src, v);
        } else {
#pragma unroll
            for (int u = 0; u < V; u++)
                v[u] = r < rows && e + u < d ? to_f32<T>(src[u]) : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < V; u += 4)
            *reinterpret_cast<float4 *>(to + u) = make_float4(v[u], v[u + 1], v[u + 2], v[u + 3]);
    }
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <typename T, int DMAX>
__global__ void __launch_bounds__(Simt<DMAX>::THREADS) attention_prompt_simt_kernel(const PromptArgs a)
{
    using C = Simt<DMAX>;
    constexpr int RT = C::RT, CT = C::CT, BN = C::BN, PITCH = C::PITCH, P_PITCH = C::P_PITCH, OC = C::OC, THREADS = C::THREADS;
    extern __shared__ __align__(16) float sm[];
    float *const qs = sm, *const ks = qs + BM * PITCH, *const vs = ks + BN * PITCH, *const pt = vs + BN * DMAX;
    __shared__ PromptTile where;
    const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
    if (tid < 32)
        find_prompt_tile<BM>(a, blockIdx.x / a.heads, gridDim.x / a.heads, where);  // the heads of a tile together, the long tiles first
    __syncthreads();
    const PromptTile w = where;
    if (w.b < 0)
        return;
    const int head = blockIdx.x % a.heads, kv_head = head / a.group, D = a.head_dim;
    const int rows = min(BM, w.n_q - w.row0);
    const int64_t first = int64_t(w.n_k) - w.n_q + w.row0;  // position of the tile's first row
    const KeyRange range = key_range(a, w, rows);
    const T *q = static_cast<const T *>(a.q) + int64_t(w.first_q + w.row0) * a.q_token + int64_t(head) * a.q_head;
    const T *k = static_cast<const T *>(a.k) + int64_t(w.first_k) * a.k_token + int64_t(kv_head) * a.k_head;
    const T *v = static_cast<const T *>(a.v) + int64_t(w.first_k) * a.v_token + int64_t(kv_head) * a.v_head;
    // K and V have one buffer each: the next K comes while the weights are computed and used, the next V beside the
    // next scores
    auto fetch_k = [&](int64_t j0) {
        if (j0 < range.end)
            load_rows<T, DMAX, BN, PITCH>(ks, k + j0 * a.k_token, a.k_token, int(min(int64_t(BN), range.end - j0)), D, a.vec);
        commit_copies();
    };
    auto fetch_v = [&](int64_t j0) {
        if (j0 < range.end)
            load_rows<T, DMAX, BN, DMAX>(vs, v + j0 * a.v_token, a.v_token, int(min(int64_t(BN), range.end - j0)), D, a.vec);
        commit_copies();
    };
    load_rows<T, DMAX, BM, PITCH>(qs, q, a.q_token, rows, D, a.vec);
    fetch_k(range.begin);
    fetch_v(range.begin);

    float o[RT][OC][4], m[RT], l[RT];
#pragma unroll
    for (int i = 0; i < RT; i++) {
        m[i] = NO_SCORE, l[i] = 0.0f;
#pragma unroll
        for (int c = 0; c < OC; c++)
            o[i][c][0] = o[i][c][1] = o[i][c][2] = o[i][c][3] = 0.0f;
    }
    for (int64_t j0 = range.begin; j0 < range.end; j0 += BN) {
        const int keys = int(min(int64_t(BN), range.end - j0));
        wait_copies<1>();  // K, and the first time Q; V may still be on its way
        __syncthreads();
        float s[RT][CT];
#pragma unroll
        for (int i = 0; i < RT; i++)
#pragma unroll
            for (int j = 0; j < CT; j++)
                s[i][j] = 0.0f;
#pragma unroll 2
        for (int d = 0; d < DMAX; d += 4) {
            float4 y[CT];
#pragma unroll
            for (int j = 0; j < CT; j++)
                y[j] = *reinterpret_cast<const float4 *>(ks + (tx + 16 * j) * PITCH + d);
#pragma unroll
            for (int i = 0; i < RT; i++) {
                const float4 x = *reinterpret_cast<const float4 *>(qs + (ty * RT + i) * PITCH + d);
#pragma unroll
                for (int j = 0; j < CT; j++)
                    s[i][j] = fmaf(x.x, y[j].x, fmaf(x.y, y[j].y, fmaf(x.z, y[j].z, fmaf(x.w, y[j].w, s[i][j]))));
            }
        }
        const bool masked = keys < BN || (a.causal && j0 + BN - 1 > first) || (a.window > 0 && j0 <= first + rows - 1 - a.window);
#pragma unroll
        for (int i = 0; i < RT; i++) {
            const int64_t p = first + ty * RT + i;
            float most = NO_SCORE;
#pragma unroll
            for (int j = 0; j < CT; j++) {
                const int64_t key = j0 + tx + 16 * j;
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
            for (int j = 0; j < CT; j++) {
                s[i][j] = exp2_approx(s[i][j] - to);
                l[i] += s[i][j];
            }
        }
#pragma unroll
        for (int j = 0; j < CT; j++)
#pragma unroll
            for (int i = 0; i < RT; i += 4)
                *reinterpret_cast<float4 *>(pt + (tx + 16 * j) * P_PITCH + ty * RT + i) = make_float4(s[i][j], s[i + 1][j], s[i + 2][j], s[i + 3][j]);
        wait_copies<0>();
        // an infinity or NaN among values that some row must not read: 0 times it is NaN, so such rows skip it
        bool odd_value = false;
        __syncthreads();
        fetch_k(j0 + BN);
        if (masked) {
            for (int i = tid; i < BN * DMAX / 4; i += THREADS) {
                const float4 x = reinterpret_cast<const float4 *>(vs)[i];
                odd_value |= !((x.x - x.x) + (x.y - x.y) + (x.z - x.z) + (x.w - x.w) == 0.0f);
            }
            odd_value = __syncthreads_or(odd_value);
        }
        if (odd_value) {
            for (int n = 0; n < keys; n++)
#pragma unroll
                for (int i = 0; i < RT; i++) {
                    const float p = pt[n * P_PITCH + ty * RT + i];
                    const int64_t key = j0 + n, at = first + ty * RT + i;
                    if ((a.causal && key > at) || (a.window > 0 && key <= at - a.window))
                        continue;
#pragma unroll
                    for (int c = 0; c < OC; c++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            o[i][c][e] = fmaf(p, vs[n * DMAX + c * 64 + tx * 4 + e], o[i][c][e]);
                }
        } else {
#pragma unroll 4
            for (int n = 0; n < BN; n++) {
                float xs[RT];
#pragma unroll
                for (int i = 0; i < RT; i += 4) {
                    const float4 x = *reinterpret_cast<const float4 *>(pt + n * P_PITCH + ty * RT + i);
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
        __syncthreads();
        fetch_v(j0 + BN);
    }
    wait_copies<0>();
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

template <typename T, int DMAX> int32_t launch_simt(ovk_ctx *ctx, const PromptArgs &a, unsigned blocks)
{
    using C = Simt<DMAX>;
    OVK_CUDA(ctx, ovk_allow_smem(attention_prompt_simt_kernel<T, DMAX>, C::SMEM, ctx->device));
    attention_prompt_simt_kernel<T, DMAX><<<blocks, C::THREADS, C::SMEM, ctx->stream>>>(a);
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
    const float factor = ovk_scale_log2e(p->scale);
    OVK_REQUIRE(ctx, factor - factor == 0.0f, "%s: scale %g is not finite, or not in powers of two", op, double(p->scale));
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
    DeviceGuard guard(ctx->device);
    PromptArgs a = {};
    a.q = q->data, a.k = k->data, a.v = v->data, a.out = out->data;
    a.q_token = q->token_stride, a.q_head = q->head_stride, a.k_token = k->token_stride, a.k_head = k->head_stride;
    a.v_token = v->token_stride, a.v_head = v->head_stride, a.o_token = out->token_stride, a.o_head = out->head_stride;
    a.cu_q = cu_q, a.cu_k = cu_k;
    a.q_tokens = int(p->q_tokens), a.k_tokens = int(p->k_tokens), a.batch = int(p->batch);
    a.heads = int(q->heads), a.group = int(q->heads / k->heads), a.head_dim = int(p->head_dim);
    a.causal = p->causal != 0, a.scale_log2e = factor;
    a.window = ovk_window(p->window);
    a.max_q = p->max_q;
    a.vec = ovk_rows_aligned(q, elem) && ovk_rows_aligned(k, elem) && ovk_rows_aligned(v, elem);
    a.status = ctx->dev_status;
    const int64_t tiles = prompt_tiles(a, BM) * a.heads;
    OVK_REQUIRE(ctx, tiles < (int64_t(1) << 31), "%s: %lld query rows of %d heads are too many for one call", op, (long long)p->q_tokens, a.heads);
    const unsigned blocks = unsigned(tiles);
    if (p->dtype == OVK_FLOAT)
        return p->head_dim <= 64    ? launch_simt<float, 64>(ctx, a, blocks)
               : p->head_dim <= 128 ? launch_simt<float, 128>(ctx, a, blocks)
                                    : launch_simt<float, 256>(ctx, a, blocks);
    bool taken = false;
    rc = ovk_prompt_tc(ctx, a, &taken);
    if (taken || rc != OVK_OK)
        return rc;
    return p->head_dim <= 64    ? launch_simt<__half, 64>(ctx, a, blocks)
           : p->head_dim <= 128 ? launch_simt<__half, 128>(ctx, a, blocks)
                                : launch_simt<__half, 256>(ctx, a, blocks);
}
