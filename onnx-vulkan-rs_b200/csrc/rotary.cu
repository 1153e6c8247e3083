// Rotary positions with several axes, for one or two tensors in one launch.
//
// Pair i of a head belongs to the axis whose section holds i and is turned by
// that axis's angle: out[a] = x[a] c - x[b] s, out[b] = x[b] c + x[a] s with
// c, s read from tables of cosines and sines.  Bytes bound it: every element is
// read and written once, three flops each; the tables are small and stay in L2.
// 16411 f16 tokens of 16 + 2 heads of 128 take 31.7 us (4.9 TB/s of 6.5 that a copy
// reaches), 33.8 when the launch waits for the whole of the kernel before.
//
// A thread owns the same few pairs (16 bytes of elements) of several heads of one
// token, so the table entries and positions are loaded once and kept in registers
// while it walks the heads.
#include "attention.cuh"

namespace {

struct RotaryView {
    const void *x[2];
    void *out[2];
    int64_t x_token[2], x_head[2], o_token[2], o_head[2];
    int heads[2];
};
struct RotaryArgs {
    RotaryView t;
    const void *positions, *cos, *sin;
    int64_t tokens, max_position;
    int items_per_row;  // turned vectors, then copied ones
    int turned, slots, heads_total;
    int pairs, rotary_dim;
    int axes, section_end[4];
    int index64, table_f16, table_vec;
    int *status;
};

__device__ __forceinline__ float table_at(const void *t, int64_t at, int f16)
{
    return f16 ? __half2float(static_cast<const __half *>(t)[at]) : static_cast<const float *>(t)[at];
}

// NP pairs a thread; IL: the two elements of a pair are neighbours.
template <typename T, bool IL, bool VEC>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs a)
{
    constexpr int V = VEC ? 16 / int(sizeof(T)) : (IL ? 2 : 1);  // elements of one access
    constexpr int NP = IL ? V / 2 : V;
    const int64_t item = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
    const int64_t row = item / a.items_per_row;
    const int vec = int(item - row * a.items_per_row);
    const int64_t token = row / a.slots;
    const int slot = int(row - token * a.slots);
    OVK_PDL_LAUNCH_DEPENDENTS();
    OVK_PDL_WAIT();
    if (token >= a.tokens)
        return;
    // a position outside the tables: the token's rows are zeros and the next flush reports it
    int64_t at[4] = {0, 0, 0, 0};
    bool bad = false;
#pragma unroll
    for (int k = 0; k < 4; k++)
        if (k < a.axes) {
            const int64_t i = k * a.tokens + token;
            at[k] = a.index64 ? static_cast<const int64_t *>(a.positions)[i] : int64_t(static_cast<const int32_t *>(a.positions)[i]);
            bad |= at[k] < 0 || at[k] >= a.max_position;
        }
    if (bad && vec == 0 && slot == 0)
        atomicExch(a.status, OVK_DEV_BAD_POSITION);
    const bool copied = vec >= a.turned;
    float c[NP], s[NP];
    const int pair0 = vec * NP;
    if (!copied && !bad) {
        int axis[NP];
#pragma unroll
        for (int e = 0; e < NP; e++) {
            axis[e] = 0;
#pragma unroll
            for (int k = 0; k < 3; k++)
                axis[e] += (k < a.axes - 1 && pair0 + e >= a.section_end[k]) ? 1 : 0;
        }
        const int64_t base[4] = {at[0] * a.pairs, at[1] * a.pairs, at[2] * a.pairs, at[3] * a.pairs};
        auto row_of = [&](int k) { return k == 0 ? base[0] : k == 1 ? base[1] : k == 2 ? base[2] : base[3]; };
        bool loaded = false;
        if constexpr (NP % 4 == 0) {
            if (a.table_vec && axis[0] == axis[NP - 1]) {
                const int64_t i = row_of(axis[0]) + pair0;
                load_row<float, NP, true>(static_cast<const float *>(a.cos) + i, c);
                load_row<float, NP, true>(static_cast<const float *>(a.sin) + i, s);
                loaded = true;
            }
        }
        if (!loaded) {
#pragma unroll
            for (int e = 0; e < NP; e++) {
                const int64_t i = row_of(axis[e]) + pair0 + e;
                c[e] = table_at(a.cos, i, a.table_f16);
                s[e] = table_at(a.sin, i, a.table_f16);
            }
        }
    } else {
        // zeros for a bad token; a copied element is one that is turned by nothing, with nothing beside it
#pragma unroll
        for (int e = 0; e < NP; e++)
            c[e] = bad ? 0.0f : 1.0f, s[e] = 0.0f;
    }
    for (int h = slot; h < a.heads_total; h += a.slots) {
        const int j = h >= a.t.heads[0] ? 1 : 0;
        const int hh = j ? h - a.t.heads[0] : h;
        const T *x = static_cast<const T *>(a.t.x[j]) + token * a.t.x_token[j] + hh * a.t.x_head[j];
        T *o = static_cast<T *>(a.t.out[j]) + token * a.t.o_token[j] + hh * a.t.o_head[j];
        if (copied) {
            const int e0 = a.rotary_dim + (vec - a.turned) * V;
            float v[V];
            load_row<T, V, VEC>(x + e0, v);
            if (bad) {
#pragma unroll
                for (int e = 0; e < V; e++)
                    v[e] = 0.0f;
            }
            store_row<T, V, VEC>(o + e0, v);
        } else if constexpr (IL) {
            float v[V];
            load_row<T, V, VEC>(x + vec * V, v);
            if (bad) {
#pragma unroll
                for (int e = 0; e < V; e++)
                    v[e] = 0.0f;
            }
#pragma unroll
            for (int e = 0; e < NP; e++) {
                const float p = v[2 * e], q = v[2 * e + 1];
                v[2 * e] = fmaf(p, c[e], -(q * s[e]));
                v[2 * e + 1] = fmaf(q, c[e], p * s[e]);
            }
            store_row<T, V, VEC>(o + vec * V, v);
        } else {
            float p[V], q[V];
            load_row<T, V, VEC>(x + pair0, p);
            load_row<T, V, VEC>(x + pair0 + a.pairs, q);
#pragma unroll
            for (int e = 0; e < V; e++) {
                if (bad)
                    p[e] = q[e] = 0.0f;
                const float t = p[e];
                p[e] = fmaf(t, c[e], -(q[e] * s[e]));
                q[e] = fmaf(q[e], c[e], t * s[e]);
            }
            store_row<T, V, VEC>(o + pair0, p);
            store_row<T, V, VEC>(o + pair0 + a.pairs, q);
        }
    }
}

template <typename T> cudaError_t launch(const RotaryArgs &a, bool il, bool vec, unsigned grid, cudaStream_t stream)
{
    void (*kernel)(RotaryArgs) = il ? (vec ? rotary_kernel<T, true, true> : rotary_kernel<T, true, false>)
                                    : (vec ? rotary_kernel<T, false, true> : rotary_kernel<T, false, false>);
    return ovk_launch_pdl(kernel, dim3(grid), dim3(256), 0, stream, a);
}

}  // namespace

extern "C" int32_t ovk_rotary(ovk_ctx *ctx, const ovk_rotary_params *p, int32_t count, const ovk_heads *x, const ovk_heads *out,
                              const void *positions, const void *cos_table, const void *sin_table)
{
    OVK_REQUIRE(ctx, p && x && out, "Rotary: null argument");
    OVK_REQUIRE(ctx, count == 1 || count == 2, "Rotary: %d tensors (1 or 2)", count);
    OVK_REFUSE(ctx, !ovk_is_activation(p->dtype), "Rotary: dtype %d (f32 or f16)", p->dtype);
    OVK_REFUSE(ctx, !ovk_is_activation(p->table_dtype), "Rotary: table dtype %d (f32 or f16)", p->table_dtype);
    OVK_REQUIRE(ctx, p->positions_dtype == OVK_INT32 || p->positions_dtype == OVK_INT64, "Rotary: position dtype %d", p->positions_dtype);
    OVK_REQUIRE(ctx, p->tokens >= 0 && p->tokens < (int64_t(1) << 31), "Rotary: %lld tokens", (long long)p->tokens);
    OVK_REQUIRE(ctx, p->head_dim >= 2 && p->head_dim <= 65536, "Rotary: head_dim %lld", (long long)p->head_dim);
    OVK_REQUIRE(ctx, p->rotary_dim >= 2 && p->rotary_dim % 2 == 0 && p->rotary_dim <= p->head_dim,
                "Rotary: rotary_dim %lld of head_dim %lld (even, at least 2)", (long long)p->rotary_dim, (long long)p->head_dim);
    OVK_REQUIRE(ctx, p->max_position >= 1 && p->max_position < (int64_t(1) << 40), "Rotary: tables of %lld positions", (long long)p->max_position);
    OVK_REQUIRE(ctx, p->axes >= 1 && p->axes <= 4, "Rotary: %d axes (1 to 4)", p->axes);
    const int64_t pairs = p->rotary_dim / 2;
    int64_t sum = 0;
    for (int k = 0; k < p->axes; k++) {
        OVK_REQUIRE(ctx, p->sections[k] >= 0, "Rotary: section %d has %d pairs", k, p->sections[k]);
        sum += p->sections[k];
    }
    OVK_REQUIRE(ctx, sum == pairs, "Rotary: the sections hold %lld pairs, rotary_dim %lld has %lld", (long long)sum,
                (long long)p->rotary_dim, (long long)pairs);
    const size_t elem = ovk_elem_bytes(p->dtype), telem = ovk_elem_bytes(p->table_dtype);
    for (int j = 0; j < count; j++) {
        int32_t rc = ovk_check_heads(ctx, "Rotary", "the input", &x[j], p->tokens, p->head_dim, elem, false);
        if (rc == OVK_OK)
            rc = ovk_check_heads(ctx, "Rotary", "the output", &out[j], p->tokens, p->head_dim, elem, true);
        if (rc != OVK_OK)
            return rc;
        OVK_REQUIRE(ctx, x[j].heads == out[j].heads, "Rotary: %lld heads in, %lld out", (long long)x[j].heads, (long long)out[j].heads);
        OVK_REQUIRE(ctx, x[j].data != out[j].data || (x[j].token_stride == out[j].token_stride && x[j].head_stride == out[j].head_stride),
                    "Rotary: in place, but with other strides");
    }
    OVK_REQUIRE(ctx, p->tokens == 0 || (positions && cos_table && sin_table), "Rotary: null positions or tables");
    OVK_REQUIRE(ctx, aligned_to(cos_table, telem) && aligned_to(sin_table, telem) &&
                         aligned_to(positions, p->positions_dtype == OVK_INT64 ? 8 : 4), "Rotary: misaligned positions or tables");
    OVK_REQUIRE(ctx, ctx, "Rotary: null context");
    if (p->tokens == 0)
        return OVK_OK;
    DeviceGuard guard(ctx->device);

    RotaryArgs a = {};
    const bool il = p->interleaved != 0;
    const int v16 = int(16 / elem);
    bool vec = (il ? p->rotary_dim : pairs) % v16 == 0 && (p->head_dim - p->rotary_dim) % v16 == 0;
    for (int j = 0; j < count; j++) {
        a.t.x[j] = x[j].data, a.t.out[j] = out[j].data;
        a.t.x_token[j] = x[j].token_stride, a.t.x_head[j] = x[j].head_stride;
        a.t.o_token[j] = out[j].token_stride, a.t.o_head[j] = out[j].head_stride;
        a.t.heads[j] = int(x[j].heads);
        a.heads_total += a.t.heads[j];
        vec = vec && ovk_rows_aligned(&x[j], elem) && ovk_rows_aligned(&out[j], elem);
    }
    const int v = vec ? v16 : (il ? 2 : 1), np = il ? v / 2 : v;
    // an element outside every pair; odd counts need single elements, which the vector of two does not give
    const int64_t rest = p->head_dim - p->rotary_dim;
    OVK_REFUSE(ctx, rest % v != 0, "Rotary: interleaved pairs with an odd number of unturned elements (%lld)", (long long)rest);
    a.positions = positions, a.cos = cos_table, a.sin = sin_table;
    a.tokens = p->tokens, a.max_position = p->max_position;
    a.turned = int(pairs / np);
    // a bad token's copied elements become zeros, so they are visited in place too
    a.items_per_row = a.turned + int(rest / v);
    a.pairs = int(pairs), a.rotary_dim = int(p->rotary_dim);
    a.axes = p->axes;
    for (int k = 0, end = 0; k < p->axes; k++)
        a.section_end[k] = end += p->sections[k];
    a.index64 = p->positions_dtype == OVK_INT64;
    a.table_f16 = p->table_dtype == OVK_FLOAT16;
    a.table_vec = !a.table_f16 && pairs % 4 == 0 && aligned_to(cos_table, 16) && aligned_to(sin_table, 16);
    a.status = ctx->dev_status;
    // head slots: as many threads as fill the machine twice, but at least one per four heads, so that
    // a thread has several independent rows in flight
    const int64_t per_slot = p->tokens * a.items_per_row, fill = int64_t(ctx->sm_count) * 4096;
    a.slots = int(std::min<int64_t>(a.heads_total, std::max<int64_t>(ceil_div64(fill, per_slot), ceil_div64(a.heads_total, 4))));
    const int64_t items = per_slot * a.slots;
    OVK_REQUIRE(ctx, ceil_div64(items, 256) < (int64_t(1) << 31), "Rotary: %lld tokens of %d heads are too many for one call",
                (long long)p->tokens, a.heads_total);
    const unsigned grid = unsigned(ceil_div64(items, 256));
    OVK_CUDA(ctx, p->dtype == OVK_FLOAT ? launch<float>(a, il, vec, grid, ctx->stream) : launch<__half>(a, il, vec, grid, ctx->stream));
    OVK_LAUNCHED(ctx, vec ? "rotary" : "rotary_scalar");
    return OVK_OK;
}
