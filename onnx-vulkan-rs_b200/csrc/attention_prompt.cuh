// Shared by the two kernels of ovk_attention_prompt: arguments, and which rows and
// keys a block works on.
#pragma once

#include "attention.cuh"

struct PromptArgs {
    const void *q, *k, *v;
    void *out;
    int64_t q_token, q_head, k_token, k_head, v_token, v_head, o_token, o_head;
    const int32_t *cu_q, *cu_k;
    int q_tokens, k_tokens, batch, heads, group, head_dim;
    int causal, vec, max_q;
    int64_t window;
    float scale_log2e;
    int *status;
};

// A tile of query rows: rows row0 .. of sequence b; b < 0: the batch has fewer tiles.
struct PromptTile {
    int b, row0, first_q, n_q, first_k, n_k;
};
struct KeyRange {
    int64_t begin, end;
};

#ifdef __CUDACC__
// The index-th tile of BM query rows of the batch, counted from the last one (under a causal mask the
// last tiles are the long ones, which go first).  One warp; the bounds are read 32 sequences at a time,
// back to front.  Bounds that leave the tensors make the sequence one without rows (or without keys); who
// reads such bounds reports them, and the last block of `blocks` reads those of the whole batch.
template <int BM> __device__ __forceinline__ void find_prompt_tile(const PromptArgs &a, int index, int blocks, PromptTile &out)
{
    const int lane = threadIdx.x & 31;
    int before = 0;
    bool found = false;
    PromptTile w = {-1, 0, 0, 0, 0, 0};
    for (int base = a.batch - 1; base >= 0; base -= 32) {
        const int b = base - lane;
        int first = 0, n = 0, first_k = 0, end_k = 0;
        if (b >= 0) {
            first = a.cu_q[b];
            const int end = a.cu_q[b + 1];
            first_k = a.cu_k[b], end_k = a.cu_k[b + 1];  // fetched with the others: one way to memory, not two
            n = end - first;
            if (first < 0 || end < first || end > a.q_tokens || (a.max_q > 0 && n > a.max_q)) {
                n = 0;
                atomicExch(a.status, OVK_DEV_BAD_SEQUENCE);
            }
        }
        const int tiles = (n + BM - 1) / BM;
        int sum = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int left = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o)
                sum += left;
        }
        const bool mine = index >= before + sum - tiles && index < before + sum;
        if (mine) {
            w.b = b, w.first_q = first, w.n_q = n;
            w.row0 = (before + sum - 1 - index) * BM;
            w.first_k = first_k;
            w.n_k = end_k - first_k;
            if (first_k < 0 || end_k < first_k || end_k > a.k_tokens) {
                w.n_k = w.first_k = 0;
                atomicExch(a.status, OVK_DEV_BAD_SEQUENCE);
            }
            out = w;
        }
        found |= __any_sync(0xffffffffu, mine);
        if (found && index < blocks - 1)
            return;
        before += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0 && !found)
        out = w;
}

// The keys that any of the tile's rows reads.
__device__ __forceinline__ KeyRange key_range(const PromptArgs &a, const PromptTile &w, int rows)
{
    const int64_t first = int64_t(w.n_k) - w.n_q + w.row0;
    KeyRange r = {0, w.n_k};
    if (a.window > 0)
        r.begin = max(int64_t(0), first - a.window + 1);
    if (a.causal)
        r.end = min(r.end, first + rows);
    return r;
}
#endif

// Tiles of BM query rows that a batch may have.
static inline int64_t prompt_tiles(const PromptArgs &a, int64_t bm)
{
    const int64_t by_rows = ceil_div64(a.q_tokens, bm) + a.batch;
    return a.max_q > 0 ? std::min(by_rows, a.batch * ceil_div64(a.max_q, bm)) : by_rows;
}

// f16 on the tensor cores; *taken says whether the call's layout is one it takes
int32_t ovk_prompt_tc(ovk_ctx *ctx, const PromptArgs &a, bool *taken);
