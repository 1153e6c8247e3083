// Attention of a few new tokens over the paged 4-bit cache: the kernel and its
// launch plan.  Instantiated per head_dim by attention_kv4_*.cu.
//
//   x[r][t] = scale * sum_d q[r][d] K[t][d],  p = 2^(x log2 e - m),
//   out[r] = sum_t p V[t] / sum_t p,          K, V[t][d] = (code - zero) * s[t][block of d]
//
// Bytes bound it: a token and key head cost head_dim bytes of codes and 2.5 bytes
// a block of 32, read once whatever the number of query heads.  At the memory's
// rate an SM must take in a token every six cycles, so what is spent per code
// decides; CUDA cores alone (three operations a code and row) cannot keep up.
//
//  - f16: codes go to mma.sync.m16n8k16 as fp16 SUBNORMALS: a nibble masked into
//    the low four bits of a half is the number code * 2^-24, into the next four
//    code * 2^-20 - exact, one logic operation for two codes, no bias to remove.
//    2^24 goes into the row's factor; elements on the second position have their
//    query value (and, for V, their output row) divided by 16.  The tensor core
//    does not normalise such products before it aligns them, which costs ten bits:
//    sums are good to about 2^-17, well below what fp16 results show.
//  - f32: codes are OR-ed into 1024 and 64, whose last bits they fill, and 1024 +
//    zero or 64 + zero subtracted: the integer code - zero, normalised, one
//    operation more.
//  - Tokens are the 16 rows of A, query rows the 8 columns of B, so a group of up
//    to eight query rows costs no more than one.
//  - K: a chunk of 32 elements has its own accumulator (f16: started at -zero *
//    sum(q) of the chunk, one product instead of a subtraction per code), then
//    scaled by its f32 scale: codes and queries enter the product exactly.
//  - V: codes minus zero (exact) times p * s rounded to fp16.
//    f32 callers get q and p * s as two fp16 parts, 22 bits.
//  - The running maximum moves only when a score passes it by 6 (p by 2^6) or a V
//    scale its own largest by 2^3: p * s starts at 2^6 to 2^7, so it stays below
//    2^16 and is a normal fp16 number down to 2^-20 of the largest, and a step
//    needs one vote, not a reduction.
//
// Every CTA takes an equal run of 64-token units of the whole batch (lengths are
// read on the device), four warps of it alternate 16-token steps, each with its
// own cp.async ring.  A run that begins or ends inside a sequence leaves a partial
// result; a second kernel joins those in CTA order, so results do not depend on
// timing.
#pragma once

#include <type_traits>

#include "attention.cuh"
#include "umma.cuh"

struct Kv4Args {
    const uint8_t *codes[2];
    const uint8_t *scales[2];
    const uint8_t *zero_points[2];
    const int32_t *cu, *lens, *table;
    const void *q;
    void *out;
    int64_t q_token, q_head, o_token, o_head;
    int64_t max_pages, window;
    int tokens, batch, pages, kv_heads, group, page_size, page_shift;  // page_shift < 0: not a power of two
    int blocks, chunk_shift;  // scales a row; log2(block_size / 32)
    float scale_log2e;
    float *partial;
    int4 *meta;
    int *status;
};

namespace kv4 {

constexpr int WARPS = 4, STEP = 16, UNIT = WARPS * STEP;
constexpr float NONE = -1e30f;  // the maximum of a row that has seen nothing (in powers of two)

template <int D_, int NT_, int PARTS_> struct Shape {
    static constexpr int D = D_, NT = NT_, PARTS = PARTS_;
    static constexpr int NCH = D / 32, ROWS = 8 * NT, ROW_BYTES = D / 2, CPR = D / 32;
    static constexpr int STAGES = (D == 256 && NT == 1) ? 3 : 4;
    static constexpr int CODES = STEP * ROW_BYTES;        // of K or of V, one stage
    static constexpr int RAW = 32 * (16 + 4 + 4);         // scales, zero points, row numbers of a stage
    static constexpr int STAGE = 2 * CODES + RAW;
    static constexpr int SZ = 2 * STEP * NCH * 4;         // {scale, zero} per token and chunk, K and V
    static constexpr int WARP_BYTES = STAGES * STAGE + SZ;
    static constexpr int QF = PARTS * NT * NCH * 512;     // query fragments
    static constexpr int MERGE = WARPS * ROWS * (D + 4) * 4;
    static constexpr int RING = WARPS * WARP_BYTES > MERGE ? WARPS * WARP_BYTES : MERGE;
    static constexpr int SMEM = RING + QF + ROWS * (NCH + 1) * 4 + WARPS * ROWS * 8 + 64;
    static constexpr bool Q_REGS = PARTS * NT * NCH * 4 <= 16;
    static constexpr int CTAS = D == 256 ? (NT == 1 ? 3 : 2) : (NT * PARTS == 1 ? 4 : 3);  // on an SM
    static constexpr bool SUBNORMAL = PARTS == 1;         // how codes enter the products
    static constexpr int SLOT = ROWS * (D + 2);           // floats of a partial result
};

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v)
{
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
template <int BYTES> __device__ __forceinline__ void copy_async(uint32_t dst, const void *src, int valid)
{
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(valid) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint32_t lds32(uint32_t a)
{
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a));
    return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t a)
{
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ void sts32(uint32_t a, uint32_t v) { asm volatile("st.shared.b32 [%0], %1;" ::"r"(a), "r"(v) : "memory"); }
__device__ __forceinline__ float half_lo(uint32_t w) { return __half2float(__ushort_as_half(uint16_t(w))); }
__device__ __forceinline__ float half_hi(uint32_t w) { return __half2float(__ushort_as_half(uint16_t(w >> 16))); }
// Two codes as halves: the nibbles at bits 0-3 and 16-19 of `w` (SECOND: 4-7 and 20-23).
template <bool SUBNORMAL, bool SECOND> __device__ __forceinline__ uint32_t codes_at(uint32_t w)
{
    return (w & (SECOND ? 0x00f000f0u : 0x000f000fu)) | (SUBNORMAL ? 0u : SECOND ? 0x54005400u : 0x64006400u);
}
// The same form of a zero point's halves, from the first position's.
template <bool SUBNORMAL> __device__ __forceinline__ uint32_t second_zero(uint32_t z)
{
    return SUBNORMAL ? z << 4 : ((z & 0x000f000fu) << 4) | 0x54005400u;
}
__device__ __forceinline__ uint32_t sub_halves(uint32_t a, uint32_t b)
{
    const __half2 h = __hsub2(*reinterpret_cast<__half2 *>(&a), *reinterpret_cast<__half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&h);
}

// What the sequence arrays say about sequence b.
struct Sequence {
    int first, n;       // packed rows
    int len, start;     // tokens in the cache; the first one that is read, on a step's boundary
    int units, tiles;   // 64-token units; tiles of query rows
};
template <int ROWS> __device__ __forceinline__ Sequence sequence(const Kv4Args &a, int b, bool report)
{
    Sequence s;
    const int end = a.cu[b + 1];
    s.first = a.cu[b];
    s.n = end - s.first;
    if (s.first < 0 || end > a.tokens || end < s.first) {
        if (report)
            atomicExch(a.status, OVK_DEV_BAD_SEQUENCE);
        s.n = 0;
    }
    s.len = a.lens[b];
    if (s.len < 0 || s.len > (1 << 30) || s.len > a.max_pages * a.page_size) {
        if (report && s.n > 0)
            atomicExch(a.status, OVK_DEV_BAD_PAGE);
        s.len = 0;
    }
    s.start = 0;
    if (a.window > 0) {
        const int64_t from = int64_t(s.len) - s.n - a.window + 1;
        s.start = from > 0 ? int(from) & ~(STEP - 1) : 0;
    }
    s.units = s.n > 0 ? max(1, (s.len - s.start + UNIT - 1) / UNIT) : 0;
    s.tiles = int((int64_t(s.n) * a.group + ROWS - 1) / ROWS);
    return s;
}

template <typename T, int D, int NT, int PARTS>
__global__ void __launch_bounds__(WARPS * 32, Shape<D, NT, PARTS>::CTAS) attention_kv4_kernel(const __grid_constant__ Kv4Args a)
{
    using S = Shape<D, NT, PARTS>;
    constexpr int NCH = S::NCH, ROWS = S::ROWS;
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    uint8_t *const qf = smem + S::RING;
    float *const q_sum = reinterpret_cast<float *>(qf + S::QF);       // [NCH][ROWS]
    float *const q_factor = q_sum + ROWS * NCH;                       // [ROWS]
    float *const stat = q_factor + ROWS;                              // [WARPS][ROWS] maxima, then sums
    int64_t *const shared64 = reinterpret_cast<int64_t *>(smem + S::SMEM - 64);
    const uint32_t ring = umma::smem_u32(smem) + warp * S::WARP_BYTES;
    const uint32_t sz = ring + S::STAGES * S::STAGE;

    OVK_PDL_LAUNCH_DEPENDENTS();
    if (tid == 0)
        a.meta[blockIdx.x] = make_int4(0, 0, 0, 0);

    // ------------------------------------------------ this CTA's run of units
    int64_t total = 0;
    for (int b = tid; b < a.batch; b += WARPS * 32) {
        const Sequence s = sequence<ROWS>(a, b, blockIdx.x == 0);
        total += int64_t(s.units) * s.tiles * a.kv_heads;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        total += __shfl_xor_sync(0xffffffffu, total, o);
    if (lane == 0)
        shared64[warp] = total;
    __syncthreads();
    total = shared64[0] + shared64[1] + shared64[2] + shared64[3];
    const int64_t ctas = min(int64_t(gridDim.x), total);  // each has at least one unit
    if (blockIdx.x >= ctas)
        return;
    int64_t at = blockIdx.x * total / ctas;
    const int64_t end = (blockIdx.x + 1) * total / ctas;
    // the sequence that holds unit `at`: a scan over the batch, 128 sequences at a time
    int b = 0;
    int64_t before = 0;  // units of the sequences before b
    for (int base = 0;; base += WARPS * 32) {
        const int mine = base + tid;
        int64_t sum = 0;
        if (mine < a.batch) {
            const Sequence s = sequence<ROWS>(a, mine, false);
            sum = int64_t(s.units) * s.tiles * a.kv_heads;
        }
        const int64_t own = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t left = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o)
                sum += left;
        }
        __syncthreads();
        if (lane == 31)
            shared64[warp] = sum;
        __syncthreads();
        int64_t offset = before;
        for (int w = 0; w < warp; w++)
            offset += shared64[w];
        const int64_t chunk_end = before + shared64[0] + shared64[1] + shared64[2] + shared64[3];
        if (at >= offset + sum - own && at < offset + sum) {
            shared64[4] = mine;
            shared64[5] = offset + sum - own;
        }
        __syncthreads();
        if (at < chunk_end) {
            b = int(shared64[4]);
            before = shared64[5];
            break;
        }
        before = chunk_end;
    }
    Sequence seq = sequence<ROWS>(a, b, false);
    int64_t in_seq = at - before;
    int item = int(in_seq / seq.units), unit = int(in_seq - int64_t(item) * seq.units);

    while (true) {
        const int units_here = int(min(int64_t(seq.units - unit), end - at));
        const int tile = item / a.kv_heads, head = item - tile * a.kv_heads;
        const int rows = int(min(int64_t(ROWS), int64_t(seq.n) * a.group - int64_t(tile) * ROWS));
        const int t_begin = seq.start + unit * UNIT, t_end = min(seq.len, seq.start + (unit + units_here) * UNIT);

        // -------------------------------------------------- query fragments
        __syncthreads();  // the segment before has been read
        if (tid < ROWS * 8) {
            const int r = tid >> 3, j = tid & 7;
            constexpr int GROUPS = D / 64;  // groups of eight elements a thread
            float v[GROUPS][8], top = 0.0f;
            if (r < rows) {
                const int64_t row = int64_t(tile) * ROWS + r;
                const int token = int(row / a.group);
                const T *src = static_cast<const T *>(a.q) + int64_t(seq.first + token) * a.q_token +
                               (int64_t(head) * a.group + (row - int64_t(token) * a.group)) * a.q_head;
#pragma unroll
                for (int i = 0; i < GROUPS; i++)
                    load_row<T, 8, true>(src + 8 * (j + 8 * i), v[i]);
            } else {
#pragma unroll
                for (int i = 0; i < GROUPS; i++)
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        v[i][e] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < GROUPS; i++)
#pragma unroll
                for (int e = 0; e < 8; e++)
                    top = fmaxf(top, fabsf(v[i][e]));
            constexpr uint32_t mask = 0xffffffffu;  // whole warps take part
#pragma unroll
            for (int o = 1; o < 8; o <<= 1)
                top = fmaxf(top, __shfl_xor_sync(mask, top, o));
            // a power of two brings the row's largest value to 2^10 .. 2^11, clear of fp16's ends
            const int exponent = int(__float_as_uint(top) >> 23);
            const int k = (exponent == 255 || top == 0.0f) ? 0 : 10 - (exponent - 127);
            const float f1 = ldexpf(1.0f, k / 2), f2 = ldexpf(1.0f, k - k / 2);
#pragma unroll
            for (int i = 0; i < GROUPS; i++) {
                const int c = (j + 8 * i) >> 2;
                float sum = 0.0f;
                float hi[8], lo[8];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float x = v[i][e] * f1 * f2;
                    // a part on the second nibble position is rounded as it will be used, divided by 16
                    const float f = S::SUBNORMAL && (e & 1) ? 0.0625f : 1.0f, fi = S::SUBNORMAL && (e & 1) ? 16.0f : 1.0f;
                    hi[e] = __half2float(__float2half_rn(x * f));
                    lo[e] = PARTS == 2 ? __half2float(__float2half_rn(x * f - hi[e])) : 0.0f;
                    sum += hi[e] * fi + lo[e] * fi;
                }
                sum += __shfl_xor_sync(mask, sum, 1);
                sum += __shfl_xor_sync(mask, sum, 2);
                const int slot = ((r >> 3) * NCH + c) * 32 + (r & 7) * 4 + (j & 3);
                uint4 *dst = reinterpret_cast<uint4 *>(qf);
                dst[slot] = make_uint4(pack_halves(hi[0], hi[4]), pack_halves(hi[1], hi[5]), pack_halves(hi[2], hi[6]),
                                       pack_halves(hi[3], hi[7]));
                if constexpr (PARTS == 2)
                    dst[NT * NCH * 32 + slot] = make_uint4(pack_halves(lo[0], lo[4]), pack_halves(lo[1], lo[5]),
                                                           pack_halves(lo[2], lo[6]), pack_halves(lo[3], lo[7]));
                if ((j & 3) == 0)
                    q_sum[c * ROWS + r] = sum;
            }
            if (j == 0)
                q_factor[r] = ldexpf(a.scale_log2e, (S::SUBNORMAL ? 24 : 0) - k);
        }
        __syncthreads();
        uint4 bq[S::Q_REGS ? PARTS : 1][S::Q_REGS ? NT : 1][S::Q_REGS ? NCH : 1];
        if constexpr (S::Q_REGS) {
#pragma unroll
            for (int p = 0; p < PARTS; p++)
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int c = 0; c < NCH; c++)
                        bq[p][n][c] = reinterpret_cast<const uint4 *>(qf)[((p * NT + n) * NCH + c) * 32 + lane];
        }
        float2 qs[S::Q_REGS ? NT : 1][S::Q_REGS ? NCH : 1];
        if constexpr (S::Q_REGS) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int c = 0; c < NCH; c++)
                    qs[n][c] = *reinterpret_cast<const float2 *>(q_sum + c * ROWS + n * 8 + 2 * t);
        }
        float factor[NT][2];
        int pos[NT][2];  // the last position that column reads; -1 for a column without a row
        const int64_t row0 = int64_t(tile) * ROWS;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int r = n * 8 + 2 * t + e;
                factor[n][e] = q_factor[r];
                pos[n][e] = r < rows ? seq.len - seq.n + int((row0 + r) / a.group) : -1;
            }
        const int pos_first = seq.len - seq.n + int(row0 / a.group);                    // of the tile's first row
        const int pos_last = seq.len - seq.n + int((row0 + rows - 1) / a.group);

        // ------------------------------------------------------ the ring
        const int steps = t_end > t_begin + warp * STEP ? (t_end - t_begin - warp * STEP + UNIT - 1) / UNIT : 0;
        auto row_of = [&](int step) -> int {  // the cache row of this lane's token of a step, -1: none
            const int token = t_begin + (warp + WARPS * step) * STEP + (lane & 15);
            if (step >= steps || token >= t_end)
                return -1;
            const int page = a.page_shift >= 0 ? token >> a.page_shift : token / a.page_size;
            const int where = a.table[int64_t(b) * a.max_pages + page];
            if (where < 0 || where >= a.pages) {
                atomicExch(a.status, OVK_DEV_BAD_PAGE);
                return -1;
            }
            return (where * a.kv_heads + head) * a.page_size + (token - page * a.page_size);
        };
        auto fetch = [&](int stage, int row) {
            const uint32_t to = ring + stage * S::STAGE;
#pragma unroll
            for (int i = 0; i < S::CPR / 2; i++) {
                const int index = lane + 32 * i, r = index / S::CPR, c = index % S::CPR;
                const int src = __shfl_sync(0xffffffffu, row, r);
                const int64_t offset = int64_t(max(src, 0)) * S::ROW_BYTES + c * 16;
                const int swizzle = S::CPR == 2 ? (r >> 2) & 1 : S::CPR == 4 ? (r >> 1) & 3 : r & 7;
                const uint32_t dst = to + r * S::ROW_BYTES + ((c ^ swizzle) << 4);
                copy_async<16>(dst, a.codes[0] + offset, src >= 0 ? 16 : 0);
                copy_async<16>(dst + S::CODES, a.codes[1] + offset, src >= 0 ? 16 : 0);
            }
            // lanes 0-15 bring the keys' scales and zero points, lanes 16-31 the values'; pieces below four
            // bytes are read from the word that holds them, up to their own end
            const int kv = lane >> 4;
            const int64_t r0 = max(row, 0);
            const uint32_t raw = to + 2 * S::CODES;
            const uint8_t *scale = a.scales[kv] + r0 * (2 * a.blocks);
            if (a.blocks == 8)
                copy_async<16>(raw + lane * 16, scale, row >= 0 ? 16 : 0);
            else if (a.blocks == 4)
                copy_async<8>(raw + lane * 16, scale, row >= 0 ? 8 : 0);
            else if (a.blocks == 2)
                copy_async<4>(raw + lane * 16, scale, row >= 0 ? 4 : 0);
            else
                copy_async<4>(raw + lane * 16, scale - 2 * (r0 & 1), row >= 0 ? 2 + 2 * int(r0 & 1) : 0);
            if (a.zero_points[0]) {
                const int bytes = (a.blocks + 1) >> 1;
                const int64_t byte = r0 * bytes;
                copy_async<4>(raw + 512 + lane * 4, a.zero_points[kv] + (byte & ~int64_t(3)), row >= 0 ? int(byte & 3) + bytes : 0);
            }
            sts32(raw + 640 + lane * 4, uint32_t(row));
        };
        {
            int row[S::STAGES - 1];
#pragma unroll
            for (int i = 0; i < S::STAGES - 1; i++)
                row[i] = row_of(i);
#pragma unroll
            for (int i = 0; i < S::STAGES - 1; i++) {
                if (i < steps)
                    fetch(i, row[i]);
                copy_commit();
            }
        }
        int next_row = row_of(S::STAGES - 1);

        float o[NCH][2][NT][4];
        float m[NT][2], l[NT][2];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            m[n][0] = m[n][1] = NONE;
            l[n][0] = l[n][1] = 0.0f;
#pragma unroll
            for (int c = 0; c < NCH; c++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    o[c][0][n][e] = o[c][1][n][e] = 0.0f;
        }
        uint32_t top_scale = 0;  // fp16 bits of the V scale that the maximum allows for

        int stage = 0, ahead = S::STAGES - 1;
        for (int step = 0; step < steps; step++) {
            copy_wait<S::STAGES - 2>();
            __syncwarp();
            if (step + S::STAGES - 1 < steps)
                fetch(ahead, next_row);
            copy_commit();
            next_row = row_of(step + S::STAGES);
            const uint32_t from = ring + stage * S::STAGE, raw = from + 2 * S::CODES;

            // ---------------- {scale, zero} of each chunk of this lane's row
            const int row = int(lds32(raw + 640 + lane * 4));
            uint32_t high = 0;
            {
                const uint4 s4 = lds128(raw + lane * 16);
                uint32_t z = a.zero_points[0] ? lds32(raw + 512 + lane * 4) : 0x88888888u;
                if (a.zero_points[0])
                    z >>= 8 * ((uint32_t(row) * ((a.blocks + 1) >> 1)) & 3);
                const uint32_t words[4] = {a.blocks == 1 && (row & 1) ? s4.x >> 16 : s4.x, s4.y, s4.z, s4.w};
                const uint32_t sign = lane < 16 ? 0x80000000u : 0u;  // subnormal: K adds -zero
                uint32_t out[NCH];
                auto expand = [&](auto shift) {
#pragma unroll
                    for (int c = 0; c < NCH; c++) {
                        const int blk = c >> decltype(shift)::value;
                        const uint32_t h = (blk & 1) ? words[blk >> 1] >> 16 : words[blk >> 1] & 0xffffu;
                        const uint32_t zero = (z >> (4 * blk)) & 15u;
                        out[c] = h | (zero << 16) | (S::SUBNORMAL ? (zero ? sign : 0u) : 0x64000000u);
                        high = max(high, h & 0x7fffu);
                    }
                };
                if (a.chunk_shift == 0)
                    expand(std::integral_constant<int, 0>());
                else if (a.chunk_shift == 1)
                    expand(std::integral_constant<int, 1>());
                else
                    expand(std::integral_constant<int, 2>());
                const uint32_t dst = sz + lane * (NCH * 4);
                if constexpr (NCH == 2) {
                    asm volatile("st.shared.v2.b32 [%0], {%1,%2};" ::"r"(dst), "r"(out[0]), "r"(out[1]) : "memory");
                } else {
#pragma unroll
                    for (int c = 0; c < NCH; c += 4)
                        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst + c * 4), "r"(out[c]), "r"(out[c + 1]),
                                     "r"(out[c + 2]), "r"(out[c + 3])
                                     : "memory");
                }
            }
            const uint32_t present = __ballot_sync(0xffffffffu, row >= 0) & 0xffffu;
            high = lane < 16 || row < 0 ? 0u : high;
            // (ballot and the vote below order the stores above before the reads)
            const bool scale_moves = __any_sync(0xffffffffu, high > top_scale + (3u << 10));
            __syncwarp();
            const int token0 = t_begin + (warp + WARPS * step) * STEP;

            // ---------------------------------------------------- scores
            float x[NT][4];
#pragma unroll
            for (int n = 0; n < NT; n++)
                x[n][0] = x[n][1] = x[n][2] = x[n][3] = 0.0f;
            const uint32_t k_row = from + g * S::ROW_BYTES + t * 4;
            const int swz = S::CPR == 2 ? (g >> 2) & 1 : S::CPR == 4 ? (g >> 1) & 3 : g & 7;
            const int swz8 = S::CPR == 2 ? ((g + 8) >> 2) & 1 : S::CPR == 4 ? ((g + 8) >> 1) & 3 : (g + 8) & 7;
            uint32_t sz_a[NCH], sz_b[NCH];  // tokens g and g + 8
            auto load_sz = [&](uint32_t base, uint32_t (&v)[NCH]) {
                if constexpr (NCH == 2) {
                    asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(base));
                } else {
#pragma unroll
                    for (int c = 0; c < NCH; c += 4) {
                        const uint4 w = lds128(base + c * 4);
                        v[c] = w.x, v[c + 1] = w.y, v[c + 2] = w.z, v[c + 3] = w.w;
                    }
                }
            };
            load_sz(sz + g * (NCH * 4), sz_a);
            load_sz(sz + (g + 8) * (NCH * 4), sz_b);
#pragma unroll
            for (int c = 0; c < NCH; c++) {
                const uint32_t w0 = lds32(k_row + ((c ^ swz) << 4)), w1 = lds32(k_row + 8 * S::ROW_BYTES + ((c ^ swz8) << 4));
                constexpr bool SUB = S::SUBNORMAL;
                const uint32_t v0 = w0 >> 8, v1 = w1 >> 8;
                uint32_t a0[4] = {codes_at<SUB, false>(w0), codes_at<SUB, false>(w1), codes_at<SUB, true>(w0), codes_at<SUB, true>(w1)};
                uint32_t a1[4] = {codes_at<SUB, false>(v0), codes_at<SUB, false>(v1), codes_at<SUB, true>(v0), codes_at<SUB, true>(v1)};
                float s0 = half_lo(sz_a[c]), s1 = half_lo(sz_b[c]), z0 = 0.0f, z1 = 0.0f;
                if constexpr (SUB) {
                    z0 = half_hi(sz_a[c]), z1 = half_hi(sz_b[c]);
                } else {
                    const uint32_t za = __byte_perm(sz_a[c], 0, 0x3232), zb = __byte_perm(sz_b[c], 0, 0x3232);
                    const uint32_t za2 = second_zero<SUB>(za), zb2 = second_zero<SUB>(zb);
                    a0[0] = sub_halves(a0[0], za), a0[1] = sub_halves(a0[1], zb), a0[2] = sub_halves(a0[2], za2), a0[3] = sub_halves(a0[3], zb2);
                    a1[0] = sub_halves(a1[0], za), a1[1] = sub_halves(a1[1], zb), a1[2] = sub_halves(a1[2], za2), a1[3] = sub_halves(a1[3], zb2);
                }
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    float2 sum = make_float2(0.0f, 0.0f);
                    if constexpr (SUB) {
                        if constexpr (S::Q_REGS)
                            sum = qs[n][c];
                        else
                            sum = *reinterpret_cast<const float2 *>(q_sum + c * ROWS + n * 8 + 2 * t);
                    }
                    float acc[4] = {z0 * sum.x, z0 * sum.y, z1 * sum.x, z1 * sum.y};
#pragma unroll
                    for (int p = 0; p < PARTS; p++) {
                        uint4 q4;
                        if constexpr (S::Q_REGS)
                            q4 = bq[p][n][c];
                        else
                            q4 = reinterpret_cast<const uint4 *>(qf)[((p * NT + n) * NCH + c) * 32 + lane];
                        mma(acc, a0, q4.x, q4.y);
                        mma(acc, a1, q4.z, q4.w);
                    }
                    x[n][0] = fmaf(s0, acc[0], x[n][0]);
                    x[n][1] = fmaf(s0, acc[1], x[n][1]);
                    x[n][2] = fmaf(s1, acc[2], x[n][2]);
                    x[n][3] = fmaf(s1, acc[3], x[n][3]);
                }
            }
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    x[n][e] *= factor[n][e & 1];
            const bool masked = present != 0xffffu || token0 + STEP - 1 > pos_first ||
                                (a.window > 0 && int64_t(token0) < int64_t(pos_last) - a.window + 1);
            if (masked) {
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int token = token0 + g + (e >= 2 ? 8 : 0), p = pos[n][e & 1];
                        const bool read = ((present >> (g + (e >= 2 ? 8 : 0))) & 1u) && token <= p &&
                                          (a.window <= 0 || int64_t(token) > int64_t(p) - a.window);
                        if (!read)
                            x[n][e] = -INFINITY;
                    }
            }
            // ------------------------------------------ the running maximum
            bool moves = scale_moves;
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    moves |= x[n][e] > m[n][e & 1] + 6.0f;
            if (__any_sync(0xffffffffu, moves)) {
                // sums and accumulators so far are brought to the new maximum and the new scale's exponent
#pragma unroll
                for (int o_ = 16; o_ > 0; o_ >>= 1)
                    high = max(high, __shfl_xor_sync(0xffffffffu, high, o_));
                const uint32_t new_scale = max(top_scale, min(high, 0x7800u) & 0x7c00u);
                const float shift = float(int(new_scale >> 10) - int(top_scale >> 10));
                top_scale = new_scale;
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float most = fmaxf(x[n][e], x[n][e + 2]);
#pragma unroll
                        for (int o_ = 4; o_ < 32; o_ <<= 1)
                            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o_));
                        const float to = fmaxf(m[n][e], most);
                        const float f = exp2_approx(m[n][e] - to - shift);
                        m[n][e] = to;
                        l[n][e] *= f;
#pragma unroll
                        for (int c = 0; c < NCH; c++) {
                            o[c][0][n][e] *= f, o[c][0][n][e + 2] *= f;
                            o[c][1][n][e] *= f, o[c][1][n][e + 2] *= f;
                        }
                    }
            }
            // p carries 2^-(exponent of the largest scale - 6): top_scale >> 10 is the exponent + 15
            const float lower = float(int(top_scale >> 10) - 21);
            float p[NT][4];
#pragma unroll
            for (int n = 0; n < NT; n++) {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    p[n][e] = exp2_approx(x[n][e] - m[n][e & 1] - lower);
                l[n][0] += p[n][0] + p[n][2];
                l[n][1] += p[n][1] + p[n][3];
            }
            // ---------------------------------------------------- values
            load_sz(sz + (STEP + g) * (NCH * 4), sz_a);
            load_sz(sz + (STEP + g + 8) * (NCH * 4), sz_b);
            uint32_t za[NCH], zb[NCH], zc[NCH], zd[NCH];  // tokens 2t, 2t + 1, 2t + 8, 2t + 9
            load_sz(sz + (STEP + 2 * t) * (NCH * 4), za);
            load_sz(sz + (STEP + 2 * t + 1) * (NCH * 4), zb);
            load_sz(sz + (STEP + 2 * t + 8) * (NCH * 4), zc);
            load_sz(sz + (STEP + 2 * t + 9) * (NCH * 4), zd);
            const uint32_t v_base = from + S::CODES + (g >> 1) * 4;
            const uint32_t select = (g & 1) ? 0x7632u : 0x5410u;
#pragma unroll
            for (int c = 0; c < NCH; c++) {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int token = 2 * t + (i & 1) + (i >> 1) * 8;
                    const int sw = S::CPR == 2 ? (token >> 2) & 1 : S::CPR == 4 ? (token >> 1) & 3 : token & 7;
                    w[i] = lds32(v_base + token * S::ROW_BYTES + ((c ^ sw) << 4));
                }
                const uint32_t y0 = __byte_perm(w[0], w[1], select), y1 = __byte_perm(w[2], w[3], select);
                const uint32_t z0 = __byte_perm(za[c], zb[c], 0x7632), z1 = __byte_perm(zc[c], zd[c], 0x7632);
                constexpr bool SUB = S::SUBNORMAL;
                const uint32_t z0s = second_zero<SUB>(z0), z1s = second_zero<SUB>(z1);
                const uint32_t h0 = y0 >> 8, h1 = y1 >> 8;
                const uint32_t a0[4] = {sub_halves(codes_at<SUB, false>(y0), z0), sub_halves(codes_at<SUB, true>(y0), z0s),
                                        sub_halves(codes_at<SUB, false>(y1), z1), sub_halves(codes_at<SUB, true>(y1), z1s)};
                const uint32_t a1[4] = {sub_halves(codes_at<SUB, false>(h0), z0), sub_halves(codes_at<SUB, true>(h0), z0s),
                                        sub_halves(codes_at<SUB, false>(h1), z1), sub_halves(codes_at<SUB, true>(h1), z1s)};
                const float s0 = half_lo(sz_a[c]), s1 = half_lo(sz_b[c]);
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    float w0 = p[n][0] * s0, w1 = p[n][1] * s0, w2 = p[n][2] * s1, w3 = p[n][3] * s1;
                    if (masked) {  // a scale that is not finite must not reach rows that do not read its token
                        w0 = p[n][0] == 0.0f ? 0.0f : w0, w1 = p[n][1] == 0.0f ? 0.0f : w1;
                        w2 = p[n][2] == 0.0f ? 0.0f : w2, w3 = p[n][3] == 0.0f ? 0.0f : w3;
                    }
                    const uint32_t h01 = pack_halves(w0, w1), h23 = pack_halves(w2, w3);
                    const uint32_t b0 = transpose8x8(h01), b1 = transpose8x8(h23);
                    mma(o[c][0][n], a0, b0, b1);
                    mma(o[c][1][n], a1, b0, b1);
                    if constexpr (PARTS == 2) {
                        const uint32_t l01 = pack_halves(w0 - half_lo(h01), w1 - half_hi(h01));
                        const uint32_t l23 = pack_halves(w2 - half_lo(h23), w3 - half_hi(h23));
                        const uint32_t c0 = transpose8x8(l01), c1 = transpose8x8(l23);
                        mma(o[c][0][n], a0, c0, c1);
                        mma(o[c][1][n], a1, c0, c1);
                    }
                }
            }
            if (++stage == S::STAGES)
                stage = 0;
            if (++ahead == S::STAGES)
                ahead = 0;
        }

        // ------------------------------------------------ join the four warps
        copy_wait<0>();
        const float lower = float(int(top_scale >> 10) - 21);
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
#pragma unroll
                for (int o_ = 4; o_ < 32; o_ <<= 1)
                    l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], o_);
                if (g == 0) {
                    stat[warp * ROWS + n * 8 + 2 * t + e] = m[n][e] + lower;
                    stat[(WARPS + warp) * ROWS + n * 8 + 2 * t + e] = l[n][e];
                }
            }
        __syncthreads();  // every ring is idle: its memory takes the accumulators
        float *const merge = reinterpret_cast<float *>(smem);
        constexpr float first = S::SUBNORMAL ? 0x1p24f : 1.0f, second = S::SUBNORMAL ? 0x1p20f : 1.0f;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                float *dst = merge + (warp * ROWS + n * 8 + 2 * t + e) * (D + 4) + 4 * g;
#pragma unroll
                for (int c = 0; c < NCH; c++)
                    *reinterpret_cast<float4 *>(dst + 32 * c) =
                        make_float4(o[c][0][n][e] * first, o[c][0][n][e + 2] * second, o[c][1][n][e] * first, o[c][1][n][e + 2] * second);
            }
        __syncthreads();
        const bool whole = unit == 0 && units_here == seq.units;
        const int which = unit == 0 ? 1 : 0;  // a partial result that begins an item, or goes on with one
        float *const slot = a.partial + (int64_t(blockIdx.x) * 2 + which) * S::SLOT;
        for (int i = tid; i < ROWS * (D / 4); i += WARPS * 32) {
            const int r = i / (D / 4), d = (i - r * (D / 4)) * 4;
            if (r >= rows)
                break;
            float most = stat[r], weight[WARPS], sum = 0.0f;
#pragma unroll
            for (int w = 1; w < WARPS; w++)
                most = fmaxf(most, stat[w * ROWS + r]);
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < WARPS; w++) {
                weight[w] = exp2_approx(stat[w * ROWS + r] - most);
                sum = fmaf(weight[w], stat[(WARPS + w) * ROWS + r], sum);
                const float4 u = *reinterpret_cast<const float4 *>(merge + (w * ROWS + r) * (D + 4) + d);
                v.x = fmaf(weight[w], u.x, v.x), v.y = fmaf(weight[w], u.y, v.y);
                v.z = fmaf(weight[w], u.z, v.z), v.w = fmaf(weight[w], u.w, v.w);
            }
            if (whole) {
                const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
                const int64_t row = row0 + r;
                const int token = int(row / a.group);
                T *dst = static_cast<T *>(a.out) + int64_t(seq.first + token) * a.o_token +
                         (int64_t(head) * a.group + (row - int64_t(token) * a.group)) * a.o_head + d;
                if constexpr (sizeof(T) == 4) {
                    *reinterpret_cast<float4 *>(dst) = make_float4(v.x * inverse, v.y * inverse, v.z * inverse, v.w * inverse);
                } else {
                    *reinterpret_cast<uint2 *>(dst) = make_uint2(pack_halves(v.x * inverse, v.y * inverse),
                                                                 pack_halves(v.z * inverse, v.w * inverse));
                }
            } else {
                *reinterpret_cast<float4 *>(slot + r * D + d) = v;
                if (d == 0) {
                    slot[ROWS * D + 2 * r] = most;
                    slot[ROWS * D + 2 * r + 1] = sum;
                }
            }
        }
        if (!whole && which == 1 && tid == 0) {
            // the CTAs that hold the rest of this item: the last is the one with its last unit
            const int64_t last_unit = at - unit + seq.units - 1;
            const int64_t last = ((last_unit + 1) * ctas - 1) / total;
            a.meta[blockIdx.x] = make_int4(int(last) + 1 - int(blockIdx.x), b, tile, head);
        }
        at += units_here;
        if (at >= end)
            break;
        unit = 0;
        if (++item == seq.tiles * a.kv_heads) {
            item = 0;
            do {
                b++;
                seq = sequence<ROWS>(a, b, false);
            } while (seq.units == 0 || seq.tiles == 0);
        }
    }
}

// Joins the partial results of items that lie in several CTAs: block (cta, row) takes the item that
// begins in `cta` and goes on behind it, if there is one, and adds its parts in CTA order.
constexpr int JOIN_THREADS = 256;
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(JOIN_THREADS) attention_kv4_join_kernel(const __grid_constant__ Kv4Args a)
{
    constexpr int LANES = D / 4, GROUPS = JOIN_THREADS / LANES, SLOT = ROWS * (D + 2);
    __shared__ float4 sums[GROUPS][LANES];
    __shared__ float tops[JOIN_THREADS / 32], group_sum[GROUPS];
    OVK_PDL_WAIT();
    const int4 meta = a.meta[blockIdx.x];
    const int count = meta.x, b = meta.y, tile = meta.z, head = meta.w, r = blockIdx.y;
    if (count == 0)
        return;
    const int first = a.cu[b], n = a.cu[b + 1] - first;
    const int64_t row = int64_t(tile) * ROWS + r;
    if (row >= int64_t(n) * a.group)
        return;
    const int tid = threadIdx.x;
    auto part = [&](int i) { return a.partial + (int64_t(blockIdx.x + i) * 2 + (i == 0 ? 1 : 0)) * SLOT; };
    float most = NONE;
    for (int i = tid; i < count; i += JOIN_THREADS)
        most = fmaxf(most, part(i)[ROWS * D + 2 * r]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    if ((tid & 31) == 0)
        tops[tid >> 5] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < JOIN_THREADS / 32; w++)
        most = fmaxf(most, tops[w]);
    const int lane = tid % LANES, group = tid / LANES;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float sum = 0.0f;
#pragma unroll 4
    for (int i = group; i < count; i += GROUPS) {
        const float *p = part(i);
        const float4 u = reinterpret_cast<const float4 *>(p + r * D)[lane];
        const float w = exp2_approx(p[ROWS * D + 2 * r] - most);
        sum = fmaf(w, p[ROWS * D + 2 * r + 1], sum);
        v.x = fmaf(w, u.x, v.x), v.y = fmaf(w, u.y, v.y), v.z = fmaf(w, u.z, v.z), v.w = fmaf(w, u.w, v.w);
    }
    sums[group][lane] = v;
    if (lane == 0)
        group_sum[group] = sum;
    __syncthreads();
    if (group != 0)
        return;
    sum = group_sum[0];
#pragma unroll
    for (int i = 1; i < GROUPS; i++) {
        const float4 u = sums[i][lane];
        v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
        sum += group_sum[i];
    }
    const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
    const int token = int(row / a.group);
    T *dst = static_cast<T *>(a.out) + int64_t(first + token) * a.o_token +
             (int64_t(head) * a.group + (row - int64_t(token) * a.group)) * a.o_head + 4 * lane;
    if constexpr (sizeof(T) == 4)
        *reinterpret_cast<float4 *>(dst) = make_float4(v.x * inverse, v.y * inverse, v.z * inverse, v.w * inverse);
    else
        *reinterpret_cast<uint2 *>(dst) = make_uint2(pack_halves(v.x * inverse, v.y * inverse), pack_halves(v.z * inverse, v.w * inverse));
}

template <typename T, int D, int NT> int32_t launch(ovk_ctx *ctx, const Kv4Args &a, int ctas)
{
    constexpr int PARTS = sizeof(T) == 4 ? 2 : 1;
    using S = Shape<D, NT, PARTS>;
    OVK_CUDA(ctx, cudaFuncSetAttribute(attention_kv4_kernel<T, D, NT, PARTS>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM));
    attention_kv4_kernel<T, D, NT, PARTS><<<ctas, WARPS * 32, S::SMEM, ctx->stream>>>(a);
    OVK_LAUNCHED(ctx, NT == 1 ? "attention_kv4" : "attention_kv4_rows16");
    if (ctas > 1) {
        OVK_CUDA(ctx, ovk_launch_pdl(attention_kv4_join_kernel<T, D, S::ROWS>, dim3(unsigned(ctas - 1), S::ROWS), dim3(JOIN_THREADS), 0,
                                     ctx->stream, a));
        ctx->launches++;
    }
    return OVK_OK;
}

}  // namespace kv4

// one per head_dim, in files of their own
int32_t ovk_kv4_launch_64(ovk_ctx *ctx, const Kv4Args &a, int32_t dtype, int tiles, int ctas);
int32_t ovk_kv4_launch_128(ovk_ctx *ctx, const Kv4Args &a, int32_t dtype, int tiles, int ctas);
int32_t ovk_kv4_launch_256(ovk_ctx *ctx, const Kv4Args &a, int32_t dtype, int tiles, int ctas);
