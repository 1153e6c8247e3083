// Attention of a few new tokens over the paged 4-bit cache: the kernel and its
// launch plan.  Instantiated per head_dim by attention_kv4_*.cu.
//
//   x[r][t] = scale * sum_d q[r][d] K[t][d],  p = 2^(x log2 e - m),
//   out[r] = sum_t p V[t] / sum_t p,          K, V[t][d] = (code - zero) * s[t][block of d]
//
// Bytes ought to bound it: a token and key head cost head_dim bytes of codes and 2.5 bytes
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
//  - ldmatrix brings the words of both operands: K's as they lie, V's transposed,
//    four codes of two neighbouring tokens in one register.
//  - K: a chunk of 32 elements has its own accumulator (f16: started at -zero *
//    sum(q) of the chunk, one product instead of a subtraction per code), then
//    scaled by its f32 scale: codes and queries enter the product exactly.
//  - V: codes minus zero (exact, so that a value of 0 adds nothing: the zeros as a
//    product of their own left 2^-17 of them behind) times p * s rounded to fp16.
//    f32 callers get q and p * s as two fp16 parts, 22 bits.
//  - f16: the running maximum moves only when a score passes it by 6 (p by 2^6) or a
//    V scale its own largest by 2^3: p * s starts at 2^6 to 2^7, so it stays below
//    2^16, has all its bits down to 2^-20 of the largest and below that steps of
//    2^-30; a step needs one vote, not a reduction.  f32: by 3 and 2^2, so that p * s
//    starts at 2^10 and the steps are 2^-34 (four drafted tokens of six sequences
//    12.4 us, 12.15 with f16's limits; with 2 and 2^1 12.7).
//
// One CTA per SM takes an equal run of units - 32 tokens for each of its consumer
// warps - of the whole batch (lengths are read on the device).  Four producer
// warps bring units into a ring with 16-byte copies, row by row, so that a page may
// have any size, and go on with the next sequence while the consumers finish one.
// (Tensor and bulk copies, six to a page of 16 tokens, were issued too slowly: 70
// instead of 37 us for 48 contexts of 4000.)  A run that begins or ends inside a
// sequence leaves a partial result, and the CTA that is the last to leave one of a
// sequence joins them, always in CTA order, so results do not depend on timing.  (A
// second kernel for that cost 5 us a call.)
//
// What does is the latency of the consumers' dependent steps: 2.9 warps a scheduler, of
// which 0.94 can issue, fill 53 % of the issue slots, no pipe is busier than 43 % and the
// memory 35 % (eight contexts of up to 100000).  The loads alone take 49 of its 67 us, the
// arithmetic alone 59.
// f16, 16 query heads on 2 key heads of 128, block 32: eight contexts of up to 100000
// tokens take 67 us (3.1 TB/s of 6.5 that a copy reaches), 48 contexts of up to 4000 31 us
// (1.8 TB/s), one context of 900 11 us, which is the way through an empty pipeline and
// back.  256-wide heads spill 28 to 184 bytes a thread: eight contexts of up to 90000, 4 query
// heads on one key head, 58 us (2.1 TB/s), 16 query heads 107; f32, up to 45000, 47 and 93.
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
    unsigned int *counters;  // one per CTA, zero between calls
    int *status;
};

namespace kv4 {

constexpr int STEP = 32;  // tokens of a warp at a time: two products' rows, independent until they meet in the sums
constexpr float NONE = NO_SCORE;  // (scores are in powers of two)

template <int D_, int NT_, int PARTS_> struct Shape {
    static constexpr int D = D_, NT = NT_, PARTS = PARTS_;
    static constexpr int NCH = D / 32, ROWS = 8 * NT, ROW_BYTES = D / 2, CPR = D / 32;
    // consumer warps, and the registers each thread of theirs and of the producer's group gets; 256-wide heads with
    // two tiles of rows hold 128 accumulators a thread
    static constexpr int WARPS = 8;
    static constexpr int REGS = WARPS == 8 ? 208 : 144, PRODUCER_REGS = WARPS == 8 ? 88 : 80;
    static constexpr int THREADS = WARPS * 32 + 128, UNIT = WARPS * STEP;
    static constexpr int STAGES = D == 256 ? 2 : 3;
    static constexpr int CODES = UNIT * ROW_BYTES;        // of K or of V, one stage
    static constexpr int SCALES = UNIT * 16, ZEROS = UNIT * 4;
    static constexpr int PRESENT = 2 * CODES + 2 * (SCALES + ZEROS) + UNIT * 4;  // behind scales, zero points and row numbers
    static constexpr int STAGE = (PRESENT + WARPS * 4 + 127) / 128 * 128;
    // of a warp: {scale, zero} of K per token and chunk, scale of V, zeros of V per pair of tokens and chunk
    static constexpr int K_SZ = STEP * NCH * 8, V_S = STEP * NCH * 4, V_Z = STEP / 2 * NCH * 4, SZ = K_SZ + V_S + V_Z;
    static constexpr int QF = PARTS * NT * NCH * 512;     // query fragments
    static constexpr int SLOTS = D == 256 && NT == 2 ? 1 : WARPS / 2;  // warps that add their sums at a time
    static constexpr int MERGE = SLOTS * ROWS * (D + 4) * 4;
    static constexpr int RING = STAGES * STAGE;
    static constexpr int SMEM = 128 + RING + WARPS * SZ + MERGE + QF + ROWS * (NCH + 1) * 4 + 2 * WARPS * ROWS * 4;
    static constexpr bool Q_REGS = PARTS * NT * NCH * 4 <= 16;
    static constexpr bool SUBNORMAL = PARTS == 1;         // how codes enter the products
    // powers of two that a score may be ahead of its row's maximum, and a V scale of its largest, before they move; and what
    // an exponent field of the scale is lowered by, so that p * s is at most 2^(AHEAD + SCALE_AHEAD + BASE - 15) = 2^15
    static constexpr int AHEAD = PARTS == 1 ? 6 : 3, BASE = PARTS == 1 ? 21 : 25;
    static constexpr uint32_t SCALE_AHEAD = PARTS == 1 ? 3 : 2;
    static constexpr int SLOT = ROWS * (D + 2);           // floats of a partial result
    static_assert(SMEM <= 227 * 1024, "shared memory");
};

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v)
{
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
// Four 8 x 8 matrices of 16-bit elements, rows at the addresses of lanes 0-7, 8-15, 16-23, 24-31
template <bool TRANS> __device__ __forceinline__ uint4 load_matrices(uint32_t a)
{
    uint4 v;
    if constexpr (TRANS)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
template <int BYTES> __device__ __forceinline__ void copy_async(uint32_t dst, const void *src, int valid)
{
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(valid) : "memory");
}
// Ordinary loads and stores of shared memory (an address in its window), which the compiler may move between barriers
__device__ __forceinline__ uint32_t lds32(uint32_t a) { return *static_cast<const uint32_t *>(__cvta_shared_to_generic(a)); }
__device__ __forceinline__ uint2 lds64(uint32_t a) { return *static_cast<const uint2 *>(__cvta_shared_to_generic(a)); }
__device__ __forceinline__ uint4 lds128(uint32_t a) { return *static_cast<const uint4 *>(__cvta_shared_to_generic(a)); }
template <typename V> __device__ __forceinline__ void sts(uint32_t a, V v) { *static_cast<V *>(__cvta_shared_to_generic(a)) = v; }
// N 32-bit words, a multiple of two
template <int N> __device__ __forceinline__ void lds_words(uint32_t a, uint32_t (&v)[N])
{
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 w = lds128(a + 4 * i);
            v[i] = w.x, v[i + 1] = w.y, v[i + 2] = w.z, v[i + 3] = w.w;
        }
    } else {
        static_assert(N == 2, "words");
        const uint2 w = lds64(a);
        v[0] = w.x, v[1] = w.y;
    }
}
template <int N> __device__ __forceinline__ void sts_words(uint32_t a, const uint32_t (&v)[N])
{
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4)
            sts(a + 4 * i, make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]));
    } else {
        static_assert(N == 2, "words");
        sts(a, make_uint2(v[0], v[1]));
    }
}
__device__ __forceinline__ float half_lo(uint32_t w) { return __half2float(__ushort_as_half(uint16_t(w))); }
__device__ __forceinline__ float half_hi(uint32_t w) { return __half2float(__ushort_as_half(uint16_t(w >> 16))); }
// Two codes as halves: the nibbles at bits 0-3 and 16-19 of `w` (SECOND: 4-7 and 20-23).
template <bool SUBNORMAL, bool SECOND> __device__ __forceinline__ uint32_t codes_at(uint32_t w)
{
    return (w & (SECOND ? 0x00f000f0u : 0x000f000fu)) | (SUBNORMAL ? 0u : SECOND ? 0x54005400u : 0x64006400u);
}
// code - zero of two codes; `z` holds the zeros as subnormal halves.
template <bool SUBNORMAL, bool SECOND> __device__ __forceinline__ uint32_t minus_zero(uint32_t w, uint32_t z)
{
    const uint32_t code = codes_at<SUBNORMAL, SECOND>(w);
    __half2 h;
    if constexpr (SUBNORMAL && SECOND)  // 16 zero * 2^-24
        h = __hfma2(*reinterpret_cast<const __half2 *>(&z), __half2half2(__ushort_as_half(0xcc00)), *reinterpret_cast<const __half2 *>(&code));
    else {
        const uint32_t zero = SUBNORMAL ? z : SECOND ? (z << 4) | 0x54005400u : z | 0x64006400u;
        h = __hsub2(*reinterpret_cast<const __half2 *>(&code), *reinterpret_cast<const __half2 *>(&zero));
    }
    return *reinterpret_cast<const uint32_t *>(&h);
}

// 2^k for -126 <= k <= 127
__device__ __forceinline__ float power_of_two(int k) { return __uint_as_float(uint32_t(k + 127) << 23); }

// a / b for b > 0; 64-bit divisions cost a hundred instructions, so the usual sizes take a 32-bit one
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b)
{
    if (((a | b) >> 32) == 0)
        return int64_t(uint32_t(a) / uint32_t(b));
    return a / b;
}
// An equal share of `total` units for each of `ctas` CTAs, the first ones one more.
struct Shares {
    int64_t base, more;
    __device__ __forceinline__ Shares(int64_t total, int64_t ctas) : base(divide(total, ctas)), more(total - base * ctas) {}
    __device__ __forceinline__ int64_t begin(int64_t cta) const { return cta * base + min(cta, more); }
    __device__ __forceinline__ int64_t holder(int64_t unit) const  // the CTA that has this unit
    {
        const int64_t large = more * (base + 1);
        return unit < large ? divide(unit, base + 1) : more + divide(unit - large, base);
    }
};

// What a CTA spends on an item beside its units - query fragments, the join of the warps - in units: the
// shares count it with each item, so that CTAs that work on two items end with the others.
constexpr int ITEM_COST = 2;

// What the sequence arrays say about sequence b.
struct Sequence {
    int first, n;       // packed rows
    int len, start;     // tokens in the cache; the first one that is read, on a step's boundary
    int units, tiles;   // units; tiles of query rows
};
template <int ROWS, int UNIT> __device__ __forceinline__ Sequence sequence(const Kv4Args &a, int b, bool report)
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
    s.tiles = (s.n * a.group + ROWS - 1) / ROWS;  // tokens x query heads < 2^31
    return s;
}

template <int N> __device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(N) : "memory"); }
// The same, and whether `ok` holds for all of them.
template <int N> __device__ __forceinline__ bool consumers_all(bool ok)
{
    uint32_t all;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %1, 0;\n\t"
        "bar.red.and.pred q, 1, %2, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(all)
        : "r"(uint32_t(ok)), "n"(N)
        : "memory");
    return all != 0;
}
// A whole warp waits.  One that has run out ends every other wait of the CTA soon after.
__device__ __forceinline__ bool wait(uint64_t *bar, uint32_t parity, volatile int *dead, int *status, int code)
{
    for (uint32_t i = 0; i < umma::WAIT_LIMIT; i++) {
        if (__all_sync(0xffffffffu, umma::mbar_try_wait(bar, parity)))
            return true;
        if ((i & 255) == 255 && __any_sync(0xffffffffu, *dead))
            return false;
    }
    *dead = 1;
    atomicExch(status, code);
    return false;
}

// A part of an item that other CTAs have parts of too.
struct Part {
    int first_cta, count;  // the CTAs that have one; count 0: no such part
    int first_row, row0, rows, head;
};

// Four elements of a result row: the item's row `row` is query head row % group of the key head, of the
// sequence's new token row / group.
template <typename T>
__device__ __forceinline__ void write_out(const Kv4Args &a, int first_row, int row, int head, int d, float4 v, float sum)
{
    const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
    const int token = row / a.group;
    T *dst = static_cast<T *>(a.out) + int64_t(first_row + token) * a.o_token + (int64_t(head) * a.group + (row - token * a.group)) * a.o_head + d;
    if constexpr (sizeof(T) == 4)
        *reinterpret_cast<float4 *>(dst) = make_float4(v.x * inverse, v.y * inverse, v.z * inverse, v.w * inverse);
    else
        *reinterpret_cast<uint2 *>(dst) = make_uint2(pack_halves(v.x * inverse, v.y * inverse), pack_halves(v.z * inverse, v.w * inverse));
}

template <typename T, int D, int NT, int PARTS>
__global__ void __launch_bounds__(Shape<D, NT, PARTS>::THREADS, 1)
attention_kv4_kernel(const __grid_constant__ Kv4Args a)
{
    using S = Shape<D, NT, PARTS>;
    constexpr int NCH = S::NCH, ROWS = S::ROWS, STAGES = S::STAGES, WARPS = S::WARPS, UNIT = S::UNIT, THREADS = S::THREADS;
    constexpr int CONSUMERS = WARPS * 32;
    extern __shared__ uint8_t smem_raw[];
    __shared__ int64_t warp_sums[THREADS / 32], found[2];
    __shared__ uint64_t full[STAGES], empty[STAGES];
    __shared__ int dead_word;
    __shared__ bool last_part;
    volatile int *const dead = &dead_word;
    const uint32_t ring = (umma::smem_u32(smem_raw) + 127u) & ~127u;
    uint8_t *const smem = smem_raw + (ring - umma::smem_u32(smem_raw));
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, g = lane >> 2, t = lane & 3;
    float *const merge = reinterpret_cast<float *>(smem + S::RING + WARPS * S::SZ);
    uint8_t *const qf = reinterpret_cast<uint8_t *>(merge) + S::MERGE;
    float *const q_sum = reinterpret_cast<float *>(qf + S::QF);       // [NCH][ROWS]
    float *const q_factor = q_sum + ROWS * NCH;                       // [ROWS]
    float *const stat = q_factor + ROWS;                              // [WARPS][ROWS] references, then sums
    const uint32_t sz = ring + S::RING + warp * S::SZ;

    OVK_PDL_LAUNCH_DEPENDENTS();
    if (tid == 0) {
        dead_word = 0;
        for (int i = 0; i < STAGES; i++) {
            umma::mbar_init(&full[i], 4 * 33);  // the producers' lanes, and one of each warp again for what it stores itself
            umma::mbar_init(&empty[i], WARPS);
        }
        umma::fence_barrier_init();
    }
    OVK_PDL_WAIT();

    // ------------------------------------------------ this CTA's run of units
    // A scan over the batch, a sequence a thread; more sequences than threads take a pass for the total first.
    auto units_of = [&](int b, bool report) -> int64_t {
        if (b >= a.batch)
            return 0;
        const Sequence s = sequence<ROWS, UNIT>(a, b, report);
        return int64_t(s.units > 0 ? s.units + ITEM_COST : 0) * s.tiles * a.kv_heads;
    };
    // the units of this thread's sequence and those before it in the chunk; the chunk's total
    auto scan = [&](int64_t own, int64_t &before) -> int64_t {
        int64_t sum = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t left = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o)
                sum += left;
        }
        __syncthreads();
        if (lane == 31)
            warp_sums[warp] = sum;
        __syncthreads();
        int64_t all = 0;
        before = sum - own;
#pragma unroll
        for (int w = 0; w < THREADS / 32; w++) {
            before += w < warp ? warp_sums[w] : 0;
            all += warp_sums[w];
        }
        return all;
    };
    int64_t own = units_of(tid, blockIdx.x == 0), place_before, total = scan(own, place_before);
    for (int base = THREADS; base < a.batch; base += THREADS) {
        int64_t unused;
        total += scan(units_of(base + tid, blockIdx.x == 0), unused);
    }
    const int64_t ctas = min(int64_t(gridDim.x), total);  // each has at least one unit
    if (blockIdx.x >= ctas)
        return;
    const Shares shares(total, ctas);
    int64_t at = shares.begin(blockIdx.x);
    const int64_t end = shares.begin(blockIdx.x + 1);
    int64_t chunk = 0;  // units of the chunks before
    for (int base = 0;; base += THREADS) {
        int64_t all = total;
        if (a.batch > THREADS) {
            own = units_of(base + tid, false);
            all = scan(own, place_before);
        }
        const int64_t mine = chunk + place_before;
        if (at >= mine && at < mine + own)
            found[0] = base + tid, found[1] = mine;
        if (at < chunk + all)
            break;
        chunk += all;
    }
    __syncthreads();
    int b = int(found[0]);
    Sequence seq = sequence<ROWS, UNIT>(a, b, false);
    int item = int(divide(at - found[1], seq.units + ITEM_COST));
    int64_t item_at = found[1] + int64_t(item) * (seq.units + ITEM_COST);  // where the item begins; its units lie behind its cost
    // both kinds of warps walk the run's segments - a piece of one item, possibly without a unit - with this
    auto segment = [&](int &unit) -> int {
        unit = int(max(int64_t(0), at - item_at - ITEM_COST));
        return int(min(int64_t(seq.units), end - item_at - ITEM_COST)) - unit;
    };
    auto next_segment = [&]() {
        at = item_at += seq.units + ITEM_COST;
        if (at >= end)
            return false;
        if (++item == seq.tiles * a.kv_heads) {
            item = 0;
            do {
                b++;
                seq = sequence<ROWS, UNIT>(a, b, false);
            } while (seq.units == 0);
        }
        return true;
    };

    if (warp >= WARPS) {
        // ----------------------------------------------------------- producers
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::PRODUCER_REGS));
        constexpr int ROUNDS = UNIT / 32, MINE = (ROUNDS + 3) / 4;  // 32 tokens a round, a lane each; rounds are dealt to the warps
        const int producer = warp - WARPS, zero_bytes = (a.blocks + 1) >> 1;
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        do {
            int unit;
            const int units_here = segment(unit);
            if (units_here <= 0)
                continue;
            const int head = item % a.kv_heads;
            const int first = seq.start + unit * UNIT + 32 * producer + lane, t_end = min(seq.len, seq.start + (unit + units_here) * UNIT);
            const int32_t *const table = a.table + int64_t(b) * a.max_pages;
            auto row_of = [&](int token) {  // the cache row of a token; -1: none
                if (token >= t_end)
                    return -1;
                const int page = a.page_shift >= 0 ? token >> a.page_shift : token / a.page_size;
                const int where = table[page];
                if (where < 0 || where >= a.pages) {
                    atomicExch(a.status, OVK_DEV_BAD_PAGE);
                    return -1;
                }
                return (where * a.kv_heads + head) * a.page_size + (token - page * a.page_size);
            };
            int row[MINE];  // of the unit that is next
#pragma unroll
            for (int i = 0; i < MINE; i++)
                row[i] = producer + 4 * i < ROUNDS ? row_of(first + 128 * i) : -1;
            for (int u = 0; u < units_here; u++) {
                ok = wait(&empty[stage], phase ^ 1, dead, a.status, OVK_DEV_TIMEOUT_SLOT);
                if (!ok)
                    break;
                const uint32_t to = ring + stage * S::STAGE, raw = to + 2 * S::CODES;
#pragma unroll
                for (int i = 0; i < MINE; i++) {
                    const int round = producer + 4 * i;
                    if (round >= ROUNDS)
                        break;
                    const int now = row[i], place = 32 * round + lane, r0 = max(now, 0);
                    const bool there = now >= 0;
#pragma unroll
                    for (int j = 0; j < S::CPR; j++) {
                        const int index = lane + 32 * j, r = index / S::CPR, c = index % S::CPR;
                        const int src = __shfl_sync(0xffffffffu, now, r);
                        const int64_t offset = int64_t(max(src, 0)) * S::ROW_BYTES + c * 16;
                        const int swizzle = S::CPR == 2 ? (r >> 2) & 1 : S::CPR == 4 ? (r >> 1) & 3 : r & 7;
                        const uint32_t dst = to + (32 * round + r) * S::ROW_BYTES + ((c ^ swizzle) << 4);
                        copy_async<16>(dst, a.codes[0] + offset, src >= 0 ? 16 : 0);
                        copy_async<16>(dst + S::CODES, a.codes[1] + offset, src >= 0 ? 16 : 0);
                    }
                    // this lane's row: scales into 16 bytes, zero points into four; pieces below four bytes are read from
                    // the word that holds them, up to their own end
                    const int64_t scale = int64_t(r0) * (2 * a.blocks), zero = int64_t(r0) * zero_bytes;
                    const uint32_t scale_to = raw + place * 16, zero_to = raw + 2 * S::SCALES + place * 4;
                    const int zero_size = there ? int(zero & 3) + zero_bytes : 0, odd = r0 & 1;
#pragma unroll
                    for (int kv = 0; kv < 2; kv++) {
                        if (a.blocks == 4)
                            copy_async<8>(scale_to + kv * S::SCALES, a.scales[kv] + scale, there ? 8 : 0);
                        else if (a.blocks == 8)
                            copy_async<16>(scale_to + kv * S::SCALES, a.scales[kv] + scale, there ? 16 : 0);
                        else if (a.blocks == 2)
                            copy_async<4>(scale_to + kv * S::SCALES, a.scales[kv] + scale, there ? 4 : 0);
                        else
                            copy_async<4>(scale_to + kv * S::SCALES, a.scales[kv] + scale - 2 * odd, there ? 2 + 2 * odd : 0);
                        if (a.zero_points[0])
                            copy_async<4>(zero_to + kv * S::ZEROS, a.zero_points[kv] + (zero & ~int64_t(3)), zero_size);
                    }
                    sts(raw + 2 * (S::SCALES + S::ZEROS) + place * 4, uint32_t(now));
                    const uint32_t present = __ballot_sync(0xffffffffu, there);
                    if (lane == 0)
                        sts(to + S::PRESENT + round * 4, present);
                    if (u + 1 < units_here)
                        row[i] = row_of(first + (u + 1) * UNIT + 128 * i);
                }
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(umma::smem_u32(&full[stage])) : "memory");
                __syncwarp();
                if (lane == 0)
                    umma::mbar_arrive(&full[stage]);
                if (++stage == STAGES)
                    stage = 0, phase ^= 1;
            }
        } while (ok && next_segment());
        asm volatile("cp.async.wait_all;" ::: "memory");
        return;
    }

    // ---------------------------------------------------------------- consumers
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::REGS));
    int stage = 0;
    uint32_t phase = 0;
    Part parts[2] = {};  // of an item that began before, and of one that goes on behind, this CTA's run
    while (true) {
        int unit;
        const int units_here = segment(unit);
        if (units_here <= 0) {
            if (!next_segment())
                break;
            continue;
        }
        const int tile = item / a.kv_heads, head = item - tile * a.kv_heads;
        const int rows = min(ROWS, seq.n * a.group - tile * ROWS);
        const int t_begin = seq.start + unit * UNIT;

        // -------------------------------------------------- query fragments
        consumers_sync<CONSUMERS>();  // the segment before has been read
        if (tid < ROWS * 8) {
            const int r = tid >> 3, j = tid & 7;
            constexpr int GROUPS = D / 64;  // groups of eight elements a thread
            float v[GROUPS][8], top = 0.0f;
            if (r < rows) {
                const int row = tile * ROWS + r, token = row / a.group;
                const T *src = static_cast<const T *>(a.q) + int64_t(seq.first + token) * a.q_token +
                               (int64_t(head) * a.group + (row - token * a.group)) * a.q_head;
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
            const float f1 = power_of_two(k / 2), f2 = power_of_two(k - k / 2);
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
                    q_sum[c * ROWS + r] = -sum;  // K's accumulators start at zero times this
            }
            if (j == 0)
                q_factor[r] = a.scale_log2e * power_of_two(-(k / 2)) * power_of_two((S::SUBNORMAL ? 24 : 0) - (k - k / 2));
        }
        consumers_sync<CONSUMERS>();
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
        const int row0 = tile * ROWS;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int r = n * 8 + 2 * t + e;
                factor[n][e] = q_factor[r];
                pos[n][e] = r < rows ? seq.len - seq.n + (row0 + r) / a.group : -1;
            }
        const int pos_first = seq.len - seq.n + row0 / a.group;                    // of the tile's first row
        const int pos_last = seq.len - seq.n + (row0 + rows - 1) / a.group;
        const int window = int(a.window);
        // where the rows that this lane addresses for ldmatrix lie: token lane % 16, and of two neighbouring chunks
        // the one that lanes 16-31 read.  Rows eight apart have the same swizzle.
        uint32_t k_at[NCH / 2];
#pragma unroll
        for (int i = 0; i < NCH / 2; i++) {
            const int r = lane & 15, c = 2 * i + (lane >> 4);
            const int swizzle = S::CPR == 2 ? (r >> 2) & 1 : S::CPR == 4 ? (r >> 1) & 3 : r & 7;
            k_at[i] = ring + (warp * STEP + r) * S::ROW_BYTES + ((c ^ swizzle) << 4);
        }
        // where the raw scales and zero points of this lane's token lie (keys'; values' lie behind all of those)
        const int place = warp * STEP + lane, zero_bytes = (a.blocks + 1) >> 1;
        const uint32_t scale_at = ring + 2 * S::CODES + place * 16;
        const uint32_t zero_at = ring + 2 * S::CODES + 2 * S::SCALES + place * 4;
        const uint32_t row_at = ring + 2 * S::CODES + 2 * (S::SCALES + S::ZEROS) + place * 4;

        float o[NCH][2][NT][4];
        // p = 2^(x - reference): the reference is the maximum m and the exponent, less BASE, of the largest scale that the row
        // has read.  A maximum beyond FAR would round that exponent away, or up to its own last place: there it is m alone, and
        // no score may be ahead of it (p is then at most 1, which leaves any scale in fp16's range).
        constexpr float FAR = 0x1p20f, AHEAD = S::AHEAD;
        float limit[NT][2], l[NT][2], reference[NT][2];  // limit: m and what a score may be ahead of it
#pragma unroll
        for (int n = 0; n < NT; n++) {
            limit[n][0] = limit[n][1] = reference[n][0] = reference[n][1] = NONE;
            l[n][0] = l[n][1] = 0.0f;
#pragma unroll
            for (int c = 0; c < NCH; c++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    o[c][0][n][e] = o[c][1][n][e] = 0.0f;
        }
        uint32_t top_scale = 0;  // fp16 bits of the V scale that every row's reference allows for
        bool ok = true;
        for (int u = 0; u < units_here; u++) {
            ok = wait(&full[stage], phase, dead, a.status, OVK_DEV_TIMEOUT_TMA);
            if (!ok)
                break;
            const uint32_t to_stage = stage * S::STAGE;
            const int token0 = t_begin + u * UNIT + warp * STEP;
            const uint32_t present = lds32(ring + to_stage + S::PRESENT + warp * 4);  // which of the step's tokens are there

            // -------- scales and zeros of each chunk of this lane's token, as the products want them
            uint32_t high;
            {
                uint32_t words[2][4] = {}, z[2] = {0x88888888u, 0x88888888u};
                const uint32_t row = lds32(row_at + to_stage);
#pragma unroll
                for (int kv = 0; kv < 2; kv++) {
                    const uint32_t where = scale_at + to_stage + kv * S::SCALES;
                    if (a.blocks == 4) {
                        const uint2 two = lds64(where);
                        words[kv][0] = two.x, words[kv][1] = two.y;
                    } else if (a.blocks == 8) {
                        lds_words(where, words[kv]);
                    } else {
                        words[kv][0] = lds32(where);
                        if (a.blocks == 1)
                            words[kv][0] = (row & 1u) ? words[kv][0] >> 16 : words[kv][0] & 0xffffu;
                    }
                    if (a.zero_points[0]) {
                        z[kv] = lds32(zero_at + to_stage + kv * S::ZEROS);
                        if (zero_bytes < 4)
                            z[kv] >>= 8 * ((row * zero_bytes) & 3);
                    }
                }
                const uint32_t z_next = __shfl_down_sync(0xffffffffu, z[1], 1);  // the next token's, for pairs of V
                auto expand = [&](auto shift) {
                    constexpr int SHIFT = decltype(shift)::value, BLOCKS = NCH >> SHIFT;
                    uint32_t out[2 * NCH];
#pragma unroll
                    for (int c = 0; c < NCH; c++) {
                        const int blk = c >> SHIFT;
                        const uint32_t zero = (z[0] >> (4 * blk)) & 15u;
                        out[2 * c] = __float_as_uint((blk & 1) ? half_hi(words[0][blk >> 1]) : half_lo(words[0][blk >> 1]));
                        // f16: what the accumulator's start multiplies; f32: the zero of a pair of codes
                        out[2 * c + 1] = S::SUBNORMAL ? __float_as_uint(half_lo(zero)) : zero * 0x00010001u;
                    }
                    sts_words(sz + lane * (NCH * 8), out);
                    uint32_t out_v[NCH];
#pragma unroll
                    for (int c = 0; c < NCH; c++) {
                        const int blk = c >> SHIFT;
                        out_v[c] = __float_as_uint((blk & 1) ? half_hi(words[1][blk >> 1]) : half_lo(words[1][blk >> 1]));
                    }
                    sts_words(sz + S::K_SZ + lane * (NCH * 4), out_v);
                    if ((lane & 1) == 0) {
                        const uint32_t low = __byte_perm(z[1], z_next, 0x5410), up = __byte_perm(z[1], z_next, 0x7632);
#pragma unroll
                        for (int c = 0; c < NCH; c++) {
                            const int blk = c >> SHIFT;
                            out_v[c] = ((blk < 4 ? low : up) >> (4 * (blk & 3))) & 0x000f000fu;
                        }
                        sts_words(sz + S::K_SZ + S::V_S + lane / 2 * (NCH * 4), out_v);
                    }
                    // the largest scale of the row (the order of fp16 numbers is that of their bits)
                    uint32_t two = words[1][0] & (BLOCKS == 1 ? 0x7fffu : 0x7fff7fffu);
#pragma unroll
                    for (int i = 1; i < BLOCKS / 2; i++)
                        two = __vmaxu2(two, words[1][i] & 0x7fff7fffu);
                    high = max(two & 0xffffu, two >> 16);
                };
                if (a.chunk_shift == 0)
                    expand(std::integral_constant<int, 0>());
                else if (a.chunk_shift == 1)
                    expand(std::integral_constant<int, 1>());
                else
                    expand(std::integral_constant<int, NCH >= 4 ? 2 : 1>());
            }
            const bool scale_moves = __any_sync(0xffffffffu, high > top_scale + (S::SCALE_AHEAD << 10));
            __syncwarp();

            // ---------------------------------------------------- scores
            float x[2][NT][4];
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int n = 0; n < NT; n++)
                    x[h][n][0] = x[h][n][1] = x[h][n][2] = x[h][n][3] = 0.0f;
#pragma unroll
            for (int i = 0; i < NCH / 2; i++) {
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    // tokens 0-7 and 8-15 of the half for chunk 2i, then for chunk 2i + 1
                    const uint4 words = load_matrices<false>(k_at[i] + to_stage + h * 16 * S::ROW_BYTES);
                    const uint4 sz_a = lds128(sz + (16 * h + g) * (NCH * 8) + 16 * i), sz_b = lds128(sz + (16 * h + g + 8) * (NCH * 8) + 16 * i);
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        constexpr bool SUB = S::SUBNORMAL;
                        const int c = 2 * i + j;
                        const uint32_t w0 = j ? words.z : words.x, w1 = j ? words.w : words.y, v0 = w0 >> 8, v1 = w1 >> 8;
                        const float s0 = __uint_as_float(j ? sz_a.z : sz_a.x), s1 = __uint_as_float(j ? sz_b.z : sz_b.x);
                        const uint32_t z0 = j ? sz_a.w : sz_a.y, z1 = j ? sz_b.w : sz_b.y;
                        uint32_t a0[4] = {codes_at<SUB, false>(w0), codes_at<SUB, false>(w1), codes_at<SUB, true>(w0), codes_at<SUB, true>(w1)};
                        uint32_t a1[4] = {codes_at<SUB, false>(v0), codes_at<SUB, false>(v1), codes_at<SUB, true>(v0), codes_at<SUB, true>(v1)};
                        if constexpr (!SUB) {
                            a0[0] = minus_zero<SUB, false>(w0, z0), a0[1] = minus_zero<SUB, false>(w1, z1);
                            a0[2] = minus_zero<SUB, true>(w0, z0), a0[3] = minus_zero<SUB, true>(w1, z1);
                            a1[0] = minus_zero<SUB, false>(v0, z0), a1[1] = minus_zero<SUB, false>(v1, z1);
                            a1[2] = minus_zero<SUB, true>(v0, z0), a1[3] = minus_zero<SUB, true>(v1, z1);
                        }
#pragma unroll
                        for (int n = 0; n < NT; n++) {
                            float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                            if constexpr (SUB) {
                                float2 sum;
                                if constexpr (S::Q_REGS)
                                    sum = qs[n][c];
                                else
                                    sum = *reinterpret_cast<const float2 *>(q_sum + c * ROWS + n * 8 + 2 * t);
                                acc[0] = __uint_as_float(z0) * sum.x, acc[1] = __uint_as_float(z0) * sum.y;
                                acc[2] = __uint_as_float(z1) * sum.x, acc[3] = __uint_as_float(z1) * sum.y;
                            }
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
                            x[h][n][0] = fmaf(s0, acc[0], x[h][n][0]);
                            x[h][n][1] = fmaf(s0, acc[1], x[h][n][1]);
                            x[h][n][2] = fmaf(s1, acc[2], x[h][n][2]);
                            x[h][n][3] = fmaf(s1, acc[3], x[h][n][3]);
                        }
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        x[h][n][e] *= factor[n][e & 1];
            const bool masked = present != 0xffffffffu || token0 + STEP - 1 > pos_first || (window > 0 && token0 < pos_last - window + 1);
            if (masked) {
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int place_in = 16 * h + g + (e >= 2 ? 8 : 0), token = token0 + place_in, p = pos[n][e & 1];
                            if (!((present >> place_in) & 1u) || token > p || (window > 0 && token <= p - window))
                                x[h][n][e] = -INFINITY;
                        }
            }
            // ------------------------------------------ the running maximum
            bool moves = scale_moves;
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    moves |= x[0][n][e] > limit[n][e & 1] || x[1][n][e] > limit[n][e & 1];
            if (__any_sync(0xffffffffu, moves)) {
                // Sums and accumulators so far are brought to the new maximum and the new scale's exponent.  A scale
                // counts for the rows that read its token: elsewhere it may be anything, and p would sink below fp16's range.
                // Tokens that only some rows read are looked through row by row where one has the largest exponent.
                uint32_t largest = high;  // of the tokens that all rows read
                bool by_row = false;
                if (masked) {
                    const int token = token0 + lane;
                    const bool there = (present >> lane) & 1u;
                    const bool by_all = there && token <= pos_first && !(window > 0 && token <= pos_last - window);
                    const bool by_some = there && token <= pos_last && !(window > 0 && token <= pos_first - window);
                    largest = by_all ? high : 0u;
                    by_row = __any_sync(0xffffffffu, by_some && !by_all);
                    if (by_row)
                        by_row = __reduce_max_sync(0xffffffffu, by_some ? high : 0u) >> 10 > __reduce_max_sync(0xffffffffu, largest) >> 10;
                }
                largest = min(__reduce_max_sync(0xffffffffu, largest) >> 10, 30u);
                uint32_t exponents = largest * 0x01010101u;  // of this lane's columns, a byte each
                if (by_row) {
#pragma unroll 1
                    for (int i = 0; i < rows; i++) {
                        const int p = seq.len - seq.n + (row0 + i) / a.group, token = token0 + lane;
                        const bool reads = ((present >> lane) & 1u) && token <= p && !(window > 0 && token <= p - window);
                        const uint32_t its = min(__reduce_max_sync(0xffffffffu, reads ? high : 0u) >> 10, 30u);
                        const int column = (i >> 3) * 2 + (i & 1);
                        if (((i & 7) >> 1) == t)
                            exponents = (exponents & ~(255u << (8 * column))) | max(its, largest) << (8 * column);
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float most = fmaxf(fmaxf(x[0][n][e], x[0][n][e + 2]), fmaxf(x[1][n][e], x[1][n][e + 2]));
#pragma unroll
                        for (int o_ = 4; o_ < 32; o_ <<= 1)
                            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o_));
                        const float m = fabsf(limit[n][e]) > FAR ? limit[n][e] : limit[n][e] - AHEAD;
                        const float before = m == NONE ? -S::BASE : rintf(reference[n][e] - m);
                        const float to = fmaxf(m, most);
                        const bool far = fabsf(to) > FAR;
                        const float next = far ? to : to + fmaxf(before, float(int((exponents >> (16 * n + 8 * e)) & 255u) - S::BASE));
                        const float f = exp2_approx(reference[n][e] - next);
                        limit[n][e] = far ? to : to + AHEAD, reference[n][e] = next;
                        l[n][e] *= f;
#pragma unroll
                        for (int c = 0; c < NCH; c++) {
                            o[c][0][n][e] *= f, o[c][0][n][e + 2] *= f;
                            o[c][1][n][e] *= f, o[c][1][n][e + 2] *= f;
                        }
                    }
                top_scale = max(top_scale, largest << 10);
            }
            float p[2][NT][4];
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int n = 0; n < NT; n++) {
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        p[h][n][e] = exp2_approx(x[h][n][e] - reference[n][e & 1]);
                    l[n][0] += p[h][n][0] + p[h][n][2];
                    l[n][1] += p[h][n][1] + p[h][n][3];
                }
            // ---------------------------------------------------- values
            auto values = [&](auto is_masked) {
#pragma unroll
                for (int i = 0; i < NCH / 2; i++) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        // pairs of the half's tokens 2t, 2t + 1 and 2t + 8, 2t + 9 for chunk 2i, then for chunk 2i + 1
                        const uint4 words = load_matrices<true>(k_at[i] + to_stage + S::CODES + h * 16 * S::ROW_BYTES);
                        const uint32_t s_at = sz + S::K_SZ + (16 * h + g) * (NCH * 4) + 8 * i, z_at = sz + S::K_SZ + S::V_S + (8 * h + t) * (NCH * 4) + 8 * i;
                        const uint2 s_a = lds64(s_at), s_b = lds64(s_at + 8 * (NCH * 4));
                        const uint2 z_a = lds64(z_at), z_b = lds64(z_at + 4 * (NCH * 4));
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            constexpr bool SUB = S::SUBNORMAL;
                            const int c = 2 * i + j;
                            const uint32_t y0 = j ? words.z : words.x, y1 = j ? words.w : words.y, h0 = y0 >> 8, h1 = y1 >> 8;
                            const uint32_t z0 = j ? z_a.y : z_a.x, z1 = j ? z_b.y : z_b.x;
                            const uint32_t a0[4] = {minus_zero<SUB, false>(y0, z0), minus_zero<SUB, true>(y0, z0), minus_zero<SUB, false>(y1, z1),
                                                    minus_zero<SUB, true>(y1, z1)};
                            const uint32_t a1[4] = {minus_zero<SUB, false>(h0, z0), minus_zero<SUB, true>(h0, z0), minus_zero<SUB, false>(h1, z1),
                                                    minus_zero<SUB, true>(h1, z1)};
                            const float s0 = __uint_as_float(j ? s_a.y : s_a.x), s1 = __uint_as_float(j ? s_b.y : s_b.x);
#pragma unroll
                            for (int n = 0; n < NT; n++) {
                                const float(&pn)[4] = p[h][n];
                                float w0 = pn[0] * s0, w1 = pn[1] * s0, w2 = pn[2] * s1, w3 = pn[3] * s1;
                                if constexpr (decltype(is_masked)::value) {  // a scale that is not finite stays with the rows that read its token
                                    w0 = pn[0] == 0.0f ? 0.0f : w0, w1 = pn[1] == 0.0f ? 0.0f : w1;
                                    w2 = pn[2] == 0.0f ? 0.0f : w2, w3 = pn[3] == 0.0f ? 0.0f : w3;
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
                    }
                }
            };
            if (masked)
                values(std::true_type());
            else
                values(std::false_type());
            __syncwarp();
            if (lane == 0)
                umma::mbar_arrive(&empty[stage]);
            if (++stage == STAGES)
                stage = 0, phase ^= 1;
        }

        // ------------------------------------------------ join the warps
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
#pragma unroll
                for (int o_ = 4; o_ < 32; o_ <<= 1)
                    l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], o_);
                if (g == 0) {
                    stat[warp * ROWS + n * 8 + 2 * t + e] = reference[n][e];
                    stat[(WARPS + warp) * ROWS + n * 8 + 2 * t + e] = l[n][e];
                }
            }
        if (!consumers_all<CONSUMERS>(ok))
            return;
        // groups of SLOTS warps add their sums, relative to the largest reference of all, one group after the other
        constexpr float first = S::SUBNORMAL ? 0x1p24f : 1.0f, second = S::SUBNORMAL ? 0x1p20f : 1.0f;
#pragma unroll
        for (int round = 0; round < WARPS / S::SLOTS; round++) {
            if (warp / S::SLOTS == round) {
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int r = n * 8 + 2 * t + e;
                        float most = NONE;
#pragma unroll
                        for (int w = 0; w < WARPS; w++)
                            most = fmaxf(most, stat[w * ROWS + r]);
                        const float f = exp2_approx(reference[n][e] - most), f1 = f * first, f2 = f * second;
                        float *dst = merge + (warp % S::SLOTS * ROWS + r) * (D + 4) + 4 * g;
#pragma unroll
                        for (int c = 0; c < NCH; c++) {
                            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            if (round > 0)
                                v = *reinterpret_cast<float4 *>(dst + 32 * c);
                            v.x = fmaf(o[c][0][n][e], f1, v.x), v.y = fmaf(o[c][0][n][e + 2], f2, v.y);
                            v.z = fmaf(o[c][1][n][e], f1, v.z), v.w = fmaf(o[c][1][n][e + 2], f2, v.w);
                            *reinterpret_cast<float4 *>(dst + 32 * c) = v;
                        }
                    }
            }
            consumers_sync<CONSUMERS>();
        }
        const bool whole = unit == 0 && units_here == seq.units;
        // a CTA has at most two parts: one that goes on with an item (slot 0), one that begins an item (slot 1)
        float *const slot = a.partial + (int64_t(blockIdx.x) * 2 + (unit == 0 ? 1 : 0)) * S::SLOT;
        for (int i = tid; i < rows * (D / 4); i += CONSUMERS) {
            const int r = i / (D / 4), d = (i - r * (D / 4)) * 4;
            float most = NONE, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < WARPS; w++)
                most = fmaxf(most, stat[w * ROWS + r]);
#pragma unroll
            for (int w = 0; w < WARPS; w++)
                sum = fmaf(exp2_approx(stat[w * ROWS + r] - most), stat[(WARPS + w) * ROWS + r], sum);
            float4 v = *reinterpret_cast<const float4 *>(merge + r * (D + 4) + d);
#pragma unroll
            for (int w = 1; w < S::SLOTS; w++) {
                const float4 u = *reinterpret_cast<const float4 *>(merge + (w * ROWS + r) * (D + 4) + d);
                v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
            }
            if (whole) {
                write_out<T>(a, seq.first, row0 + r, head, d, v, sum);
            } else {
                *reinterpret_cast<float4 *>(slot + r * D + d) = v;
                if (d == 0)
                    *reinterpret_cast<float2 *>(slot + ROWS * D + 2 * r) = make_float2(most, sum);
            }
        }
        if (!whole) {
            // the CTAs that hold this item: from the one that has its first unit to the one that has its last
            Part &part = parts[unit == 0 ? 1 : 0];
            part.first_cta = int(shares.holder(item_at + ITEM_COST));
            part.count = int(shares.holder(item_at + ITEM_COST + seq.units - 1)) - part.first_cta + 1;
            part.first_row = seq.first, part.row0 = row0, part.rows = rows, part.head = head;
        }
        if (!next_segment())
            break;
    }

    // ------------------------------------------- join items, where this CTA is the last to have left its part
#pragma unroll 1
    for (int which = 0; which < 2; which++) {
        const Part part = parts[which];
        if (part.count == 0)
            continue;
        __threadfence();
        consumers_sync<CONSUMERS>();
        if (tid == 0) {
            last_part = atomicAdd(&a.counters[part.first_cta], 1u) == unsigned(part.count - 1);
            if (last_part)
                a.counters[part.first_cta] = 0;
        }
        consumers_sync<CONSUMERS>();
        if (!last_part)
            continue;
        __threadfence();
        // a lane of sixteen fetches the maximum and sum of one part, and all of them their elements of sixteen parts
        const uint32_t half = (lane & 16) ? 0xffff0000u : 0x0000ffffu;
        for (int i = tid; i < part.rows * (D / 4); i += CONSUMERS) {
            const int r = i / (D / 4), d = (i - r * (D / 4)) * 4;
            float top = NONE, sum = 0.0f;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (int base = 0; base < part.count; base += 16) {
                auto slot_of = [&](int k) { return a.partial + (int64_t(part.first_cta + k) * 2 + (k == 0 ? 1 : 0)) * S::SLOT; };
                float2 ml = make_float2(NONE, 0.0f);
                if (base + (lane & 15) < part.count)
                    ml = __ldcg(reinterpret_cast<const float2 *>(slot_of(base + (lane & 15)) + ROWS * D + 2 * r));
                float4 u[16];
#pragma unroll
                for (int k = 0; k < 16; k++)
                    u[k] = base + k < part.count ? __ldcg(reinterpret_cast<const float4 *>(slot_of(base + k) + r * D + d)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                float most = ml.x;
#pragma unroll
                for (int o = 1; o < 16; o <<= 1)
                    most = fmaxf(most, __shfl_xor_sync(half, most, o));
                const float to = fmaxf(top, most), f = exp2_approx(top - to), mine = exp2_approx(ml.x - to);
                top = to;
                sum *= f;
                v.x *= f, v.y *= f, v.z *= f, v.w *= f;
#pragma unroll
                for (int k = 0; k < 16; k++) {
                    const float w = __shfl_sync(half, mine, k, 16);
                    sum = fmaf(w, __shfl_sync(half, ml.y, k, 16), sum);
                    v.x = fmaf(w, u[k].x, v.x), v.y = fmaf(w, u[k].y, v.y), v.z = fmaf(w, u[k].z, v.z), v.w = fmaf(w, u[k].w, v.w);
                }
            }
            write_out<T>(a, part.first_row, part.row0 + r, part.head, d, v, sum);
        }
    }
}

template <typename T, int D, int NT> int32_t launch(ovk_ctx *ctx, const Kv4Args &a, int ctas)
{
    constexpr int PARTS = sizeof(T) == 4 ? 2 : 1;
    using S = Shape<D, NT, PARTS>;
    OVK_CUDA(ctx, ovk_allow_smem(attention_kv4_kernel<T, D, NT, PARTS>, S::SMEM, ctx->device));
    OVK_CUDA(ctx, ovk_launch_pdl(attention_kv4_kernel<T, D, NT, PARTS>, dim3(unsigned(ctas)), dim3(S::THREADS), S::SMEM, ctx->stream, a));
    OVK_LAUNCHED(ctx, NT == 1 ? "attention_kv4" : "attention_kv4_rows16");
    return OVK_OK;
}

}  // namespace kv4

// one per head_dim, in files of their own
int32_t ovk_kv4_launch_64(ovk_ctx *ctx, const Kv4Args &a, int32_t dtype, int tiles, int ctas);
int32_t ovk_kv4_launch_128(ovk_ctx *ctx, const Kv4Args &a, int32_t dtype, int tiles, int ctas);
int32_t ovk_kv4_launch_256(ovk_ctx *ctx, const Kv4Args &a, int32_t dtype, int tiles, int ctas);
