// f16 attention over packed prompts on the 5th-generation tensor cores.
//
//   S = Q K^T (128 query rows x 64 or 128 keys, f32 in tensor memory),
//   P = 2^(scale' S - m) (f16, written back over S),  O = O + P V (f32 in tensor memory),
//
// m a per-row reference that follows the running maximum, out = O / sum of P.
// The two products are 4 head_dim operations per score, the exponential one of 16
// a cycle and SM: at head_dim 128 both pipes need the same 1024 cycles for 128 x 128
// scores, so the point of the layout is that neither waits for the other.
//
//   softmax groups of four warps   a thread owns a row: tcgen05.ld, maximum, exp2,
//                                  tcgen05.st, and at the end its row of the result
//   control group: warp 0          TMA: Q once, then K and V tiles into one ring in
//                                  the order the products use them
//                  warps 1, 2      issue tcgen05.mma
//   guards                         look through V tiles that some row of the block
//                                  does not read entirely (below): warp 3 of the
//                                  control group, or a group of their own
//
// Up to 128 elements a head two independent query tiles share each K and V tile
// (two heads of a group, or neighbouring rows where the group is odd), each with
// its own issuing warp and two S buffers of 64 keys: while the one half of a tile's
// softmax runs, the tensor core works for the other half and for the other tile.
// (The core's queue is short - a warp that issues runs at the core's pace - and a
// wait costs some 300 cycles even where nothing is to be waited for: one issuer for
// both tiles took 308 us for 8192 tokens of 16 heads, two 294, with two buffers 280:
// 980 TFLOP/s, 416000 cycles; replayed for a few milliseconds 239 us, 1150 TFLOP/s.
// What is left is the softmax's own latency: 128 rows are four warps, one to a
// scheduler, and the two tiles run in step.)  256-wide heads fill tensor
// memory with one tile's O, so there one tile has two S buffers of 128 keys, one warp
// issues Q K^T and the other P V, and the next scores are computed before the last
// weights are used: 408 us for 8192 tokens of 16 heads so replayed, 1350 TFLOP/s.
//
// A block is one query tile (or two) from its first load to its last store, one on
// an SM at a time: some 15000 cycles pass outside the products (lookup 1200, first
// tiles 4000, store 3800, the next block's start 1700, half of the first and last
// softmax), which is what short prompts and windows cost: 8192 tokens of 16 heads
// of 256 take 150 to 171 us with a window of 1024, 750 to 860 TFLOP/s.
//
// The reference m lies 7 below the row's maximum and moves only when that passes it by 15, so O is rarely rescaled;
// the softmax group does it itself, between the products that write O.  P then has 2^7 to 2^15 where the row's largest
// score is: fp16 holds weights down to 2^-21 of that in full and counts what is below in steps of 2^-31, so that a long
// flat tail is not lost (sums are f32).
//
// Masked weights are exactly 0, and 0 times an infinity is NaN: in tiles that are
// not read whole, the guards zero the V rows behind the sequence's end and every
// V element that is not finite, and note its column.  A row adds such elements of
// the keys that it does read when it stores its result.
#include "attention_prompt.cuh"
#include "umma.cuh"

namespace {

constexpr int BM = 128;

template <int DP_> struct Tc {
    static constexpr int DP = DP_;                       // head_dim rounded up; TMA fills the rest with zeros
    static constexpr int NS = DP == 256 ? 1 : 2;         // query tiles of a block
    static constexpr int BN = DP == 256 ? 128 : 64;      // keys of a tile; each query tile has two S buffers of as many columns
    static constexpr int CH = DP == 256 ? 2 : 1;         // ring stages of a K or V tile
    static constexpr int ATOMS = DP / 64;                // 128-byte columns of a row
    static constexpr int Q_BYTES = BM * DP * 2;
    static constexpr int STAGE = BN * DP * 2 / CH;
    static constexpr int STAGES = DP == 256 ? 5 : 10;
    static constexpr int GUARDS = NS == 2 ? 1 : 4;       // warps
    static constexpr int THREADS = 384;
    static constexpr int SOFTMAX_REGS = NS == 2 ? 208 : 232, OTHER_REGS = NS == 2 ? 88 : 104;
    static constexpr int SMEM = NS * Q_BYTES + STAGES * STAGE + 1024;
    static constexpr int O_COL = 256;                    // S of the two tiles (or buffers) at 0 and 128
};

struct TcParams {
    PromptArgs a;
    int pairs;     // blocks along the heads
    int by_heads;  // the two query tiles are two heads of a group; else neighbouring rows
    int window, vec_out;
};

struct Shared {
    // s_full, p_full, pv_done: of each S buffer, 2 * query tile + buffer
    uint64_t q_full[2], full[10], empty[10], raw[10], s_full[4], p_full[4], pv_done[4], drain[2];
    uint32_t tmem;
    int dead;
    uint32_t odd[8];  // columns in which a V element that is not finite was zeroed
    PromptTile tile;
};

__device__ __forceinline__ bool wait(uint64_t *bar, uint32_t parity, volatile int *dead, int *status, int code)
{
    for (uint32_t i = 0; i < umma::WAIT_LIMIT; i++) {
        if (umma::mbar_try_wait(bar, parity))
            return true;
        if ((i & 255) == 255 && *dead)
            return false;
    }
    *dead = 1;
    atomicExch(status, code);
    return false;
}

// A whole warp waits; what it returns is the same for all lanes, and the compiler knows it.
__device__ __forceinline__ bool wait_warp(uint64_t *bar, uint32_t parity, volatile int *dead, int *status, int code)
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

template <int DP>
__global__ void __launch_bounds__(Tc<DP>::THREADS, 1)
attention_prompt_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                           const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ TcParams p)
{
    using C = Tc<DP>;
    constexpr int NS = C::NS, SB = 2, CH = C::CH, BN = C::BN;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Shared sh;
    const uint32_t smem_base = (umma::smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *const smem = smem_raw + (smem_base - umma::smem_u32(smem_raw));
    uint8_t *const ring = smem + NS * C::Q_BYTES;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, group = warp >> 2;
    volatile int *const dead = &sh.dead;
    int *const status = p.a.status;
    const PromptArgs &a = p.a;

    const int index = blockIdx.x / p.pairs, pair = blockIdx.x - index * p.pairs;
    const bool rows_split = NS == 2 && !p.by_heads;
    OVK_PDL_LAUNCH_DEPENDENTS();
    if (tid == 32) {
        umma::prefetch_tmap(&tm_q);
        umma::prefetch_tmap(&tm_k);
        umma::prefetch_tmap(&tm_v);
    }
    OVK_PDL_WAIT();
    if (warp == 0) {
        if (rows_split)
            find_prompt_tile<2 * BM>(a, index, gridDim.x / p.pairs, sh.tile);
        else
            find_prompt_tile<BM>(a, index, gridDim.x / p.pairs, sh.tile);
        __syncwarp();
        if (lane == 0) {
            // how many threads give a ring stage back: one for each query tile that there is
            const int users = NS == 1 || (rows_split && sh.tile.n_q - sh.tile.row0 <= BM) ? 1 : 2;
            sh.dead = 0;
            for (int i = 0; i < 8; i++)
                sh.odd[i] = 0;
            for (int i = 0; i < 2; i++) {
                umma::mbar_init(&sh.q_full[i], 1);
                umma::mbar_init(&sh.drain[i], 1);
            }
            for (int i = 0; i < 4; i++) {
                umma::mbar_init(&sh.s_full[i], 1);
                umma::mbar_init(&sh.p_full[i], 4);
                umma::mbar_init(&sh.pv_done[i], 1);
            }
            for (int i = 0; i < C::STAGES; i++) {
                umma::mbar_init(&sh.full[i], 1);
                umma::mbar_init(&sh.empty[i], users);
                umma::mbar_init(&sh.raw[i], 1);
            }
            umma::fence_barrier_init();
        }
    }
    __syncthreads();
    const PromptTile w = sh.tile;
    if (w.b < 0)
        return;  // the batch has fewer tiles; nothing is allocated or in flight yet
    // a block's query tiles: head and first row of each, and how many rows are left for it
    const int head0 = NS == 2 && p.by_heads ? 2 * pair : pair;
    const int kv_head = head0 / a.group;
    const int rows_all = min(rows_split ? 2 * BM : BM, w.n_q - w.row0);
    const int streams = NS == 1 || (rows_split && rows_all <= BM) ? 1 : 2;
    const int pos0 = w.n_k - w.n_q + w.row0;  // position of the block's first row
    const int key_begin = p.window > 0 ? max(0, pos0 - p.window + 1) : 0;
    const int key_end = a.causal ? min(w.n_k, pos0 + rows_all) : w.n_k;
    const int tiles = key_end > key_begin ? (key_end - key_begin + BN - 1) / BN : 0;
    // whether some of the rows first .. last do not read the whole of tile i
    auto partial = [&](int i, int first, int last) {
        const int j0 = key_begin + i * BN;
        return j0 + BN > key_end || (a.causal && j0 + BN - 1 > first) || (p.window > 0 && j0 <= last - p.window);
    };
    const int pos_last = pos0 + rows_all - 1;

    if (group >= NS) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::OTHER_REGS));
        const int role = warp - NS * 4;
        if (role == 1) {
            umma::tmem_alloc(&sh.tmem, 512);
            umma::tmem_relinquish();
        }
        uint32_t tmem = 0;
        if (role != 0) {  // the loads need no tensor memory
            umma::tc_fence_before();
            asm volatile("bar.sync 1, %0;" ::"n"(C::THREADS - 32) : "memory");
            umma::tc_fence_after();
            tmem = sh.tmem;
        }
        if (role == 0) {
            // ------------------------------------------------------------ loads
            if (lane == 0 && tiles > 0) {
                auto load_q = [&](int s) {
                    umma::mbar_expect_tx(&sh.q_full[s], C::Q_BYTES);
                    for (int x = 0; x < C::ATOMS; x++)
                        umma::tma_load_3d(smem + s * C::Q_BYTES + x * BM * 128, &tm_q, &sh.q_full[s], 64 * x,
                                          rows_split ? head0 : head0 + s, w.first_q + w.row0 + (rows_split ? s * BM : 0));
                };
                load_q(0);
                int stage = 0, issued = 0;
                uint32_t phase = 0;
                uint32_t in_raw = 0, raw_phase = 0;  // a bit per stage: its last copy is counted at `raw`; uses of `raw` so far
                bool ok = true;
                auto load = [&](bool value, int tile) {
                    for (int c = 0; c < CH && ok; c++) {
                        ok = wait(&sh.empty[stage], phase ^ 1, dead, status, OVK_DEV_TIMEOUT_SLOT);
                        if (!ok)
                            return;
                        uint8_t *dst = ring + stage * C::STAGE;
                        // a V tile that the guards look through first is theirs to pass on
                        uint64_t *const bar = value && partial(tile, pos0, pos_last) ? &sh.raw[stage] : &sh.full[stage];
                        umma::mbar_expect_tx(bar, C::STAGE);
                        const int row = w.first_k + key_begin + tile * BN;
                        if (CH == 1 || !value) {  // whole rows, or (K) half of the columns of each
                            for (int x = 0; x < C::ATOMS / CH; x++)
                                umma::tma_load_3d(dst + x * BN * 128, value ? &tm_v : &tm_k, bar,
                                                  64 * (c * (C::ATOMS / CH) + x), kv_head, row);
                        } else {  // V: half of the keys; its box has half the rows
                            for (int x = 0; x < C::ATOMS; x++)
                                umma::tma_load_3d(dst + x * (BN / CH) * 128, &tm_v, bar, 64 * x, kv_head, row + c * (BN / CH));
                        }
                        issued++;
                        in_raw = bar == &sh.raw[stage] ? in_raw | (1u << stage) : in_raw & ~(1u << stage);
                        raw_phase ^= bar == &sh.raw[stage] ? 1u << stage : 0u;
                        if (++stage == C::STAGES)
                            stage = 0, phase ^= 1;
                    }
                };
                load(false, 0);
                if (streams == 2)
                    load_q(1);
                if (tiles > 1)
                    load(false, 1);
                for (int i = 0; i < tiles && ok; i++) {
                    load(true, i);
                    if (i + SB < tiles)
                        load(false, i + SB);
                }
                if (!ok) {  // copies in flight end before the block does
                    for (int k = max(0, issued - C::STAGES); k < issued; k++)
                        if ((in_raw >> (k % C::STAGES)) & 1)
                            umma::mbar_wait(&sh.raw[k % C::STAGES], ((raw_phase >> (k % C::STAGES)) & 1) ^ 1);
                        else
                            umma::mbar_wait(&sh.full[k % C::STAGES], (k / C::STAGES) & 1);
                    for (int s = 0; s < streams; s++)
                        umma::mbar_wait(&sh.q_full[s], 0);
                }
            }
        } else if (role <= 2) {
            // --------------------------------------------------------- products
            const int self = role - 1;  // of two query tiles the one; of one tile, 0 issues P V and 1 issues Q K^T
            if (tiles > 0 && (NS == 1 || self < streams)) {
                const bool leader = umma::elect_one();  // the whole warp keeps step, so that descriptors stay in uniform registers
                constexpr uint32_t k_hi = ((1024u >> 4) & 0x3fffu) | (1u << 14) | (umma::LAYOUT_SW128 << 29);
                constexpr uint32_t qk_desc = umma::instr_desc(1, 0, 0, BM, BN);
                constexpr uint32_t pv_desc = umma::instr_desc(1, 0, 0, BM, DP) | (1u << 16);  // V: keys along the rows
                constexpr uint32_t v_lbo = DP == 64 ? 1u : uint32_t(BN / CH) * 128u >> 4;
                const uint32_t q_lo = (((umma::smem_u32(smem) + (NS == 2 ? self * C::Q_BYTES : 0)) >> 4) & 0x3fffu) | (1u << 16);
                const uint32_t ring_lo = umma::smem_u32(ring) >> 4;
                int stage = 0;
                uint32_t phase = 0;
                bool ok = true;
                auto next_tile = [&](int (&at)[CH], bool mine) {  // the ring's next tile; waits for it if it is this thread's
#pragma unroll
                    for (int c = 0; c < CH; c++) {
                        if (mine)
                            ok = ok && wait_warp(&sh.full[stage], phase, dead, status, OVK_DEV_TIMEOUT_TMA);
                        at[c] = stage;
                        if (++stage == C::STAGES)
                            stage = 0, phase ^= 1;
                    }
                };
                auto qk = [&](int buffer, const int (&at)[CH]) {
                    const uint32_t d = tmem + buffer * BN;
#pragma unroll
                    for (int c = 0; c < CH; c++) {
                        const uint32_t b_lo = ((ring_lo + uint32_t(at[c]) * (C::STAGE >> 4)) & 0x3fffu) | (1u << 16);
                        const uint32_t a_lo = q_lo + c * (C::ATOMS / CH) * (BM * 128 >> 4);
#pragma unroll
                        for (int k = 0; k < DP / CH / 16; k++) {
                            const uint32_t step = (k & 3) * 2, a_off = (k >> 2) * (BM * 128 >> 4) + step, b_off = (k >> 2) * (BN * 128 >> 4) + step;
                            if (leader)
                                umma::mma_f16_lohi(d, a_lo + a_off, k_hi, b_lo + b_off, k_hi, qk_desc, c > 0 || k > 0);
                        }
                    }
                    if (leader) {
                        umma::mma_commit(&sh.s_full[buffer]);
#pragma unroll
                        for (int c = 0; c < CH; c++)
                            umma::mma_commit(&sh.empty[at[c]]);
                    }
                };
                auto pv = [&](int buffer, const int (&at)[CH], bool accumulate, bool announce) {
                    const uint32_t d = tmem + C::O_COL + (NS == 2 ? self * DP : 0), pt = tmem + buffer * BN;
#pragma unroll
                    for (int c = 0; c < CH; c++) {
                        const uint32_t b_lo = ((ring_lo + uint32_t(at[c]) * (C::STAGE >> 4)) & 0x3fffu) | (v_lbo << 16);
#pragma unroll
                        for (int k = 0; k < BN / CH / 16; k++)
                            if (leader)
                                umma::mma_f16_ts(d, pt + c * (BN / CH / 2) + 8 * k, b_lo + k * (2048 >> 4), k_hi, pv_desc, accumulate || c > 0 || k > 0);
                    }
                    if (leader) {
                        if (announce)
                            umma::mma_commit(&sh.pv_done[buffer]);
#pragma unroll
                        for (int c = 0; c < CH; c++)
                            umma::mma_commit(&sh.empty[at[c]]);
                    }
                };
                int k_at[CH], v_at[CH];
                if constexpr (NS == 2) {
                    // tile i's scores go into buffer i & 1, behind the product that uses the weights of tile i - 2 there
                    ok = wait_warp(&sh.q_full[self], 0, dead, status, OVK_DEV_TIMEOUT_TMA);
                    for (int j = 0; j < SB && j < tiles; j++) {
                        next_tile(k_at, true);
                        if (ok)
                            qk(2 * self + j, k_at);
                    }
                    for (int i = 0; i < tiles && ok; i++) {
                        const bool more = i + SB < tiles;
                        next_tile(v_at, true);
                        if (more)
                            next_tile(k_at, true);
                        ok = ok && wait_warp(&sh.p_full[2 * self + (i & 1)], (i >> 1) & 1, dead, status, OVK_DEV_TIMEOUT_SLOT);
                        if (!ok)
                            break;
                        umma::tc_fence_after();
                        pv(2 * self + (i & 1), v_at, i > 0, true);
                        if (more)
                            qk(2 * self + (i & 1), k_at);
                    }
                } else {
                    // tile i's scores go into buffer i & 1 once the weights of tile i - 2, which lay there, are used
                    const bool scores = self == 1;
                    if (scores)
                        ok = wait_warp(&sh.q_full[0], 0, dead, status, OVK_DEV_TIMEOUT_TMA);
                    for (int j = 0; j < SB && j < tiles; j++) {
                        next_tile(k_at, scores);
                        if (scores && ok)
                            qk(j, k_at);
                    }
                    for (int i = 0; i < tiles && ok; i++) {
                        next_tile(v_at, !scores);
                        if (!scores) {
                            ok = ok && wait_warp(&sh.p_full[i & 1], (i >> 1) & 1, dead, status, OVK_DEV_TIMEOUT_SLOT);
                            if (!ok)
                                break;
                            umma::tc_fence_after();
                            pv(i & 1, v_at, i > 0, true);
                        }
                        if (i + SB < tiles) {
                            next_tile(k_at, scores);
                            if (scores) {
                                ok = ok && wait_warp(&sh.pv_done[i & 1], (i >> 1) & 1, dead, status, OVK_DEV_TIMEOUT_MMA);
                                if (!ok)
                                    break;
                                umma::tc_fence_after();
                                qk(i & 1, k_at);
                            }
                        }
                    }
                }
                if (!ok) {  // products in flight end before tensor memory is freed
                    if (leader)
                        umma::mma_commit(&sh.drain[self]);
                    umma::mbar_wait(&sh.drain[self], 0);
                }
            }
            __syncwarp();
        } else if (tiles > 0 && (NS == 2 || group == 2)) {
            // ------------------------------------------------------------ guards
            const int guard = NS == 2 ? 0 : warp & 3;
            int n = CH * min(SB, tiles);  // place in the ring
            uint32_t raw_phase = 0;       // a bit per stage
            bool ok = true;
            for (int i = 0; i < tiles && ok; i++) {
                for (int c = 0; c < CH && ok; c++, n++) {
                    if (!partial(i, pos0, pos_last))
                        continue;
                    const int stage = n % C::STAGES;
                    ok = wait_warp(&sh.raw[stage], (raw_phase >> stage) & 1, dead, status, OVK_DEV_TIMEOUT_TMA);
                    raw_phase ^= 1u << stage;
                    // in each 128-byte column the chunk's rows lie one after the other, eight 16-byte words a row
                    constexpr int KEYS = BN / CH, STEP = 32 * C::GUARDS, WORDS = C::STAGE / 16 / STEP;
                    const int left = min(KEYS, max(0, key_end - (key_begin + i * BN + c * KEYS)));  // rows before the end
                    const int self = guard * 32 + lane;
                    if (ok) {
                        uint4 *const words = reinterpret_cast<uint4 *>(ring + stage * C::STAGE) + self;
                        bool wrote = false;
                        if (left < KEYS)
                            for (int k = 0; k < WORDS; k++)
                                if ((((self + STEP * k) >> 3) & (KEYS - 1)) >= left)
                                    words[STEP * k] = make_uint4(0, 0, 0, 0), wrote = true;
                        uint32_t bad = 0;
#pragma unroll 8
                        for (int k = 0; k < WORDS; k++) {
                            const uint4 v = words[STEP * k];  // a carry into the sign bit marks an exponent of ones
                            bad |= ((v.x & 0x7c007c00u) + 0x04000400u) | ((v.y & 0x7c007c00u) + 0x04000400u) |
                                   ((v.z & 0x7c007c00u) + 0x04000400u) | ((v.w & 0x7c007c00u) + 0x04000400u);
                        }
                        if (bad & 0x80008000u) {
                            wrote = true;
#pragma unroll 1
                            for (int k = 0; k < WORDS; k++) {
                                const int at = self + STEP * k;
                                const int col = at / (KEYS * 8) * 64 + (((at & 7) ^ ((at >> 3) & 7)) << 3);  // of the word's first element
                                __half *const z = reinterpret_cast<__half *>(&words[STEP * k]);
                                for (int e = 0; e < 8; e++)
                                    if ((__half_as_ushort(z[e]) & 0x7c00u) == 0x7c00u) {
                                        z[e] = __ushort_as_half(0);
                                        atomicOr(&sh.odd[(col + e) >> 5], 1u << ((col + e) & 31));
                                    }
                            }
                        }
                        if (wrote)
                            umma::fence_proxy_async();
                    }
                    // all of them, also after a wait that gave up: then all leave
                    uint32_t all;
                    asm volatile(
                        "{\n\t.reg .pred p, q;\n\t"
                        "setp.ne.b32 p, %1, 0;\n\t"
                        "bar.red.and.pred q, 2, %2, p;\n\t"
                        "selp.u32 %0, 1, 0, q;\n\t}"
                        : "=r"(all)
                        : "r"(uint32_t(ok)), "n"(32 * C::GUARDS)
                        : "memory");
                    ok = all != 0;
                    if (ok && guard == 0 && lane == 0)
                        umma::mbar_arrive(&sh.full[stage]);
                }
                n += i + SB < tiles ? CH : 0;
            }
        }
    } else {
        // ---------------------------------------------------------------- softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::SOFTMAX_REGS));
        umma::tc_fence_before();
        asm volatile("bar.sync 1, %0;" ::"n"(C::THREADS - 32) : "memory");
        umma::tc_fence_after();
        const uint32_t tmem = sh.tmem;
        const int s = group;
        if (s < streams) {
            const int r = tid & 127, rows = min(BM, rows_all - (rows_split ? s * BM : 0));
            const int first = pos0 + (rows_split ? s * BM : 0), pos = first + r;
            const uint32_t lanes = uint32_t(warp & 3) << 21;  // 32 lanes a warp
            const uint32_t t_o = tmem + lanes + C::O_COL + s * DP;
            const float scale = a.scale_log2e;
            float m = NO_SCORE, l = 0.0f;
            float ahead = 15.0f;  // how far a score may pass m; less than any where m is so large that scores have to be rounded (below)
            bool ok = true;
            for (int i = 0; i < tiles; i++) {
                const int buffer = 2 * s + (i & 1);
                const uint32_t t_s = tmem + lanes + buffer * BN;
                ok = wait_warp(&sh.s_full[buffer], (i >> 1) & 1, dead, status, OVK_DEV_TIMEOUT_MMA);
                if (!ok)
                    break;
                umma::tc_fence_after();
                uint32_t x[BN / 32][32];
#pragma unroll
                for (int c = 0; c < BN / 32; c++)
                    umma::tmem_ld_32x32(t_s + 32 * c, x[c]);
                umma::tmem_ld_wait();
                const int j0 = key_begin + i * BN;
                if (j0 + BN > w.n_k || (a.causal && j0 + BN - 1 > first)) {
                    const int hi = (a.causal ? min(pos, w.n_k - 1) : w.n_k - 1) - j0;
#pragma unroll
                    for (int c = 0; c < BN / 32; c++)
#pragma unroll
                        for (int e = 0; e < 32; e++)
                            if (32 * c + e > hi)
                                x[c][e] = 0xff800000u;  // -infinity
                }
                if (p.window > 0 && j0 <= first + rows - 1 - p.window) {
                    const int lo = pos - p.window + 1 - j0;
#pragma unroll
                    for (int c = 0; c < BN / 32; c++)
#pragma unroll
                        for (int e = 0; e < 32; e++)
                            if (32 * c + e < lo)
                                x[c][e] = 0xff800000u;
                }
                float most[4];
#pragma unroll
                for (int e = 0; e < 4; e++)
                    most[e] = __uint_as_float(x[0][e]);
#pragma unroll
                for (int e = 4; e < BN; e++)
                    most[e & 3] = fmaxf(most[e & 3], __uint_as_float(x[e >> 5][e & 31]));
                const float top = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * scale;
                float factor = scale;
                if (__any_sync(0xffffffffu, top - m > ahead)) {  // the difference is exact where it matters
                    const float to = fmaxf(m, top - 7.0f), f = exp2_approx(m - to);
                    m = to;
                    // m is a rounded product, off by up to 2^-25 |m|; the multiply-add below uses unrounded ones.  That is a
                    // factor common to all of a row's weights, but far from zero it passes fp16's range: there scores are
                    // rounded too.
                    ahead = fabsf(m) > 0x1p22f && m != NO_SCORE ? -INFINITY : 15.0f;
                    if (__any_sync(0xffffffffu, ahead < 0.0f)) {
                        factor = 1.0f;
#pragma unroll
                        for (int e = 0; e < BN; e++)
                            x[e >> 5][e & 31] = __float_as_uint(__uint_as_float(x[e >> 5][e & 31]) * scale);
                    }
                    l *= f;
                    if (i > 0) {
                        // the product before this one may still be writing O
                        ok = wait_warp(&sh.pv_done[2 * s + ((i - 1) & 1)], ((i - 1) >> 1) & 1, dead, status, OVK_DEV_TIMEOUT_MMA);
                        if (!ok)
                            break;
                        umma::tc_fence_after();
#pragma unroll
                        for (int c = 0; c < DP / 16; c++) {
                            uint32_t o[16];
                            umma::tmem_ld_32x16(t_o + 16 * c, o);
                            umma::tmem_ld_wait();
#pragma unroll
                            for (int e = 0; e < 16; e++)
                                o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                            umma::tmem_st_32x16(t_o + 16 * c, o);
                        }
                    }
                }
                float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int c = 0; c < BN / 64; c++) {
                    uint32_t out[32];
#pragma unroll
                    for (int e = 0; e < 32; e++) {
                        const int at = 64 * c + 2 * e;
                        const float p0 = exp2_approx(fmaf(__uint_as_float(x[at >> 5][at & 31]), factor, -m));
                        const float p1 = exp2_approx(fmaf(__uint_as_float(x[at >> 5][(at & 31) + 1]), factor, -m));
                        sum[(2 * e) & 3] += p0;
                        sum[(2 * e + 1) & 3] += p1;
                        out[e] = pack_halves(p0, p1);
                    }
                    umma::tmem_st_32x32(t_s + 32 * c, out);
                }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                umma::tmem_st_wait();
                umma::tc_fence_before();
                __syncwarp();
                if (lane == 0)
                    umma::mbar_arrive(&sh.p_full[buffer]);
            }
            if (ok && tiles > 0) {
                ok = wait_warp(&sh.pv_done[2 * s + ((tiles - 1) & 1)], ((tiles - 1) >> 1) & 1, dead, status, OVK_DEV_TIMEOUT_MMA);
                umma::tc_fence_after();
            }
            if (ok) {
                // By way of the queries' place in shared memory, which no product reads any more: a warp lays its 32 rows
                // there, 16-byte words exchanged by row so that neither side meets in a bank, and stores them row by row.
                // (Straight from registers a store touched 32 lines: 6300 cycles a tile of 256-wide rows, now 3800.)
                const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
                uint8_t *const stage = smem + s * C::Q_BYTES;
                bool any_odd = false;
                for (int i = 0; i < DP / 32; i++)
                    any_odd |= sh.odd[i] != 0;
#pragma unroll 1  // run once a tile, so what it costs is fetching its instructions
                for (int c = 0; c < DP / 64; c++) {
                    uint32_t o[2][32];
                    if (tiles > 0) {
                        umma::tmem_ld_32x32(t_o + 64 * c, o[0]);
                        umma::tmem_ld_32x32(t_o + 64 * c + 32, o[1]);
                        umma::tmem_ld_wait();
                    } else {
#pragma unroll
                        for (int e = 0; e < 64; e++)
                            o[e >> 5][e & 31] = 0;
                    }
                    if (any_odd && (sh.odd[2 * c] | sh.odd[2 * c + 1])) {
                        // elements that the guards took out, of the keys that this row reads
                        for (int i = 0; i < tiles; i++) {
                            if (r >= rows || !partial(i, pos0, pos_last))
                                continue;
                            const int j0 = key_begin + i * BN;
                            const int from = p.window > 0 ? max(j0, pos - p.window + 1) : j0;
                            const int to = min(j0 + BN, a.causal ? min(w.n_k, pos + 1) : w.n_k);
                            for (int j = from; j < to; j++) {
                                const __half *v = static_cast<const __half *>(a.v) + int64_t(w.first_k + j) * a.v_token +
                                                  int64_t(kv_head) * a.v_head + 64 * c;
#pragma unroll
                                for (int e = 0; e < 64; e++)
                                    if ((sh.odd[2 * c + (e >> 5)] >> (e & 31)) & 1) {
                                        const float x = __half2float(v[e]);
                                        if (!(x - x == 0.0f))
                                            o[e >> 5][e & 31] = __float_as_uint(__uint_as_float(o[e >> 5][e & 31]) + x);
                                    }
                            }
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        uint32_t h[4];
#pragma unroll
                        for (int u = 0; u < 4; u++)
                            h[u] = pack_halves(__uint_as_float(o[e >> 2][8 * (e & 3) + 2 * u]) * inverse,
                                               __uint_as_float(o[e >> 2][8 * (e & 3) + 2 * u + 1]) * inverse);
                        *reinterpret_cast<uint4 *>(stage + r * (DP * 2) + c * 128 + ((e ^ (r & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
                    }
                }
                __syncwarp();
                constexpr int WORDS = DP / 8;  // of a row
                const int word = lane % WORDS, r0 = (warp & 3) * 32;
                __half *const out = static_cast<__half *>(a.out) +
                                    int64_t(w.first_q + w.row0 + (rows_split ? s * BM : 0)) * a.o_token +
                                    int64_t(rows_split ? head0 : head0 + s) * a.o_head + 8 * word;
                const int left = a.head_dim - 8 * word;  // elements of the row from this word on: it may end inside the word
                auto store = [&](int k, bool whole) {
                    const int row = r0 + k * (32 / WORDS) + lane / WORDS;
                    if (row >= rows)
                        return false;
                    const uint8_t *const from = stage + row * (DP * 2) + ((word ^ (row & 7)) << 4);
                    __half *const to = out + int64_t(row) * a.o_token;
                    if (whole)
                        *reinterpret_cast<uint4 *>(to) = *reinterpret_cast<const uint4 *>(from);
                    else
#pragma unroll 1
                        for (int e = 0; e < min(left, 8); e++)
                            to[e] = reinterpret_cast<const __half *>(from)[e];
                    return true;
                };
                if (p.vec_out && left >= 8) {
#pragma unroll 8
                    for (int k = 0; k < WORDS; k++)
                        if (!store(k, true))
                            break;
                } else if (left > 0) {
#pragma unroll 1
                    for (int k = 0; k < WORDS; k++)
                        if (!store(k, false))
                            break;
                }
            }
        }
    }
    umma::tc_fence_before();
    __syncthreads();
    umma::tc_fence_after();
    if (warp == NS * 4 + 1)
        umma::tmem_dealloc(sh.tmem, 512);
}

bool make_map(CUtensorMap *map, const void *base, int64_t tokens, int64_t heads, int64_t head_dim, int64_t token_stride,
              int64_t head_stride, uint32_t rows)
{
    ovk_encode_tiled_fn fn = ovk_get_encode_tiled();
    if (!fn)
        return false;
    // a stride that no step uses may be anything; the map wants a positive one
    const int64_t hs = heads > 1 ? head_stride * 2 : 16, ts = tokens > 1 ? token_stride * 2 : 16;
    cuuint64_t dims[3] = {cuuint64_t(head_dim), cuuint64_t(heads), cuuint64_t(tokens)};
    cuuint64_t strides[2] = {cuuint64_t(hs), cuuint64_t(ts)};
    cuuint32_t box[3] = {64, 1, rows}, step[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void *>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DP> int32_t launch(ovk_ctx *ctx, const PromptArgs &a, bool *taken)
{
    using C = Tc<DP>;
    CUtensorMap q, k, v;
    const int kv_heads = a.heads / a.group;
    if (!make_map(&q, a.q, a.q_tokens, a.heads, a.head_dim, a.q_token, a.q_head, BM) ||
        !make_map(&k, a.k, a.k_tokens, kv_heads, a.head_dim, a.k_token, a.k_head, C::BN) ||
        !make_map(&v, a.v, a.k_tokens, kv_heads, a.head_dim, a.v_token, a.v_head, C::BN / C::CH))
        return OVK_OK;
    TcParams p = {};
    p.a = a;
    p.by_heads = C::NS == 2 && a.group % 2 == 0;
    p.pairs = p.by_heads ? a.heads / 2 : a.heads;
    p.window = int(a.window);
    p.vec_out = aligned_to(a.out, 16) && a.o_token % 8 == 0 && a.o_head % 8 == 0;
    const int64_t rows = C::NS == 2 && !p.by_heads ? 2 * BM : BM;
    const int64_t grid = prompt_tiles(a, rows) * p.pairs;
    if (grid >= (int64_t(1) << 31))
        return OVK_OK;
    OVK_CUDA(ctx, ovk_allow_smem(attention_prompt_tc_kernel<DP>, C::SMEM, ctx->device));
    OVK_CUDA(ctx, ovk_launch_pdl(attention_prompt_tc_kernel<DP>, dim3(unsigned(grid)), dim3(C::THREADS), C::SMEM, ctx->stream, q, k, v, p));
    *taken = true;
    OVK_LAUNCHED(ctx, "attention_prompt_tc");
    return OVK_OK;
}

}  // namespace

// *taken stays false where the layout is not one that a tensor map describes, or the scale is not positive
// (the maximum is taken before scaling).
int32_t ovk_prompt_tc(ovk_ctx *ctx, const PromptArgs &a, bool *taken)
{
    *taken = false;
    if (!a.vec || !(a.scale_log2e > 0.0f) || a.k_tokens == 0)
        return OVK_OK;
    return a.head_dim <= 64 ? launch<64>(ctx, a, taken) : a.head_dim <= 128 ? launch<128>(ctx, a, taken) : launch<256>(ctx, a, taken);
}
