// Shared by the attention operators: argument checks, the device guard, packed
// sequences, and f32 <-> element conversions.
#pragma once

#include "ovk_internal.h"

// The caller's current device is put back when the call returns.
struct DeviceGuard {
    int before = -1;
    explicit DeviceGuard(int device)
    {
        int now = -1;
        if (cudaGetDevice(&now) == cudaSuccess && now != device && cudaSetDevice(device) == cudaSuccess)
            before = now;
    }
    ~DeviceGuard()
    {
        if (before >= 0)
            cudaSetDevice(before);
    }
};

// Lets a kernel use `bytes` of dynamic shared memory on this device: once per kernel and device, since the
// call costs about as much as a launch.  Threads that ask at the same time set the same value.
template <typename... A> static inline cudaError_t ovk_allow_smem(void (*kernel)(A...), size_t bytes, int device)
{
    struct Done {
        void (*kernel)(A...);
        uint64_t devices;
    };
    constexpr int MOST = 16;  // kernels of one signature
    static thread_local Done done[MOST] = {};
    for (int i = 0; i < MOST; i++) {
        if (done[i].kernel == kernel || !done[i].kernel) {
            if (device < 64 && done[i].kernel == kernel && (done[i].devices >> device & 1))
                return cudaSuccess;
            const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes));
            if (e == cudaSuccess && device < 64)
                done[i].kernel = kernel, done[i].devices |= uint64_t(1) << device;
            return e;
        }
    }
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes));
}

// The factor that brings scores to powers of two; not finite where the scale, or this product, is not.
static inline float ovk_scale_log2e(float scale) { return scale * 1.4426950408889634f; }

// Positions are below 2^30: a window of that and more leaves out none, which is what 0 says.  (Beside the largest 64-bit
// numbers the kernels' differences would wrap.)
static inline int64_t ovk_window(int64_t window) { return window >= (int64_t(1) << 30) ? 0 : window; }

constexpr int64_t OVK_MAX_HEADS = (1 << 16) - 1;  // heads are a grid dimension

// A [tokens, heads, head_dim] tensor with contiguous heads; `what` names it in the message.  Strides
// may have any order (a [heads, tokens] tensor is one too); an output's rows must not overlap.
static inline int32_t ovk_check_heads(ovk_ctx *ctx, const char *op, const char *what, const ovk_heads *t, int64_t tokens,
                                      int64_t head_dim, size_t elem, bool output)
{
    OVK_REQUIRE(ctx, t, "%s: %s is null", op, what);
    OVK_REQUIRE(ctx, t->heads >= 1 && t->heads <= OVK_MAX_HEADS, "%s: %s has %lld heads", op, what, (long long)t->heads);
    OVK_REQUIRE(ctx, t->token_stride >= 0 && t->head_stride >= 0 && t->token_stride < (int64_t(1) << 40) &&
                         t->head_stride < (int64_t(1) << 40),
                "%s: %s has strides %lld and %lld", op, what, (long long)t->token_stride, (long long)t->head_stride);
    if (output && tokens > 0) {
        // rows of head_dim elements at token_stride and head_stride: disjoint when the larger stride
        // steps over everything the smaller one covers
        const bool heads_inside = t->token_stride >= t->head_stride;
        const int64_t inner = heads_inside ? t->head_stride : t->token_stride;
        const int64_t outer = heads_inside ? t->token_stride : t->head_stride;
        const int64_t n_inner = heads_inside ? t->heads : tokens, n_outer = heads_inside ? tokens : t->heads;
        OVK_REQUIRE(ctx, (n_inner == 1 || inner >= head_dim) &&
                             (n_outer == 1 || outer >= (n_inner == 1 ? head_dim : inner * (n_inner - 1) + head_dim)),
                    "%s: rows of %s overlap (strides %lld and %lld)", op, what, (long long)t->token_stride,
                    (long long)t->head_stride);
    }
    OVK_REQUIRE(ctx, tokens == 0 || t->data, "%s: %s has no data", op, what);
    OVK_REQUIRE(ctx, aligned_to(t->data, elem), "%s: %s is not aligned to its elements", op, what);
    return OVK_OK;
}
// Whether every row of `t` starts on a 16-byte boundary.
static inline bool ovk_rows_aligned(const ovk_heads *t, size_t elem)
{
    return aligned_to(t->data, 16) && (t->token_stride * int64_t(elem)) % 16 == 0 && (t->head_stride * int64_t(elem)) % 16 == 0;
}
static inline bool ovk_is_activation(int32_t dtype) { return dtype == OVK_FLOAT || dtype == OVK_FLOAT16; }
static inline size_t ovk_elem_bytes(int32_t dtype) { return dtype == OVK_FLOAT ? 4 : 2; }

int32_t ovk_check_kv4(ovk_ctx *ctx, const char *op, const ovk_kv4_cache *c);
int32_t ovk_check_kv4_batch(ovk_ctx *ctx, const char *op, const ovk_kv4_batch *b);

#ifdef __CUDACC__
// The index of the sequence that holds packed row `token` of `tokens`, or -1: the last b with cu[b] <= token,
// if its end lies behind it (empty sequences share their start with the next one).  Where the sequences bring
// about as many rows each - one in decode - the first place looked at is the right one.
__device__ __forceinline__ int sequence_of(const int32_t *__restrict__ cu, int batch, int token, int tokens)
{
    const int guess = int(float(token) * (float(batch) / float(tokens)));  // any will do; batch < 2^24
    if (guess < batch && cu[guess] <= token && token < cu[guess + 1])
        return guess;
    int lo = 0, hi = batch;  // cu[lo] <= token < cu[hi] once both are inside
    if (token < cu[0] || token >= cu[batch])
        return -1;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cu[mid] <= token)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// The running maximum of a row that has seen nothing.  Finite, so that a masked score (-infinity) less it is -infinity and
// not NaN; no score is lower but one that has overflowed.
constexpr float NO_SCORE = -3.402823466e38f;

__device__ __forceinline__ float exp2_approx(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack_halves(float lo, float hi)
{
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// N consecutive elements of 4 or 2 bytes, in 16-byte accesses where VEC says that the address allows it
template <typename T, int N, bool VEC> __device__ __forceinline__ void load_row(const T *p, float (&v)[N])
{
    if constexpr (VEC) {
        constexpr int PER = 16 / sizeof(T);
        static_assert(N % PER == 0, "whole 16-byte words");
#pragma unroll
        for (int i = 0; i < N / PER; i++) {
            const uint4 w = reinterpret_cast<const uint4 *>(p)[i];
            if constexpr (sizeof(T) == 4) {
                v[4 * i] = __uint_as_float(w.x), v[4 * i + 1] = __uint_as_float(w.y);
                v[4 * i + 2] = __uint_as_float(w.z), v[4 * i + 3] = __uint_as_float(w.w);
            } else {
                const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[e]));
                    v[8 * i + 2 * e] = f.x, v[8 * i + 2 * e + 1] = f.y;
                }
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++)
            v[i] = to_f32<T>(p[i]);
    }
}
template <typename T, int N, bool VEC> __device__ __forceinline__ void store_row(T *p, const float (&v)[N])
{
    if constexpr (VEC) {
        constexpr int PER = 16 / sizeof(T);
        static_assert(N % PER == 0, "whole 16-byte words");
#pragma unroll
        for (int i = 0; i < N / PER; i++) {
            uint4 w;
            if constexpr (sizeof(T) == 4) {
                w = make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]),
                               __float_as_uint(v[4 * i + 3]));
            } else {
                w = make_uint4(pack_halves(v[8 * i], v[8 * i + 1]), pack_halves(v[8 * i + 2], v[8 * i + 3]),
                               pack_halves(v[8 * i + 4], v[8 * i + 5]), pack_halves(v[8 * i + 6], v[8 * i + 7]));
            }
            reinterpret_cast<uint4 *>(p)[i] = w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++)
            p[i] = from_f32<T>(v[i]);
    }
}
#endif
