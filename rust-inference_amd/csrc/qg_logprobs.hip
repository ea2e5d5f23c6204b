// qg_logprobs.hip -- log probabilities of given tokens, entropy and the most
// likely tokens of rows of logits (qg_logprobs_dev, include/qgops.h).
#include <hip/hip_runtime.h>

#include <cmath>

#include "qg_common.h"
#include "qg_internal.h"
#include "qgops.h"

namespace qgl {
namespace {

// A row's numbers: m = max x, z = sum e, s = sum d e with d = (x - m) log2(e) and
// e = 2^d, so that log p_t = x_t - m - ln z and the entropy is ln z - ln(2) s / z.
//
// A row is read once, in parts of one workgroup each (several where there are
// few rows; joined by final_k), 256 E elements at a time in registers: the maximum
// of a thread's own elements, then their sums under it, then the threads' sums
// are joined.  For the alternatives every element is a key (value, then the
// smaller id first), all keys distinct.  The k-th largest of the threads' largest
// keys is a floor: no more than k threads hold keys at or above it, so at most k E
// candidates leave the registers, usually little more than k; they are ranked by
// counting the larger ones.
//
// Bound by the read of the logits where there are many rows (2048 rows of 151936
// in f16, no alternatives: 152 us, 4.1 TB/s, what a plain sum of them reads at), by
// two dependent launches where there are few: one row of 152064 with 8 alternatives
// 8.8 us and 7.3 (64 of them: 9.8 and 15.2), 64 rows of 128256 with 20 14.0 and 5.2.
constexpr uint32_t kThreads = 256;
constexpr uint32_t kMaxParts = 64, kMaxK = QG_LOGPROBS_MAX_TOP;
constexpr float kLowest = -3.402823466e38f, kLog2e = 1.44269504f, kLn2 = 0.693147181f;

struct Args {
    const void *x;
    uint64_t ld;
    uint32_t n_cols, n_given, k;
    uint32_t parts, len;             // elements of a part
    const uint32_t *tokens;
    float *logprobs, *entropy;
    uint32_t *top_ids;
    float *top_logprobs;
    float *sums;                     // [row][part][4]: m, z, s
    uint64_t *keys;                  // [row][part][k]
};

struct Sums {
    float m, z, s;
};

// The sums of two sets of logits.  m is at least kLowest, so that a set of
// nothing (or of -inf) adds nothing.
__device__ __forceinline__ Sums join(Sums a, Sums b)
{
    const float m = fmaxf(a.m, b.m);
    const float da = fmaxf(a.m - m, -1e30f) * kLog2e, db = fmaxf(b.m - m, -1e30f) * kLog2e;
    // inf - inf is NaN and stays one
    const float ea = __builtin_amdgcn_exp2f((a.m - m) * kLog2e), eb = __builtin_amdgcn_exp2f((b.m - m) * kLog2e);
    return Sums{m, a.z * ea + b.z * eb, ea * (a.s + da * a.z) + eb * (b.s + db * b.z)};
}

// Over the workgroup, to all threads.
__device__ Sums join_all(Sums a, Sums *red)
{
#pragma unroll 1
    for (int o = 32; o > 0; o >>= 1)
        a = join(a, Sums{__shfl_xor(a.m, o, 64), __shfl_xor(a.z, o, 64), __shfl_xor(a.s, o, 64)});
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) red[threadIdx.x >> 6] = a;
    __syncthreads();
    a = red[0];
#pragma unroll 1
    for (uint32_t i = 1; i < kThreads / 64; i++) a = join(a, red[i]);
    return a;
}

// Larger keys first: larger values, then smaller ids.  0: no key (NaN).
__device__ __forceinline__ uint64_t key_of(float x, uint32_t id)
{
    const uint32_t b = __float_as_uint(x + 0.f);              // -0 as 0
    const uint32_t o = b & 0x80000000u ? ~b : b | 0x80000000u;
    return x == x ? (uint64_t)o << 32 | (uint32_t)~id : 0ull;
}
__device__ __forceinline__ float value_of(uint64_t key)
{
    const uint32_t o = (uint32_t)(key >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}

// LDS of the selection: the threads' largest keys, candidates and what is left of
// them, the best so far, floor_of's answer, the number of candidates.
template <uint32_t CAP> struct Pick {
    static constexpr uint32_t kRounds = (CAP + kThreads - 1) / kThreads;
    uint64_t top[kThreads], cand[CAP], left[CAP > kThreads ? kMaxK * kRounds : 1], best[kMaxK], floor;
    uint32_t n;
};

// How many of n keys (16-byte aligned, zeros up to a multiple of 16) are larger:
// sixteen at a time, their reads one behind the other.
__device__ __forceinline__ uint32_t count_larger(const uint64_t *keys, uint32_t n, uint64_t key)
{
    uint32_t c = 0;
#pragma unroll 2
    for (uint32_t i = 0; i < n; i += 16) {
        ulonglong2 t[8];
#pragma unroll
        for (uint32_t j = 0; j < 8; j++) t[j] = *(const ulonglong2 *)&keys[i + 2 * j];
#pragma unroll
        for (uint32_t j = 0; j < 8; j++) c += (t[j].x > key ? 1u : 0u) + (t[j].y > key ? 1u : 0u);
    }
    return c;
}

// The k-th largest of the threads' keys (0: fewer than k have one).
template <uint32_t CAP> __device__ uint64_t floor_of(Pick<CAP> &p, uint64_t key, uint32_t k)
{
    __syncthreads();
    p.top[threadIdx.x] = key;
    if (threadIdx.x == 0) p.floor = 0;
    __syncthreads();
    const uint32_t larger = count_larger(p.top, kThreads, key);
    if (key && larger == k - 1) p.floor = key;               // one thread, or none
    __syncthreads();
    return p.floor;
}

// The k largest of p.cand[0 .. p.n), in order, into p.best (0 behind them).
template <uint32_t CAP> __device__ void rank(Pick<CAP> &p, uint32_t k)
{
    uint64_t *from = p.cand, *to = p.left;
    __syncthreads();
    uint32_t n = p.n;
    while (n > kThreads) {                    // at most k ceil(n / 256) are left each time
        uint64_t top = 0;
#pragma unroll 1
        for (uint32_t i = threadIdx.x; i < n; i += kThreads) top = from[i] > top ? from[i] : top;
        const uint64_t f = floor_of(p, top, k);
        if (threadIdx.x == 0) p.n = 0;
        __syncthreads();
        if (top && top >= f)
#pragma unroll 1
            for (uint32_t i = threadIdx.x; i < n; i += kThreads)
                if (from[i] && from[i] >= f) to[atomicAdd(&p.n, 1u)] = from[i];
        __syncthreads();
        n = p.n;
        uint64_t *const t = from;
        from = to;
        to = t;
    }
    const uint64_t own = threadIdx.x < n ? from[threadIdx.x] : 0ull;
    p.top[threadIdx.x] = own;
    if (threadIdx.x < k) p.best[threadIdx.x] = 0;
    __syncthreads();
    const uint32_t larger = count_larger(p.top, n, own);
    if (own && larger < k) p.best[larger] = own;
    __syncthreads();
}

// What a row answers with, from its sums and the keys in `best`.
__device__ void answer(const Args &a, uint64_t row, const void *x, bool f16, Sums t, const uint64_t *best)
{
    // no token of positive probability: no distribution
    const float lz = t.z > 0.f ? logf(t.z) : __uint_as_float(0x7FC00000u);
    for (uint32_t i = threadIdx.x; i < a.n_given; i += kThreads) {
        const uint32_t id = a.tokens[row * a.n_given + i];
        float y = id == QG_TOKEN_NONE ? 0.f : __uint_as_float(0x7FC00000u);
        if (id < a.n_cols) y = (f16 ? (float)((const _Float16 *)x)[id] : ((const float *)x)[id]) - t.m - lz;
        a.logprobs[row * a.n_given + i] = y;
    }
    if (a.entropy && threadIdx.x == 0) a.entropy[row] = lz - kLn2 * (t.s / t.z);
    for (uint32_t i = threadIdx.x; i < a.k; i += kThreads) {
        const uint64_t key = best[i];
        a.top_ids[row * a.k + i] = key ? ~(uint32_t)key : QG_TOKEN_NONE;
        a.top_logprobs[row * a.k + i] = key ? value_of(key) - t.m - lz : -INFINITY;
    }
}

// Grid: (rows, parts).  TOP: with alternatives.
template <int E, bool F16, bool TOP> __global__ void __launch_bounds__(kThreads) part_k(Args a)
{
    constexpr uint32_t VE = F16 ? 8 : 4, NV = E / VE, CAP = TOP ? kMaxK * E + kMaxK : 1;
    __shared__ __attribute__((aligned(16))) Pick<CAP> pick;
    __shared__ Sums red[kThreads / 64];
    typedef _Float16 h8 __attribute__((ext_vector_type(8)));
    const uint64_t row = blockIdx.x;
    const uint32_t es = F16 ? 2 : 4, lo = blockIdx.y * a.len, hi = min(lo + a.len, a.n_cols);
    const char *x = (const char *)a.x + row * a.ld * es;
    // the first element of a 16-byte word at or before lo
    const int64_t begin = (int64_t)lo - (int64_t)(((uintptr_t)x / es + lo) % VE);
    Sums all{kLowest, 0.f, 0.f};
    uint64_t least = 0;                                        // the k-th best so far
    if (TOP && threadIdx.x < kMaxK) pick.best[threadIdx.x] = 0;
    for (int64_t c = begin; c < (int64_t)hi; c += (int64_t)kThreads * E) {
        float v[NV][VE];
#pragma unroll
        for (uint32_t i = 0; i < NV; i++) {
            const int64_t at = c + (int64_t)(i * kThreads + threadIdx.x) * VE;
            if (at >= (int64_t)lo && at + VE <= (int64_t)hi) {
                if (F16) {
                    const h8 w = *(const h8 *)(x + at * 2);
#pragma unroll
                    for (uint32_t j = 0; j < VE; j++) v[i][j] = (float)w[j];
                } else {
                    const float4 w = *(const float4 *)(x + at * 4);
                    v[i][0] = w.x; v[i][1] = w.y; v[i][2] = w.z; v[i][3] = w.w;
                }
            } else {
#pragma unroll
                for (uint32_t j = 0; j < VE; j++) {
                    const int64_t k = at + j;
                    v[i][j] = k < (int64_t)lo || k >= (int64_t)hi ? -INFINITY
                              : F16 ? (float)((const _Float16 *)x)[k] : ((const float *)x)[k];
                }
            }
        }
        Sums t{kLowest, 0.f, 0.f};
#pragma unroll
        for (uint32_t i = 0; i < NV; i++)
#pragma unroll
            for (uint32_t j = 0; j < VE; j++) t.m = fmaxf(t.m, v[i][j]);
#pragma unroll
        for (uint32_t i = 0; i < NV; i++)
#pragma unroll
            for (uint32_t j = 0; j < VE; j++) {
                const float d = (v[i][j] - t.m) * kLog2e, e = __builtin_amdgcn_exp2f(d);
                t.z += e;
                t.s = __builtin_fmaf(fmaxf(d, -1000.f), e, t.s);
            }
        all = join(all, t);
        if (TOP) {
            // element n of the thread (vector n / VE)
            const int64_t own0 = c + (int64_t)threadIdx.x * VE;
            auto id_of = [&](uint32_t n) { return own0 + (int64_t)(n / VE) * (kThreads * VE) + n % VE; };
            // its key, read once more (0 outside of the part)
            auto key_at = [&](uint32_t n) {
                const int64_t k = id_of(n);
                if (k < (int64_t)lo || k >= (int64_t)hi) return 0ull;
                return (unsigned long long)key_of(F16 ? (float)((const _Float16 *)x)[k] : ((const float *)x)[k], (uint32_t)k);
            };
            // the thread's largest key: the first of its largest values (t.m is
            // kLowest at least: where it is, every element is looked at)
            uint64_t top = 0;
            if (t.m > kLowest) {
                uint32_t n = 0;
#pragma unroll
                for (int i = E - 1; i >= 0; i--) n = v[i / VE][i % VE] == t.m ? (uint32_t)i : n;
                top = key_of(t.m, (uint32_t)id_of(n));
            } else {
#pragma unroll 1
                for (uint32_t n = 0; n < E; n++) {
                    const uint64_t key = key_at(n);
                    top = key > top ? key : top;
                }
            }
            if (__syncthreads_or(top > least)) {
                const uint64_t f = floor_of(pick, top, a.k);
                const uint64_t from = f > least ? f : least + 1;
                if (threadIdx.x == 0) pick.n = 0;
                __syncthreads();
                if (threadIdx.x < a.k && pick.best[threadIdx.x])
                    pick.cand[atomicAdd(&pick.n, 1u)] = pick.best[threadIdx.x];
                if (top >= from) {
                    // the elements that are as large as the floor's value by their
                    // bits, then their keys
                    const float y = from >> 32 ? value_of(from) : -INFINITY;
                    uint64_t some = 0;
#pragma unroll
                    for (int i = 0; i < E; i++) some |= v[i / VE][i % VE] >= y ? 1ull << i : 0ull;
#pragma unroll 1
                    for (; some; some &= some - 1) {
                        const uint64_t key = key_at((uint32_t)__ffsll((unsigned long long)some) - 1);
                        if (key >= from) pick.cand[atomicAdd(&pick.n, 1u)] = key;
                    }
                }
                rank(pick, a.k);
                least = pick.best[a.k - 1];
            }
        }
    }
    all = join_all(all, red);
    if (a.parts == 1) {
        answer(a, row, x, F16, all, TOP ? pick.best : nullptr);
        return;
    }
    const uint64_t at = row * a.parts + blockIdx.y;
    if (threadIdx.x == 0) *(float4 *)(a.sums + at * 4) = make_float4(all.m, all.z, all.s, 0.f);
    if (TOP && threadIdx.x < a.k) a.keys[at * a.k + threadIdx.x] = pick.best[threadIdx.x];
}

// Joins the parts of a row.
template <bool F16, bool TOP> __global__ void __launch_bounds__(kThreads) final_k(Args a)
{
    constexpr uint32_t CAP = TOP ? kMaxParts * kMaxK : 1;
    __shared__ __attribute__((aligned(16))) Pick<CAP> pick;
    __shared__ Sums red[kThreads / 64];
    const uint64_t row = blockIdx.x;
    Sums t{kLowest, 0.f, 0.f};
    if (threadIdx.x < a.parts) {
        const float4 w = *(const float4 *)(a.sums + (row * a.parts + threadIdx.x) * 4);
        t = Sums{w.x, w.y, w.z};
    }
    if (TOP) {
        if (threadIdx.x == 0) pick.n = a.parts * a.k;
#pragma unroll 8
        for (uint32_t i = threadIdx.x; i < a.parts * a.k; i += kThreads)
            pick.cand[i] = a.keys[row * a.parts * a.k + i];
        rank(pick, a.k);
    }
    t = join_all(t, red);
    answer(a, row, (const char *)a.x + row * a.ld * (F16 ? 2 : 4), F16, t, TOP ? pick.best : nullptr);
}

// Parts of a row: enough for about two workgroups per compute unit, of 2048
// elements at least (64 rows of 128256 with 20 alternatives 19.8 us; three and four
// a compute unit 29 and 23).
uint32_t parts_of(size_t n_rows, size_t n_cols, int n_cu)
{
    const size_t want = 2u * (size_t)(n_cu > 0 ? n_cu : 256) / (n_rows ? n_rows : 1), most = (n_cols + 2047) / 2048;
    size_t s = want < most ? want : most;
    s = s < 1 ? 1 : s > kMaxParts ? kMaxParts : s;
    return (uint32_t)s;
}

template <bool F16, bool TOP> void launch(const Args &a, uint32_t n_rows, hipStream_t st)
{
    const dim3 grid(n_rows, a.parts), block(kThreads);
    // up to 7 elements more for the rows' alignment
    const uint32_t per = (a.len + 7 + kThreads - 1) / kThreads;
    if (per <= 8) hipLaunchKernelGGL((part_k<8, F16, TOP>), grid, block, 0, st, a);
    else if (per <= 16) hipLaunchKernelGGL((part_k<16, F16, TOP>), grid, block, 0, st, a);
    else if (per <= 32) hipLaunchKernelGGL((part_k<32, F16, TOP>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((part_k<64, F16, TOP>), grid, block, 0, st, a);
    if (a.parts > 1) hipLaunchKernelGGL((final_k<F16, TOP>), dim3(n_rows), block, 0, st, a);
}

}  // namespace
}  // namespace qgl

extern "C" {

int qg_logprobs_work(qg_ctx *ctx, size_t n_rows, size_t n_cols, size_t k, size_t *bytes)
{
    if (!ctx || !bytes) return qg_fail(ctx, QG_ERR_INVALID_ARG, "ctx or bytes is NULL");
    // a launch counts its threads in 32 bits, 256 for each row
    if (n_rows >> 24 || n_cols < 1 || n_cols > 0x7FFFFFFFu || k > QG_LOGPROBS_MAX_TOP)
        return qg_fail(ctx, QG_ERR_SHAPE, "logits or alternatives");
    // what calls of fewer rows need too: parts * rows is largest just before the
    // rows alone are enough workgroups
    const size_t cus = (size_t)(ctx->n_cu > 0 ? ctx->n_cu : 256), cells = n_rows * qgl::kMaxParts;
    *bytes = n_cols > 2048 ? (cells < 2 * cus ? cells : 2 * cus) * (16 + 8 * k) : 0;
    return QG_OK;
}

int qg_logprobs_dev(qg_ctx *ctx, const void *d_logits, uint32_t type, size_t n_rows, size_t n_cols, size_t ld,
                    const uint32_t *d_tokens, size_t n_given, float *d_logprobs, float *d_entropy, size_t k,
                    uint32_t *d_top_ids, float *d_top_logprobs, void *d_work, size_t work_bytes, void *stream)
{
    size_t need = 0;
    const int rc = qg_logprobs_work(ctx, n_rows, n_cols, k, &need);
    if (rc) return rc;
    if (type != qg::T_F32 && type != qg::T_F16)
        return qg_fail(ctx, QG_ERR_UNSUPPORTED_TYPE, "logits are neither f32 nor f16");
    size_t all;
    if (n_given > 0x7FFFFFFFu || (n_rows > 1 && ld < n_cols) ||
        __builtin_mul_overflow(n_rows, ld > n_cols ? ld : n_cols, &all) || all >> 58)
        return qg_fail(ctx, QG_ERR_SHAPE, "logits or given tokens");
    if (n_rows == 0) return QG_OK;
    const size_t es = type == qg::T_F16 ? 2 : 4;
    if (!d_logits || (n_given && (!d_tokens || !d_logprobs)) || (k && (!d_top_ids || !d_top_logprobs)))
        return qg_fail(ctx, QG_ERR_INVALID_ARG, "logits, tokens or an output is NULL");
    if ((uintptr_t)d_logits % es ||
        ((uintptr_t)d_tokens | (uintptr_t)d_logprobs | (uintptr_t)d_entropy | (uintptr_t)d_top_ids | (uintptr_t)d_top_logprobs) % 4)
        return qg_fail(ctx, QG_ERR_INVALID_ARG, "an array is not aligned to its elements");
    if (need > work_bytes) return qg_fail(ctx, QG_ERR_SHAPE, "workspace too small");
    if (need && (!d_work || (uintptr_t)d_work % 16))
        return qg_fail(ctx, QG_ERR_INVALID_ARG, "workspace missing or not 16-byte aligned");
    hipError_t e = hipSetDevice(ctx->device);
    if (e != hipSuccess) return qg_fail(ctx, QG_ERR_HIP, "hipSetDevice", e);
    qgl::Args a{};
    a.x = d_logits;
    a.ld = ld;
    a.n_cols = (uint32_t)n_cols;
    a.n_given = (uint32_t)n_given;
    a.k = (uint32_t)k;
    a.tokens = d_tokens;
    a.logprobs = d_logprobs;
    a.entropy = d_entropy;
    a.top_ids = d_top_ids;
    a.top_logprobs = d_top_logprobs;
    a.parts = qgl::parts_of(n_rows, n_cols, ctx->n_cu);
    a.len = (uint32_t)((n_cols + a.parts - 1) / a.parts);
    a.sums = (float *)d_work;
    a.keys = (uint64_t *)(a.sums + (size_t)n_rows * a.parts * 4);
    const hipStream_t st = stream ? (hipStream_t)stream : ctx->stream;
    if (type == qg::T_F16) k ? qgl::launch<true, true>(a, (uint32_t)n_rows, st) : qgl::launch<true, false>(a, (uint32_t)n_rows, st);
    else k ? qgl::launch<false, true>(a, (uint32_t)n_rows, st) : qgl::launch<false, false>(a, (uint32_t)n_rows, st);
    e = hipGetLastError();
    return e == hipSuccess ? QG_OK : qg_fail(ctx, QG_ERR_HIP, "log probabilities", e);
}

}  // extern "C"
