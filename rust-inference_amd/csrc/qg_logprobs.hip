// qg_logprobs.hip -- log probabilities of given tokens, entropy and the most
// likely tokens of rows of logits (qg_logprobs_dev, include/qgops.h).
#include <hip/hip_runtime.h>

#include <cmath>

#include "qg_common.h"
#include "qg_internal.h"
#include "qgops.h"

namespace qgl {
namespace {

struct Args {
    const void *x;
    uint64_t ld;
    uint32_t f16, n_cols, n_given, k;
    const uint32_t *tokens;
    float *logprobs, *entropy;
    uint32_t *top_ids;
    float *top_logprobs;
};

__device__ __forceinline__ float at(const Args &a, uint64_t row, uint32_t i)
{
    return a.f16 ? (float)((const _Float16 *)a.x)[row * a.ld + i] : ((const float *)a.x)[row * a.ld + i];
}

// x before y among the alternatives: larger, or equal with a smaller id
__device__ __forceinline__ bool before(float x, uint32_t i, float y, uint32_t j)
{
    return j == QG_TOKEN_NONE || x > y || (x == y && i < j);
}

template <class F> __device__ __forceinline__ float block_fold(float v, float *red, F f)
{
    for (int o = 32; o > 0; o >>= 1) v = f(v, __shfl_xor(v, o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
    for (uint32_t i = 1; i < blockDim.x >> 6; i++) v = f(v, red[i]);
    return v;
}

// One workgroup per row.
__global__ void __launch_bounds__(256) row_k(Args a)
{
    __shared__ float red[4], bx[4];
    __shared__ uint32_t bi[4];
    const uint64_t row = blockIdx.x;
    float m = -INFINITY;
    for (uint32_t i = threadIdx.x; i < a.n_cols; i += 256) m = fmaxf(m, at(a, row, i));
    m = block_fold(m, red, [](float x, float y) { return fmaxf(x, y); });
    float z = 0.f, s = 0.f;
    for (uint32_t i = threadIdx.x; i < a.n_cols; i += 256) {
        const float d = at(a, row, i) - m, e = expf(d);
        z += e;
        if (!(e == 0.f)) s += d * e;
    }
    z = block_fold(z, red, [](float x, float y) { return x + y; });
    s = block_fold(s, red, [](float x, float y) { return x + y; });
    const float lz = logf(z);
    for (uint32_t i = threadIdx.x; i < a.n_given; i += 256) {
        const uint32_t t = a.tokens[row * a.n_given + i];
        a.logprobs[row * a.n_given + i] = t == QG_TOKEN_NONE ? 0.f : t < a.n_cols ? at(a, row, t) - m - lz : NAN;
    }
    if (a.entropy && threadIdx.x == 0) a.entropy[row] = lz - s / z;
    float px = INFINITY;
    uint32_t pi = QG_TOKEN_NONE;
    for (uint32_t r = 0; r < a.k; r++) {
        float x = -INFINITY;
        uint32_t id = QG_TOKEN_NONE;
        for (uint32_t i = threadIdx.x; i < a.n_cols; i += 256) {
            const float y = at(a, row, i);
            // behind the last one taken (r > 0), a number, and before the best so far
            if (y == y && (r == 0 || before(px, pi, y, i)) && (r == 0 || i != pi) && before(y, i, x, id)) { x = y; id = i; }
        }
        for (int o = 32; o > 0; o >>= 1) {
            const float ox = __shfl_xor(x, o, 64);
            const uint32_t oi = (uint32_t)__shfl_xor((int)id, o, 64);
            if (oi != QG_TOKEN_NONE && before(ox, oi, x, id)) { x = ox; id = oi; }
        }
        __syncthreads();
        if ((threadIdx.x & 63) == 0) { bx[threadIdx.x >> 6] = x; bi[threadIdx.x >> 6] = id; }
        __syncthreads();
        x = bx[0];
        id = bi[0];
        for (int i = 1; i < 4; i++)
            if (bi[i] != QG_TOKEN_NONE && before(bx[i], bi[i], x, id)) { x = bx[i]; id = bi[i]; }
        if (threadIdx.x == 0) {
            a.top_ids[row * a.k + r] = id;
            a.top_logprobs[row * a.k + r] = id == QG_TOKEN_NONE ? -INFINITY : x - m - lz;
        }
        px = x;
        pi = id;
        if (id == QG_TOKEN_NONE) {
            for (uint32_t j = r + 1 + threadIdx.x; j < a.k; j += 256) {
                a.top_ids[row * a.k + j] = QG_TOKEN_NONE;
                a.top_logprobs[row * a.k + j] = -INFINITY;
            }
            break;
        }
    }
}

}  // namespace
}  // namespace qgl

extern "C" {

int qg_logprobs_work(qg_ctx *ctx, size_t n_rows, size_t n_cols, size_t k, size_t *bytes)
{
    if (!ctx || !bytes) return qg_fail(ctx, QG_ERR_INVALID_ARG, "ctx or bytes is NULL");
    if (n_rows > 0x7FFFFFFFu || n_cols < 1 || n_cols > 0x7FFFFFFFu || k > QG_LOGPROBS_MAX_TOP)
        return qg_fail(ctx, QG_ERR_SHAPE, "logits or alternatives");
    *bytes = 0;
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
    a.f16 = type == qg::T_F16;
    a.n_cols = (uint32_t)n_cols;
    a.n_given = (uint32_t)n_given;
    a.k = (uint32_t)k;
    a.tokens = d_tokens;
    a.logprobs = d_logprobs;
    a.entropy = d_entropy;
    a.top_ids = d_top_ids;
    a.top_logprobs = d_top_logprobs;
    hipLaunchKernelGGL(qgl::row_k, dim3((uint32_t)n_rows), dim3(256), 0, stream ? (hipStream_t)stream : ctx->stream, a);
    e = hipGetLastError();
    return e == hipSuccess ? QG_OK : qg_fail(ctx, QG_ERR_HIP, "log probabilities", e);
}

}  // extern "C"
