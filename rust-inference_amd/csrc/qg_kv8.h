// qg_kv8.h -- the 8-bit KV cache of include/qgops.h inside the library: its
// layout on the device, shared by the kernels that write, read and attend
// (qg_kv8.hip, qg_kv8_attention.hip) and by the decode step's model.
#pragma once

#include <hip/hip_runtime.h>

#include "qg_internal.h"
#include "qgops.h"

namespace qg8 {

constexpr uint32_t kBlock = QG_KV8_BLOCK;
constexpr int kZero = 128;                   // a code's byte is the code + 128 (qg_kv8_attention.hip, halves)
constexpr uint32_t kZeros = 0x80808080u;

// A cache as the kernels see it.  A head's elements are padded with zeros to
// dp, a multiple of 64.  Index sh = seq * n_heads + head.
//
// Codes: one block of 32 positions of one head is 32 dp bytes at
// ((kv * n_seqs * n_heads + sh) * n_blocks + block) * 32 dp (kv: 0 keys, 1
// values), arranged so that a lane's 16 bytes are operands of
// v_mfma_f32_16x16x32 (lane l holds row l % 16 and k = 8 (l / 16) .. + 8 of A):
//   keys    position t, element d: A's rows are positions, so lane (g, t % 16),
//           g = d % 64 / 16, holds elements 16 g .. + 16 of every 64 -- the first
//           eight for one product, the others for the next (q is laid the same
//           way, so the order of the contraction does not matter);
//   values  A's rows are elements and k the positions: lane (g, r) holds
//           elements 32 u + 2 r and + 1, each at the positions 4 g .. + 4 and
//           16 + 4 g .. + 4 -- the positions whose scores the lane has after
//           two products of 16 positions each.
struct View {
    uint8_t *codes;          // [2][sh][n_blocks][32 dp]
    float *scale;            // [2][sh][n_blocks]
    float *tail;             // [2][sh][2][32][dp]: f32 values of the blocks that are or were open
    uint32_t *tail_max;      // [2][sh][2][32]: bits of each position's largest magnitude
    int32_t *tail_at;        // [2][sh][4]: block of slot 0, of slot 1 (-1: none), positions held by each
    uint32_t n_seqs, n_heads, hd, dp, max_len, n_blocks;
};

__host__ __device__ __forceinline__ uint32_t key_at(uint32_t t, uint32_t d, uint32_t dp)
{
    return (((t >> 4) * (dp >> 6) + (d >> 6)) << 10) + (((d >> 4 & 3u) * 16u + (t & 15u)) << 4) + (d & 15u);
}
__host__ __device__ __forceinline__ uint32_t value_at(uint32_t t, uint32_t d)
{
    return ((d >> 5) << 10) + (((t >> 2 & 3u) * 16u + (d >> 1 & 15u)) << 4) + ((d & 1u) << 3) + (t >> 4 << 2) + (t & 3u);
}

// The rows of a call: qg_batch, or (lens NULL) the rows 0 .. n_rows of the one
// sequence of a cache, ending at len0.
struct Batch {
    const uint32_t *starts, *lens;
    uint32_t n_rows, len0;
};

// Rows of a sequence: first row, count, position of the first row (may be
// below 0), number of positions.
struct Span {
    uint32_t row, n;
    int64_t pos;
    uint32_t len;
};

__device__ __forceinline__ Span span_of(const Batch &b, uint32_t s)
{
    Span p;
    if (b.starts) {
        p.row = min(b.starts[s], b.n_rows);
        const uint32_t end = min(b.starts[s + 1], b.n_rows);
        p.n = end > p.row ? end - p.row : 0u;
    } else {
        p.row = b.lens ? s : 0u;
        p.n = b.lens ? 1u : b.n_rows;
    }
    p.len = b.lens ? b.lens[s] : b.len0;
    p.pos = (int64_t)p.len - (int64_t)p.n;
    return p;
}

// Rows of qg_rows for the kernels; vec: 16-byte accesses of 16 elements.
struct Rows {
    void *p;
    uint64_t ld_row, ld_head;
    uint32_t f16, vec;
};

__device__ __forceinline__ float load1(const Rows &r, uint64_t at)
{
    return r.f16 ? (float)((const _Float16 *)r.p)[at] : ((const float *)r.p)[at];
}

// Elements d .. d + 16 of a row that starts at element `at`; zero from hd on.
__device__ __forceinline__ void load16(const Rows &r, uint64_t at, uint32_t d, uint32_t hd, float *x)
{
    if (r.vec) {
        if (d >= hd) {
#pragma unroll
            for (int i = 0; i < 16; i++) x[i] = 0.f;
        } else if (r.f16) {
            typedef _Float16 h8 __attribute__((ext_vector_type(8)));
            const h8 *p = (const h8 *)((const _Float16 *)r.p + at + d);
            const h8 a = p[0], b = p[1];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[i] = (float)a[i];
                x[8 + i] = (float)b[i];
            }
        } else {
            const float4 *p = (const float4 *)((const float *)r.p + at + d);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float4 a = p[i];
                x[4 * i] = a.x; x[4 * i + 1] = a.y; x[4 * i + 2] = a.z; x[4 * i + 3] = a.w;
            }
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 16; i++) x[i] = d + i < hd ? load1(r, at + d + i) : 0.f;
    }
}

__device__ __forceinline__ void store1(const Rows &r, uint64_t at, float v)
{
    if (r.f16) ((_Float16 *)r.p)[at] = (_Float16)v;
    else ((float *)r.p)[at] = v;
}

// A decode step's projections of one token, on the device: q [kv head][n_rep][hd]
// is rotated in place, k and v [kv head][hd] are left as they are.  pos: of the
// rotation (rows of the tables, hd / 2 each); slot: in the cache; *len becomes
// slot + 1.
struct Append {
    float *q;
    const float *k, *v, *bq, *bk, *bv, *cos_t, *sin_t;
    const uint32_t *pos, *slot;
    uint32_t *len, n_rep;
};

// Launchers; 0, or -1 for a failed launch (hipGetLastError holds it).
int launch_write(const View &c, const Batch &b, const Rows &k, const Rows &v, int n_cu, hipStream_t st);
int launch_append(const View &c, const Append &a, hipStream_t st);
int launch_read(const View &c, uint32_t seq, uint32_t n_seqs, uint32_t pos, uint32_t n, const Rows *k, const Rows *v,
                hipStream_t st);
int launch_attention(const View &c, const Batch &b, uint32_t n_heads, const Rows &q, float scale, uint32_t window,
                     const Rows &out, void *work, int n_cu, hipStream_t st);
size_t attention_work(const View &c, size_t n_rows, size_t n_heads, int n_cu);

}  // namespace qg8

struct qg_kv8 {
    qg_ctx *ctx = nullptr;
    qg8::View v{};
    void *mem = nullptr;
    size_t bytes = 0;
};

// qg_kv8_create / qg_kv8_free without the context's list of handles.
int qg_kv8_make(qg_ctx *ctx, size_t n_seqs, size_t n_kv_heads, size_t head_dim, size_t max_len, qg_kv8 **out);
void qg_kv8_drop(qg_kv8 *kv);
