// qg_kv8_attention.hip -- attention over the 8-bit KV cache (include/qgops.h).
#include "qg_kv8.h"

#include <cmath>

namespace qg8 {
namespace {

// One wave per (row, query head): lane (t, half) scores position t of a block
// over half of the head's elements, then lanes hold output elements.  The
// softmax's running maximum and sum are kept in the exponent's base 2.
__global__ void __launch_bounds__(64) row_k(View v, Batch b, uint32_t n_rep, Rows q, float scale2, uint32_t window, Rows out)
{
    __shared__ float qs[256], ps[32];
    const uint32_t row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, dp = v.dp;
    uint32_t seq = 0;
    Span s{};
    bool found = false;
    for (seq = 0; seq < v.n_seqs; seq++) {
        s = span_of(b, seq);
        if (row >= s.row && row < s.row + s.n) { found = true; break; }
    }
    if (!found) return;
    const int64_t p = s.pos + (int64_t)(row - s.row);
    const int64_t end = p + 1 < (int64_t)min(s.len, v.max_len) ? p + 1 : (int64_t)min(s.len, v.max_len);
    const int64_t from = window && p + 1 > (int64_t)window ? p + 1 - (int64_t)window : 0;
    for (uint32_t d = lane; d < dp; d += 64)
        qs[d] = d < v.hd ? load1(q, (uint64_t)row * q.ld_row + (uint64_t)h * q.ld_head + d) : 0.f;
    __syncthreads();
    const uint64_t sh = (uint64_t)seq * v.n_heads + h / n_rep, all = (uint64_t)v.n_seqs * v.n_heads;
    float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int64_t blk = from / 32; blk * 32 < end; blk++) {
        const uint8_t *kc = v.codes + (sh * v.n_blocks + (uint64_t)blk) * 32 * dp;
        const uint8_t *vc = v.codes + ((all + sh) * v.n_blocks + (uint64_t)blk) * 32 * dp;
        const float ks = v.scale[sh * v.n_blocks + (uint64_t)blk], vs = v.scale[(all + sh) * v.n_blocks + (uint64_t)blk];
        const uint32_t t = lane & 31u;
        float x = 0.f;
        for (uint32_t d = (lane >> 5) * (dp / 2); d < (lane >> 5) * (dp / 2) + dp / 2; d++)
            x += qs[d] * (float)(int8_t)kc[key_at(t, d, dp)];
        x += __shfl_xor(x, 32, 64);
        const int64_t j = blk * 32 + t;
        const bool seen = j >= from && j < end;
        x = seen ? x * ks * scale2 : -INFINITY;
        float bm = x;
        for (int o = 16; o > 0; o >>= 1) bm = fmaxf(bm, __shfl_xor(bm, o, 64));
        const float mn = fmaxf(m, bm);
        const float pt = seen ? exp2f(x - mn) : 0.f;
        const float alpha = m == mn ? 1.f : exp2f(m - mn);
        float bs = pt;
        for (int o = 16; o > 0; o >>= 1) bs += __shfl_xor(bs, o, 64);
        l = l * alpha + bs;
        m = mn;
        __syncthreads();
        if (lane < 32) ps[lane] = pt;
        __syncthreads();
        for (uint32_t i = 0; i < dp / 64; i++) {
            const uint32_t d = lane + 64 * i;
            float a = 0.f;
            for (uint32_t u = 0; u < 32; u++) {
                const int64_t ju = blk * 32 + u;
                if (ju >= from && ju < end) a += ps[u] * ((float)(int8_t)vc[value_at(u, d)] * vs);
            }
            acc[i] = acc[i] * alpha + a;
        }
    }
    const float inv = end > from ? 1.f / l : 0.f;
    for (uint32_t i = 0; i < dp / 64; i++) {
        const uint32_t d = lane + 64 * i;
        if (d < v.hd) store1(out, (uint64_t)row * out.ld_row + (uint64_t)h * out.ld_head + d, end > from ? acc[i] * inv : 0.f);
    }
}

}  // namespace

size_t attention_work(const View &, size_t, size_t, int)
{
    return 0;
}

int launch_attention(const View &v, const Batch &b, uint32_t n_heads, const Rows &q, float scale, uint32_t window,
                     const Rows &out, void *, int, hipStream_t st)
{
    if (b.n_rows == 0) return 0;
    hipLaunchKernelGGL(row_k, dim3(b.n_rows, n_heads), dim3(64), 0, st, v, b, n_heads / v.n_heads, q,
                       scale * 1.44269504f, window, out);
    return hipPeekAtLastError() == hipSuccess ? 0 : -1;
}

}  // namespace qg8
