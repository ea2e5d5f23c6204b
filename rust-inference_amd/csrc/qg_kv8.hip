// qg_kv8.hip -- the 8-bit KV cache of include/qgops.h: handles, and the
// kernels that quantise new keys and values into it and read them back.
#include "qg_kv8.h"

#include <algorithm>
#include <new>

namespace qg8 {
namespace {

__device__ __forceinline__ uint32_t wave_max_u(uint32_t v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, 64));
    return v;
}

// What a call does to one sequence: the positions first .. last of blocks b0 ..
// bl.  Items are what one workgroup per head takes: item 0 block b0 and, where
// the last block stays open, that one too (they share the f32 tail); item j >
// 0 the `group` whole blocks from b0 + 1 + (j - 1) group on.
struct Piece {
    Span s;
    uint32_t first, end, b0, bl, items;   // positions first .. end
};

__device__ __forceinline__ Piece piece_of(const Batch &b, uint32_t seq, uint32_t max_len, uint32_t group)
{
    Piece p;
    p.s = span_of(b, seq);
    p.end = min(p.s.len, max_len);
    p.first = p.s.pos > 0 ? (uint32_t)min(p.s.pos, (int64_t)0xFFFFFFFFll) : 0u;
    p.b0 = p.bl = p.items = 0;
    if (p.s.n == 0 || p.first >= p.end) return p;
    p.b0 = p.first / kBlock;
    p.bl = (p.end - 1) / kBlock;
    const uint32_t whole = p.bl - p.b0 - ((p.bl > p.b0 && p.end % kBlock) ? 1u : 0u);
    p.items = 1 + (whole + group - 1) / group;
    return p;
}

__device__ __forceinline__ uint32_t lane_of(uint32_t v, uint32_t l)
{
    return (uint32_t)__builtin_amdgcn_readlane((int)v, (int)l);
}

// The sequence, its piece and the item of workgroup `want`: the items of the
// sequences before it are counted 64 sequences at a time, by every wave on its
// own.  False behind the last item.
__device__ bool find_item(const Batch &b, uint32_t n_seqs, uint32_t max_len, uint32_t group, uint32_t want,
                          uint32_t *seq, uint32_t *item, Piece *piece)
{
    const uint32_t lane = threadIdx.x & 63u;
    if (b.lens && !b.starts) {                       // one row each
        *seq = want;
        *item = 0;
        *piece = piece_of(b, want, max_len, group);
        return piece->items != 0;
    }
    uint32_t before = 0;
    for (uint32_t s0 = 0; s0 < n_seqs; s0 += 64) {
        Piece p{};
        if (s0 + lane < n_seqs) p = piece_of(b, s0 + lane, max_len, group);
        uint32_t n = p.items;
#pragma unroll
        for (uint32_t o = 1; o < 64; o <<= 1) {
            const uint32_t up = (uint32_t)__shfl_up((int)n, o, 64);
            if (lane >= o) n += up;
        }
        const uint64_t past = __ballot(before + n > want);
        if (past) {
            const uint32_t l = (uint32_t)__ffsll((unsigned long long)past) - 1;
            *seq = s0 + l;
            *item = want - (before + lane_of(n - p.items, l));
            piece->s.row = lane_of(p.s.row, l);
            piece->s.n = lane_of(p.s.n, l);
            piece->s.len = lane_of(p.s.len, l);
            piece->s.pos = (int64_t)piece->s.len - (int64_t)piece->s.n;
            piece->first = lane_of(p.first, l);
            piece->end = lane_of(p.end, l);
            piece->b0 = lane_of(p.b0, l);
            piece->bl = lane_of(p.bl, l);
            piece->items = lane_of(p.items, l);
            return true;
        }
        before += lane_of(n, 63);
    }
    return false;
}

// x / s to the nearest, ties to even, as a code: the f32 product with 1 / s can
// be one off next to a half; the remainder x - q s is exact (q s has bits no
// lower than s / 2's last, and the difference is at most about s / 2), so it
// decides.
__device__ __forceinline__ int code_of(float x, float s, float inv)
{
    float q = rintf(x * inv);
    const float r = __builtin_fmaf(-q, s, x), h = 0.5f * s, a = fabsf(r);
    if (a >= h && s > 0.f) {
        if (a > h || ((int)q & 1)) q += r > 0.f ? 1.f : -1.f;
    }
    return (int)q;
}

// The codes of 16 elements as bytes (code + 128), s > 0.  The product's integer is
// the low byte of its sum with 1.5 2^23 + 128 (rounded once, ties to even); where
// any remainder reaches s / 2, code_of decides for all of them.
__device__ __forceinline__ uint4 codes_of(const float *x, float s, float inv)
{
    constexpr float kMagic = 12582912.f + (float)kZero;
    const float h = 0.5f * s;
    float most = 0.f;
    union { uint32_t w[4]; uint8_t b[16]; uint4 u; } r;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t t[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float y = __builtin_fmaf(x[4 * i + j], inv, kMagic);
            most = fmaxf(most, fabsf(__builtin_fmaf(kMagic - y, s, x[4 * i + j])));
            t[j] = __float_as_uint(y);
        }
        const uint32_t lo = __builtin_amdgcn_perm(t[1], t[0], 0x0C0C0400u), hi = __builtin_amdgcn_perm(t[3], t[2], 0x04000C0Cu);
        r.w[i] = lo | hi;
    }
    if (most >= h)
        for (int j = 0; j < 16; j++) r.b[j] = (uint8_t)(code_of(x[j], s, inv) + kZero);
    return r.u;
}

constexpr uint32_t kInf = 0x7F800000u;

// A block's scale from the bits of its largest magnitude.
__device__ __forceinline__ float scale_of(uint32_t m)
{
    const float s = __uint_as_float(m) / 127.0f;
    return m >= kInf ? __uint_as_float(0x7FC00000u) : s < 0x1p-126f ? 0.f : s;
}

// Values of a block from LDS (rows of dp + 16 bytes) into the cache's order, 16
// bytes at a time: two elements at eight positions.
__device__ __forceinline__ void put_values(const uint8_t *stage, uint8_t *codes, uint32_t dp)
{
    for (uint32_t u = threadIdx.x; u < 2 * dp; u += 256) {
        const uint32_t g = u >> 4 & 3u, d = (u >> 6) * 32u + 2u * (u & 15u);
        uint32_t two[8], w[4];
#pragma unroll
        for (uint32_t j = 0; j < 8; j++)
            two[j] = *(const uint16_t *)(stage + (4u * g + (j & 3u) + (j >> 2) * 16u) * (dp + 16) + d);
#pragma unroll
        for (uint32_t j = 0; j < 2; j++) {                // four positions: their first elements, their second ones
            const uint32_t a = two[4 * j] | two[4 * j + 1] << 16, b = two[4 * j + 2] | two[4 * j + 3] << 16;
            w[j] = __builtin_amdgcn_perm(b, a, 0x06040200u);
            w[2 + j] = __builtin_amdgcn_perm(b, a, 0x07050301u);
        }
        *(uint4 *)(codes + u * 16u) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// The slots of f32 rows of a head: their blocks (-1: none) and the positions held
// of each; the one that block b0 takes, and whether it holds what lies before the
// call's rows lo .. hi of that block.
struct Tail {
    int32_t tag0, tag1, fill0, fill1;
    uint32_t slot;
    bool held;
};

// The slot holds positions 0 .. n of block b.
__device__ __forceinline__ void hold(Tail &a, uint32_t b, uint32_t n)
{
    a.tag0 = a.slot ? a.tag0 : (int32_t)b;
    a.fill0 = a.slot ? a.fill0 : (int32_t)n;
    a.tag1 = a.slot ? (int32_t)b : a.tag1;
    a.fill1 = a.slot ? (int32_t)n : a.fill1;
}

__device__ __forceinline__ Tail take_tail(int4 at, uint32_t b0, uint32_t lo, uint32_t hi)
{
    const int32_t b = (int32_t)b0, n = (int32_t)lo;
    Tail a;
    // what is held of this block from lo on, or of later ones, is written anew
    a.fill0 = at.x == b ? min(at.z, n) : at.z;
    a.fill1 = at.y == b ? min(at.w, n) : at.w;
    a.tag0 = at.x > b || (at.x == b && a.fill0 < n) || (at.x == b && n == 0) ? -1 : at.x;
    a.tag1 = at.y > b || (at.y == b && a.fill1 < n) || (at.y == b && n == 0) ? -1 : at.y;
    a.held = a.tag0 == b || a.tag1 == b;
    a.slot = a.held ? (a.tag0 == b ? 0u : 1u) : (a.tag0 <= a.tag1 ? 0u : 1u);      // else the older one gives way
    if (hi < kBlock) hold(a, b0, hi);
    return a;
}

__device__ __forceinline__ void put_tail(int32_t *at, const Tail &a)
{
    if (threadIdx.x == 0) *(int4 *)at = make_int4(a.tag0, a.tag1, a.fill0, a.fill1);
}

// Block `b`'s positions lo .. hi (of 32) from the rows (load(r, i, d, y): elements
// d = 16 (c + 8 i) .. + 16 of the r-th one, zero from head_dim on), those before
// lo from what the cache holds.  One workgroup of 256: thread (t, c): position t =
// tid / 8, elements 16 (c + 8 i) .. + 16.  FIRST: the call's first block, which
// takes its slot; else a new one (lo = 0) in the slot of `tail`.  All that may be
// needed of the head is asked for before any of it is looked at.
template <int NC, bool FIRST, class Load>
__device__ void write_block(const View &v, Load load, uint64_t base, uint32_t b, uint32_t lo, uint32_t hi, Tail &tail,
                            bool key, uint32_t *maxes, uint32_t *red, uint8_t *stage)
{
    const uint32_t tid = threadIdx.x, t = tid >> 3, c = tid & 7u, dp = v.dp;
    uint8_t *codes = v.codes + (base * v.n_blocks + b) * kBlock * dp;
    float *scale = v.scale + base * v.n_blocks + b;
    uint32_t *maxes_of = v.tail_max + base * 2 * kBlock;
    const bool fresh = t >= lo && t < hi, old = t < lo, open = hi < kBlock;
    float s_old = 0.f;
    uint32_t m0 = 0, m1 = 0;
    int4 at;
    if (FIRST) {
        at = *(const int4 *)(v.tail_at + base * 4);
        s_old = *scale;
        m0 = maxes_of[t];
        m1 = maxes_of[kBlock + t];
    }
    float val[NC][16], top = 0.f;
#pragma unroll
    for (int i = 0; i < NC; i++) {
        const uint32_t d = 16u * (c + 8u * i);
        if (d >= dp) break;
#pragma unroll
        for (int j = 0; j < 16; j++) val[i][j] = 0.f;
        if (fresh) load(t - lo, i, d, val[i]);
    }
    if (FIRST) tail = take_tail(at, b, lo, hi);
    const bool held = FIRST && tail.held;
    float *rows = v.tail + (base * 2 + tail.slot) * kBlock * dp + t * dp;
    uint32_t m;
#pragma unroll
    for (int i = 0; i < NC; i++) {
        const uint32_t d = 16u * (c + 8u * i);
        if (d >= dp) break;
        if (old && !held)              // a block reopened from its codes
            for (uint32_t j = 0; j < 16; j++) {
                const int q = (int)codes[key ? key_at(t, d + j, dp) : value_at(t, d + j)] - kZero;
                val[i][j] = (float)q * s_old;
            }
#pragma unroll
        for (int j = 0; j < 16; j++) top = __builtin_elementwise_maximum(top, fabsf(val[i][j]));    // NaN if any is
    }
    m = __float_as_uint(top) & 0x7FFFFFFFu;
    // a position's largest magnitude, over its eight threads
    m = max(m, (uint32_t)__shfl_xor((int)m, 1, 64));
    m = max(m, (uint32_t)__shfl_xor((int)m, 2, 64));
    m = max(m, (uint32_t)__shfl_xor((int)m, 4, 64));
    if (old && held) m = tail.slot ? m1 : m0;
    if (c == 0) maxes[t] = m;
    m = wave_max_u(m);
    if ((tid & 63u) == 0) red[tid >> 6] = m;
    __syncthreads();
    m = max(max(red[0], red[1]), max(red[2], red[3]));
    const float s = scale_of(m);
    const float inv = s > 0.f ? 1.0f / s : 0.f;              // NaN: no codes
    // the block's codes of the positions before lo stand while the scale does
    const bool again = lo > 0 && (__float_as_uint(s) != __float_as_uint(s_old) || !held);
    if (again && old && held) {
#pragma unroll
        for (int i = 0; i < NC; i++) {
            const uint32_t d = 16u * (c + 8u * i);
            if (d >= dp) break;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float4 a = *(const float4 *)(rows + d + 4 * j);
                val[i][4 * j] = a.x; val[i][4 * j + 1] = a.y; val[i][4 * j + 2] = a.z; val[i][4 * j + 3] = a.w;
            }
        }
    }
    const bool whole = lo == 0 || again;
    const bool put = fresh || (old && again);
#pragma unroll
    for (int i = 0; i < NC; i++) {
        const uint32_t d = 16u * (c + 8u * i);
        if (d >= dp) break;
        union { uint8_t b[16]; uint4 u; } w;
        w.u = make_uint4(kZeros, kZeros, kZeros, kZeros);
        if (s > 0.f && put) w.u = codes_of(val[i], s, inv);
        if (key) {
            if (put) *(uint4 *)(codes + key_at(t, d, dp)) = w.u;
        } else if (whole) {
            *(uint4 *)(stage + t * (dp + 16) + d) = w.u;
        } else if (fresh) {
            for (uint32_t j = 0; j < 16; j++) codes[value_at(t, d + j)] = w.b[j];
        }
        // the f32 values of a block that stays open
        if (open && (fresh || (old && !held)))
#pragma unroll
            for (int j = 0; j < 4; j++)
                *(float4 *)(rows + d + 4 * j) = make_float4(val[i][4 * j], val[i][4 * j + 1], val[i][4 * j + 2],
                                                            val[i][4 * j + 3]);
    }
    if (!key && whole) {
        __syncthreads();
        put_values(stage, codes, dp);
    }
    if (tid == 0) *scale = s;
    if (open && tid < hi && (tid >= lo || !held)) maxes_of[tail.slot * kBlock + tid] = maxes[tid];
    __syncthreads();
}

// A thread's 16 elements of a row as they lie in memory: f16 in two words, else
// as f32.
struct Raw {
    uint4 w[4];
};

__device__ __forceinline__ Raw load_raw(const Rows &x, uint64_t at, uint32_t d, uint32_t hd)
{
    Raw r;
    if (x.vec) {
#pragma unroll
        for (int i = 0; i < 4; i++) r.w[i] = make_uint4(0, 0, 0, 0);
        if (d >= hd) return r;
        const uint4 *p = (const uint4 *)((const char *)x.p + (at + d) * (x.f16 ? 2 : 4));
        r.w[0] = p[0];
        r.w[1] = p[1];
        if (!x.f16) {
            r.w[2] = p[2];
            r.w[3] = p[3];
        }
    } else {
        union { float f[16]; uint4 w[4]; } u;
        load16(x, at, d, hd, u.f);
#pragma unroll
        for (int i = 0; i < 4; i++) r.w[i] = u.w[i];
    }
    return r;
}

__device__ __forceinline__ void floats_of(const Rows &x, const Raw &r, float *y)
{
    typedef _Float16 h8 __attribute__((ext_vector_type(8)));
    if (x.vec && x.f16) {
        const h8 a = __builtin_bit_cast(h8, r.w[0]), b = __builtin_bit_cast(h8, r.w[1]);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            y[i] = (float)a[i];
            y[8 + i] = (float)b[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            y[4 * i] = __uint_as_float(r.w[i].x); y[4 * i + 1] = __uint_as_float(r.w[i].y);
            y[4 * i + 2] = __uint_as_float(r.w[i].z); y[4 * i + 3] = __uint_as_float(r.w[i].w);
        }
    }
}

// `count` whole blocks from b on (rows from element row_at on): nothing of them is
// kept but codes and scales.  The next block's rows are on their way while one is
// worked on.  red: two sets in turn, so that a block of keys takes one barrier.
template <int NC>
__device__ void write_whole(const View &v, const Rows &x, uint64_t row_at, uint64_t base, uint32_t b, uint32_t count, bool key,
                            uint32_t (*red)[4], uint8_t *stage)
{
    const uint32_t tid = threadIdx.x, t = tid >> 3, c = tid & 7u, dp = v.dp;
    uint8_t *codes = v.codes + (base * v.n_blocks + b) * kBlock * dp;
    float *scale = v.scale + base * v.n_blocks + b;
    const uint64_t at = row_at + (uint64_t)t * x.ld_row;
    Raw raw[NC];
#pragma unroll
    for (int i = 0; i < NC; i++)
        if (16u * (c + 8u * i) < dp) raw[i] = load_raw(x, at, 16u * (c + 8u * i), v.hd);
    for (uint32_t k = 0; k < count; k++) {
        float val[NC][16], top = 0.f;
#pragma unroll
        for (int i = 0; i < NC; i++) {
            if (16u * (c + 8u * i) >= dp) break;
            floats_of(x, raw[i], val[i]);
#pragma unroll
            for (int j = 0; j < 16; j++) top = __builtin_elementwise_maximum(top, fabsf(val[i][j]));    // NaN if any is
        }
        if (k + 1 < count)
#pragma unroll
            for (int i = 0; i < NC; i++)
                if (16u * (c + 8u * i) < dp)
                    raw[i] = load_raw(x, at + (uint64_t)(k + 1) * kBlock * x.ld_row, 16u * (c + 8u * i), v.hd);
        uint32_t m = wave_max_u(__float_as_uint(top) & 0x7FFFFFFFu);
        if ((tid & 63u) == 0) red[k & 1u][tid >> 6] = m;
        __syncthreads();
        m = max(max(red[k & 1u][0], red[k & 1u][1]), max(red[k & 1u][2], red[k & 1u][3]));
        const float s = scale_of(m), inv = s > 0.f ? 1.0f / s : 0.f;
#pragma unroll
        for (int i = 0; i < NC; i++) {
            const uint32_t d = 16u * (c + 8u * i);
            if (d >= dp) break;
            const uint4 w = s > 0.f ? codes_of(val[i], s, inv) : make_uint4(kZeros, kZeros, kZeros, kZeros);
            if (key) *(uint4 *)(codes + key_at(t, d, dp)) = w;
            else *(uint4 *)(stage + t * (dp + 16) + d) = w;
        }
        if (!key) {
            __syncthreads();
            put_values(stage, codes, dp);
        }
        if (tid == 0) scale[k] = s;
        codes += kBlock * dp;
    }
}

// Grid: (items, heads, keys / values).  Bound by the latency of a few dependent
// loads where there is little (one token 3.6 us, 1001 tokens of 8 heads of 128 in
// f32 7.5), by the memory and its latency where there is much (32 prompts of up to
// 2048 tokens, 8 heads of 128 in f16, 194 MB: 53 us, 3.7 TB/s).
//
// The scale of a block follows from its largest magnitude, so a new token in a
// block that is partly there costs its own row and 32 remembered magnitudes
// while it is not the largest, and the block's f32 rows (kept in one of two
// slots) when it is.  Two slots, because a call that ends one block and opens
// another must leave the values of the first: the same call may come again.
template <int NC>
__global__ void __launch_bounds__(256, NC == 1 ? 5 : 2) write_k(View v, Batch b, Rows k, Rows val, uint32_t group)
{
    __shared__ uint32_t maxes[kBlock], red[2][4];
    __shared__ __attribute__((aligned(16))) uint8_t stage[kBlock * (128 * NC + 16)];
    uint32_t seq, item;
    Piece p;
    if (!find_item(b, v.n_seqs, v.max_len, group, blockIdx.x, &seq, &item, &p)) return;
    const bool key = blockIdx.z == 0;
    const Rows &x = key ? k : val;
    const uint32_t head = blockIdx.y, sh = seq * v.n_heads + head;
    const uint64_t base = (uint64_t)blockIdx.z * v.n_seqs * v.n_heads + sh;
    // element of the row that holds position pos
    auto row_at = [&](uint32_t pos) {
        return (uint64_t)(p.s.row + (uint32_t)((int64_t)pos - p.s.pos)) * x.ld_row + head * x.ld_head;
    };
    if (item) {
        const uint32_t blk = p.b0 + 1 + (item - 1) * group;
        const uint32_t count = min(group, p.end / kBlock - blk);
        write_whole<NC>(v, x, row_at(blk * kBlock), base, blk, count, key, red, stage);
        return;
    }
    const uint32_t lo = p.first % kBlock, hi = p.bl == p.b0 ? p.end - p.b0 * kBlock : kBlock;
    Tail tail;
    auto rows_from = [&](uint32_t pos) {
        const uint64_t first = row_at(pos);
        return [&, first](uint32_t r, int, uint32_t d, float *y) { load16(x, first + (uint64_t)r * x.ld_row, d, v.hd, y); };
    };
    write_block<NC, true>(v, rows_from(p.first), base, p.b0, lo, hi, tail, key, maxes, red[0], stage);
    if (p.bl > p.b0 && p.end % kBlock) {
        tail.slot = tail.held ? 1 - tail.slot : tail.tag0 <= tail.tag1 ? 0 : 1;
        hold(tail, p.bl, p.end % kBlock);
        write_block<NC, false>(v, rows_from(p.bl * kBlock), base, p.bl, 0, p.end % kBlock, tail, key, maxes, red[0], stage);
    }
    put_tail(v.tail_at + base * 4, tail);
}

// A decode step's projections of one token (Append): q and k with their biases
// rotated, v with its own, k and v written as the token's place of a cache of one
// sequence.  Grid: (1, kv heads, keys / values / the kv head's query heads).
// One launch for what was two (the rotation, then write_k), each a chain of dependent
// loads: 5 to 6 us inside a decode step.
template <int NC> __global__ void __launch_bounds__(256) append_k(View v, Append a)
{
    __shared__ uint32_t maxes[kBlock], red[4];
    __shared__ __attribute__((aligned(16))) uint8_t stage[kBlock * (128 * NC + 16)];
    const uint32_t head = blockIdx.y, hd = v.hd;
    const bool key = blockIdx.z == 0;
    const float *x = (key ? a.k : a.v) + head * hd, *b = (key ? a.bk : a.bv) + head * hd;
    float own[NC][16];                                        // asked for before the position is known
    if (blockIdx.z < 2)
#pragma unroll
        for (int i = 0; i < NC; i++) {
            const uint32_t d = 16u * ((threadIdx.x & 7u) + 8u * i);
#pragma unroll
            for (uint32_t j = 0; j < 16; j++) own[i][j] = d + j < hd ? x[d + j] + b[d + j] : 0.f;
        }
    const uint32_t pos = *a.pos, at = *a.slot;
    const float *cs = a.cos_t + (size_t)pos * (hd / 2), *sn = a.sin_t + (size_t)pos * (hd / 2);
    if (blockIdx.z == 2) {
        for (uint32_t i = 2 * threadIdx.x; i < a.n_rep * hd; i += 512) {
            const uint32_t e = head * a.n_rep * hd + i, j = i % hd / 2;
            const float x0 = a.q[e] + a.bq[e], x1 = a.q[e + 1] + a.bq[e + 1];
            a.q[e] = x0 * cs[j] - x1 * sn[j];
            a.q[e + 1] = x0 * sn[j] + x1 * cs[j];
        }
        if (head == 0 && threadIdx.x == 0) *a.len = at + 1;
        return;
    }
    if (at >= v.max_len) return;
    const uint64_t base = (uint64_t)blockIdx.z * v.n_heads + head;
    const uint32_t lo = at % kBlock;
    Tail tail;
    auto row = [&](uint32_t, int i, uint32_t d, float *y) {
#pragma unroll
        for (uint32_t j = 0; j < 16; j += 2) {
            const bool turn = key && d + j < hd;              // hd is even
            const float x0 = own[i][j], x1 = own[i][j + 1];
            const float c = turn ? cs[(d + j) / 2] : 1.f, s = turn ? sn[(d + j) / 2] : 0.f;
            y[j] = turn ? x0 * c - x1 * s : x0;
            y[j + 1] = turn ? x0 * s + x1 * c : x1;
        }
    };
    write_block<NC, true>(v, row, base, at / kBlock, lo, lo + 1, tail, key, maxes, red, stage);
    put_tail(v.tail_at + base * 4, tail);
}

// Grid: (blocks, heads * keys / values, sequences); 256 threads.  A thread takes 16
// bytes of the cache as they lie: 16 elements of a key, or two elements of eight
// values, which it stores as pairs (16 lanes fill 64 or 128 bytes of a row).
// Bound by the stores where there is much: 71 us for 32 sequences of 2048 tokens
// of 8 heads of 128 in f16, 268 MB written and 134 MB read at 5.7 TB/s (94 with an
// element a store); 2.6 us for one token, a launch.
__global__ void __launch_bounds__(256) read_k(View v, uint32_t seq0, uint32_t pos, uint32_t n, Rows k, Rows val)
{
    const uint32_t blk = pos / kBlock + blockIdx.x, head = blockIdx.y % v.n_heads;
    const bool key = k.p && blockIdx.y < v.n_heads;
    const Rows &x = key ? k : val;
    const uint32_t seq = seq0 + blockIdx.z, dp = v.dp;
    const uint64_t base = (uint64_t)(key ? 0 : 1) * v.n_seqs * v.n_heads + (uint64_t)seq * v.n_heads + head;
    const uint8_t *codes = v.codes + (base * v.n_blocks + blk) * kBlock * dp;
    const float s = v.scale[base * v.n_blocks + blk];
    const uint64_t out = (uint64_t)blockIdx.z * n, p0 = (uint64_t)blk * kBlock;
    auto at = [&](uint32_t t, uint32_t d) {
        return (out + (p0 + t - pos)) * x.ld_row + head * x.ld_head + d;
    };
    for (uint32_t u = threadIdx.x; u < 2 * dp; u += 256) {
        union { uint8_t b[16]; uint4 u; } w;
        w.u = *(const uint4 *)(codes + u * 16u);
        auto val_of = [&](int j) { return (float)((int)w.b[j] - kZero) * s; };
        if (key) {
            // unit u of 16 bytes: position and 16 elements
            const uint32_t t = (u >> 6) / (dp >> 6) * 16u + (u & 15u), d = (u >> 6) % (dp >> 6) * 64u + (u >> 4 & 3u) * 16u;
            if (p0 + t < pos || p0 + t >= (uint64_t)pos + n) continue;
            if (x.vec && d < v.hd) {
                if (x.f16) {
                    union { _Float16 h[16]; uint4 u[2]; } y;
#pragma unroll
                    for (int j = 0; j < 16; j++) y.h[j] = (_Float16)val_of(j);
                    uint4 *o = (uint4 *)((_Float16 *)x.p + at(t, d));
                    o[0] = y.u[0];
                    o[1] = y.u[1];
                } else {
                    float4 *o = (float4 *)((float *)x.p + at(t, d));
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        o[j] = make_float4(val_of(4 * j), val_of(4 * j + 1), val_of(4 * j + 2), val_of(4 * j + 3));
                }
            } else {
                for (uint32_t j = 0; j < 16; j++)
                    if (d + j < v.hd) store1(x, at(t, d + j), val_of((int)j));
            }
        } else {
            const uint32_t g = u >> 4 & 3u, d = (u >> 6) * 32u + 2u * (u & 15u);
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) {
                const uint32_t t = 4u * g + (j & 3u) + (j >> 2) * 16u;
                if (p0 + t < pos || p0 + t >= (uint64_t)pos + n) continue;
                if (x.vec && d < v.hd) {
                    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
                    const float lo = val_of((int)j), hi = val_of(8 + (int)j);
                    if (x.f16) *(h2 *)((_Float16 *)x.p + at(t, d)) = h2{(_Float16)lo, (_Float16)hi};
                    else *(float2 *)((float *)x.p + at(t, d)) = make_float2(lo, hi);
                    continue;
                }
                if (d < v.hd) store1(x, at(t, d), val_of((int)j));
                if (d + 1 < v.hd) store1(x, at(t, d + 1), val_of(8 + (int)j));
            }
        }
    }
}

int launched()
{
    return hipPeekAtLastError() == hipSuccess ? 0 : -1;
}

}  // namespace

int launch_write(const View &v, const Batch &b, const Rows &k, const Rows &x, int n_cu, hipStream_t st)
{
    if (b.n_rows == 0) return 0;
    const uint64_t seqs = b.starts ? std::min(v.n_seqs, b.n_rows) : 1u;
    const bool one = b.lens && !b.starts;                     // one row, one item for each sequence
    // one block a workgroup while all of them are there at once (5 a compute unit
    // fit); else four, each block's rows loaded during the one before (us, 32
    // prompts of up to 2048 tokens: 54 against 66, two 62, eight 56; with 6
    // workgroups a compute unit 68)
    const uint64_t room = 5ull * (uint32_t)(n_cu > 0 ? n_cu : 256);
    const uint32_t group = !one && ((uint64_t)b.n_rows / kBlock + 2 * seqs) * v.n_heads * 2 > room ? 4u : 1u;
    // items of a sequence of n rows: at most n / (32 group) + 2
    const dim3 grid(one ? b.n_rows : (uint32_t)(b.n_rows / (kBlock * group) + 2 * seqs), v.n_heads, 2);
    if (v.dp > 128) hipLaunchKernelGGL((write_k<2>), grid, dim3(256), 0, st, v, b, k, x, group);
    else hipLaunchKernelGGL((write_k<1>), grid, dim3(256), 0, st, v, b, k, x, group);
    return launched();
}

int launch_append(const View &v, const Append &a, hipStream_t st)
{
    const dim3 grid(1, v.n_heads, 3);
    if (v.dp > 128) hipLaunchKernelGGL((append_k<2>), grid, dim3(256), 0, st, v, a);
    else hipLaunchKernelGGL((append_k<1>), grid, dim3(256), 0, st, v, a);
    return launched();
}

int launch_read(const View &v, uint32_t seq, uint32_t n_seqs, uint32_t pos, uint32_t n, const Rows *k, const Rows *x,
                hipStream_t st)
{
    if (n == 0 || n_seqs == 0 || (!k && !x)) return 0;
    const uint32_t blocks = (pos + n - 1) / kBlock - pos / kBlock + 1;
    hipLaunchKernelGGL(read_k, dim3(blocks, v.n_heads * ((k ? 1u : 0u) + (x ? 1u : 0u)), n_seqs), dim3(256), 0, st, v, seq,
                       pos, n, k ? *k : Rows{}, x ? *x : Rows{});
    return launched();
}

}  // namespace qg8

// ------------------------------------------------------------------- C ABI

namespace {

// One of the context's caches.
int check_kv8(qg_ctx *ctx, const qg_kv8 *kv)
{
    if (!ctx || !kv) return qg_fail(ctx, QG_ERR_INVALID_ARG, "ctx or cache is NULL");
    if (!ctx->kv8s.count(const_cast<qg_kv8 *>(kv))) return qg_fail(ctx, QG_ERR_INVALID_ARG, "not a cache of this context");
    return QG_OK;
}

// Rows of a call, positions of a read: a launch counts its threads in 32 bits,
// and 256 of them take 32 positions (and two part blocks of every sequence).
constexpr size_t kMostRows = (size_t)1 << 28;

// a * b + c, below 2^58: addresses in bytes fit
bool fits(size_t a, size_t b, size_t c, size_t *out)
{
    size_t t;
    if (__builtin_mul_overflow(a, b, &t) || __builtin_add_overflow(t, c, &t) || t >> 58) return false;
    *out = t;
    return true;
}

// qg_rows of n rows of `heads` heads of hd elements
int check_rows(qg_ctx *ctx, const qg_rows *r, size_t n, size_t heads, size_t hd, bool written, qg8::Rows *out)
{
    if (!r) return qg_fail(ctx, QG_ERR_INVALID_ARG, "rows are NULL");
    if (r->type != qg::T_F32 && r->type != qg::T_F16)
        return qg_fail(ctx, QG_ERR_UNSUPPORTED_TYPE, "rows are neither f32 nor f16");
    const size_t es = r->type == qg::T_F16 ? 2 : 4;
    if (n && !r->data) return qg_fail(ctx, QG_ERR_INVALID_ARG, "rows without data");
    if ((uintptr_t)r->data % es) return qg_fail(ctx, QG_ERR_INVALID_ARG, "rows not aligned to their elements");
    size_t by_head, all;
    if (!fits(heads - 1, r->ld_head, hd, &by_head) || !fits(n ? n - 1 : 0, r->ld_row, by_head, &all))
        return qg_fail(ctx, QG_ERR_SHAPE, "rows too large");
    if (written && n) {
        size_t by_row;
        const bool heads_in_rows = (heads == 1 || r->ld_head >= hd) && (n == 1 || r->ld_row >= by_head);
        const bool rows_in_heads = fits(n - 1, r->ld_row, hd, &by_row) && (n == 1 || r->ld_row >= hd) &&
                                   (heads == 1 || r->ld_head >= by_row);
        if (!heads_in_rows && !rows_in_heads) return qg_fail(ctx, QG_ERR_SHAPE, "written rows overlap");
    }
    const size_t per = 16 / es;
    out->p = r->data;
    out->ld_row = r->ld_row;
    out->ld_head = r->ld_head;
    out->f16 = r->type == qg::T_F16;
    out->vec = (uintptr_t)r->data % 16 == 0 && r->ld_row % per == 0 && r->ld_head % per == 0 && hd % 16 == 0;
    return QG_OK;
}

int check_batch(qg_ctx *ctx, const qg_kv8 *kv, const qg_batch *b, qg8::Batch *out)
{
    if (!b) return qg_fail(ctx, QG_ERR_INVALID_ARG, "batch is NULL");
    if (b->n_rows >= kMostRows) return qg_fail(ctx, QG_ERR_SHAPE, "too many rows");
    if (!b->d_lens || ((uintptr_t)b->d_lens | (uintptr_t)b->d_starts) % 4)
        return qg_fail(ctx, QG_ERR_INVALID_ARG, "batch lengths missing or not aligned");
    if (!b->d_starts && b->n_rows != kv->v.n_seqs)
        return qg_fail(ctx, QG_ERR_SHAPE, "without starts a batch has one row per sequence");
    *out = qg8::Batch{b->d_starts, b->d_lens, (uint32_t)b->n_rows, 0};
    return QG_OK;
}

hipStream_t pick(qg_ctx *ctx, void *stream)
{
    return stream ? (hipStream_t)stream : ctx->stream;
}

int launch_status(qg_ctx *ctx, int r, const char *what)
{
    return r == 0 ? QG_OK : qg_fail(ctx, QG_ERR_HIP, what, hipGetLastError());
}

}  // namespace

int qg_kv8_make(qg_ctx *ctx, size_t n_seqs, size_t n_kv_heads, size_t head_dim, size_t max_len, qg_kv8 **out)
{
    if (n_seqs < 1 || n_seqs > 65535 || n_kv_heads < 1 || n_kv_heads > 65535 || head_dim < 1 || head_dim > 256 ||
        max_len < 1 || max_len > 0x7FFFFFE0u || n_seqs * n_kv_heads > (size_t)1 << 26)
        return qg_fail(ctx, QG_ERR_SHAPE, "cache sizes");
    qg8::View v{};
    v.n_seqs = (uint32_t)n_seqs;
    v.n_heads = (uint32_t)n_kv_heads;
    v.hd = (uint32_t)head_dim;
    v.dp = (v.hd + 63u) / 64u * 64u;
    v.max_len = (uint32_t)max_len;
    v.n_blocks = (v.max_len + qg8::kBlock - 1) / qg8::kBlock;
    const size_t sh = 2 * n_seqs * n_kv_heads, block = (size_t)qg8::kBlock * v.dp;
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    size_t codes;
    if (!fits(sh * v.n_blocks, block, 0, &codes)) return qg_fail(ctx, QG_ERR_SHAPE, "cache sizes");
    const size_t scale = up(sh * v.n_blocks * 4), tail = up(sh * 2 * block * 4), tmax = up(sh * 2 * qg8::kBlock * 4),
                 at = up(sh * 16);
    const size_t bytes = codes + scale + tail + tmax + at;
    hipError_t e = hipSetDevice(ctx->device);
    if (e != hipSuccess) return qg_fail(ctx, QG_ERR_HIP, "hipSetDevice", e);
    qg_kv8 *kv = new (std::nothrow) qg_kv8;
    if (!kv) return qg_fail(ctx, QG_ERR_OUT_OF_MEMORY, "host allocation");
    kv->ctx = ctx;
    kv->bytes = bytes;
    e = qg_alloc_injected(ctx) ? hipErrorOutOfMemory : hipMalloc(&kv->mem, bytes);
    if (e != hipSuccess) {
        (void)hipGetLastError();
        delete kv;
        return qg_fail(ctx, QG_ERR_OUT_OF_MEMORY, "hipMalloc cache", e);
    }
    uint8_t *p = (uint8_t *)kv->mem;
    v.codes = p;
    v.scale = (float *)(p += codes);
    v.tail = (float *)(p += scale);
    v.tail_max = (uint32_t *)(p += tail);
    v.tail_at = (int32_t *)(p += tmax);
    kv->v = v;
    e = hipMemsetAsync(kv->mem, qg8::kZero, codes, ctx->stream);
    if (e == hipSuccess) e = hipMemsetAsync(v.scale, 0, bytes - at - codes, ctx->stream);
    if (e == hipSuccess) e = hipMemsetAsync(v.tail_at, 0xFF, at, ctx->stream);      // -1: no block
    const hipError_t es = hipStreamSynchronize(ctx->stream);
    if (e == hipSuccess) e = es;
    if (e != hipSuccess) {
        qg_kv8_drop(kv);
        return qg_fail(ctx, QG_ERR_HIP, "clearing the cache", e);
    }
    *out = kv;
    return QG_OK;
}

void qg_kv8_drop(qg_kv8 *kv)
{
    if (!kv) return;
    if (kv->mem) (void)hipFree(kv->mem);
    delete kv;
}

void qg_kv8_free_all(qg_ctx *ctx)
{
    for (qg_kv8 *kv : ctx->kv8s) qg_kv8_drop(kv);
    ctx->kv8s.clear();
}

extern "C" {

int qg_kv8_create(qg_ctx *ctx, size_t n_seqs, size_t n_kv_heads, size_t head_dim, size_t max_len, qg_kv8 **out)
{
    if (!ctx || !out) return qg_fail(ctx, QG_ERR_INVALID_ARG, "ctx or out is NULL");
    *out = nullptr;
    qg_kv8 *kv = nullptr;
    const int rc = qg_kv8_make(ctx, n_seqs, n_kv_heads, head_dim, max_len, &kv);
    if (rc) return rc;
    try {
        ctx->kv8s.insert(kv);
    } catch (...) {
        qg_kv8_drop(kv);
        return qg_fail(ctx, QG_ERR_OUT_OF_MEMORY, "host allocation");
    }
    *out = kv;
    return QG_OK;
}

int qg_kv8_free(qg_ctx *ctx, qg_kv8 *kv)
{
    const int rc = check_kv8(ctx, kv);
    if (rc) return rc;
    (void)hipSetDevice(ctx->device);
    (void)hipStreamSynchronize(ctx->stream);
    ctx->kv8s.erase(kv);
    qg_kv8_drop(kv);
    return QG_OK;
}

int qg_kv8_info(const qg_kv8 *kv, size_t *n_seqs, size_t *n_kv_heads, size_t *head_dim, size_t *max_len, size_t *bytes)
{
    if (!kv) return QG_ERR_INVALID_ARG;
    if (n_seqs) *n_seqs = kv->v.n_seqs;
    if (n_kv_heads) *n_kv_heads = kv->v.n_heads;
    if (head_dim) *head_dim = kv->v.hd;
    if (max_len) *max_len = kv->v.max_len;
    if (bytes) *bytes = kv->bytes;
    return QG_OK;
}

int qg_kv8_write_dev(qg_ctx *ctx, qg_kv8 *kv, const qg_batch *batch, const qg_rows *k, const qg_rows *v, void *stream)
{
    int rc = check_kv8(ctx, kv);
    qg8::Batch b{};
    qg8::Rows rk{}, rv{};
    if (rc || (rc = check_batch(ctx, kv, batch, &b)) ||
        (rc = check_rows(ctx, k, b.n_rows, kv->v.n_heads, kv->v.hd, false, &rk)) ||
        (rc = check_rows(ctx, v, b.n_rows, kv->v.n_heads, kv->v.hd, false, &rv)))
        return rc;
    if (rk.f16 != rv.f16) return qg_fail(ctx, QG_ERR_UNSUPPORTED_TYPE, "k and v of two types");
    if (b.n_rows == 0) return QG_OK;
    const hipError_t e = hipSetDevice(ctx->device);
    if (e != hipSuccess) return qg_fail(ctx, QG_ERR_HIP, "hipSetDevice", e);
    return launch_status(ctx, qg8::launch_write(kv->v, b, rk, rv, ctx->n_cu, pick(ctx, stream)), "cache write");
}

int qg_kv8_read_dev(qg_ctx *ctx, const qg_kv8 *kv, size_t seq, size_t n_seqs, size_t pos, size_t n, const qg_rows *k,
                    const qg_rows *v, void *stream)
{
    int rc = check_kv8(ctx, kv);
    if (rc) return rc;
    const qg8::View &c = kv->v;
    if (seq > c.n_seqs || n_seqs > c.n_seqs - seq || pos > c.max_len || n > c.max_len - pos ||
        n >= kMostRows)
        return qg_fail(ctx, QG_ERR_SHAPE, "positions outside the cache, or too many");
    qg8::Rows rk{}, rv{};
    if ((k && (rc = check_rows(ctx, k, n_seqs * n, c.n_heads, c.hd, true, &rk))) ||
        (v && (rc = check_rows(ctx, v, n_seqs * n, c.n_heads, c.hd, true, &rv))))
        return rc;
    if (n == 0 || n_seqs == 0 || (!k && !v)) return QG_OK;
    if (c.n_heads * 2ull > 65535) return qg_fail(ctx, QG_ERR_SHAPE, "too many heads to read at once");
    const hipError_t e = hipSetDevice(ctx->device);
    if (e != hipSuccess) return qg_fail(ctx, QG_ERR_HIP, "hipSetDevice", e);
    return launch_status(ctx, qg8::launch_read(c, (uint32_t)seq, (uint32_t)n_seqs, (uint32_t)pos, (uint32_t)n,
                                               k ? &rk : nullptr, v ? &rv : nullptr, pick(ctx, stream)), "cache read");
}

int qg_kv8_attention_work(qg_ctx *ctx, const qg_kv8 *kv, size_t n_rows, size_t n_heads, size_t *bytes)
{
    const int rc = check_kv8(ctx, kv);
    if (rc) return rc;
    if (!bytes) return qg_fail(ctx, QG_ERR_INVALID_ARG, "bytes is NULL");
    if (n_heads == 0 || n_heads % kv->v.n_heads || n_heads > 65535 || n_rows >= kMostRows ||
        n_rows * n_heads > 0x7FFFFFFFu)
        return qg_fail(ctx, QG_ERR_SHAPE, "rows or heads");
    *bytes = qg8::attention_work(kv->v, n_rows, n_heads, ctx->n_cu);
    return QG_OK;
}

int qg_kv8_attention_dev(qg_ctx *ctx, const qg_kv8 *kv, const qg_batch *batch, size_t n_heads, const qg_rows *q,
                         float scale, size_t window, const qg_rows *out, void *d_work, size_t work_bytes, void *stream)
{
    int rc = check_kv8(ctx, kv);
    if (rc) return rc;
    if (n_heads == 0 || n_heads % kv->v.n_heads || n_heads > 65535)
        return qg_fail(ctx, QG_ERR_SHAPE, "query heads are no multiple of the cache's heads");
    qg8::Batch b{};
    qg8::Rows rq{}, ro{};
    if ((rc = check_batch(ctx, kv, batch, &b)) || (rc = check_rows(ctx, q, b.n_rows, n_heads, kv->v.hd, false, &rq)) ||
        (rc = check_rows(ctx, out, b.n_rows, n_heads, kv->v.hd, true, &ro)))
        return rc;
    if (b.n_rows * n_heads > 0x7FFFFFFFu) return qg_fail(ctx, QG_ERR_SHAPE, "too many rows");
    if (rq.f16 != ro.f16) return qg_fail(ctx, QG_ERR_UNSUPPORTED_TYPE, "q and out of two types");
    if (b.n_rows == 0) return QG_OK;
    const size_t need = qg8::attention_work(kv->v, b.n_rows, n_heads, ctx->n_cu);
    if (need > work_bytes) return qg_fail(ctx, QG_ERR_SHAPE, "workspace too small");
    if (need && (!d_work || (uintptr_t)d_work % 16))
        return qg_fail(ctx, QG_ERR_INVALID_ARG, "workspace missing or not 16-byte aligned");
    const hipError_t e = hipSetDevice(ctx->device);
    if (e != hipSuccess) return qg_fail(ctx, QG_ERR_HIP, "hipSetDevice", e);
    // no row stands at 2^32 or above: a wider window hides nothing
    const uint32_t win = window > 0xFFFFFFFFull ? 0u : (uint32_t)window;
    return launch_status(ctx, qg8::launch_attention(kv->v, b, (uint32_t)n_heads, rq, scale, win, ro, d_work, ctx->n_cu,
                                                    pick(ctx, stream)), "attention");
}

}  // extern "C"
