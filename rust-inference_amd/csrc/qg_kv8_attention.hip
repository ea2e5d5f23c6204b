// qg_kv8_attention.hip -- attention over the 8-bit KV cache (include/qgops.h).
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = 2^(s_j - m),  s_j = scale log2(e) q . k_j,
//   k_j = ks c_j, v_j = vs d_j: codes c, d under the scales of j's block.
//
// One pass over the positions with a running reference m of every row.  The
// products run on v_mfma_f32_16x16x32_f16: the codes are exact in f16, and q, p
// are f16 pieces (one for f16 rows, hi + lo for f32 rows: 22 bits).  Both
// products are taken transposed, S^T = K Q^T and O^T = V^T P^T, so that a lane
// holds one row's scores (column l % 16 of S^T) in the places in which the second
// product wants them (its B operand), and row statistics need no broadcast; the
// cache is laid out so that a lane's 16-byte load is the A operand of two
// products of either kind (qg_kv8.h).
//
//   * q is scaled by a power of two per row (largest magnitude into [1024,
//     2048)), its sign by that of `scale`; s = f acc with one factor f >= 0 per row
//     and block.
//   * m moves only when a score passes it by more than kLift (then the row's sums
//     are rescaled): no cross-lane step otherwise.  p = 2^(s - m + kBias) lies as
//     high in f16's range as it can, for the low pieces' bits.
//   * vs goes into p as a ratio to a running reference scale that moves only when
//     the ratio leaves 2^-6 .. 2, so the accumulators are not touched per block.
//   * masked positions: a score of -inf, p = 0 whatever their codes; a block with a
//     NaN scale reaches the rows that see a position of it.
//
// Rows are (token, query head) pairs of one kv head: pair r of a sequence is token
// r / n_rep, head r % n_rep (the callers keep n_rows * n_heads below 2^31, and the
// cache's sequences * heads within 2^26).  Tiles of pairs of one sequence and kv
// head are the items; an item's work is its visible blocks in chunks of a few.  All items'
// chunks, end to end, are dealt out evenly to the workgroups (about two per
// compute unit) whatever the sequences' lengths; a workgroup's share may end
// inside an item, then the parts' (m, sum, unnormalised output) go to the
// workspace and merge_k joins them.
#include "qg_kv8.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace qg8 {
namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));

constexpr float kBias = 12.f, kLift = 2.f;   // 2^(12 + 2) times a ratio of 2: f16's largest power
constexpr float kLow = -3.0e38f;              // below any score
constexpr uint32_t kNone = 0xFFFFFFFFu;

// Where a workgroup's share begins inside an item: the item and the workgroups
// that have its first and last part.
struct Split {
    uint32_t first, last, seq, head, tile, pad[3];
};

struct Work {
    Split *split;      // [workgroup]
    float *ml;         // [workgroup][2][kM][2]
    float *part;       // [workgroup][2][kM][dp]
};

// The blocks that a tile of pairs sees, and its chunks (one at least: rows
// that see nothing are written too).
struct Tile {
    uint32_t blk0, blocks, chunks;
};

struct Problem {
    View v;
    Batch b;
    Rows q, out;
    uint32_t n_rep, rep_mul, rep_shift;    // x / n_rep = (mulhi(x, rep_mul) + x) >> rep_shift for x < 2^31
    uint32_t window;
    uint32_t chunk, lead;                  // blocks that are dealt out together; see width
    float scale2;      // |scale| log2(e)
    float sign;
    Work w;
};

__device__ __forceinline__ uint32_t over_rep(const Problem &a, uint32_t x)
{
    return (__umulhi(x, a.rep_mul) + x) >> a.rep_shift;
}

// First position and one past the last that the token at position p sees.
__device__ __forceinline__ void sight(const Problem &a, const Span &s, int64_t p, int64_t *lo, int64_t *hi)
{
    const int64_t len = min(s.len, a.v.max_len);
    *hi = p + 1 < len ? p + 1 : len;
    *lo = a.window && p + 1 > (int64_t)a.window ? p + 1 - (int64_t)a.window : 0;
}

template <uint32_t M> __device__ __forceinline__ uint32_t tiles_of(const Problem &a, const Span &s)
{
    return (s.n * a.n_rep + M - 1) / M;
}

template <uint32_t M> __device__ __forceinline__ Tile tile_of(const Problem &a, const Span &s, uint32_t t)
{
    const uint32_t r0 = t * M, r1 = min(r0 + M, s.n * a.n_rep) - 1;
    int64_t lo, hi, x, y;
    sight(a, s, s.pos + (int64_t)over_rep(a, r0), &lo, &x);
    sight(a, s, s.pos + (int64_t)over_rep(a, r1), &y, &hi);
    Tile k;
    k.blk0 = 0;
    k.blocks = 0;
    if (hi > lo) {
        k.blk0 = (uint32_t)(lo / kBlock);
        k.blocks = (uint32_t)((hi - 1) / kBlock) - k.blk0 + 1;
    }
    k.chunks = max(1u, (k.blocks + a.chunk - 1) / a.chunk);
    return k;
}

// Lane l's sequence, to all.
__device__ __forceinline__ Span span_at(const Span &s, uint32_t l)
{
    Span r;
    r.row = (uint32_t)__builtin_amdgcn_readlane((int)s.row, (int)l);
    r.n = (uint32_t)__builtin_amdgcn_readlane((int)s.n, (int)l);
    r.len = (uint32_t)__builtin_amdgcn_readlane((int)s.len, (int)l);
    r.pos = (int64_t)r.len - (int64_t)r.n;
    return r;
}

// Sums over the lanes up to each (DPP: shifts within the rows of 16, then the
// rows' last lanes to the rows behind them), and the last one's.
template <int CTRL, int ROWS = 0xF> __device__ __forceinline__ uint32_t dpp0(uint32_t v)
{
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ uint32_t scan64(uint32_t v)
{
    v += dpp0<0x111>(v);
    v += dpp0<0x112>(v);
    v += dpp0<0x114>(v);
    v += dpp0<0x118>(v);
    v += dpp0<0x142, 0xA>(v);
    v += dpp0<0x143, 0xC>(v);
    return v;
}
__device__ __forceinline__ uint32_t lane_of(uint32_t v, uint32_t l)
{
    return (uint32_t)__builtin_amdgcn_readlane((int)v, (int)l);
}

// What an item takes of the order: its chunks, and `lead` places before them
// that stand for what every item costs whatever its length (its rows' way in and
// out).
__device__ __forceinline__ uint32_t width(const Problem &a, const Tile &t) { return t.chunks + a.lead; }

// Places of all tiles of a sequence (one kv head), by the whole wave.
template <uint32_t M> __device__ uint32_t seq_places(const Problem &a, const Span &s)
{
    const uint32_t n = tiles_of<M>(a, s), lane = threadIdx.x & 63u;
    uint32_t c = 0;
    for (uint32_t t = lane; t < n; t += 64) c += width(a, tile_of<M>(a, s, t));
    return lane_of(scan64(c), 63);
}

// Places of 64 sequences from s0 on, a sequence per lane, all kv heads; and the
// lanes' sequences.
template <uint32_t M> __device__ uint32_t lane_places(const Problem &a, uint32_t s0, Span *own)
{
    const uint32_t lane = threadIdx.x & 63u, s = s0 + lane;
    uint32_t n = 0, c = 0;
    *own = Span{};
    if (s < a.v.n_seqs) {
        *own = span_of(a.b, s);
        n = tiles_of<M>(a, *own);
        if (n == 1) c = width(a, tile_of<M>(a, *own, 0));
    }
    uint64_t many = __ballot(n > 1);
    while (many) {
        const uint32_t l = (uint32_t)__ffsll((unsigned long long)many) - 1;
        many &= many - 1;
        const uint32_t t = seq_places<M>(a, span_at(*own, l));
        if (lane == l) c = t;
    }
    return c * a.v.n_heads;
}

// The order: its length, the running sums and the sequences of the first 64.
struct Order {
    uint32_t total, first;
    Span own;
};

template <uint32_t M> __device__ Order order_of(const Problem &a)
{
    Order o;
    o.total = 0;
    for (uint32_t s0 = 0; s0 < a.v.n_seqs; s0 += 64) {
        Span own;
        const uint32_t c = scan64(lane_places<M>(a, s0, &own));
        if (s0 == 0) {
            o.first = c;
            o.own = own;
        }
        o.total += lane_of(c, 63);
    }
    return o;
}

struct Item {
    uint32_t seq, head, tile, tiles;
    uint32_t start;                     // place of its first chunk
    uint32_t s0, before;                // its 64 sequences' first, and the places before them
    Tile t;
    Span s;
};

// The item that holds place `at` (less than the total); `before` places lie
// before the sequences from s0 on, a multiple of 64, and `at` is none of them.
template <uint32_t M>
__device__ Item find(const Problem &a, uint32_t at, const Order &o, uint32_t s0 = 0, uint32_t before = 0)
{
    const uint32_t lane = threadIdx.x & 63u;
    Item it{};
    for (; s0 < a.v.n_seqs; s0 += 64) {
        Span own = o.own;
        const uint32_t c = s0 == 0 ? o.first : scan64(lane_places<M>(a, s0, &own));
        const uint64_t past = __ballot(before + c > at);
        if (!past) {
            before += lane_of(c, 63);
            continue;
        }
        const uint32_t l = (uint32_t)__ffsll((unsigned long long)past) - 1;
        const uint32_t up_to = lane_of(c, l), below = l ? lane_of(c, l - 1) : 0u;
        it.seq = s0 + l;
        it.s0 = s0;
        it.before = before;
        it.s = span_at(own, l);
        before += below;
        const uint32_t per_head = (up_to - below) / a.v.n_heads;
        it.head = (at - before) / per_head;
        before += it.head * per_head;
        it.tiles = tiles_of<M>(a, it.s);
        for (uint32_t t0 = 0; t0 < it.tiles; t0 += 64) {
            const uint32_t d = it.tiles == 1 ? per_head
                               : scan64(t0 + lane < it.tiles ? width(a, tile_of<M>(a, it.s, t0 + lane)) : 0u);
            const uint64_t in = __ballot(before + d > at);
            if (!in) {
                before += lane_of(d, 63);
                continue;
            }
            const uint32_t k = (uint32_t)__ffsll((unsigned long long)in) - 1;
            it.tile = t0 + k;
            it.start = before + (k ? lane_of(d, k - 1) : 0u) + a.lead;
            it.t = tile_of<M>(a, it.s, it.tile);
            return it;
        }
        return it;
    }
    return it;
}

// The item behind `it`: the next tile, else the next head, else the next sequence.
template <uint32_t M> __device__ void advance(const Problem &a, Item &it, const Order &o)
{
    const uint32_t end = it.start + it.t.chunks;
    if (it.tile + 1 < it.tiles) {
        it.tile++;
    } else if (it.head + 1 < a.v.n_heads) {
        it.head++;
        it.tile = 0;
    } else {
        it = find<M>(a, end, o, it.s0, it.before);
        return;
    }
    it.start = end + a.lead;
    it.t = tile_of<M>(a, it.s, it.tile);
}

// Eight codes (bytes code + 128) as f16: 1024 + byte by its bits, less 1152.
__device__ __forceinline__ h8 halves(uint32_t a, uint32_t b)
{
    const h2 bias = {(_Float16)1152.f, (_Float16)1152.f};
    union { h2 p[4]; h8 v; } r;
    r.p[0] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u)) - bias;
    r.p[1] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u)) - bias;
    r.p[2] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u)) - bias;
    r.p[3] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)) - bias;
    return r.v;
}

__device__ __forceinline__ v4f mfma(h8 a, h8 b, v4f c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// A row's q in the B operand's layout: lane (r, g) holds elements 64 c + 16 g ..
// + 16, the first eight for product 2 c, the others for 2 c + 1.
template <int DP, int NP> struct QFrag {
    h8 h[NP][DP / 32];
    float f;                  // s = f * (key scale) * acc
};

// x: the lane's elements 64 c' + 16 g + 4 c'' .. + 4 at 4 c' + c''
template <int DP, int NP> __device__ __forceinline__ void load_q(const Problem &a, const float4 *x, QFrag<DP, NP> &q)
{
    uint32_t m = 0;
#pragma unroll
    for (int c = 0; c < DP / 16; c++) {
        m = max(max(m, __float_as_uint(x[c].x) & 0x7FFFFFFFu), __float_as_uint(x[c].y) & 0x7FFFFFFFu);
        m = max(max(m, __float_as_uint(x[c].z) & 0x7FFFFFFFu), __float_as_uint(x[c].w) & 0x7FFFFFFFu);
    }
    m = max(m, (uint32_t)__shfl_xor((int)m, 16, 64));
    m = max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
    // largest magnitude into [1024, 2048): 2^up, within what keeps 2^-up and q 2^up normal
    const bool bad = m >= 0x7F800000u;
    const int up = bad ? 0 : min(137 - (int)(m >> 23), 110);
    const float s = ldexpf(a.sign, up);
    q.f = bad ? __uint_as_float(0x7FC00000u) : ldexpf(a.scale2, -up);
#pragma unroll
    for (int c = 0; c < DP / 16; c++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float y = bad ? 0.f : (j == 0 ? x[c].x : j == 1 ? x[c].y : j == 2 ? x[c].z : x[c].w) * s;
            const _Float16 hi = (_Float16)y;
            q.h[0][c / 2][c % 2 * 4 + j] = hi;
            if (NP == 2) q.h[NP - 1][c / 2][c % 2 * 4 + j] = (_Float16)(y - (float)hi);
        }
}

// A wave's running state for 16 rows: lane (r, g) holds row r's reference, the
// sum over its own positions, and elements of the output.
template <int DP> struct State {
    v4f o[DP / 16];
    float m, l;
};

// The scale of values that o is held in (0: none yet) and its inverse; the same
// in all lanes.
struct Ref {
    float ref, inv;
};

// Keeps the largest of the next blocks' scales within 2^-6 .. 2 of the reference;
// o is rescaled where it is not.
template <int DP, int NT> __device__ __forceinline__ void refer(float vs, Ref &r, State<DP> *st)
{
    const float q = vs * r.inv;
    if ((q <= 2.f && q >= 0x1p-6f) || !(vs > 0.f)) return;
    const float next = r.ref > 0.f ? fmaxf(vs, r.ref * 0x1p-60f) : vs, k = r.ref / next;
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int i = 0; i < DP / 16; i++) st[t].o[i] *= k;
    r.ref = next;
    r.inv = 1.f / next;
}

// vs / ref as a power of two, and inverted.  A scale of 0 (all codes zero) or NaN
// (see mask) counts as 1; one that is nothing beside the reference as 2^-100,
// which f16 does not hold either.
__device__ __forceinline__ void ratio_of(float vs, const Ref &r, float *log, float *inv)
{
    const float q = vs > 0.f ? fmaxf(vs * r.inv, 0x1p-100f) : 1.f;
    *log = __builtin_amdgcn_logf(q);
    *inv = __builtin_amdgcn_rcpf(q);
}

// Which of a block's positions 4 g + i and 16 + 4 g + i a row sees that sees lo
// .. hi of it: bit 4 k + i.
__device__ __forceinline__ uint32_t seen_of(int32_t lo, int32_t hi, uint32_t g)
{
    uint32_t s = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int32_t at = (int32_t)(16 * (j / 4) + 4 * g) + j % 4;
        s |= at >= lo && at < hi ? 1u << j : 0u;
    }
    return s;
}

// Largest of a lane's eight scores; NaN if one is (the row is then NaN whatever
// its reference).  maximum, not fmaxf: one instruction for three values, which
// need not be made quiet first.
__device__ __forceinline__ float top_of(const v4f *x)
{
    auto top = [](float a, float b, float c) { return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c); };
    return top(top(x[0][0], x[0][1], x[0][2]), top(x[0][3], x[1][0], x[1][1]), __builtin_elementwise_maximum(x[1][2], x[1][3]));
}

// Moves the rows' references up where `top` (a lane's largest score) is past them.
template <int DP> __device__ __forceinline__ void lift(float top, State<DP> &st)
{
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float m = fmaxf(st.m, top), k = exp2_(st.m - m);
    st.m = m;
    st.l *= k;
#pragma unroll
    for (int i = 0; i < DP / 16; i++) st.o[i] *= k;
}

// The factor of a row's scores of a block; never 0, so that a masked score of
// -inf stays one (NaN for a row of q that is not finite).
__device__ __forceinline__ float factor(float ks, float f)
{
    const float x = ks * f;
    return x < 0x1p-126f ? 0x1p-126f : x;
}

// Scores of positions outside lo .. hi of a block to -inf.  A block whose scale
// is not a number makes the sum of every row that sees of it NaN, and is then as
// if masked for all (its scales become 1).
__device__ __forceinline__ void mask(v4f *x, int32_t lo, int32_t hi, uint32_t g, bool nan, float &l)
{
    const uint32_t seen = seen_of(lo, hi, g);
#pragma unroll
    for (int j = 0; j < 8; j++) x[j / 4][j % 4] = !nan && (seen >> j & 1u) ? x[j / 4][j % 4] : -INFINITY;
    if (nan && seen) l = __uint_as_float(0x7FC00000u);
}

// Weights of a block's scores: w_j = 2^(f x_j + c), kBias above the row's reference
// (c = kBias - m + log2 of the block's value ratio), as f16 pieces p.  Two at a
// time, so that they can be spread between products.
template <int NP> __device__ __forceinline__ float weigh2(float x, float y, float f, float c, int j, h8 *p)
{
    const float a = exp2_(__builtin_fmaf(x, f, c)), b = exp2_(__builtin_fmaf(y, f, c));
    if (NP == 1) {
        p[0][j] = (_Float16)a;
        p[0][j + 1] = (_Float16)b;
    } else {
        // the high piece by one instruction of its own, so that the low piece is
        // the rest of that very value
        const h2 h = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(a, b));
        p[0][j] = h[0];
        p[0][j + 1] = h[1];
        p[NP - 1][j] = (_Float16)(a - (float)h[0]);
        p[NP - 1][j + 1] = (_Float16)(b - (float)h[1]);
    }
    return a + b;
}

// What rows see of the blocks from position `base` on, in 32 bits: a row's lo ..
// hi there.
__device__ __forceinline__ int32_t from(int64_t p, int64_t base)
{
    return (int32_t)max((int64_t)0, min(p - base, (int64_t)0x40000000));
}

// Row r of a tile of M pairs: its row of q and out, and its positions.
struct Row {
    bool valid;
    uint64_t row;
    uint32_t head;
    int64_t lo, hi;
};

template <uint32_t M> __device__ __forceinline__ Row row_of(const Problem &a, const Span &s, uint32_t head, uint32_t tile, uint32_t r)
{
    Row w;
    const uint32_t pair = tile * M + r;
    w.valid = pair < s.n * a.n_rep;
    const uint32_t i = w.valid ? over_rep(a, pair) : 0;
    w.row = s.row + i;
    w.head = w.valid ? head * a.n_rep + (pair - i * a.n_rep) : 0;
    sight(a, s, s.pos + (int64_t)i, &w.lo, &w.hi);
    if (!w.valid) {                              // masks nothing, and is not stored
        w.lo = 0;
        w.hi = INT64_MAX;
    }
    return w;
}

// Elements d .. d + 4 of a row (d a multiple of 4).
__device__ __forceinline__ void store4v(const Rows &r, uint64_t at, uint32_t d, uint32_t hd, float4 x)
{
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    if (d >= hd) return;
    if (r.f16) *(h4 *)((_Float16 *)r.p + at + d) = h4{(_Float16)x.x, (_Float16)x.y, (_Float16)x.z, (_Float16)x.w};
    else *(float4 *)((float *)r.p + at + d) = x;
}
__device__ __forceinline__ void store4(const Rows &r, uint64_t at, uint32_t d, uint32_t hd, float4 x)
{
    if (r.vec) {
        store4v(r, at, d, hd, x);
        return;
    }
    if (d < hd) store1(r, at + d, x.x);
    if (d + 1 < hd) store1(r, at + d + 1, x.y);
    if (d + 2 < hd) store1(r, at + d + 2, x.z);
    if (d + 3 < hd) store1(r, at + d + 3, x.w);
}

// What a wave's lanes have written to LDS is there for its other lanes.
__device__ __forceinline__ void wave_sync()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// A wave's 16 rows r0 .. of a tile's q (`row` the lane's) as load_q takes them:
// straight from memory, or, where the rows take no 16-byte accesses, element by
// element through LDS (rows of DP + 4 floats at `to`).
template <uint32_t M, int DP>
__device__ __forceinline__ void take_q(const Problem &a, const Item &it, uint32_t r0, const Row &row, float *to, float4 *x)
{
    const uint32_t lane = threadIdx.x & 63u, r = lane & 15u, g = lane >> 4;
    if (a.q.vec) {
        const uint64_t at = row.row * a.q.ld_row + row.head * a.q.ld_head;
#pragma unroll
        for (int c = 0; c < DP / 16; c++) x[c] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (!row.valid) return;
        if (a.q.f16) {
#pragma unroll
            for (int c = 0; c < DP / 16; c += 2) {
                const uint32_t d = 64 * (c / 4) + 16 * g + 4 * (c % 4);
                if (d >= a.v.hd) continue;
                const h8 h = *(const h8 *)((const _Float16 *)a.q.p + at + d);
                x[c] = make_float4((float)h[0], (float)h[1], (float)h[2], (float)h[3]);
                x[c + 1] = make_float4((float)h[4], (float)h[5], (float)h[6], (float)h[7]);
            }
        } else {
#pragma unroll
            for (int c = 0; c < DP / 16; c++) {
                const uint32_t d = 64 * (c / 4) + 16 * g + 4 * (c % 4);
                if (d < a.v.hd) x[c] = *(const float4 *)((const float *)a.q.p + at + d);
            }
        }
        return;
    }
#pragma unroll 1
    for (uint32_t u = lane; u < 16u * DP; u += 64) {
        const uint32_t k = u / DP, d = u % DP;
        const Row w = row_of<M>(a, it.s, it.head, it.tile, r0 + k);
        to[k * (DP + 4) + d] = w.valid && d < a.v.hd ? load1(a.q, w.row * a.q.ld_row + w.head * a.q.ld_head + d) : 0.f;
    }
    wave_sync();
#pragma unroll
    for (int c = 0; c < DP / 16; c++) x[c] = *(const float4 *)(to + r * (DP + 4) + 64 * (c / 4) + 16 * g + 4 * (c % 4));
    wave_sync();
}

// cut: a workgroup's share begins inside `it`.  (Not a pointer to an item or none:
// the item would have to lie in memory, and every use of it read it from there.)
__device__ __forceinline__ void put_split(const Problem &a, uint32_t wg, bool cut, const Item &it, uint32_t per)
{
    if (threadIdx.x) return;
    Split s{};
    s.first = cut ? it.start / per : kNone;
    s.last = (it.start + it.t.chunks - 1) / per;
    s.seq = it.seq;
    s.head = it.head;
    s.tile = it.tile;
    a.w.split[wg] = s;
}

// Workgroup id -> place in the order of the chunks: ids go round the 8 XCDs, and
// neighbours in the order (the same keys and values) belong on one.
__device__ __forceinline__ uint32_t place_of(uint32_t id, uint32_t n)
{
    const uint32_t each = n / 8;
    return id < each * 8 ? (id % 8) * each + id / 8 : id;
}

// Few rows: tiles of 16 pairs.  The four waves take an item's blocks in turn, each
// with all 16 rows and operands straight from the cache (the next block's 64 dp
// bytes are requested before a block is used); their sums are joined in LDS.  A
// part's fixed cost (its rows, the first loads, the join) hides behind the next
// part's loads, which are requested before the join.
//
// Bound by the read of the cache where it is long: 64 sequences of up to 8192
// tokens, 8 kv heads of 128, f16 rows 107 us (the 0.55 GB of codes at 5.2 TB/s; a
// large copy does 5.0), one of 131072 tokens 45 (6 TB/s, half of it from the last
// level cache).  Short ones are a chain of latencies: lengths, codes, products,
// join, 5.9 us at 49 tokens, 9.5 at 2256 (four kv heads of 18 parts each).  Two workgroups a compute unit; three (with half
// the registers) were slower, and so were parts of 8 or 16 blocks.
constexpr uint32_t kFewM = 16;

template <int DP, int NP> __global__ void __launch_bounds__(256, DP <= 128 ? 2 : 1) few_k(Problem a)
{
    constexpr int NK = DP / 32, NV = DP / 32;             // 16-byte loads of a lane per block
    constexpr int LD = DP + 4;
    __shared__ __attribute__((aligned(16))) float so[4][16][LD], sm[4][16], sl[4][16];
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63u, r = lane & 15u, g = lane >> 4;
    const uint32_t wg = place_of(blockIdx.x, gridDim.x);
    const Order order = order_of<kFewM>(a);
    const uint32_t per = max((order.total + gridDim.x - 1) / gridDim.x, 1u);
    uint32_t at = wg * per;
    const uint32_t end = min(at + per, order.total);
    if (at >= end) {
        put_split(a, wg, false, Item{}, per);
        return;
    }
    Item it = find<kFewM>(a, at, order);
    put_split(a, wg, at > it.start, it, per);
    if (it.start >= end) return;                             // only its lead is here
    const uint64_t all = (uint64_t)a.v.n_seqs * a.v.n_heads;
    const uint8_t *kb, *vb;
    const float *ks, *vs;
    uint32_t c0, nc, blk0, last, blk;
    uint4 k[NK], v[NV];
    float ksc = 0.f, vsc = 0.f;
    Row row;
    float4 qx[DP / 16];
    auto fetch_k = [&](uint32_t b) {
        const uint64_t off = (uint64_t)b * (kBlock * DP);
#pragma unroll
        for (int i = 0; i < NK; i++) k[i] = *(const uint4 *)(kb + off + i * 1024);
        ksc = ks[b];
    };
    auto fetch_v = [&](uint32_t b) {
        const uint64_t off = (uint64_t)b * (kBlock * DP);
#pragma unroll
        for (int i = 0; i < NV; i++) v[i] = *(const uint4 *)(vb + off + i * 1024);
        vsc = vs[b];
    };
    // the part of `it` that is here, and its first loads
    auto begin = [&]() {
        c0 = at > it.start ? at - it.start : 0u;
        nc = min(it.t.chunks, end - it.start) - c0;
        const uint64_t sh = (uint64_t)it.seq * a.v.n_heads + it.head;
        kb = a.v.codes + sh * a.v.n_blocks * (kBlock * DP) + lane * 16u;
        vb = a.v.codes + (all + sh) * a.v.n_blocks * (kBlock * DP) + lane * 16u;
        ks = a.v.scale + sh * a.v.n_blocks;
        vs = a.v.scale + (all + sh) * a.v.n_blocks;
        last = it.t.blk0 + min(it.t.blocks, (c0 + nc) * a.chunk);
        blk0 = it.t.blk0 + c0 * a.chunk;
        blk = blk0 + wave;
        row = row_of<kFewM>(a, it.s, it.head, it.tile, r);
        if (blk < last) {
            fetch_k(blk);
            fetch_v(blk);
        }
        if (a.q.vec) take_q<kFewM, DP>(a, it, 0, row, nullptr, qx);
    };
    begin();
    for (;;) {
        if (!a.q.vec) {
            __syncthreads();                      // the part before is done with so
            take_q<kFewM, DP>(a, it, 0, row, &so[wave][0][0], qx);
        }
        QFrag<DP, NP> q;
        load_q<DP, NP>(a, qx, q);
        const int32_t lo = from(row.lo, (int64_t)blk0 * kBlock), hi = from(row.hi, (int64_t)blk0 * kBlock);
        State<DP> st;
        st.m = kLow;
        st.l = 0.f;
#pragma unroll
        for (int i = 0; i < DP / 16; i++) st.o[i] = v4f{0.f, 0.f, 0.f, 0.f};
        Ref ref{0.f, 0.f};
        while (blk < last) {
            // the next block's loads are in flight while a block is worked on: its
            // keys' from where these are used up, its values' likewise
            const float kcs = ksc;
            const bool more = blk + 4 < last;
            v4f acc[2] = {v4f{0.f, 0.f, 0.f, 0.f}, v4f{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int c = 0; c < DP / 64; c++)
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    const uint4 w = k[t * (DP / 64) + c];
                    const h8 x = halves(w.x, w.y), y = halves(w.z, w.w);
#pragma unroll
                    for (int n = 0; n < NP; n++) {
                        acc[t] = mfma(x, q.h[n][2 * c], acc[t]);
                        acc[t] = mfma(y, q.h[n][2 * c + 1], acc[t]);
                    }
                }
            if (more) fetch_k(blk + 4);
            const float vcs = vsc;
            float log, inv;
            refer<DP, 1>(vcs, ref, &st);
            ratio_of(vcs, ref, &log, &inv);
            const int32_t off = (int32_t)(blk - blk0) * (int32_t)kBlock;
            const bool nan = kcs != kcs || vcs != vcs;
            const float f = factor(nan ? 1.f : kcs, q.f);
            if (__any(lo > off || hi < off + (int32_t)kBlock) || nan) mask(acc, lo - off, hi - off, g, nan, st.l);
            const float top = top_of(acc) * f;
            if (__any(top > st.m + kLift)) lift(top, st);
            h8 p[NP];
            const float c = kBias - st.m + log;
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 8; j += 2) sum += weigh2<NP>(acc[j / 4][j % 4], acc[j / 4][j % 4 + 1], f, c, j, p);
            st.l = __builtin_fmaf(sum, inv, st.l);
#pragma unroll
            for (int i = 0; i < DP / 32; i++) {
                const h8 x = halves(v[i].x, v[i].y), y = halves(v[i].z, v[i].w);
#pragma unroll
                for (int n = 0; n < NP; n++) {
                    st.o[2 * i] = mfma(x, p[n], st.o[2 * i]);
                    st.o[2 * i + 1] = mfma(y, p[n], st.o[2 * i + 1]);
                }
            }
            if (more) fetch_v(blk + 4);
            blk += 4;
        }
        // the next part's loads are in flight while this one's waves are joined
        const Item done = it;
        const bool from0 = c0 == 0, whole = from0 && nc == it.t.chunks;
        bool go = it.start + it.t.chunks < end;
        if (go) {
            advance<kFewM>(a, it, order);
            go = it.start < end;
            if (go) begin();
        }
        // lane (r, g) holds elements 32 i + 8 g .. + 8 of row r
        st.l += __shfl_xor(st.l, 16, 64);
        st.l += __shfl_xor(st.l, 32, 64);
        __syncthreads();
        if (g == 0) {
            sm[wave][r] = st.m;
            sl[wave][r] = st.l;
        }
#pragma unroll
        for (int i = 0; i < DP / 32; i++) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                float4 w;
                w.x = st.o[2 * i][2 * h] * ref.ref;
                w.y = st.o[2 * i + 1][2 * h] * ref.ref;
                w.z = st.o[2 * i][2 * h + 1] * ref.ref;
                w.w = st.o[2 * i + 1][2 * h + 1] * ref.ref;
                *(float4 *)&so[wave][r][32 * i + 8 * g + 4 * h] = w;
            }
        }
        __syncthreads();
        const uint64_t slot = (uint64_t)wg * 2 + (from0 ? 1u : 0u);
        for (uint32_t u = threadIdx.x; u < 16u * (DP / 4); u += 256) {
            const uint32_t rr = u / (DP / 4), d = u % (DP / 4) * 4u;
            const float m = fmaxf(fmaxf(sm[0][rr], sm[1][rr]), fmaxf(sm[2][rr], sm[3][rr]));
            float l = 0.f;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const float e = exp2_(sm[w][rr] - m);
                l += e * sl[w][rr];
                const float4 o = *(const float4 *)&so[w][rr][d];
                x.x += e * o.x; x.y += e * o.y; x.z += e * o.z; x.w += e * o.w;
            }
            if (whole) {
                const Row w = row_of<kFewM>(a, done.s, done.head, done.tile, rr);
                if (!w.valid) continue;
                const float inv = 1.f / l;
                x = w.hi > w.lo ? make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv) : make_float4(0.f, 0.f, 0.f, 0.f);
                store4(a.out, w.row * a.out.ld_row + w.head * a.out.ld_head, d, a.v.hd, x);
            } else {
                *(float4 *)(a.w.part + (slot * kFewM + rr) * DP + d) = x;
                if (d == 0) {
                    a.w.ml[(slot * kFewM + rr) * 2] = m;
                    a.w.ml[(slot * kFewM + rr) * 2 + 1] = l;
                }
            }
        }
        if (!go) break;
    }
}

// Many rows: tiles of 64 RT pairs, 16 RT a wave.  The workgroup's waves share
// an item's blocks: a block's codes are loaded into registers three blocks ahead,
// turned into f16 once and put into a ring of three in LDS in the order of the
// operands, from where every wave feeds its products (an operand is read once
// for RT tiles of rows).  Within a wave the matrix cores and the vector units
// work at the same time: the scores of block j + 1 while block j's are turned
// into weights, the outputs of block j while the codes of block j + 2 are turned
// into f16.
//
// Bound by the matrix cores and the vector units together (16 of the latter's
// instructions a block and tile are exponentials): 1001 tokens of 32 heads of 128
// in f32, two pieces of q and p, 41 us, 0.20 PFLOP/s of the formula and twice that
// of products; up to 2048 new tokens of four sequences in f16 over 4096 positions
// each 406 us with the merge, 0.76 PFLOP/s, where a large f16 matrix product does
// 1.11: matrix cores busy in 33 % of the cycles, vector units in 56 %, waves waiting
// (data, barriers) in 27 % of theirs.  Two workgroups of 48 KB a compute unit; larger tiles (256
// pairs) spill: 744 against 480 us at that stage.  Rows that take 16-byte accesses
// go straight from and to memory; through LDS they cost a part 10000 cycles more.
template <int DP, int NP, int RT> __global__ void __launch_bounds__(256, 2) many_k(Problem a)
{
    constexpr uint32_t M = 64 * RT;
    constexpr int NU = DP / 64;                           // 16-byte units of codes a thread stages per block
    extern __shared__ __attribute__((aligned(16))) h8 stage[];        // [3][keys, values][DP / 32 * 2][64]
    constexpr uint32_t kOne = DP * 4;                                 // operands of 16 bytes: keys or values of a block
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63u, r = lane & 15u, g = lane >> 4;
    float *const mine = (float *)(stage + wave * (kOne * 3 / 2));        // 16 rows of DP + 4 floats fit
    const uint32_t wg = place_of(blockIdx.x, gridDim.x);
    const Order order = order_of<M>(a);
    const uint32_t per = max((order.total + gridDim.x - 1) / gridDim.x, 1u);
    uint32_t at = wg * per;
    const uint32_t end = min(at + per, order.total);
    if (at >= end) {
        put_split(a, wg, false, Item{}, per);
        return;
    }
    Item it = find<M>(a, at, order);
    put_split(a, wg, at > it.start, it, per);
    const uint64_t all = (uint64_t)a.v.n_seqs * a.v.n_heads;
    for (;;) {
        if (it.start >= end) break;                      // only its lead is here
        const uint32_t c0 = at > it.start ? at - it.start : 0u, nc = min(it.t.chunks, end - it.start) - c0;
        const uint64_t sh = (uint64_t)it.seq * a.v.n_heads + it.head;
        // the part's first block; n of them (0: an item that sees nothing)
        const uint32_t blk0 = it.t.blk0 + c0 * a.chunk;
        const uint32_t n = it.t.blk0 + min(it.t.blocks, (c0 + nc) * a.chunk) - blk0;
        const uint8_t *kb = a.v.codes + (sh * a.v.n_blocks + blk0) * (kBlock * DP);
        const uint8_t *vb = a.v.codes + ((all + sh) * a.v.n_blocks + blk0) * (kBlock * DP);
        const float *ks = a.v.scale + sh * a.v.n_blocks + blk0, *vs = a.v.scale + (all + sh) * a.v.n_blocks + blk0;
        uint4 code[NU];
        // the blocks' codes; the last one's again behind it
        auto fetch = [&](uint32_t b) {
            const uint64_t off = (uint64_t)min(b, n - 1) * (kBlock * DP);
#pragma unroll
            for (int i = 0; i < NU; i++) {
                const uint32_t u = threadIdx.x + 256u * i;
                code[i] = *(const uint4 *)(u < 2 * DP ? kb + off + u * 16u : vb + off + (u - 2 * DP) * 16u);
            }
        };
        auto put = [&](uint32_t slot, int half, uint4 w) {        // half: of 2 NU
            const uint32_t u = threadIdx.x + 256u * (half / 2);
            h8 *to = stage + slot * 2 * kOne + (u >> 6) * 128u + lane + half % 2 * 64;
            *to = half % 2 ? halves(w.z, w.w) : halves(w.x, w.y);
        };
        Row row[RT];
        float4 qx[RT][DP / 16];
#pragma unroll
        for (int t = 0; t < RT; t++) {
            row[t] = row_of<M>(a, it.s, it.head, it.tile, (wave * RT + t) * 16u + r);
            // LDS: the wave's quarter of the ring (every part ends with a barrier)
            take_q<M, DP>(a, it, (wave * RT + t) * 16u, row[t], mine, qx[t]);
        }
        uint4 code0[NU], code1[NU];
        if (n) {
            fetch(0);
#pragma unroll
            for (int i = 0; i < NU; i++) code0[i] = code[i];
            fetch(1);
#pragma unroll
            for (int i = 0; i < NU; i++) code1[i] = code[i];
            fetch(2);
        }
        QFrag<DP, NP> q[RT];
        State<DP> st[RT];
        int32_t lo[RT], hi[RT], lo_all = 0, hi_all = 0x7FFFFFFF;
#pragma unroll
        for (int t = 0; t < RT; t++) {
            load_q<DP, NP>(a, qx[t], q[t]);
            lo[t] = from(row[t].lo, (int64_t)blk0 * kBlock);
            hi[t] = from(row[t].hi, (int64_t)blk0 * kBlock);
            lo_all = max(lo_all, lo[t]);
            hi_all = min(hi_all, hi[t]);
            st[t].m = kLow;
            st[t].l = 0.f;
#pragma unroll
            for (int i = 0; i < DP / 16; i++) st[t].o[i] = v4f{0.f, 0.f, 0.f, 0.f};
        }
        Ref ref{0.f, 0.f};
        // S^T of the block in `slot`
        auto scores = [&](uint32_t slot, v4f (&x)[RT][2]) {
            const h8 *kf = stage + slot * 2 * kOne + lane;
#pragma unroll
            for (int t = 0; t < RT; t++) x[t][0] = x[t][1] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < DP / 32; c++)
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const h8 w = kf[(k * (DP / 32) + c) * 64];
#pragma unroll
                    for (int t = 0; t < RT; t++)
#pragma unroll
                        for (int i = 0; i < NP; i++) x[t][k] = mfma(w, q[t].h[i][c], x[t][k]);
                }
        };
        float ksn = 0.f, vsn = 0.f;
        // block j, its scores in x; the next one's into y.  slot: j % 3
        auto block = [&](uint32_t j, uint32_t slot, v4f (&x)[RT][2], v4f (&y)[RT][2]) {
            const float ksc = ksn, vsc = vsn;
            const uint32_t next = min(j + 1, n - 1), s1 = slot == 2 ? 0u : slot + 1, s2 = slot == 0 ? 2u : slot - 1;
            ksn = ks[next];
            vsn = vs[next];
            constexpr int kOps = DP / 16, kAhead = 4;     // operands of keys, and of values; in flight
            const h8 *kf = stage + s1 * 2 * kOne + lane, *vf = stage + slot * 2 * kOne + kOne + lane;
            h8 ops[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; i++) ops[i] = kf[i * 64];
            // what may branch first: the value scale's reference, masks, the rows' references
            refer<DP, RT>(vsc, ref, st);
            float log, inv;
            ratio_of(vsc, ref, &log, &inv);
            const bool nan = ksc != ksc || vsc != vsc;
            const int32_t off = (int32_t)(j * kBlock);
            if (__any(lo_all > off || hi_all < off + (int32_t)kBlock) || nan) {
#pragma unroll
                for (int t = 0; t < RT; t++) mask(x[t], lo[t] - off, hi[t] - off, g, nan, st[t].l);
            }
            float f[RT], top[RT];
            bool past = false;
#pragma unroll
            for (int t = 0; t < RT; t++) {
                f[t] = factor(nan ? 1.f : ksc, q[t].f);
                top[t] = top_of(x[t]) * f[t];
                past = past || top[t] > st[t].m + kLift;
            }
            if (__any(past)) {
#pragma unroll
                for (int t = 0; t < RT; t++) lift(top[t], st[t]);
            }
            // operand by operand: its products, the read of the one kAhead behind it,
            // and a share of the vector work (the order is held by barriers to the
            // scheduler, which would put each part in one piece and wait for every
            // read)
            h8 p[RT][NP];
            float c[RT], sum[RT];
#pragma unroll
            for (int t = 0; t < RT; t++) {
                c[t] = kBias - st[t].m + log;
                sum[t] = 0.f;
                y[t][0] = y[t][1] = v4f{0.f, 0.f, 0.f, 0.f};
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < kOps; i++) {
                const h8 w = ops[i % kAhead];
                if (i + kAhead < kOps) ops[i % kAhead] = kf[(i + kAhead) * 64];
                else if (i + kAhead < 2 * kOps) ops[i % kAhead] = vf[(i + kAhead - kOps) * 64];
#pragma unroll
                for (int t = 0; t < RT; t++)
#pragma unroll
                    for (int k = 0; k < NP; k++)
                        y[t][i / (kOps / 2)] = mfma(w, q[t].h[k][i % (kOps / 2)], y[t][i / (kOps / 2)]);
#pragma unroll
                for (int e = i * 4 / kOps; e < (i + 1) * 4 / kOps; e++)
#pragma unroll
                    for (int t = 0; t < RT; t++)
                        sum[t] += weigh2<NP>(x[t][e / 2][e % 2 * 2], x[t][e / 2][e % 2 * 2 + 1], f[t], c[t], 2 * e, p[t]);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int i = 0; i < kOps; i++) {
                const h8 w = ops[i % kAhead];
                if (i + kAhead < kOps) ops[i % kAhead] = vf[(i + kAhead) * 64];
#pragma unroll
                for (int t = 0; t < RT; t++)
#pragma unroll
                    for (int k = 0; k < NP; k++) st[t].o[i] = mfma(w, p[t][k], st[t].o[i]);
                if (i % 2) put(s2, i / 2, code[i / 4]);   // block j + 2, where j - 1 was
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int t = 0; t < RT; t++) st[t].l = __builtin_fmaf(sum[t], inv, st[t].l);
            fetch(j + 3);
            __syncthreads();
        };
        if (n) {
            __syncthreads();                              // the part before is done with the ring
#pragma unroll
            for (int i = 0; i < 2 * NU; i++) {
                put(0, i, code0[i / 2]);
                put(1, i, code1[i / 2]);
            }
            ksn = ks[0];
            vsn = vs[0];
            __syncthreads();
            v4f x[RT][2], y[RT][2];
            scores(0, x);
            uint32_t slot = 0;
            for (uint32_t j = 0;; j += 2) {
                block(j, slot, x, y);
                slot = slot == 2 ? 0u : slot + 1;
                if (j + 1 >= n) break;
                block(j + 1, slot, y, x);
                slot = slot == 2 ? 0u : slot + 1;
                if (j + 2 >= n) break;
            }
        }
        const bool whole = c0 == 0 && nc == it.t.chunks;
        const uint64_t slot = (uint64_t)wg * 2 + (c0 ? 0u : 1u);
#pragma unroll
        for (int t = 0; t < RT; t++) {
            const uint32_t rr = (wave * RT + t) * 16u + r;
            float l = st[t].l;
            l += __shfl_xor(l, 16, 64);
            l += __shfl_xor(l, 32, 64);
            const float k = whole ? ref.ref / l : ref.ref;
            if (!whole && g == 0) {
                a.w.ml[(slot * M + rr) * 2] = st[t].m;
                a.w.ml[(slot * M + rr) * 2 + 1] = l;
            }
            // lane (r, g) holds elements 32 i + 8 g .. + 8 of row r
            const Row w = row_of<M>(a, it.s, it.head, it.tile, rr);
            const uint64_t to = w.row * a.out.ld_row + w.head * a.out.ld_head;
            float *const part = a.w.part + (slot * M + rr) * DP;
            const bool sees = !whole || w.hi > w.lo, direct = !whole || a.out.vec;
#pragma unroll
            for (int i = 0; i < DP / 32; i++) {
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint32_t d = 32 * i + 8 * g + 4 * h;
                    float4 x = make_float4(st[t].o[2 * i][2 * h] * k, st[t].o[2 * i + 1][2 * h] * k,
                                           st[t].o[2 * i][2 * h + 1] * k, st[t].o[2 * i + 1][2 * h + 1] * k);
                    if (!sees) x = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (!whole) *(float4 *)(part + d) = x;
                    else if (!direct) *(float4 *)(mine + r * (DP + 4) + d) = x;
                    else if (w.valid) store4v(a.out, to, d, a.v.hd, x);
                }
            }
            if (!direct) {                                // element by element, through LDS
                wave_sync();
#pragma unroll 1
                for (uint32_t u = lane; u < 16u * DP; u += 64) {
                    const uint32_t x = u / DP, d = u % DP;
                    const Row y = row_of<M>(a, it.s, it.head, it.tile, (wave * RT + t) * 16u + x);
                    if (y.valid && d < a.v.hd)
                        store1(a.out, y.row * a.out.ld_row + y.head * a.out.ld_head + d, mine[x * (DP + 4) + d]);
                }
                wave_sync();
            }
        }
        if (!n) __syncthreads();                          // as every part ends
        if (it.start + it.t.chunks >= end) break;
        advance<M>(a, it, order);
    }
}

// Joins the parts of an item that workgroups first .. last hold (the first one's
// in slot 1, the others' in slot 0).  Grid: (workgroups - 1, row groups); the
// workgroup of the second part does it.  DP / 4 lanes take a row's elements; few
// rows of many parts (PARTS): the other threads take parts in turn; else they
// take rows.  Bound by its launch and a few dependent reads where there are few
// parts: 4 to 5.5 us behind few_k, 7.6 and 14 behind many_k's tiles of 64 and 128
// pairs (up to 67 MB of parts).  A short prompt over a long cache has many parts a
// tile: 32 of them 8.6 us with eight on their way together and eight row groups (25.8
// one after the other, 13.0 with four groups).
template <uint32_t M, int DP, bool PARTS> __global__ void __launch_bounds__(256) merge_k(Problem a)
{
    constexpr uint32_t L = DP / 4, N = 256 / L;            // 192 / 4 = 48: 5 groups, 16 lanes idle
    __shared__ __attribute__((aligned(16))) float sm[N], sl[N], so[N][DP];
    const uint32_t wg = blockIdx.x + 1;
    const Split s = a.w.split[wg];
    if (s.first == kNone || s.first + 1 != wg) return;
    const Span span = span_of(a.b, s.seq);
    const uint32_t lane = threadIdx.x % L, grp = threadIdx.x / L, d = lane * 4;
    for (uint32_t r = PARTS ? blockIdx.y : blockIdx.y * N + grp; r < M; r += PARTS ? M : gridDim.y * N) {
        float m = kLow, l = 0.f;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        auto add = [&](float n, float k, float4 o) {
            const float top = fmaxf(m, n), e = exp2_(m - top), f = exp2_(n - top);
            m = top;
            l = l * e + k * f;
            x.x = x.x * e + o.x * f; x.y = x.y * e + o.y * f; x.z = x.z * e + o.z * f; x.w = x.w * e + o.w * f;
        };
        // the thread's parts, AT of them on their way together
        auto take = [&](auto at_once) {
            constexpr uint32_t AT = decltype(at_once)::value, step = PARTS ? N : 1;
            for (uint32_t w0 = s.first + (PARTS ? grp : 0); w0 <= s.last; w0 += AT * step) {
                float2 t[AT];
                float4 o[AT];
#pragma unroll
                for (uint32_t j = 0; j < AT; j++) {              // the last one again behind it
                    const uint32_t w = min(w0 + j * step, s.last);
                    const uint64_t at = ((uint64_t)w * 2 + (w == s.first ? 1u : 0u)) * M + r;
                    t[j] = *(const float2 *)(a.w.ml + at * 2);
                    o[j] = *(const float4 *)(a.w.part + at * DP + d);
                }
#pragma unroll
                for (uint32_t j = 0; j < AT; j++)
                    if (w0 + j * step <= s.last) add(t[j].x, t[j].y, o[j]);
            }
        };
        if (grp < N) {
            if (s.last - s.first < 2 * (PARTS ? N : 1)) take(std::integral_constant<uint32_t, 2>{});
            else take(std::integral_constant<uint32_t, 8>{});
        }
        if (PARTS) {
            if (grp < N) {
                if (lane == 0) { sm[grp] = m; sl[grp] = l; }
                *(float4 *)&so[grp][d] = x;
            }
            __syncthreads();
            if (grp) return;
            for (uint32_t w = 1; w < N; w++) add(sm[w], sl[w], *(const float4 *)&so[w][d]);
        }
        if (grp >= N) return;
        const Row w = row_of<M>(a, span, s.head, s.tile, r);
        if (!w.valid) continue;
        const float inv = 1.f / l;
        x = w.hi > w.lo ? make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv) : make_float4(0.f, 0.f, 0.f, 0.f);
        store4(a.out, w.row * a.out.ld_row + w.head * a.out.ld_head, d, a.v.hd, x);
    }
}

// Workgroups of a call, and its workspace.
uint32_t workgroups(int n_cu)
{
    return 2u * (uint32_t)(n_cu > 0 ? n_cu : 256);
}

size_t work_bytes(uint32_t wgs, uint32_t m, uint32_t dp)
{
    return (size_t)wgs * (sizeof(Split) + 2u * m * (dp + 2u) * sizeof(float));
}

Work work_at(void *p, uint32_t wgs, uint32_t m)
{
    Work w;
    w.split = (Split *)p;
    w.ml = (float *)(w.split + wgs);
    w.part = w.ml + (size_t)wgs * 2 * m * 2;
    return w;
}

// Which tiles a call takes, by its (token, head) pairs per sequence and kv
// head: what is not a sequence's is computed for nothing, while fewer, larger
// tiles read and convert the cache less often.
enum Kind { kFew, kMany64, kMany128 };

Kind kind_of(const View &v, uint64_t n_rows, bool starts, uint64_t n_rep, int n_cu)
{
    const uint64_t pairs = starts ? n_rows * n_rep / std::min<uint64_t>(v.n_seqs, n_rows ? n_rows : 1) : n_rep;
    // two tiles of 16 rather than half of one of 64 (us: 24 pairs over 8000 positions
    // 21 against 54, 32 of eight sequences 33 against 43; 56 of 16 sequences 72
    // against 62)
    if (pairs <= 32) return kFew;
    // tiles of 128 pairs where there are enough of them for the workgroups: with
    // fewer, the items are cut anyway, and the smaller ones have less to begin and
    // end with (1001 tokens of 32 heads 41 against 47 us, f32; 5200 of them over four
    // sequences 610 against 459, f16)
    const uint64_t tiles = (n_rows * n_rep + 127) / 128 * v.n_heads;
    return pairs <= 64 || v.dp > 128 || tiles < workgroups(n_cu) ? kMany64 : kMany128;
}

uint32_t tile_rows(Kind k)
{
    return k == kFew ? kFewM : k == kMany64 ? 64u : 128u;
}

template <int DP, int NP, int RT> int launch_many(Problem &a, uint32_t wgs, hipStream_t st)
{
    const size_t lds = 3u * 2u * DP * 4u * 16u;
    hipLaunchKernelGGL((many_k<DP, NP, RT>), dim3(wgs), dim3(256), lds, st, a);
    if (hipPeekAtLastError() != hipSuccess) return -1;
    if (a.v.n_blocks > a.chunk)
        hipLaunchKernelGGL((merge_k<64 * RT, DP, false>), dim3(wgs - 1, 8), dim3(256), 0, st, a);
    return hipPeekAtLastError() == hipSuccess ? 0 : -1;
}

template <int DP> int launch_dp(Problem &a, Kind kind, int n_cu, hipStream_t st)
{
    const uint32_t wgs = workgroups(n_cu);
    if (kind == kFew) {
        if (a.q.f16) hipLaunchKernelGGL((few_k<DP, 1>), dim3(wgs), dim3(256), 0, st, a);
        else hipLaunchKernelGGL((few_k<DP, 2>), dim3(wgs), dim3(256), 0, st, a);
        if (hipPeekAtLastError() != hipSuccess) return -1;
        // no item of a cache of one chunk is ever cut
        if (a.v.n_blocks > a.chunk) {
            const uint32_t rows = a.b.lens && !a.b.starts ? std::min(kFewM, a.n_rep) : kFewM;
            hipLaunchKernelGGL((merge_k<kFewM, DP, true>), dim3(wgs - 1, rows), dim3(256), 0, st, a);
        }
        return hipPeekAtLastError() == hipSuccess ? 0 : -1;
    }
    if (kind == kMany64)
        return a.q.f16 ? launch_many<DP, 1, 1>(a, wgs, st) : launch_many<DP, 2, 1>(a, wgs, st);
    if constexpr (DP <= 128)
        return a.q.f16 ? launch_many<DP, 1, 2>(a, wgs, st) : launch_many<DP, 2, 2>(a, wgs, st);
    return -1;
}

}  // namespace

size_t attention_work(const View &v, size_t n_rows, size_t n_heads, int n_cu)
{
    // calls of fewer rows take no larger tiles
    const uint32_t m = std::max(tile_rows(kind_of(v, n_rows, true, n_heads / v.n_heads, n_cu)),
                                tile_rows(kind_of(v, n_rows, false, n_heads / v.n_heads, n_cu)));
    return work_bytes(workgroups(n_cu), m, v.dp);
}

int launch_attention(const View &v, const Batch &b, uint32_t n_heads, const Rows &q, float scale, uint32_t window,
                     const Rows &out, void *work, int n_cu, hipStream_t st)
{
    if (b.n_rows == 0) return 0;
    Problem a{};
    a.v = v;
    a.b = b;
    a.q = q;
    a.out = out;
    a.n_rep = n_heads / v.n_heads;
    a.window = window;
    a.sign = std::signbit(scale) ? -1.f : 1.f;
    a.scale2 = fabsf(scale) * 1.44269504f;
    const Kind kind = kind_of(v, b.n_rows, b.starts || !b.lens, a.n_rep, n_cu);
    while ((1ull << a.rep_shift) < a.n_rep) a.rep_shift++;
    a.rep_mul = (uint32_t)((((1ull << a.rep_shift) - a.n_rep) << 32) / a.n_rep + 1);
    // a block for each wave of few_k, two of many_k; more where the chunks
    // would not be counted in 31 bits (all tiles seeing the whole cache)
    a.chunk = kind == kFew ? 4u : 2u;
    // what an item costs whatever its length, in chunks (us at 2, 3, 4, 6: 1001
    // tokens of 32 heads 42.7, 41.2, 42.0, 45.0; 64 sequences' tokens 107, 108, 108, 111);
    // single tokens of one sequence are items of one length and need no balance
    a.lead = kind == kFew && v.n_seqs == 1 ? 0u : 3u;
    const uint64_t tiles = ((uint64_t)b.n_rows * a.n_rep + tile_rows(kind) - 1) / tile_rows(kind) + v.n_seqs;
    while (tiles * v.n_heads * (v.n_blocks / a.chunk + 1 + a.lead) >> 31) a.chunk *= 2;
    a.w = work_at(work, workgroups(n_cu), tile_rows(kind));
    switch (v.dp) {
    case 64: return launch_dp<64>(a, kind, n_cu, st);
    case 128: return launch_dp<128>(a, kind, n_cu, st);
    case 192: return launch_dp<192>(a, kind, n_cu, st);
    case 256: return launch_dp<256>(a, kind, n_cu, st);
    default: return -1;
    }
}

}  // namespace qg8
