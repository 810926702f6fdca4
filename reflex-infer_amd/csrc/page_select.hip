// page_select.hip -- which pages of a paged cache a token attends to: bounds of each
// page's keys, and the pages of the largest score against them, on the gfx950 matrix
// cores.
//
//   bounds  a page's smallest and largest key of each dim over its filled positions, lo
//           and hi, in steps of scale = max(|lo|, |hi|) * fp32(1 / 127): rint(lo / scale),
//           rint(hi / scale).  NaN keys are left out, infinities count as the largest
//           fp32 numbers.
//   score   of a page for a query q: no key of it has a larger product than
//           sum_d max(q_d lo_d, q_d hi_d) (up to the steps).  The query in steps of its
//           own, max |q| * fp32(1 / 127): with q- = min(q, 0), q+ = max(q, 0) the sum is q- . lo +
//           q+ . hi, a product of whole numbers below 2^23, exact in any order; times the
//           query's step, times the page's scale, both rounded.  A page's score for a token
//           is the largest over the heads of the KV head's group.
//   choice  the first n_first pages and the last n_last always, then the largest scores,
//           equal ones by index, in order.  Two rounded products and comparisons: the
//           same lists whichever way the work is cut.
// Bound: the bytes of the bounds (264 a page and head of 128 with its scale and entry), in
// pieces of 256: a loop that does nothing else reads those of 64 sequences of 500 to 30000
// positions, pages of 16, in 14 us, of sequences alike in 10 (5.8 TB/s); for a prompt's chunk,
// whose tokens share them, waiting (vector instructions and products are 12 of its 25 us: all
// workgroups score first and choose then, two a CU); for a few tokens the chain of lengths,
// table, bounds and choice.  So a row of bounds is loaded by lanes beside one another and turned in LDS (16
// rows at a time by the operand's layout 21), a chunk's tokens share a workgroup's, and a
// few tokens' scores and choice are two launches, the first over more workgroups.
// Measured: those 64 sequences, 32 / 8 heads, lists of 64, 24 us (the longest sequences' steps
// are its end; two launches 31); one token of 16 / 2 heads after 60000 positions, lists of
// 128, 5.7 + 7.2; a chunk of 512 tokens of 28 / 4 heads after 30000, pages of 32, 25.5.
// Bounds: the pages of 64 new tokens in an int8 cache 5.5 us, those of 8536, pages of 64, 11
// (their bytes at the rate of a copy 3.5).
#include <float.h>
#include <math.h>

#include <algorithm>

#include "launch.h"
#include "mfma_util.h"
#include "paged.h"
#include "q4k_device.h"

namespace rxq4 {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr float kStepOfMax = 1.0f / 127.0f;
__device__ __forceinline__ int to_step(float x, float scale) {
    const float z = scale > 0.0f ? rintf(x / scale) : 0.0f;  // (IEEE: the bytes follow from x alone)
    return (int)fminf(fmaxf(z, -127.0f), 127.0f);
}

// ------------------------------------------------------------------ bounds
// A workgroup takes 32 pieces of 8 dims of one page, whole heads, by 8 groups of threads
// that share the page's positions.
constexpr int kPieces = 32, kGroups = 8;

struct BoundsParams {
    PageBounds out;
    SeqBatch b;
    PagedCache c;
    int rows_wg;  // rows of the batch that a workgroup looks for pages' first new tokens in
};

// Positions [0, held) of pool page `page`, heads head0 .. of it.
template <bool I8>
__device__ __forceinline__ void bound_page(const BoundsParams &p, int page, int held, int head0) {
    __shared__ float part[4][2][8][kPieces];
    __shared__ float most[kPieces];
    const int tid = threadIdx.x, pc = tid % kPieces, grp = tid / kPieces;
    const int hd = p.c.hd, n_ch = hd / 8, heads = min(kPieces / n_ch, p.c.n_kv - head0);
    const int ch = pc % n_ch, h = pc / n_ch;
    const bool live = h < heads;
    const int row_bytes = p.c.n_kv * hd * (I8 ? 1 : 2);
    const int head = head0 + (live ? h : 0);
    const uint8_t *src = p.c.k + (int64_t)page * p.c.page_bytes + (int64_t)(head * hd + 8 * ch) * (I8 ? 1 : 2);
    float lo[8], hi[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        lo[i] = INFINITY;
        hi[i] = -INFINITY;
    }
    constexpr int U = 8;
    for (int at = grp; at < held; at += U * kGroups) {
        u32x4 x[U];
        float s[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {  // (places past the end repeat the last)
            const int pos = min(at + u * kGroups, held - 1);
            if constexpr (I8) {
                const u32x2 y = *reinterpret_cast<const u32x2 *>(src + (int64_t)pos * row_bytes);
                x[u] = u32x4{y.x, y.y, 0u, 0u};
                s[u] = p.c.ks ? p.c.ks[(((int64_t)page << p.c.shift) + pos) * p.c.n_kv + head] : 1.0f;
            } else {
                x[u] = load16(src + (int64_t)pos * row_bytes);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float y;
                if constexpr (I8) y = (float)(int8_t)(x[u][i >> 2] >> (8 * (i & 3))) * s[u];
                else y = f16_bits_to_f32(x[u][i >> 1] >> (16 * (i & 1)) & 0xFFFFu);
                lo[i] = fminf(lo[i], y);  // (of a NaN and a number the number)
                hi[i] = fmaxf(hi[i], y);
            }
    }
    __syncthreads();  // the page before is read
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float l = fminf(lo[i], __shfl_xor(lo[i], 32, 64)), m = fmaxf(hi[i], __shfl_xor(hi[i], 32, 64));
        if ((tid & 32) == 0) {
            part[tid >> 6][0][i][pc] = l;
            part[tid >> 6][1][i][pc] = m;
        }
    }
    __syncthreads();
    // a thread a dim: of piece tid / 8
    const int c = tid >> 3, i = tid & 7;
    float l = part[0][0][i][c], m = part[0][1][i][c];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
        l = fminf(l, part[w][0][i][c]);
        m = fmaxf(m, part[w][1][i][c]);
    }
    const bool none = !(l <= m);  // NaN at every position
    l = none ? 0.0f : fminf(fmaxf(l, -FLT_MAX), FLT_MAX);
    m = none ? 0.0f : fminf(fmaxf(m, -FLT_MAX), FLT_MAX);
    float top = fmaxf(fabsf(l), fabsf(m));
#pragma unroll
    for (int off = 4; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
    if (i == 0) most[c] = top;
    __syncthreads();
    const int hc = c / n_ch;
    if (hc >= heads) return;
    for (int j = 0; j < n_ch; ++j) top = fmaxf(top, most[hc * n_ch + j]);
    const float scale = top * kStepOfMax;
    const int64_t row = (int64_t)page * p.c.n_kv + head0 + hc;
    int8_t *dst = p.out.bounds + row * 2 * hd + 16 * (c % n_ch) + i;
    dst[0] = (int8_t)to_step(l, scale);
    dst[8] = (int8_t)to_step(m, scale);
    if (c % n_ch == 0 && i == 0) p.out.scales[row] = scale;
}

// A page belongs to the row of its sequence's first new token in it.
template <bool I8>
__global__ __launch_bounds__(256) void kv_bounds_kernel(BoundsParams p) {
    const int head0 = blockIdx.y * (kPieces / (p.c.hd / 8)), mask = (1 << p.c.shift) - 1;
    const int t_end = min(((int)blockIdx.x + 1) * p.rows_wg, p.b.n_tokens), limit = position_limit(p.b, p.c);
    for (int t = blockIdx.x * p.rows_wg; t < t_end;) {  // uniform
        SeqSpan span;
        const int s = seq_of_row(p.b, t, span);
        if (s >= p.b.n_seqs) return;
        const int n = min(span.n, p.b.max_new), last = span.row0 + n;
        const int end = min(span.pos0 + n, limit);
        for (int r = max(t, span.row0); r < min(last, t_end);) {
            const int pos = span.pos0 + (r - span.row0);
            if (pos >= end) break;
            if (pos >= 0 && ((pos & mask) == 0 || r == span.row0)) {
                const int page = slot_of(p.c, s, pos) >> p.c.shift;  // -1 stays -1
                if (page >= 0) bound_page<I8>(p, page, min(mask + 1, end - (pos & ~mask)), head0);
            }
            r += pos < 0 ? -pos : mask + 1 - (pos & mask);
        }
        t = max(t + 1, span.row0 + span.n);
    }
}

// ------------------------------------------------------------------ scores
constexpr uint32_t kAlways = 0xFFFFFFFFu;  // above every score's key; 0: no candidate

struct SelectParams {
    int32_t *pages;
    const uint16_t *q;
    PageBounds bounds;
    SeqBatch b;
    PagedCache c;
    int n_heads, group, n_select, n_first, n_last;
    int tokens;      // of a tile at most
    int room;        // keys of a token in LDS
    uint32_t *keys;  // split: [n_tokens][n_kv][stride]
    int stride;
    int parts;       // split: workgroups of a token and KV head
};

// Bits that order as the numbers do, above 0; -0 as 0, and NaN, which of a score is an infinite
// scale times 0.
__device__ __forceinline__ uint32_t key_of(float x) {
    // (not by adding 0: that becomes one rounding with the product before it, which is -0 yet)
    const uint32_t u = __builtin_islessgreater(x, 0.0f) ? __builtin_bit_cast(uint32_t, x) : 0u;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The KV head and the unit (a token or a tile, for all its KV heads) of a workgroup.  The
// heads of a unit go to one XCD (workgroups are dealt to the eight in turn): their rows of a
// page, and its scales, lie beside one another.
__device__ __forceinline__ int unit_of(const SelectParams &p, int &kvh) {
    const int x8 = blockIdx.x / 8;
    kvh = x8 % p.c.n_kv;
    return x8 / p.c.n_kv * 8 + blockIdx.x % 8;
}
int64_t units_grid(int64_t units, int n_kv) { return (units + 7) / 8 * 8 * n_kv; }
constexpr int64_t kMostWorkgroups = 0x7FFFFF;  // of a launch: of up to 512 threads each, 2^32 in all

__device__ __forceinline__ float score_of(uint32_t key) {
    return __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

// The tokens of a tile: rows [t0, t0 + n) of the batch, all of sequence s; the first at pos0.
struct Tile {
    int s, t0, n, pos0;
};
__device__ __forceinline__ int pages_of(const SelectParams &p, int pos) {
    const int sees = min(position_limit(p.b, p.c), pos + 1);
    return sees > 0 ? ((sees - 1) >> p.c.shift) + 1 : 0;
}
__device__ __forceinline__ bool token_of(const SelectParams &p, int t, Tile &tile) {
    if (t >= p.b.n_tokens) return false;
    SeqSpan span;
    tile.s = seq_of_row(p.b, t, span);
    if (tile.s >= p.b.n_seqs || t < span.row0 || t - span.row0 >= min(span.n, p.b.max_new)) return false;
    tile.t0 = t;
    tile.n = 1;
    tile.pos0 = span.pos0 + (t - span.row0);
    return true;
}
__device__ __forceinline__ bool tile_of(const SelectParams &p, int u, Tile &tile) {
    const TileRows t = tile_rows(p.b, p.tokens, u);
    tile = Tile{t.s, t.row0, t.n, t.span.pos0 + (t.row0 - t.span.row0)};
    return t.n > 0;
}

// What the waves of a workgroup share while they score.  The queries of a tile in steps, for
// the matrix operands: a row's 8 dims' values below 0, then above, and its step.  A token has
// GP rows, the heads h0 .. of the KV head's group (those past the group the last again).  And
// each wave's 16 pages of bounds, the other operand.  (A row's start moves through the banks.)
template <int KS>
constexpr int kRowLanes = KS > 4 ? 32 : KS > 2 ? 16 : 8;  // lanes that load a row's chunks
template <int KS, int ROWS, int WAVES>
struct ScoreShared {
    u32x4 query[ROWS][4 * KS + 1];
    u32x4 bound[WAVES][16][kRowLanes<KS> + 1];
    float steps[ROWS];
};

// A row's chunks of 8 dims, sub and sub + 16, by 16 lanes.
template <int KS>
struct QueryRow {
    u32x4 raw[KS > 4 ? 2 : 1];
};
template <int KS, int GP>
__device__ __forceinline__ QueryRow<KS> load_query(const SelectParams &p, const Tile &tile, int kvh, int h0, int row) {
    const int sub = threadIdx.x & 15, n_ch = p.c.hd / 8;
    const int tok = min(row / GP, tile.n - 1), head = kvh * p.group + min(h0 + row % GP, p.group - 1);
    const uint16_t *q = p.q + ((int64_t)(tile.t0 + tok) * p.n_heads + head) * p.c.hd;
    QueryRow<KS> x;
#pragma unroll
    for (int c = 0; c < (KS > 4 ? 2 : 1); ++c) x.raw[c] = load16(q + 8 * min(sub + 16 * c, n_ch - 1));
    return x;
}
template <int KS, typename Shared>
__device__ __forceinline__ void store_query(const SelectParams &p, const QueryRow<KS> &q, int row, Shared &out) {
    constexpr int C = KS > 4 ? 2 : 1;
    const int sub = threadIdx.x & 15, n_ch = p.c.hd / 8;
    float x[C][8], top = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) {  // NaN as 0, infinities as fp16's largest, dims past the head's 0
            const float v = f16_bits_to_f32(q.raw[c][i >> 1] >> (16 * (i & 1)) & 0xFFFFu);
            x[c][i] = ((v == v) & (sub + 16 * c < n_ch)) ? fminf(fmaxf(v, -65504.0f), 65504.0f) : 0.0f;
            top = fmaxf(top, fabsf(x[c][i]));
        }
    top = dpp_row_max<0x128>(top);
    top = dpp_row_max<0x124>(top);
    top = dpp_row_max<0x122>(top);
    top = dpp_row_max<0x121>(top);
    const float step = top * kStepOfMax, inv = 1.0f / step;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        // rint of the rounded quotient, from a product with the reciprocal: the two are at
        // most 127.5 * 3 * 2^-24 = 2.3e-5 apart, so the nearest whole number is the same
        // unless the product is that near to a half (one wave in ten has one)
        float z[8];
        bool near = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float y = x[c][i] * inv;
            z[i] = rintf(y);
            near |= !(fabsf(y - z[i]) <= 0.4999f);
        }
        if (__builtin_amdgcn_ballot_w64(near) != 0)
#pragma unroll 1
            for (int i = 0; i < 8; ++i) {
                float v = x[c][0];
#pragma unroll
                for (int k = 1; k < 8; ++k) v = i == k ? x[c][k] : v;
                v = (float)to_step(v, step);
#pragma unroll
                for (int k = 0; k < 8; ++k) z[k] = i == k ? v : z[k];
            }
        u32x4 b{0u, 0u, 0u, 0u};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int n = (int)z[i];
            b[i >> 2] |= ((uint32_t)min(n, 0) & 0xFFu) << (8 * (i & 3));
            b[2 + (i >> 2)] |= (uint32_t)max(n, 0) << (8 * (i & 3));
        }
        if (sub + 16 * c < 4 * KS) out.query[row][sub + 16 * c] = b;
    }
    if (sub == 0) out.steps[row] = step;
}

// The waves' LDS accesses so far, and nothing of memory.
__device__ __forceinline__ void lds_sync() {
    wave_lds_fence();
    wait_lgkmcnt0();
    lds_barrier();
    wave_lds_fence();
}

// The scores of pages [j0, j1) for the tile's tokens, as keys, that of token i and page j
// to at(i)[j].  KS: chunks of 8 dims of a lane; QT operands of 16 rows; ONE: of one token.
// A wave takes 64 pages a step, `step` pages apart, a lane the table's entry and the scale of
// one.  They are four operands of 16 pages, loaded a row by lanes beside one another (by the
// operand's layout, 16 rows beside one another, the same loads take half as long again) and
// turned in the wave's own LDS: lane 16 g + r then holds chunks g + 4 ks of row r and of page
// r, and receives rows 4 g .. + 3 of page r.  The same operand of the next step is loaded
// once this one's is in LDS, the entries a step ahead of that.  Where DUP lanes hold the same
// token and page after the maximum over the heads, each finishes another operand's.
template <int KS, int GP, int QT, bool ONE, int WAVES, typename At>
__device__ __forceinline__ void score_pages(const SelectParams &p, const Tile &tile, int kvh, int j0, int j1,
                                            int step, ScoreShared<KS, ONE ? GP : 16 * QT, WAVES> &sh, At at) {
    static_assert(!ONE || (GP >= 4 && QT == 1), "one token's rows");
    constexpr int ROWS = ONE ? GP : 16 * QT;
    constexpr int RING = ONE || KS > 4 ? 2 : 4;       // operands that are loaded ahead
    constexpr int PER = GP >= 4 ? 1 : 4 / GP;  // a lane's tokens of an operand
    constexpr int DUP = ONE ? 4 : GP >= 4 ? GP / 4 : 1;
    constexpr int LW = kRowLanes<KS>, NL = LW / 4;  // loads of an operand
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15, g = lane >> 4;
    const int hd = p.c.hd, n_ch = hd / 8;
    const int32_t *const table = p.c.table ? p.c.table + (int64_t)tile.s * p.c.width : p.b.lens;
    const bool has_table = p.c.table != nullptr;
    // (No load stands in a branch: the compiler would wait for all of them there.  Pages past
    // the end are the last one again: one row for all workgroups would be one channel of L2.)
    const auto entry = [&](int j) {
        const int e = table[has_table ? min(j, j1 - 1) : 0];
        return has_table ? e : min(j, j1 - 1);
    };
    const float *const scales = p.bounds.scales + kvh;
    const int8_t *const bounds = p.bounds.bounds + (int64_t)kvh * 2 * hd + 16 * min(lane % LW, n_ch - 1);
    const uint32_t page_step = p.c.n_kv * 2 * hd;
    struct Operand {
        u32x4 b[NL];
    };
    // a hole's row is the pool's first
    const auto in_pool = [&](int e) { return (unsigned)e < (unsigned)p.c.n_pages ? e : 0; };
    const auto load_scale = [&](int e) { return scales[(uint64_t)(uint32_t)in_pool(e) * (uint32_t)p.c.n_kv]; };
    const auto load = [&](int e, int o, Operand &S) {  // operand o of the 64 entries
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const uint32_t page = in_pool(__shfl(e, 16 * o + (64 * i + lane) / LW, 64));
            S.b[i] = load16(bounds + (uint64_t)page * page_step);
        }
    };
    for (int h0 = 0; h0 < p.group; h0 += GP) {
        int j = j0 + 64 * w;
        constexpr int QW = WAVES * 4;  // rows of queries at a time
        QueryRow<KS> q;
        if (tid / 16 < ROWS) q = load_query<KS, GP>(p, tile, kvh, h0, tid / 16);
        int ent = entry(j + lane), ent1 = entry(j + step + lane);
        // this lane's tokens and the pages that they see (-1: no token)
        int sees[QT][PER];
        uint32_t *dst[QT][PER];
#pragma unroll
        for (int t = 0; t < QT; ++t)
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int token = ONE ? 0 : t * (16 / GP) + 4 * g / GP + i;
                const bool mine = token < tile.n;
                sees[t][i] = mine ? pages_of(p, tile.pos0 + token) : -1;
                dst[t][i] = at(mine ? token : 0);
            }
        Operand S[RING];
#pragma unroll
        for (int o = 0; o < RING; ++o) load(ent, o, S[o]);
        float scale = load_scale(ent);
        lds_sync();  // the queries before are read
        if (tid / 16 < ROWS) store_query<KS>(p, q, tid / 16, sh);
        for (int row = tid / 16 + QW; row < ROWS; row += QW)
            store_query<KS>(p, load_query<KS, GP>(p, tile, kvh, h0, row), row, sh);
        lds_sync();
        i32x4 qa[QT][KS];
        f32x4 qs[QT];
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            const int row = ONE ? r % GP : 16 * t + r;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) qa[t][ks] = __builtin_bit_cast(i32x4, sh.query[row][4 * ks + g]);
            qs[t] = *reinterpret_cast<const f32x4 *>(&sh.steps[ONE ? 4 * g % GP : 16 * t + 4 * g]);
        }
        for (; j < j1; j += step) {
            const float scale1 = load_scale(ent1);
            const int ent2 = entry(j + 2 * step + lane);
            // -1: a hole, NaN: a page that is not chosen for its score
            const float mine = (unsigned)ent < (unsigned)p.c.n_pages ? (scale >= 0.0f ? scale : __builtin_nanf("")) : -1.0f;
            float x[4][QT][PER];
#pragma unroll
            for (int o = 0; o < 4; ++o) {
                wave_lds_fence();
#pragma unroll
                for (int i = 0; i < NL; ++i) sh.bound[w][(64 * i + lane) / LW][lane % LW] = S[o % RING].b[i];
                load(o + RING < 4 ? ent : ent1, (o + RING) % 4, S[o % RING]);
                wave_lds_fence();
                i32x4 dot[QT];
#pragma unroll
                for (int t = 0; t < QT; ++t) dot[t] = i32x4{0, 0, 0, 0};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    // (chunks past head_dim: any, the query's are zeros)
                    const i32x4 b = __builtin_bit_cast(i32x4, sh.bound[w][r][4 * ks + g]);
#pragma unroll
                    for (int t = 0; t < QT; ++t) dot[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(qa[t][ks], b, dot[t], 0, 0, 0);
                }
                // The largest over the heads, then times the page's scale: the order of the two
                // does not matter, rounding keeps the order of products with the same scale.
#pragma unroll
                for (int t = 0; t < QT; ++t) {
                    float y[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) y[i] = (float)dot[t][i] * qs[t][i];
                    if (GP == 1) {
#pragma unroll
                        for (int i = 0; i < PER; ++i) x[o][t][i] = y[i];
                    } else if (GP == 2) {
                        x[o][t][0] = fmaxf(y[0], y[1]);
                        x[o][t][PER - 1] = fmaxf(y[2], y[3]);
                    } else {
                        y[0] = fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]));
                        if (GP >= 8) y[0] = max_xor_rows<16>(y[0]);
                        if (GP >= 16) y[0] = max_xor_rows<32>(y[0]);
                        x[o][t][0] = y[0];
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < 4 / DUP; ++k) {
                const int o = DUP == 1 ? k : k * DUP + g % DUP;  // the operand of this lane's page
                const int page = j + 16 * o + r;
                const float s = DUP == 4 ? mine : __shfl(mine, 16 * o + r, 64);
#pragma unroll
                for (int t = 0; t < QT; ++t)
#pragma unroll
                    for (int i = 0; i < PER; ++i) {
                        float y = x[k * DUP][t][i];
#pragma unroll
                        for (int d = 1; d < DUP; ++d) y = g % DUP == d ? x[k * DUP + d][t][i] : y;
                        const int n = sees[t][i];
                        const bool always = (page < p.n_first) | (page >= n - p.n_last);
                        uint32_t key = always ? kAlways : key_of(y * s);
                        key = ((s < 0.0f) | (page >= n) | (!always & !(s >= 0.0f))) ? 0u : key;
                        if (n >= 0 && page < j1) {
                            if (GP == 16 && h0 > 0) key = max(key, dst[t][i][page]);  // (of the heads before, the same lane's)
                            dst[t][i][page] = key;
                        }
                    }
            }
            ent = ent1;
            ent1 = ent2;
            scale = scale1;
        }
    }
}

// ------------------------------------------------------------------ the choice
// The waves that share a token's keys: all of a workgroup, or one by itself.
template <int WAVES>
__device__ __forceinline__ void sync_waves() {
    if constexpr (WAVES > 1) __syncthreads();
    else wave_lds_fence();
}

// The largest over a wave, every lane getting it.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_max_from(uint32_t x) {
    return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
    x = dpp_max_from<0x111, 0xF>(x);  // row_shr:1
    x = dpp_max_from<0x112, 0xF>(x);
    x = dpp_max_from<0x114, 0xF>(x);
    x = dpp_max_from<0x118, 0xF>(x);
    x = dpp_max_from<0x142, 0xA>(x);  // row_bcast:15 into rows 1 and 3
    x = dpp_max_from<0x143, 0xC>(x);  // row_bcast:31 into rows 2 and 3
    return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}

constexpr int kTokenWaves = 8, kSplitWaves = 16;  // of a workgroup with one token
template <int WAVES>
constexpr int kHold = WAVES > 1 ? 128 / WAVES : 16;  // keys of a lane at most
template <int WAVES>
constexpr int kKeys = 64 * kHold<WAVES> * WAVES;
// (a list's pages and as many more: each time round takes some)
static_assert(kKeys<kTokenWaves> >= 2 * RXQ4_MAX_SELECT && kKeys<kSplitWaves> >= 2 * RXQ4_MAX_SELECT, "keys of a token");
constexpr int kBins = 256;
template <int WAVES>
struct PickShared {
    int hist[3][kBins];  // zeros in the first
    int sums[WAVES][4];
    uint32_t few[64];
    int n_few;           // 0
    uint32_t lowest;     // 0
    int counts[kHold<WAVES> * WAVES];  // by 64 keys: those in, and of the border's key << 16
};

// The n_select largest of a token's n <= 64 HOLD WAVES keys (0 is none), equal ones from
// the front, in order to keep(place, key, index of the key); how many.  Every key is read
// before the first is kept.
//   border  counts of 256 equal parts of the scores' range say in which one the border
//           lies; the few keys of that part are ranked (many: counts again, of the keys')
//   places  the kept of each 64 keys, and before them
template <int WAVES, int HOLD, typename Keep>
__device__ __forceinline__ int pick_of(const uint32_t *keys, int n, int n_select, PickShared<WAVES> &sh, Keep keep) {
    constexpr int T = 64 * WAVES;
    const int lane = threadIdx.x & 63, w = WAVES > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
    const int tid = WAVES > 1 ? threadIdx.x : lane;
    uint32_t x[HOLD];
    int some = 0, always = 0;
    uint32_t high = 0, low = 0;  // the largest, and of ~key
#pragma unroll
    for (int c = 0; c < HOLD; ++c) x[c] = keys[max(min(c * T + tid, n - 1), 0)];
#pragma unroll
    for (int c = 0; c < HOLD; ++c) {
        if (c * T + tid >= n) x[c] = 0;
        if (c * T >= n) continue;  // uniform
        some += __builtin_popcountll(__builtin_amdgcn_ballot_w64(x[c] != 0));
        always += __builtin_popcountll(__builtin_amdgcn_ballot_w64(x[c] == kAlways));
        const uint32_t v = x[c] == kAlways ? 0u : x[c];
        high = max(high, v);
        low = max(low, v ? ~v : 0u);
    }
    high = wave_max(high);
    low = wave_max(low);
    if constexpr (WAVES > 1) {
        if (lane == 0) *reinterpret_cast<i32x4 *>(sh.sums[w]) = i32x4{some, always, (int)high, (int)low};
        __syncthreads();
        some = always = 0;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) {
            const i32x4 v = *reinterpret_cast<const i32x4 *>(sh.sums[i]);
            some += v[0];
            always += v[1];
            high = max(high, (uint32_t)v[2]);
            low = max(low, (uint32_t)v[3]);
        }
        some = __builtin_amdgcn_readfirstlane(some);
        always = __builtin_amdgcn_readfirstlane(always);
        high = __builtin_amdgcn_readfirstlane(high);
        low = __builtin_amdgcn_readfirstlane(low);
    }
    // keys from `above` on are kept, and of those equal to `tie` the first `ties`
    uint32_t above = 1u, tie = 0u;
    int ties = 0;
    int need = n_select - always;  // of the keys in [lo, hi]: at least as many
    if (some > n_select && need <= 0) above = kAlways;
    if (some > n_select && need > 0) {
        const uint32_t lo = ~low;
        // The part of the counts that the border lies in: `need` are still needed from it, of
        // `count`.  From the top: lane l has parts 255 - 4 l, .. - 3.
        const auto part_of_border = [&](const int *hist, int &count) {
            const i32x4 c = *reinterpret_cast<const i32x4 *>(hist + kBins - 4 - 4 * lane);
            const int upto = wave_prefix(c[0] + c[1] + c[2] + c[3]);
            const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto >= need));
            need -= __builtin_amdgcn_readlane(upto - (c[0] + c[1] + c[2] + c[3]), at);
            int part = kBins - 1 - 4 * at;
#pragma unroll
            for (int i = 3; i >= 0; --i) {
                count = __builtin_amdgcn_readlane(c[i], at);
                if (need <= count) break;
                need -= count;
                --part;
            }
            return part;
        };
        // Equal parts of the scores' range first (of the keys' range most scores would be in
        // one, and LDS counts one address's a lane at a time): a score's part never falls as
        // its key rises.  Infinite scores are left to the keys.
        const float from = score_of(lo), width = score_of(high) - from, rcp = (float)kBins / width;
        const auto part_of = [&](uint32_t key) {
            return min(max((int)((score_of(key) - from) * rcp), 0), kBins - 1);
        };
        int part = -1, count = 0;
        if (width < INFINITY && rcp < INFINITY) {
#pragma unroll
            for (int c = 0; c < HOLD; ++c) {
                if (c * T >= n) continue;
                if (x[c] != 0 && x[c] != kAlways) atomicAdd(&sh.hist[0][part_of(x[c])], 1);
            }
            sync_waves<WAVES>();
            part = part_of_border(sh.hist[0], count);
        }
        if (part >= 0 && count <= 64) {
            // The part's keys, in any order; its need-th largest is the border.
#pragma unroll
            for (int c = 0; c < HOLD; ++c) {
                if (c * T >= n) continue;
                if (x[c] != 0 && x[c] != kAlways && part_of(x[c]) == part) sh.few[atomicAdd(&sh.n_few, 1)] = x[c];
            }
            sync_waves<WAVES>();
            const uint32_t v = lane < count ? sh.few[lane] : 0u;
            int larger = 0, alike = 0;
            for (int i = 0; i < count; ++i) {
                const uint32_t u = (uint32_t)__builtin_amdgcn_readlane((int)v, i);
                larger += u > v;
                alike += u == v;
            }
            const bool border = lane < count && larger < need && need <= larger + alike;
            const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(border));
            tie = (uint32_t)__builtin_amdgcn_readlane((int)v, at);
            above = tie + 1u;
            ties = need - __builtin_amdgcn_readlane(larger, at);
        } else {
            // Many in one part, or infinities: parts of the keys' range, narrowed to one key.  From
            // the part's own least key on: those below it are of the parts before, and not in the
            // counts.
            uint32_t least = lo, most = high;
            if (part >= 0) {
                uint32_t lowest = 0;
#pragma unroll
                for (int c = 0; c < HOLD; ++c)
                    if (x[c] != 0 && x[c] != kAlways && part_of(x[c]) == part) lowest = max(lowest, ~x[c]);
                lowest = wave_max(lowest);
                if (lane == 0) atomicMax(&sh.lowest, lowest);
                sync_waves<WAVES>();
                least = ~sh.lowest;
            }
            const auto mine = [&](uint32_t key) {
                return key >= least && key <= most && key != 0 && key != kAlways && (part < 0 || part_of(key) == part);
            };
            for (int turn = 1;; turn = turn == 2 ? 0 : turn + 1) {
                const int shift = max(0, 24 - __builtin_clz(most - least | 1u));
                int *const hist = sh.hist[turn];
                for (int i = tid; i < kBins; i += T) hist[i] = 0;  // (read three turns ago)
                sync_waves<WAVES>();
#pragma unroll
                for (int c = 0; c < HOLD; ++c) {
                    if (c * T >= n) continue;
                    if (mine(x[c])) atomicAdd(&hist[(x[c] - least) >> shift], 1);
                }
                sync_waves<WAVES>();
                least += (uint32_t)part_of_border(hist, count) << shift;
                if (count == need || shift == 0) break;
                most = least + min(most - least, (1u << shift) - 1u);  // (their sum may pass 2^32)
            }
            above = count == need ? least : least + 1u;
            tie = count == need ? 0u : least;
            ties = count == need ? 0 : need;
        }
    }
    // the kept of each 64 keys, in the keys' order
    int mine = 0;
#pragma unroll
    for (int c = 0; c < HOLD; ++c) {
        if (c * T >= n) continue;
        const int in = __builtin_popcountll(__builtin_amdgcn_ballot_w64(x[c] >= above));
        const int tied = ties ? __builtin_popcountll(__builtin_amdgcn_ballot_w64(x[c] == tie)) : 0;
        mine = lane == c ? in | tied << 16 : mine;
    }
    int both[2] = {mine, 0};
    if constexpr (WAVES > 1) {
        if (lane < HOLD) sh.counts[lane * WAVES + w] = mine;
        __syncthreads();
        constexpr int PL = HOLD * WAVES > 64 ? 2 : 1;  // counts of a lane
        static_assert(HOLD * WAVES <= 128, "counts of a lane");
#pragma unroll
        for (int i = 0; i < PL; ++i) both[i] = PL * lane < HOLD * WAVES ? sh.counts[lane * PL + i] : 0;
    }
    const int tied = (both[0] >> 16) + (both[1] >> 16);
    int tied_before = wave_prefix(tied) - tied, kept[2], free[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        free[i] = max(ties - tied_before, 0);  // of the ties that may still be kept
        kept[i] = (both[i] & 0xFFFF) + min(free[i], both[i] >> 16);
        tied_before += both[i] >> 16;
    }
    const int upto = wave_prefix(kept[0] + kept[1]);
    const int first[2] = {upto - kept[0] - kept[1], upto - kept[1]};
    const uint64_t below = (uint64_t(1) << lane) - 1;
#pragma unroll
    for (int c = 0; c < HOLD; ++c) {
        if (c * T >= n) continue;
        int from, room;
        if constexpr (HOLD * WAVES > 64) {  // two counts a lane
            const int e = c * WAVES + w;
            const int f0 = __builtin_amdgcn_readlane(first[0], e >> 1), f1 = __builtin_amdgcn_readlane(first[1], e >> 1);
            const int r0 = __builtin_amdgcn_readlane(free[0], e >> 1), r1 = __builtin_amdgcn_readlane(free[1], e >> 1);
            from = e & 1 ? f1 : f0;
            room = e & 1 ? r1 : r0;
        } else {
            from = __builtin_amdgcn_readlane(first[0], c * WAVES + w);
            room = __builtin_amdgcn_readlane(free[0], c * WAVES + w);
        }
        const bool over = x[c] >= above, tied_here = ties && x[c] == tie;
        const uint64_t in = __builtin_amdgcn_ballot_w64(over), same = __builtin_amdgcn_ballot_w64(tied_here);
        const int rank = __builtin_popcountll(same & below);
        if (over || (tied_here && rank < room))
            keep(from + __builtin_popcountll(in & below) + min(rank, room), x[c], c * T + tid, c);
    }
    return __builtin_amdgcn_readlane(upto, 63);
}

template <int WAVES, typename Keep>
__device__ __forceinline__ int pick(const uint32_t *keys, int n, int n_select, PickShared<WAVES> &sh, Keep keep) {
    return n <= 64 * WAVES * 4 ? pick_of<WAVES, 4>(keys, n, n_select, sh, keep)
                               : pick_of<WAVES, kHold<WAVES>>(keys, n, n_select, sh, keep);
}

// A token's list from its keys: the first `kept` with their pages in idx, key e behind them
// of page base + e - kept.  The last time into `out`, else in place; how many were kept.
template <int WAVES>
__device__ __forceinline__ int narrow(const SelectParams &p, uint32_t *keys, int *idx, int n, int kept, int base,
                                      bool last, int32_t *out, PickShared<WAVES> &sh) {
    const int tid = WAVES > 1 ? threadIdx.x : threadIdx.x & 63;
    for (int i = tid; i < kBins; i += 64 * WAVES) sh.hist[0][i] = 0;
    if (tid == 0) {
        sh.n_few = 0;
        sh.lowest = 0;
    }
    sync_waves<WAVES>();
    // (a key is kept at or before its own place, its page is that of a place as far or farther)
    const auto page = [&](int e) { return e < kept ? idx[e] : base + e - kept; };
    int m;
    if (last) {
        m = pick<WAVES>(keys, n, p.n_select, sh, [&](int at, uint32_t, int e, int) { out[at] = page(e); });
        for (int i = m + tid; i < p.n_select; i += 64 * WAVES) out[i] = -1;
    } else {
        int old[kHold<WAVES>];  // the pages of this lane's kept keys, read before any is written
#pragma unroll
        for (int c = 0; c < kHold<WAVES>; ++c) {
            const int e = c * 64 * WAVES + tid;
            old[c] = e < kept ? idx[e] : base + e - kept;
        }
        sync_waves<WAVES>();
        m = pick<WAVES>(keys, n, p.n_select, sh, [&](int at, uint32_t key, int, int c) {
            keys[at] = key;
            idx[at] = old[c];
        });
    }
    return m;
}

// A token and KV head a workgroup.  Parts of the pages one after the other, where there are
// more than LDS holds keys of.
template <int WAVES, typename Fill>
__device__ __forceinline__ void list_of_token(const SelectParams &p, const Tile &tile, int kvh, uint32_t *dyn,
                                              PickShared<WAVES> &sh, Fill fill) {
    uint32_t *const keys = dyn;
    int *const idx = reinterpret_cast<int *>(dyn + p.room);
    const int n_pages = pages_of(p, tile.pos0), part = p.room - p.n_select;  // (1 or more)
    int32_t *const out = p.pages + ((int64_t)tile.t0 * p.c.n_kv + kvh) * p.n_select;
    for (int j0 = 0, kept = 0;;) {
        const int j1 = min(n_pages, j0 + part);
        if (j1 > j0) fill(keys + kept - j0, j0, j1);
        const bool last = j1 >= n_pages;
        kept = narrow<WAVES>(p, keys, idx, kept + j1 - j0, kept, j0, last, out, sh);
        if (last) break;
        __syncthreads();
        j0 = j1;
    }
}

template <int KS, int GP>
__global__ __launch_bounds__(64 * kTokenWaves, KS > 4 ? 2 : 4) void select_token_kernel(SelectParams p) {
    extern __shared__ __attribute__((aligned(16))) uint32_t dyn[];
    __shared__ __attribute__((aligned(16))) PickShared<kTokenWaves> sh;
    __shared__ __attribute__((aligned(16))) ScoreShared<KS, GP, kTokenWaves> score;
    int kvh;
    const int t = unit_of(p, kvh);
    Tile tile;
    if (!token_of(p, t, tile)) return;  // uniform
    list_of_token<kTokenWaves>(p, tile, kvh, dyn, sh, [&](uint32_t *dst, int j0, int j1) {
        score_pages<KS, GP, 1, true, kTokenWaves>(p, tile, kvh, j0, j1, 64 * kTokenWaves, score, [&](int) { return dst; });
    });
}

// The same in two launches: the scores, a token's and KV head's pages over p.parts
// workgroups, and the choice.
constexpr int kPart = 4 * 64;
template <int KS, int GP>
__global__ __launch_bounds__(256) void score_pages_kernel(SelectParams p) {
    __shared__ __attribute__((aligned(16))) ScoreShared<KS, GP, 4> score;
    int kvh;
    const int at = unit_of(p, kvh);
    Tile tile;
    if (at >= p.b.n_tokens * p.parts || !token_of(p, at % p.b.n_tokens, tile)) return;
    const int n_pages = pages_of(p, tile.pos0);
    uint32_t *const dst = p.keys + ((int64_t)tile.t0 * p.c.n_kv + kvh) * p.stride;
    const int j0 = at / p.b.n_tokens * kPart;
    if (j0 < n_pages)
        score_pages<KS, GP, 1, true, 4>(p, tile, kvh, j0, n_pages, p.parts * kPart, score, [&](int) { return dst; });
}
__global__ __launch_bounds__(64 * kSplitWaves) void pick_pages_kernel(SelectParams p) {
    extern __shared__ __attribute__((aligned(16))) uint32_t dyn[];
    __shared__ __attribute__((aligned(16))) PickShared<kSplitWaves> sh;
    int kvh;
    const int t = unit_of(p, kvh);
    Tile tile;
    if (!token_of(p, t, tile)) return;  // uniform
    const uint32_t *src = p.keys + ((int64_t)tile.t0 * p.c.n_kv + kvh) * p.stride;
    list_of_token<kSplitWaves>(p, tile, kvh, dyn, sh, [&](uint32_t *dst, int j0, int j1) {
        for (int j = j0 + threadIdx.x; j < j1; j += 64 * kSplitWaves) dst[j] = src[j];
    });
}

// Several tokens of a sequence and a KV head a workgroup, which share the pages' bounds;
// then a wave a token.
template <int GP>
constexpr int kTileOperands = GP >= 4 ? 2 : 1;
template <int KS, int GP>
__global__ __launch_bounds__(256) void select_tile_kernel(SelectParams p) {
    constexpr int QT = kTileOperands<GP>, TOKENS = 16 * QT / GP;
    extern __shared__ __attribute__((aligned(16))) uint32_t dyn[];
    __shared__ __attribute__((aligned(16))) PickShared<1> sh[4];
    __shared__ __attribute__((aligned(16))) ScoreShared<KS, 16 * QT, 4> score;
    __shared__ int kept[TOKENS];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int kvh;
    const int u = unit_of(p, kvh);
    Tile tile;
    if (!tile_of(p, u, tile)) return;  // uniform
    uint32_t *const keys = dyn;
    int *const idx = reinterpret_cast<int *>(dyn + p.tokens * p.room);
    if (threadIdx.x < TOKENS) kept[threadIdx.x] = 0;
    __syncthreads();
    const int n_pages = pages_of(p, tile.pos0 + tile.n - 1), part = p.room - p.n_select;
    for (int j0 = 0;;) {
        const int j1 = min(n_pages, j0 + part);
        if (j1 > j0)
            score_pages<KS, GP, QT, false, 4>(p, tile, kvh, j0, j1, 256, score,
                                    [&](int i) { return keys + i * p.room + kept[i] - j0; });
        __syncthreads();
        const bool last = j1 >= n_pages;
        for (int i = w; i < tile.n; i += 4) {
            const int before = kept[i];
            const int n = narrow<1>(p, keys + i * p.room, idx + i * p.n_select, before + j1 - j0, before, j0, last,
                                    p.pages + ((int64_t)(tile.t0 + i) * p.c.n_kv + kvh) * p.n_select, sh[w]);
            wave_lds_fence();
            if ((threadIdx.x & 63) == 0) kept[i] = n;
        }
        if (last) break;
        __syncthreads();
        j0 = j1;
    }
}

template <int KS, int GP>
hipError_t launch_tiles(SelectParams &p, int64_t pages, hipStream_t st) {
    p.tokens = 16 * kTileOperands<GP> / GP;
    p.room = (int)std::min<int64_t>(kKeys<1>, pages + p.n_select);
    const int64_t units = (p.b.n_tokens + p.tokens - 1) / p.tokens + p.b.n_seqs;
    const int64_t grid = units_grid(units, p.c.n_kv);
    if (grid > kMostWorkgroups) return hipErrorInvalidValue;
    select_tile_kernel<KS, GP><<<(unsigned)grid, 256, (size_t)p.tokens * (p.room + p.n_select) * 4, st>>>(p);
    return hipGetLastError();
}

template <int KS, int GP>
hipError_t launch_tokens(SelectParams &p, int64_t pages, hipStream_t st) {
    const int cus = device_info().cu_count > 0 ? device_info().cu_count : 256;
    const int64_t heads = (int64_t)p.b.n_tokens * p.c.n_kv;
    if (units_grid(p.b.n_tokens, p.c.n_kv) > kMostWorkgroups) return hipErrorInvalidValue;
    const unsigned grid = (unsigned)units_grid(p.b.n_tokens, p.c.n_kv);
    // Few tokens with many pages: the scores on more workgroups than one a token and KV head, as
    // many as two a CU.  Measured, us of one launch / two, pages of 16, one token of 32 / 8 heads:
    // 384 pages 9.5 / 10.8, 512 9.7 / 10.8, 768 11.1 / 10.9, 2048 18 / 12, 4096 30 / 13; 12 tokens 512
    // 10.6 / 11.2, 1024 14 / 13, 2048 20 / 20, 4096 34 / 28, 24 tokens 2048 26 / 27, 4096 45 / 44; at
    // head_dim 64 two launches pay later (512 7.2 / 9.3, 1024 8.5 / 9.9, 2048 11.1 / 10.6).
    const int64_t parts = std::min<int64_t>((pages + kPart - 1) / kPart, 2 * cus / heads);
    if (pages >= 512 && parts > 1 && heads * pages * 4 <= (int64_t)kWorkspaceBytes) {
        float *ws = nullptr;
        const hipError_t e = Scratch{}.get(st, heads * pages * 4, &ws);
        if (e != hipSuccess) return e;
        p.keys = reinterpret_cast<uint32_t *>(ws);
        p.stride = (int)pages;
        p.parts = (int)parts;
        p.room = (int)std::min<int64_t>(kKeys<kSplitWaves>, pages + p.n_select);
        score_pages_kernel<KS, GP><<<(unsigned)units_grid(p.b.n_tokens * parts, p.c.n_kv), 256, 0, st>>>(p);
        pick_pages_kernel<<<grid, 64 * kSplitWaves, (size_t)(p.room + p.n_select) * 4, st>>>(p);
    } else {
        p.room = (int)std::min<int64_t>(kKeys<kTokenWaves>, pages + p.n_select);
        select_token_kernel<KS, GP><<<grid, 64 * kTokenWaves, (size_t)(p.room + p.n_select) * 4, st>>>(p);
    }
    return hipGetLastError();
}

// Tiles where the tokens' KV heads are enough to fill the CUs: a token's whole workgroup scores
// and chooses for it, a tile's wave walks a token's keys part after part.  So about one and a half
// a CU for few pages (3/4 of the two workgroups of a CU), two more for each part of pages, three at
// most (max_len may be far above the lengths); at head_dim above 128, where a CU holds one of the
// tokens' workgroups, 3/4 of that, with groups of one head, of which a tile has 16, 3/2.  Groups
// above 8 heads leave a tile one or two tokens: tiles in one part alone.
// Measured, us of tokens / tiles, pages of 16, lists of 64, one sequence of 32 / 8 heads after
// 60000 positions: 4 new tokens 15 / 74, 32 30 / 106, 256 150 / 107; after 30000, 64 28 / 55, 128 48 /
// 55, 256 86 / 57; after 5000, 64 13 / 19, 128 22 / 20; 28 / 4 heads after 30000, 128 25 / 39, 256 44 / 39;
// 8 / 8 heads of 64, 256 55 / 80, 512 97 / 80; 64 / 4 heads of 64, 512 54 / 73, after 1000 29 / 19.  256
// sequences of two new tokens 76 / 54, 32 of three 38 / 40, 32 of eight 64 / 52.  Over 1042 such calls
// the side taken is at worst 1.6 times the better one, 1.01 in the mean, in 42 more than 1.1.
bool takes_tiles(const SelectParams &p, int64_t pages) {
    const int64_t cus = device_info().cu_count > 0 ? device_info().cu_count : 256;
    if (p.n_select > kKeys<1> / 2) return false;
    if (units_grid(p.b.n_tokens, p.c.n_kv) > kMostWorkgroups) return true;  // (a token a workgroup is too many)
    if (p.b.max_new < 2 || p.b.n_tokens < 2 * (int64_t)p.b.n_seqs) return false;
    const int64_t part = kKeys<1> - p.n_select, heads = (int64_t)p.b.n_tokens * p.c.n_kv;
    if (p.group > 8 && pages > part) return false;
    // heads >= (3/4 + pages / part) * 2 cus * (3/4 or 1) * (3/2 or 1)
    return 16 * heads * part >= (3 * part + 4 * std::min(pages, 3 * part)) * cus * (p.c.hd > 128 ? 3 : 4) * (p.group == 1 ? 3 : 2);
}

template <int KS>
hipError_t launch_select(SelectParams p, hipStream_t st) {
    // the pages that a sequence may have
    const int64_t most = (std::min<int64_t>(p.b.max_len, (int64_t)p.c.width << p.c.shift) + (1 << p.c.shift) - 1) >> p.c.shift;
    const int64_t pages = std::max<int64_t>(128, (most + 127) / 128 * 128);
    if (takes_tiles(p, most)) {
        if (p.group == 1) return launch_tiles<KS, 1>(p, pages, st);
        if (p.group == 2) return launch_tiles<KS, 2>(p, pages, st);
        if (p.group <= 4) return launch_tiles<KS, 4>(p, pages, st);
        if (p.group <= 8) return launch_tiles<KS, 8>(p, pages, st);
        return launch_tiles<KS, 16>(p, pages, st);
    }
    if (p.group <= 4) return launch_tokens<KS, 4>(p, pages, st);
    if (p.group <= 8) return launch_tokens<KS, 8>(p, pages, st);
    return launch_tokens<KS, 16>(p, pages, st);
}

}  // namespace

hipError_t launch_kv_bounds(const PageBounds &bounds, const SeqBatch &batch, const PagedCache &cache,
                            int kv_int8, hipStream_t st) {
    // Few rows: one a workgroup; many: as many as leave a thousand workgroups, a page's at most
    // (those without a page's first row end after the lookup of their sequence).
    const int heads = kPieces / (cache.hd / 8), parts = (cache.n_kv + heads - 1) / heads;
    const int64_t rows = (int64_t)batch.n_tokens * parts / 1024;
    BoundsParams p{bounds, batch, cache, (int)std::max<int64_t>(1, std::min<int64_t>(1 << cache.shift, rows))};
    const dim3 grid((batch.n_tokens + p.rows_wg - 1) / p.rows_wg, parts);
    if (kv_int8) kv_bounds_kernel<true><<<grid, 256, 0, st>>>(p);
    else kv_bounds_kernel<false><<<grid, 256, 0, st>>>(p);
    return hipGetLastError();
}

hipError_t launch_select_pages(int32_t *pages, int n_select, int n_first, int n_last, const uint16_t *q,
                               int n_heads, const PageBounds &bounds, const SeqBatch &batch,
                               const PagedCache &cache, hipStream_t st) {
    SelectParams p{};
    p.pages = pages;
    p.q = q;
    p.bounds = bounds;
    p.b = batch;
    p.c = cache;
    p.n_heads = n_heads;
    p.group = n_heads / cache.n_kv;
    p.n_select = n_select;
    p.n_first = n_first;
    p.n_last = n_last;
    if (cache.hd <= 64) return launch_select<2>(p, st);
    if (cache.hd <= 96) return launch_select<3>(p, st);
    if (cache.hd <= 128) return launch_select<4>(p, st);
    return launch_select<8>(p, st);
}

}  // namespace rxq4
