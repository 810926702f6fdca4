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
    constexpr int U = 4;
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
    int gp;       // rows of a token in a tile: the group's heads, a power of two up to 16
    int tokens;   // of a tile at most
    int room;     // keys of a token in LDS
    uint32_t *keys;  // split: [n_tokens][n_kv][stride]
    int stride;
    int parts;    // split: workgroups of a token and KV head
};

// Bits that order as the numbers do, above 0; -0 as 0.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The tokens of a tile: rows [t0, t0 + n) of the batch, all of sequence s; the first at pos0.
struct Tile {
    int s, t0, n, pos0;
};
__device__ __forceinline__ int pages_of(const SelectParams &p, int pos) {
    const int sees = min(position_limit(p.b, p.c), pos + 1);
    return sees > 0 ? ((sees - 1) >> p.c.shift) + 1 : 0;
}
// Unit u of the first ceil(n_tokens / tokens): the rows from u * tokens up to the next such
// row that are of the sequence of the first; the units behind them: a sequence's rows
// before its first multiple of `tokens`.  Every row is in one.
__device__ __forceinline__ bool tile_of(const SelectParams &p, int u, Tile &tile) {
    const int whole = (p.b.n_tokens + p.tokens - 1) / p.tokens;
    SeqSpan span;
    int from;
    if (u < whole) {
        from = u * p.tokens;
        tile.s = seq_of_row(p.b, from, span);
        if (tile.s >= p.b.n_seqs || from < span.row0) return false;
    } else {
        tile.s = u - whole;
        span = seq_span(p.b, tile.s);
        from = span.row0;
        if (from % p.tokens == 0) return false;  // a unit of the first kind
    }
    const int to = min((from / p.tokens + 1) * p.tokens, span.row0 + min(span.n, p.b.max_new));
    tile.t0 = from;
    tile.n = to - from;
    tile.pos0 = span.pos0 + (from - span.row0);
    return tile.n > 0;
}

// The scores of pages [j0, j1) for the tile's tokens, as keys: of token i, page j at
// dst[i * pitch + j - j0 + skip[i]].  KS: chunks of 8 dims of a lane.  A wave takes 32 pages
// at a time, the operand's columns; its rows are the queries, lane 16 g + r holding chunks
// g + 4 ks of row and page r and receiving rows 4 g .. + 3 of page r.
template <int KS, typename Place>
__device__ __forceinline__ void score_pages(const SelectParams &p, const Tile &tile, int kvh, int j0, int j1,
                                            int step, float *qsteps, Place place) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const int hd = p.c.hd, n_ch = hd / 8;
    const int32_t *const table = p.c.table ? p.c.table + (int64_t)tile.s * p.c.width : nullptr;
    const auto page_of = [&](int j) {
        const int page = table ? table[min(j, j1 - 1)] : j;
        return j < j1 && (unsigned)page < (unsigned)p.c.n_pages ? page : -1;
    };
    // this lane's tokens of a page: those of rows 4 g .. + 3
    const int per = p.gp >= 4 ? 1 : 4 / p.gp, first = 4 * g / p.gp;
    const bool mine = p.gp < 8 || g % (p.gp / 4) == 0;
    for (int h0 = 0; h0 < p.group; h0 += p.gp) {
        const int tok = min(r / p.gp, tile.n - 1), head = kvh * p.group + min(h0 + r % p.gp, p.group - 1);
        const uint16_t *q = p.q + ((int64_t)(tile.t0 + tok) * p.n_heads + head) * hd;
        u32x4 raw[KS];
        float top = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int ch = 4 * ks + g;
            raw[ks] = ch < n_ch ? load16(q + 8 * ch) : u32x4{0u, 0u, 0u, 0u};
        }
        const auto value = [&](int ks, int i) {  // NaN as 0, infinities as fp16's largest
            const float x = f16_bits_to_f32(raw[ks][i >> 1] >> (16 * (i & 1)) & 0xFFFFu);
            return x == x ? fminf(fmaxf(x, -65504.0f), 65504.0f) : 0.0f;
        };
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(value(ks, i)));
        top = max_xor_rows<16>(top);
        top = max_xor_rows<32>(top);
        const float qstep = top * kStepOfMax;
        i32x4 qa[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            uint32_t b[4] = {0u, 0u, 0u, 0u};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int z = to_step(value(ks, i), qstep);
                b[i >> 2] |= ((uint32_t)min(z, 0) & 0xFFu) << (8 * (i & 3));
                b[2 + (i >> 2)] |= (uint32_t)max(z, 0) << (8 * (i & 3));
            }
            qa[ks] = i32x4{(int)b[0], (int)b[1], (int)b[2], (int)b[3]};
        }
        float *const mysteps = qsteps + 16 * w;
        wave_lds_fence();
        if (g == 0) mysteps[r] = qstep;
        wave_lds_fence();
        const f32x4 qs = *reinterpret_cast<const f32x4 *>(mysteps + 4 * g);

        int j = j0 + 32 * w;
        int page[2] = {page_of(j + r), page_of(j + 16 + r)};
        for (; j < j1; j += step) {
            const int next[2] = {page_of(j + step + r), page_of(j + step + 16 + r)};
            i32x4 bound[2][KS];
            float scale[2];
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                const int64_t row = (int64_t)max(page[st], 0) * p.c.n_kv + kvh;
                scale[st] = p.bounds.scales[row];
                const int8_t *src = p.bounds.bounds + row * 2 * hd;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
                    bound[st][ks] = __builtin_bit_cast(i32x4, load16(src + 16 * min(4 * ks + g, n_ch - 1)));
            }
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                i32x4 dot{0, 0, 0, 0};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)  // (chunks past head_dim: the query's are zeros)
                    dot = __builtin_amdgcn_mfma_i32_16x16x64_i8(qa[ks], bound[st][ks], dot, 0, 0, 0);
                float x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = (float)dot[i] * qs[i] * scale[st];
                if (p.gp >= 2) {
                    x[0] = fmaxf(x[0], x[1]);
                    x[1] = fmaxf(x[2], x[3]);
                }
                if (p.gp >= 4) x[0] = fmaxf(x[0], x[1]);
                if (p.gp >= 8) x[0] = max_xor_rows<16>(x[0]);
                if (p.gp >= 16) x[0] = max_xor_rows<32>(x[0]);
                const int at = j + 16 * st + r;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int token = first + i;
                    if (i >= per || !mine || token >= tile.n || at >= j1) continue;
                    const int n = pages_of(p, tile.pos0 + token);
                    uint32_t key = page[st] < 0 || at >= n ? 0u
                                   : at < p.n_first || at >= n - p.n_last ? kAlways : key_of(x[i]);
                    uint32_t *dst = place(token, at);
                    if (h0 > 0) key = max(key, *dst);  // (the same lane's, of the heads before)
                    *dst = key;
                }
            }
            page[0] = next[0];
            page[1] = next[1];
        }
    }
}

// ------------------------------------------------------------------ the choice
// Keys of a token, in the order of their pages: the first `kept` with their pages in idx,
// key e behind them of page base + e - kept.
struct Keys {
    uint32_t *key;
    int *idx;
    int n, kept, base;
};

// WAVES waves: all four of a workgroup, or one by itself.
template <int WAVES>
__device__ __forceinline__ void sync_waves() {
    if constexpr (WAVES == 4) __syncthreads();
    else wave_lds_fence();
}

struct Border {
    uint32_t above;  // keys from it on are kept whatever their number
    uint32_t tie;    // of the keys equal to it
    int ties;        // the first so many
};

// The border of the n_select largest keys (0 is none): counts of 256 equal parts of the
// range that the border lies in, until a part is one key or is kept whole.
template <int WAVES>
__device__ __forceinline__ Border find_border(const Keys &k, int n_select, int *hist, int *sums) {
    const int lane = threadIdx.x & 63, tid = WAVES == 4 ? threadIdx.x : lane, w = threadIdx.x >> 6;
    int some = 0, always = 0;
    uint32_t lo = kAlways, hi = 0;
    for (int e = tid; e < k.n; e += 64 * WAVES) {
        const uint32_t x = k.key[e];
        some += x != 0;
        always += x == kAlways;
        if (x != 0 && x != kAlways) {
            lo = min(lo, x);
            hi = max(hi, x);
        }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        some += __shfl_xor(some, off, 64);
        always += __shfl_xor(always, off, 64);
        lo = min(lo, (uint32_t)__shfl_xor((int)lo, off, 64));
        hi = max(hi, (uint32_t)__shfl_xor((int)hi, off, 64));
    }
    if constexpr (WAVES == 4) {
        __syncthreads();
        if (lane == 0) {
            sums[w] = some;
            sums[4 + w] = always;
            sums[8 + w] = (int)lo;
            sums[12 + w] = (int)hi;
        }
        __syncthreads();
        some = sums[0] + sums[1] + sums[2] + sums[3];
        always = sums[4] + sums[5] + sums[6] + sums[7];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            lo = min(lo, (uint32_t)sums[8 + i]);
            hi = max(hi, (uint32_t)sums[12 + i]);
        }
    }
    if (some <= n_select) return Border{1u, 0u, 0};
    int need = n_select - always;  // of the keys in [lo, hi]: at least as many
    if (need <= 0) return Border{kAlways, 0u, 0};
    for (;;) {
        const int shift = max(0, 24 - __builtin_clz(hi - lo | 1u));
        sync_waves<WAVES>();  // the counts before are read
        for (int i = tid; i < 256; i += 64 * WAVES) hist[i] = 0;
        sync_waves<WAVES>();
        for (int e = tid; e < k.n; e += 64 * WAVES) {
            const uint32_t x = k.key[e];
            if (x >= lo && x <= hi) atomicAdd(&hist[(x - lo) >> shift], 1);
        }
        sync_waves<WAVES>();
        // from the top: lane l has parts 255 - 4 l, .. - 3
        const i32x4 c = *reinterpret_cast<const i32x4 *>(hist + 252 - 4 * lane);
        const int upto = wave_prefix(c[0] + c[1] + c[2] + c[3]);
        const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto >= need));
        int above = __builtin_amdgcn_readlane(upto - (c[0] + c[1] + c[2] + c[3]), at);
        int part = 255 - 4 * at, count = 0;
#pragma unroll
        for (int i = 3; i >= 0; --i) {
            count = __builtin_amdgcn_readlane(c[i], at);
            if (above + count >= need) break;
            above += count;
            --part;
        }
        need -= above;
        lo += (uint32_t)part << shift;
        if (count == need) return Border{lo, 0u, 0};
        if (shift == 0) return Border{lo + 1u, lo, need};
        hi = min(hi, lo + ((1u << shift) - 1u));
    }
}

// The keys within the border, in order, to keep(place, key, page); how many.  (`keep` may
// write the keys' own first places: a key's place is not behind it, and what lies there has
// been read.)
template <int WAVES, typename Keep>
__device__ __forceinline__ int keep_keys(const Keys &k, const Border &b, int *sums, Keep keep) {
    const int lane = threadIdx.x & 63, tid = WAVES == 4 ? threadIdx.x : lane, w = threadIdx.x >> 6;
    const uint64_t below = (uint64_t(1) << lane) - 1;
    int out = 0, ties = 0;
    if constexpr (WAVES == 4) __syncthreads();
    for (int e0 = 0, odd = 0; e0 < k.n; e0 += 64 * WAVES, odd ^= 8) {
        const int e = e0 + tid;
        const uint32_t x = e < k.n ? k.key[e] : 0u;
        const int page = e < k.kept ? k.idx[e] : k.base + e - k.kept;
        const bool tie = x != 0u && x == b.tie;
        const uint64_t in = __builtin_amdgcn_ballot_w64(x >= b.above), tied = __builtin_amdgcn_ballot_w64(tie);
        int in_before = 0, ties_before = 0, in_all = __builtin_popcountll(in), ties_all = __builtin_popcountll(tied);
        if constexpr (WAVES == 4) {
            if (lane == 0) {
                sums[odd + w] = in_all;
                sums[odd + 4 + w] = ties_all;
            }
            __syncthreads();
            in_all = ties_all = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int a = sums[odd + i], c = sums[odd + 4 + i];
                in_before += i < w ? a : 0;
                ties_before += i < w ? c : 0;
                in_all += a;
                ties_all += c;
            }
        } else {
            wave_lds_fence();
        }
        // of the ties those that are still free
        const int free = max(b.ties - ties, 0);
        const int my_tie = ties_before + __builtin_popcountll(tied & below);
        if (x >= b.above || (tie && my_tie < free))
            keep(out + in_before + __builtin_popcountll(in & below) + min(my_tie, free), x, page);
        out += in_all + min(ties_all, free);
        ties += ties_all;
    }
    return out;
}

// The tokens' lists.  LDS: room keys and n_select kept pages a token.
struct SelectShared {
    int hist[4][256];
    int sums[4][16];
    float qsteps[64];
};

template <int WAVES>
__device__ __forceinline__ int narrow(const SelectParams &p, Keys &k, bool last, int32_t *out, SelectShared &sh) {
    const int w = WAVES == 4 ? 0 : threadIdx.x >> 6;
    const Border b = find_border<WAVES>(k, p.n_select, sh.hist[w], sh.sums[w]);
    int n;
    if (last) {
        n = keep_keys<WAVES>(k, b, sh.sums[w], [&](int at, uint32_t, int page) { out[at] = page; });
        for (int i = n + (WAVES == 4 ? threadIdx.x : threadIdx.x & 63); i < p.n_select; i += 64 * WAVES) out[i] = -1;
    } else {
        n = keep_keys<WAVES>(k, b, sh.sums[w], [&](int at, uint32_t key, int page) {
            k.key[at] = key;
            k.idx[at] = page;
        });
    }
    return n;
}

// SPLIT: the keys are read from p.keys, a token and KV head a workgroup.
template <int KS, bool SPLIT>
__global__ __launch_bounds__(256) void select_pages_kernel(SelectParams p) {
    extern __shared__ __attribute__((aligned(16))) uint32_t dyn[];
    __shared__ __attribute__((aligned(16))) SelectShared sh;
    __shared__ int kept[16];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), kvh = blockIdx.x % p.c.n_kv;
    Tile tile;
    if (!tile_of(p, blockIdx.x / p.c.n_kv, tile)) return;  // uniform
    uint32_t *const keys = dyn;
    int *const idx = reinterpret_cast<int *>(dyn + p.tokens * p.room);
    if (threadIdx.x < 16) kept[threadIdx.x] = 0;
    __syncthreads();
    const int n_pages = pages_of(p, tile.pos0 + tile.n - 1);
    const int part = p.room - p.n_select;  // pages at a time
    int j0 = 0;
    do {
        const int j1 = min(n_pages, j0 + part);
        const bool last = j1 >= n_pages;
        if constexpr (SPLIT) {
            const uint32_t *src = p.keys + ((int64_t)tile.t0 * p.c.n_kv + kvh) * p.stride;
            const int k0 = kept[0] - j0;
            for (int j = j0 + threadIdx.x; j < j1; j += 256) keys[k0 + j] = src[j];
        } else if (j1 > j0) {
            score_pages<KS>(p, tile, kvh, j0, j1, 128, sh.qsteps,
                            [&](int token, int j) { return keys + token * p.room + kept[token] + j - j0; });
        }
        __syncthreads();
        const auto token = [&](int i) {
            return Keys{keys + i * p.room, idx + i * p.n_select, kept[i] + j1 - j0, kept[i], j0};
        };
        const auto out = [&](int i) {
            return p.pages + ((int64_t)(tile.t0 + i) * p.c.n_kv + kvh) * p.n_select;
        };
        // several tokens: a wave each; else all waves on one after the other
        if (tile.n > 2) {
            for (int i = w; i < tile.n; i += 4) {
                Keys k = token(i);
                const int n = narrow<1>(p, k, last, out(i), sh);
                wave_lds_fence();
                if ((threadIdx.x & 63) == 0) kept[i] = n;
            }
        } else {
            for (int i = 0; i < tile.n; ++i) {
                Keys k = token(i);
                const int n = narrow<4>(p, k, last, out(i), sh);
                __syncthreads();
                if (threadIdx.x == 0) kept[i] = n;
            }
        }
        __syncthreads();
        j0 = j1;
    } while (j0 < n_pages);
}

// SPLIT: the scores alone, parts of 128 pages over p.parts workgroups.
template <int KS>
__global__ __launch_bounds__(256) void score_pages_kernel(SelectParams p) {
    __shared__ __attribute__((aligned(16))) float qsteps[64];
    const int kvh = blockIdx.x % p.c.n_kv, at = blockIdx.x / p.c.n_kv;
    Tile tile;
    if (!tile_of(p, at / p.parts, tile)) return;
    const int n_pages = pages_of(p, tile.pos0);
    uint32_t *const dst = p.keys + ((int64_t)tile.t0 * p.c.n_kv + kvh) * p.stride;
    const int j0 = at % p.parts * 128;
    if (j0 < n_pages)
        score_pages<KS>(p, tile, kvh, j0, n_pages, p.parts * 128, qsteps, [&](int, int j) { return dst + j; });
}

template <int KS>
hipError_t launch_select(SelectParams p, hipStream_t st) {
    const int cus = device_info().cu_count > 0 ? device_info().cu_count : 256;
    // the pages that a sequence may have, in whole parts of 128
    const int64_t most = (std::min<int64_t>(p.b.max_len, (int64_t)p.c.width << p.c.shift) + (1 << p.c.shift) - 1) >> p.c.shift;
    const int64_t pages = std::max<int64_t>(128, (most + 127) / 128 * 128);
    p.gp = 1;
    while (p.gp < p.group && p.gp < 16) p.gp *= 2;
    // tokens of a tile: the rows of the operand, where the sequences have some
    p.tokens = p.b.n_tokens < 4 * (int64_t)p.b.n_seqs || p.b.max_new == 1 ? 1 : 16 / p.gp;
    constexpr int kLds = 48 << 10;
    const auto room = [&](int tokens) { return (int64_t)kLds / 4 / tokens - p.n_select; };
    while (p.tokens > 1 && room(p.tokens) < p.n_select + 256) p.tokens /= 2;
    p.room = (int)std::min<int64_t>(room(p.tokens), pages + p.n_select);
    const int64_t units = (p.b.n_tokens + p.tokens - 1) / p.tokens + (p.tokens > 1 ? p.b.n_seqs : 0);
    // Few tokens with many pages: the scores on more workgroups than one a token and KV head.
    const int64_t heads = (int64_t)p.b.n_tokens * p.c.n_kv;
    const int64_t parts = std::min<int64_t>(pages / 128, 2 * cus / std::max<int64_t>(heads, 1));
    if (p.tokens == 1 && pages >= 1024 && parts > 1 && heads * pages * 4 <= (int64_t)kWorkspaceBytes) {
        float *ws = nullptr;
        const hipError_t e = Scratch{}.get(st, heads * pages * 4, &ws);
        if (e != hipSuccess) return e;
        p.keys = reinterpret_cast<uint32_t *>(ws);
        p.stride = (int)pages;
        p.parts = (int)parts;
        score_pages_kernel<KS><<<(unsigned)(units * p.c.n_kv * parts), 256, 0, st>>>(p);
        select_pages_kernel<2, true><<<(unsigned)(units * p.c.n_kv), 256, (p.room + p.n_select) * 4, st>>>(p);
        return hipGetLastError();
    }
    if (units * p.c.n_kv > 0x7FFFFF) return hipErrorInvalidValue;
    select_pages_kernel<KS, false><<<(unsigned)(units * p.c.n_kv), 256, (size_t)p.tokens * (p.room + p.n_select) * 4, st>>>(p);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_kv_bounds(const PageBounds &bounds, const SeqBatch &batch, const PagedCache &cache,
                            int kv_int8, hipStream_t st) {
    // Few rows: one a workgroup; many: as many as leave some thousand workgroups, a page's at most.
    BoundsParams p{bounds, batch, cache, std::max(1, std::min(1 << cache.shift, batch.n_tokens / 1024))};
    const int heads = kPieces / (cache.hd / 8);
    const dim3 grid((batch.n_tokens + p.rows_wg - 1) / p.rows_wg, (cache.n_kv + heads - 1) / heads);
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
