// attn_paged.hip -- attention of a batch's new tokens over a paged KV cache, on
// the gfx950 matrix cores.
//
// Token at position p, head h: out = sum_j e^(s_j) v_j / sum_j e^(s_j) over the
// positions j <= p whose page is in the pool, s_j = scale q.k_j, KV head h /
// group; the sums relative to a running maximum, in fp32.
//
// Query rows.  The rows of a sequence and KV head are numbered t * group + j (new
// token t, j-th head of the group).  A workgroup takes 16 of them, the columns of
// a 16 x 16 MFMA tile, and one chunk of positions: each K and V row is read once
// for all of them.
//
// Bound: reading the cache, in pieces of a head's row (256 bytes at head_dim 128,
// fp16).  Loops that do nothing else read such pieces, 8 heads' rows together, at 5.3 to
// 5.8 TB/s, by which lane and XCD takes what, 128-byte pieces of int8 at 4.9 to 5.4, and
// 4 KB pieces at 6.0.  So a step's loads are issued a step ahead, nothing of K passes
// LDS, and the chunks are cut from the batch's own lengths, which only the device knows
// (up to kSeqs sequences).
// Attention over listed pages is the same walk over the places of a list (`Lists` below).
// Measured, 32 / 8 heads of 128, one new token a sequence, pages of 16: 512
// sequences of 1023 positions 372 us (5.8 TB/s), 256 of 2047 397 (5.4), 64 of 64 to
// 8000 92 (4.7); int8 512 of 1023 231 (4.8; pages of 64 221), 256 of 2047 246 (4.5), 16
// of 20000 to 40000, pages of 64, 202 (4.9).  A call's fixed part (launch, first loads,
// the chunks' ends, the combine) is about 20 us at 64 sequences and 8 at one.
#include <math.h>

#include <algorithm>

#include "attn_paged.h"
#include "attn_tile.h"
#include "launch.h"
#include "mfma_util.h"
#include "paged.h"
#include "q4k_device.h"

namespace rxq4 {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int kStep = 128;      // positions per step of a workgroup
constexpr int kNoStep = 1 << 22;  // past every position (2^24 at most): its loads are past the end
constexpr int kMaxChunks = 64;  // chunks of positions per sequence
constexpr int kSeqs = 256;      // sequences whose chunks a workgroup counts itself

typedef const float __attribute__((address_space(1))) *GlobalFloat;
__device__ const float g_one = 1.0f;  // int8 caches without scales: read with stride 0

__device__ __forceinline__ float log2_scale(float vs) {
    return fminf(fmaxf(__builtin_amdgcn_logf(fabsf(vs)), kMinScale), kMaxScale);
}

// Waves per SIMD that the registers are cut to: what is in flight is what counts, and
// an int8 step holds half the bytes of an fp16 one.  (With a list's page beside the entry,
// small fp16 pages spill at four.)
enum Lists { kNoLists, kTokenLists, kTileLists, kWideTileLists };  // (at the kernel)
constexpr int rows_waves(int hd, bool i8, bool big, Lists lists) {
    if (hd > 128) return 1;
    if (lists == kWideTileLists) return hd == 64 ? 3 : 2;
    if (lists == kTileLists) return hd == 64 ? 4 : 3;
    return hd == 64 ? (lists == kTokenLists && !i8 && !big ? 3 : 4) : i8 ? 3 : 2;
}

// Steps of the walk over a sequence (0: not this kernel's; one where its tokens see
// nothing, to write their zeros).
__device__ __forceinline__ int seq_steps(const PagedParams &p, const SeqSpan &span) {
    const int n = min(span.n, p.b.max_new);
    if (n == 0 || n * p.group > kPagedRows) return 0;
    return (max(min(span.pos0 + n, position_limit(p.b, p.c)), 1) + kStep - 1) / kStep;
}

// The chunks of the batch, sequence after sequence: of at most so many steps that there
// are about p.max_units, a sequence's about equally long.  Lane l holds the sequences
// per l, .. per l + per - 1; the same in every wave, from the same sums.
constexpr int kPer = kSeqs / 64;
struct RowsUnits {
    int per;
    SeqSpan span[kPer];
    int steps[kPer], chunks[kPer];
    int upto;  // chunks up to the lane's last
};
__device__ __forceinline__ RowsUnits rows_units(const PagedParams &p) {
    RowsUnits u{};
    const int lane = threadIdx.x & 63;
    u.per = (p.b.n_seqs + 63) >> 6;
    int all = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
        if (i < u.per) {  // uniform
            const int s = lane * u.per + i;
            u.span[i] = seq_span(p.b, min(s, p.b.n_seqs - 1));
            u.steps[i] = s < p.b.n_seqs ? seq_steps(p, u.span[i]) : 0;
            all += u.steps[i];
        }
    all = __builtin_amdgcn_readlane(wave_prefix(all), 63);
    // (a few short sequences: one step a chunk, no division)
    const int most = all <= p.max_units ? p.min_tiles : max(p.min_tiles, (all + p.max_units - 1) / p.max_units);
#pragma unroll
    for (int i = 0; i < kPer; ++i)
        if (i < u.per) {
            u.chunks[i] = most == 1 ? u.steps[i] : (u.steps[i] + most - 1) / most;
            u.upto += u.chunks[i];
        }
    u.upto = wave_prefix(u.upto);
    return u;
}

// A chunk of a sequence's steps.  With more than kSeqs sequences the chunks are of
// p.chunk positions, every sequence with p.n_chunks of them.
struct RowsUnit {
    SeqSpan span;
    int s, c;           // sequence (-1: none), chunk
    int chunks, chunk;  // chunks of the sequence; positions of each
    int64_t slot;       // of the chunk's partials
    int tok;            // listed pages: the (first) token of the sequence
    int tokens;         // a tile's
};
__device__ __forceinline__ RowsUnit rows_unit(const PagedParams &p, int idx) {
    RowsUnit r{};
    r.s = -1;
    if (p.n_chunks == 1 || p.b.n_seqs > kSeqs) {
        // (a sequence's chunks on different XCDs)
        r.c = idx / p.b.n_seqs;
        if (r.c >= p.n_chunks) return r;
        const int s = (idx + 3 * r.c) % p.b.n_seqs;
        r.span = seq_span(p.b, s);
        r.chunk = p.chunk;
        r.chunks = (seq_steps(p, r.span) * kStep + p.chunk - 1) / p.chunk;
        r.slot = (int64_t)s * p.n_chunks + r.c;
        if (r.c < r.chunks) r.s = s;
        return r;
    }
    const RowsUnits u = rows_units(p);
    const uint64_t past = __builtin_amdgcn_ballot_w64(u.upto > idx);
    if (past == 0) return r;
    const int at = __builtin_ctzll(past);
    int c = idx - __builtin_amdgcn_readlane(u.upto, at);
#pragma unroll
    for (int i = 0; i < kPer; ++i) c += __builtin_amdgcn_readlane(u.chunks[i], at);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int chunks = __builtin_amdgcn_readlane(u.chunks[i], at);
        if (c >= 0 && c < chunks) {
            const int n = __builtin_amdgcn_readlane(u.steps[i], at);
            r.span = SeqSpan{__builtin_amdgcn_readlane(u.span[i].row0, at), __builtin_amdgcn_readlane(u.span[i].n, at),
                             __builtin_amdgcn_readlane(u.span[i].pos0, at)};
            r.s = at * u.per + i;
            r.c = c;
            r.chunks = chunks;
            r.chunk = n == chunks ? kStep : __builtin_amdgcn_readfirstlane((n + chunks - 1) / chunks) * kStep;
        }
        c -= chunks;
    }
    r.slot = idx;
    return r;
}

// Listed pages: a token, its KV head kvh, the heads of the group from head0 on, and a chunk
// of the places.  An XCD (workgroups are dealt to the eight in turn) takes the tokens of one
// KV head one after another: the lists of two heads have no pages in common (64 sequences'
// tokens with 1024 positions each 50.7 us; all heads of a token on one XCD 52.7).
__device__ __forceinline__ RowsUnit selected_unit(const PagedParams &p, int &kvh, int &head0) {
    RowsUnit r{};
    r.s = -1;
    const int per = gridDim.x / 8;  // (a multiple of 8)
    const int idx = (int)(blockIdx.x % 8) * per + (int)(blockIdx.x / 8);
    r.c = idx % p.n_chunks;
    int at = idx / p.n_chunks;
    const int block = at % p.head_blocks;
    at /= p.head_blocks;
    const int t = at % p.b.n_tokens;
    kvh = at / p.b.n_tokens;
    head0 = block * kPagedRows;
    if (kvh >= p.c.n_kv) return r;
    const int s = seq_of_row(p.b, t, r.span);
    r.tok = t - r.span.row0;
    if (s >= p.b.n_seqs || r.tok < 0 || r.tok >= min(r.span.n, p.b.max_new)) return r;
    r.s = s;
    r.chunk = p.chunk;
    r.chunks = p.n_chunks;
    r.slot = ((int64_t)t * p.n_chunks + r.c) * p.head_blocks + block;
    return r;
}

// Listed pages: the tokens of a tile and their KV head kvh; an XCD takes tiles one after
// another, with all of their KV heads.
__device__ __forceinline__ RowsUnit tile_unit(const PagedParams &p, int &kvh) {
    RowsUnit r{};
    r.s = -1;
    // the whole tiles first, as many on each XCD, then those at the sequences' starts (mostly none)
    const int whole = (p.b.n_tokens + p.tile - 1) / p.tile, n = whole * p.c.n_kv, per = (n + 7) / 8;
    const int x = blockIdx.x % 8, k = blockIdx.x / 8, starts = (gridDim.x / 8) - per;
    const int idx = k < per ? x * per + k : n + x * starts + (k - per);
    if (k < per && idx >= n) return r;
    kvh = idx % p.c.n_kv;
    const TileRows t = tile_rows(p.b, p.tile, idx / p.c.n_kv);
    if (t.n == 0) return r;
    r.span = t.span;
    r.tok = t.row0 - t.span.row0;
    r.tokens = t.n;
    r.s = t.s;
    r.chunks = 1;
    r.chunk = 1 << 30;
    return r;
}

// The pages that a tile's tokens list, in order, each once with the tokens that do: work[k]
// the page of the pool, work[tile * n_select + k] its place in the table | tokens << 24; how
// many.  A byte of `marks` (LDS of so many bytes) a page of the sequence takes the tokens'
// bits, part after part of a long one.  Where a list has a page twice every entry of all
// stays its own.  By the whole workgroup.
__device__ __forceinline__ int merge_lists(const PagedParams &p, const RowsUnit &unit, int kvh, int *work,
                                           uint32_t *marks, int bytes) {
    __shared__ int counts[2][4], twice;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, n = p.n_select, total = unit.tokens * n;
    const int limit = position_limit(p.b, p.c);
    const int32_t *const table = p.c.table ? p.c.table + (int64_t)unit.s * p.c.width : nullptr;
    const auto pages_of = [&](int t) {
        const int sees = min(limit, unit.span.pos0 + unit.tok + t + 1);
        return sees > 0 ? ((sees - 1) >> p.c.shift) + 1 : 0;
    };
    const auto value = [&](int e, int &t) {  // -1: none that the token sees
        t = e / n;
        const int x = p.lists[((int64_t)(unit.span.row0 + unit.tok + t) * p.c.n_kv + kvh) * n + e % n];
        return x >= 0 && x < pages_of(t) ? x : -1;
    };
    int found = 0, odd = 0;
    // the places of the workgroup's `mine` entries a thread, behind those found
    const auto place = [&](int mine) {
        const int upto = wave_prefix(mine);
        if (lane == 63) counts[odd][w] = upto;
        __syncthreads();
        int at = found + upto - mine;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            at += i < w ? counts[odd][i] : 0;
            found += counts[odd][i];
        }
        odd ^= 1;
        return at;
    };
    const auto keep = [&](int at, int page, int x, uint32_t tokens) {
        work[at] = page;
        work[p.tile * n + at] = x | (int)(tokens << 24);
    };
    if (tid == 0) twice = 0;
    const int pages = pages_of(unit.tokens - 1);
    for (int base = 0; base < pages; base += bytes) {
        const int words = (min(bytes, pages - base) + 3) / 4;
        __syncthreads();  // the part before is read
        for (int i = tid; i < words; i += 256) marks[i] = 0;
        __syncthreads();
        for (int e = tid; e < total; e += 256) {
            int t;
            const int x = value(e, t) - base;
            if (x < 0 || x >= bytes) continue;
            const uint32_t bit = 1u << (8 * (x & 3) + t);
            if (atomicOr(&marks[x >> 2], bit) & bit) twice = 1;
        }
        __syncthreads();
        if (twice) break;
        for (int i0 = 0; i0 < words; i0 += 256) {
            const uint32_t m = i0 + tid < words ? marks[i0 + tid] : 0u;
            int page[4], mine = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int x = base + 4 * (i0 + tid) + i;
                page[i] = m >> (8 * i) & 0xFFu ? table ? table[x] : x : -1;
                if ((unsigned)page[i] >= (unsigned)p.c.n_pages) page[i] = -1;
                mine += page[i] >= 0;
            }
            int at = place(mine);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (page[i] >= 0) keep(at++, page[i], base + 4 * (i0 + tid) + i, m >> (8 * i) & 0xFFu);
        }
    }
    if (pages > 0 && twice) {  // uniform
        __syncthreads();
        found = 0;
        for (int e0 = 0; e0 < total; e0 += 256) {
            int t = 0, page = -1;
            const int x = e0 + tid < total ? value(e0 + tid, t) : -1;
            if (x >= 0) page = table ? table[x] : x;
            const bool there = (unsigned)page < (unsigned)p.c.n_pages;
            const int at = place(there);
            if (there) keep(at, page, x, 1u << t);
        }
    }
    __syncthreads();
    return found;
}

// Wave w takes positions 32 w .. + 31 of every 128-position step of the chunk with
// its own online softmax; the four waves merge at the end.  Per step, lane l =
// 16 g + r:
//   S^T = K . Q^T    v_mfma_f32_16x16x32_f16, src0 = 16 positions x 32 dims of K
//                    straight from memory (16 bytes a lane), src1 = Q^T; the lane
//                    gets positions 16 st + 4 g + i of row r;
//   softmax          as in attn_prefill.hip: the reference point m moves when the
//                    row's maximum has outgrown it by 2^kLazy; a lane's sums stay its
//                    own to the end; int8: P holds the V scales and m follows the
//                    maximum of score + log2 |scale|;
//   O^T += V^T P^T   the same MFMA, src0 = 16 dims x 32 positions of V^T (two
//                    ds_read_tr16_b64 of the wave's V rows in LDS), src1 = P^T as the
//                    score registers hold it (k of a lane group: its positions), in
//                    fp16 hi + lo parts (22 bits).
// The next step's K and V are loaded before this step's arithmetic.  Pages of 16
// positions or more (BIG): the 16 rows of an operand lie in one page, a buffer resource
// of the wave, so that a load needs no address arithmetic, and the lanes hold the table
// entries of 32 steps; smaller ones: lane i looks up position i, a step ahead, and the
// rows' offsets go through LDS.
// Rows past the end or in holes are zeros (BIG: past the end of the operand's buffer
// resource; else the pool's first row in their place, cleared), their scores
// -infinity.
//
// Listed pages.  kTokenLists: a workgroup takes one token, up to 16 heads of a KV head's group,
// and one chunk of the places of its listed pages, page_size a list entry; all rows see the
// same, so the masks are the entries'.  kTileLists: several tokens of a sequence, as many as 16
// rows hold, and the pages that any of them lists, each read once (the lists of a prompt's
// neighbours agree on most); a row's mask is its token's bit beside the page.  kWideTileLists:
// of two blocks of 16 rows, which share K and V and what is done to them.
// Bound: a token's reads of the cache, in the pieces above; a tile's pages come from the L2,
// and the chain of a step bounds it, of which 32 KB of K and V in and out of LDS are a
// half; a wide one's step issues 270 vector instructions and 48 products, which end to end
// would be three fifths of its time (27 and 17 of 74 us at 2.4 GHz): the rest is waiting, two
// waves a SIMD.
// Measured, head_dim 128: 64 tokens of 32 / 8 heads, 64 pages of 16 each, 51 us (5.3 TB/s; 256
// pages each 190, 5.65), 16 in an int8 cache, 32 pages of 64, 17 + 4 for the combine; a chunk of
// 512 tokens of 28 / 4 heads, 64 pages of 32, 78 us wide, 87 narrow (a token a workgroup 150,
// with K by the operand's rows 134); of 1000 of 32 / 8, pages of 16, 99 and 117.
template <int HD, bool I8, bool BIG, Lists LISTS>
__global__ __launch_bounds__(256, rows_waves(HD, I8, BIG, LISTS)) void attn_paged_rows_kernel(PagedParams p) {
    constexpr bool SEL = LISTS == kTokenLists, TILE = LISTS == kTileLists || LISTS == kWideTileLists;
    constexpr int RB = LISTS == kWideTileLists ? 2 : 1;  // rows, in blocks of 16
    // A chunk is 16 bytes: 8 dims of fp16, 16 of int8, which are two k steps of a
    // product (a lane's dims need only be the same in K and Q).
    constexpr int EC = I8 ? 16 : 8;                     // dims of a chunk
    constexpr int KL = (HD + 4 * EC - 1) / (4 * EC);    // K chunks of a lane and operand
    constexpr int KS = I8 ? 2 * KL : KL;                // k steps
    constexpr int DT = HD / 16, VROW = HD + 16, CH = HD / EC, NV = (32 * CH + 63) / 64;
    constexpr int esz = I8 ? 1 : 2;
    constexpr int NM = DT * 4 + 2;  // merge values per lane: O, m, l
    constexpr int kV = 4 * 32 * VROW * 2, kM = 4 * NM * 64 * 4;
    __shared__ __attribute__((aligned(16))) uint8_t smem[kV > kM ? kV : kM];
    __shared__ int64_t rowoff[BIG ? 1 : 4][32];
    __shared__ __attribute__((aligned(16))) float scl[4][3][I8 ? 32 : 1];
    __shared__ __attribute__((aligned(16))) int tokens_of[TILE && !BIG ? 4 : 1][32];  // that see each position

    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4;
    uint16_t *const vl = reinterpret_cast<uint16_t *>(smem) + w * 32 * VROW;
    // The KV heads of a sequence's chunk go to one XCD (workgroups are dealt to the eight in
    // turn): they read the same pages and scales (int8, 512 sequences of 1023 positions, 244
    // us with the heads on all, 216 so).  A sequence's chunks go to different ones.
    int kvh, head0 = 0;
    RowsUnit unit;
    int listed_pages = 0;  // TILE: pages that the tile's tokens list
    extern __shared__ int work[];  // TILE: their pages of the pool; their places | tokens << 24
    if constexpr (SEL) {
        unit = selected_unit(p, kvh, head0);
    } else if constexpr (TILE) {
        unit = tile_unit(p, kvh);
        if (unit.s >= 0) listed_pages = merge_lists(p, unit, kvh, work, reinterpret_cast<uint32_t *>(smem), sizeof(smem));
    } else {
        const int x8 = blockIdx.x / 8;
        kvh = x8 % p.c.n_kv;
        unit = rows_unit(p, x8 / p.c.n_kv * 8 + blockIdx.x % 8);
    }
    const int s = unit.s, c = unit.c, beg = c * unit.chunk;
    if (s < 0) return;  // uniform
    if (LISTS == kNoLists && p.n_chunks > 1 && c == 0 && kvh == 0 && tid == 0) {
        p.firsts[2 * s] = (int)unit.slot;
        p.firsts[2 * s + 1] = unit.chunks;
    }
    const int limit = position_limit(p.b, p.c);

    // (No load of the walk stands in a branch: the compiler would wait for all of them.)
    const bool has_table = p.c.table != nullptr && limit > 0;
    const int32_t *const table = has_table ? p.c.table + (int64_t)s * p.c.width : p.b.lens;
    const int p_lane = beg + 32 * w + (lane & 31);  // the lane's position of the first step
    auto entry = [&](int pos) {
        const int i = max(min(pos, limit - 1), 0) >> p.c.shift;
        const int x = table[has_table ? i : 0];
        return has_table ? x : i;
    };
    // BIG: lane 2 j + st holds the entry of operand st of step j, for 32 steps; else the
    // lane's position's, one step ahead
    const SeqSpan span = unit.span;
    // SEL: the list's page at place `at` (-1: none that the token sees), its page of the pool
    // (-1: a hole), and how many of its positions from the place on the token sees
    const int sees = SEL ? min(limit, span.pos0 + unit.tok + 1) : 0;
    const int pages_seen = sees > 0 ? ((sees - 1) >> p.c.shift) + 1 : 0;
    const int32_t *const list =
        SEL ? p.lists + ((int64_t)(span.row0 + unit.tok) * p.c.n_kv + kvh) * p.n_select : nullptr;
    auto listed = [&](int at) {
        const int i = at >> p.c.shift, x = list[min(i, p.n_select - 1)];
        return i < p.n_select && x >= 0 && x < pages_seen ? x : -1;
    };
    auto page_of = [&](int x) {
        const int e = table[has_table ? max(x, 0) : 0], page = has_table ? e : x;
        return x >= 0 && (unsigned)page < (unsigned)p.c.n_pages ? page : -1;
    };
    auto seen_from = [&](int x, int at) { return sees - (x << p.c.shift) - (at & ((1 << p.c.shift) - 1)); };
    int there = 0;    // SEL, BIG: beside the entry, the operand's positions that the token sees
    int x_ahead = 0;  // SEL, small pages: the list's page of the step after the newest entry's
    int of_tokens = 0;  // TILE: beside the entry, its place and tokens
    auto entries = [&](int j) {
        const int at = beg + 32 * w + kStep * (j + (lane >> 1)) + 16 * (lane & 1);
        if constexpr (TILE) {
            const int i = at >> p.c.shift, k = min(i, max(listed_pages - 1, 0));
            of_tokens = work[p.tile * p.n_select + k];
            const int last = min(limit, span.pos0 + unit.tok + unit.tokens);  // positions that the last token sees
            const int place = ((of_tokens & 0xFFFFFF) << p.c.shift) + (at & ((1 << p.c.shift) - 1));
            there = i < listed_pages ? min(max(last - place, 0), 16) : 0;
            return work[k];
        } else if constexpr (SEL) {
            const int x = listed(at), page = page_of(x);
            there = page >= 0 ? min(max(seen_from(x, at), 0), 16) : 0;
            return page;
        } else {
            return entry(at);
        }
    };
    auto next_entry = [&](int j) {  // small pages: the lane's position's of step j, asked for in order
        const int at = p_lane + kStep * j;
        if constexpr (TILE) {
            return 0;  // (in LDS: looked up with the loads)
        } else if constexpr (SEL) {
            const int x = j == 0 ? listed(at) : x_ahead;
            x_ahead = listed(at + kStep);
            const int page = page_of(x);
            return seen_from(x, at) > 0 ? page : -1;
        } else {
            return entry(at);
        }
    };
    int ent = BIG ? entries(0) : next_entry(0), ent_next = BIG ? 0 : next_entry(1);
    const int rows = SEL ? min(p.group - head0, kPagedRows) : (TILE ? unit.tokens : min(span.n, p.b.max_new)) * p.group;
    const int end_seq = TILE ? listed_pages << p.c.shift : SEL ? (limit > 0 ? p.n_select << p.c.shift : 0) : min(span.pos0 + (rows - 1) / p.group + 1, limit);
    const int end = min(end_seq, beg + unit.chunk);
    const int hd = p.c.hd, n_ch = hd / EC;
    // of the lane's rows the token, its position and where the row's output is
    int mine[RB], qpos[RB];
    int64_t orow[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        const int row = min(16 * b + r, rows - 1);  // (columns past the last row repeat it)
        mine[b] = SEL ? 0 : row / p.group;
        const int tok = LISTS != kNoLists ? unit.tok + mine[b] : mine[b];
        const int head = kvh * p.group + (SEL ? head0 + row : row % p.group);
        qpos[b] = span.pos0 + tok;
        orow[b] = ((int64_t)(span.row0 + tok) * p.n_heads + head) * hd;
    }
    if (end <= beg) {  // uniform
#pragma unroll
        for (int b = 0; b < RB; ++b)
            if (c == 0 && w == 0 && 16 * b + r < rows)  // the tokens see nothing
                for (int ch = g; ch < hd / 8; ch += 4)
                    *reinterpret_cast<u32x4 *>(p.out + orow[b] + 8 * ch) = u32x4{0u, 0u, 0u, 0u};
        return;
    }
    const int row_bytes = p.c.n_kv * hd * esz;
    const uint8_t *kb = p.c.k + (int64_t)kvh * hd * esz, *vb = p.c.v + (int64_t)kvh * hd * esz;

    u32x4 qf[RB][KS];
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int ch = I8 ? 2 * (4 * (ks / 2) + g) + ks % 2 : 4 * ks + g;  // of 8 dims
            qf[b][ks] = ch < hd / 8 ? load16(p.q + orow[b] + 8 * ch) : u32x4{0u, 0u, 0u, 0u};
        }
    // Byte offsets within a 16-row operand: K row r, dims 32 ks + 8 g; V row of the
    // lane's chunks.  Chunks past head_dim are past the operand's end (BIG), or the
    // last one again.
    constexpr int kPast = 0x7FFF0000;
    int ko[KL], vo[NV];
#pragma unroll
    for (int i = 0; i < KL; ++i) {
        const int ch = 4 * i + g;
        ko[i] = BIG ? (ch < n_ch ? r * row_bytes + 16 * ch : kPast) : 16 * min(ch, n_ch - 1);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int id = lane + 64 * j, ch = id % CH;
        vo[j] = BIG ? (ch < n_ch && id < 32 * CH ? (id / CH & 15) * row_bytes + 16 * ch : kPast) : 16 * min(ch, n_ch - 1);
    }
    // (global pointers: a generic load would be waited for with the LDS reads)
    const GlobalFloat ksp = p.c.ks ? (GlobalFloat)(p.c.ks + kvh) : (GlobalFloat)&g_one;
    const GlobalFloat vsp = p.c.vs ? (GlobalFloat)(p.c.vs + kvh) : (GlobalFloat)&g_one;
    const int s_stride = p.c.ks ? p.c.n_kv : 0, v_stride = p.c.vs ? p.c.n_kv : 0;
    // K as the products take it; TILE: by rows as V, turned in LDS (16 rows side by side are 64
    // lookups of the L1 a load and bound a tile whose pages come from the L2, rows one after
    // another 16)
    struct Rows {
        u32x4 k[TILE ? 1 : 2][TILE ? NV : KL], v[NV];
    };
    struct Step {
        float ks, vs;
        uint32_t seen;  // which of the wave's 32 positions there are
        int of[2];      // TILE: an operand's page and tokens; small pages: the lane's position's tokens
        bool all[2];    // TILE: every token sees all of the operand (small pages: of both)
    };
    // TILE: the loads of K and of V are left to the caller, from the operands' buffers
    struct Operands {
        __amdgpu_buffer_rsrc_t k[2], v[2];
    };
    auto load_rows = [&](const __amdgpu_buffer_rsrc_t *from, const uint8_t *base, u32x4 *x) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if constexpr (!BIG) {
                x[j] = load16(base + rowoff[w][min((lane + 64 * j) / CH, 31)] + vo[j]);
                continue;
            }
            constexpr bool kSplit = 64 % CH != 0 || 64 / CH > 16;  // a load's rows may be in both operands
            if constexpr (kSplit) {
                const bool first = (lane + 64 * j) / CH < 16;
                x[j] = buffer_load16(from[0], first ? vo[j] : kPast) | buffer_load16(from[1], first ? kPast : vo[j]);
            } else {
                x[j] = buffer_load16(from[64 * j / CH / 16], vo[j]);
            }
        }
    };
    auto load_k = [&](const Operands &from, Rows &R) {
        if constexpr (TILE) {
            load_rows(from.k, kb, R.k[0]);
        } else {
#pragma unroll
            for (int st = 0; st < 2; ++st)
#pragma unroll
                for (int i = 0; i < KL; ++i) R.k[st][i] = buffer_load16(from.k[st], ko[i]);
        }
    };
    auto load_v = [&](const Operands &from, Rows &R) { load_rows(from.v, vb, R.v); };
    auto load_step = [&](int j, [[maybe_unused]] int e, Step &S, Rows &R, Operands &from) {
        const int mask = (1 << p.c.shift) - 1;
        if constexpr (BIG) {
            // an operand's rows: those of its positions that there are, from the first
            S.seen = 0;
            int page[2], place[2];
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                const int pos = beg + 32 * w + kStep * j + 16 * st;
                page[st] = __builtin_amdgcn_readlane(e, (2 * j + st) & 63);
                const int n = LISTS != kNoLists ? (pos < end ? __builtin_amdgcn_readlane(there, (2 * j + st) & 63) : 0)
                              : (unsigned)page[st] < (unsigned)p.c.n_pages ? max(min(end - pos, 16), 0) : 0;
                S.seen |= ((1u << n) - 1) << (16 * st);
                page[st] = n > 0 ? page[st] : 0;
                place[st] = pos & mask;
                if constexpr (TILE) {
                    S.of[st] = __builtin_amdgcn_readlane(of_tokens, (2 * j + st) & 63);
                    const int first = ((S.of[st] & 0xFFFFFF) << p.c.shift) + place[st];
                    S.all[st] = n > 0 && (uint32_t)S.of[st] >> 24 == (1u << unit.tokens) - 1u &&
                                first + 16 <= min(limit, span.pos0 + unit.tok + 1);
                }
                const int64_t base = (int64_t)page[st] * p.c.page_bytes + (int64_t)place[st] * row_bytes;
                const int bytes = n > 0 ? (n - 1) * row_bytes + hd * esz : 0;
                from.k[st] = make_rsrc(kb + base, bytes);
                from.v[st] = make_rsrc(vb + base, bytes);
            }
            if constexpr (I8) {
                const bool ok = (S.seen >> (lane & 31)) & 1;
                const int64_t at = ok ? ((int64_t)(lane & 16 ? page[1] : page[0]) << p.c.shift) +
                                            (lane & 16 ? place[1] : place[0]) + (lane & 15) : 0;
                S.ks = ksp[at * s_stride];
                S.vs = vsp[at * v_stride];
            }
            if constexpr (!TILE) {
                load_k(from, R);
                load_v(from, R);
            }
        } else {
            const int pos = p_lane + kStep * j;
            bool ok = pos < end && (unsigned)e < (unsigned)p.c.n_pages;
            if constexpr (TILE) {
                const int k = min(pos >> p.c.shift, listed_pages - 1), of = work[p.tile * p.n_select + k];
                const int at = ((of & 0xFFFFFF) << p.c.shift) + (pos & mask);  // the place of the sequence
                // of the tokens that list it those that are not before it
                const int before = max(at - (span.pos0 + unit.tok), 0);
                S.of[0] = pos < end && at < limit && before < 8 ? (of >> 24 & 0xFF) >> before << before : 0;
                ok = S.of[0] != 0;
                e = ok ? work[k] : 0;
                S.all[0] = __builtin_amdgcn_ballot_w64(S.of[0] != (1 << unit.tokens) - 1) == 0;
            }
            S.seen = (uint32_t)__builtin_amdgcn_ballot_w64(ok);
            const int place = pos & mask;
            if constexpr (I8) {
                const int64_t at = ok ? ((int64_t)e << p.c.shift) + place : 0;
                S.ks = ksp[at * s_stride];
                S.vs = vsp[at * v_stride];
            }
            if constexpr (TILE) wave_lds_fence();  // the rows before are asked for
            if (lane < 32) rowoff[w][lane] = ok ? (int64_t)e * p.c.page_bytes + (int64_t)place * row_bytes : 0;
            wave_lds_fence();
            if constexpr (TILE) return;
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                const uint8_t *src = kb + rowoff[w][16 * st + r];
#pragma unroll
                for (int i = 0; i < KL; ++i) R.k[st][i] = load16(src + ko[i]);
            }
#pragma unroll
            for (int j = 0; j < NV; ++j) R.v[j] = load16(vb + rowoff[w][min((lane + 64 * j) / CH, 31)] + vo[j]);
            wave_lds_fence();
        }
    };
    auto widen = [](uint32_t a, uint32_t b) {  // 8 int8
        const u32x2 x = i8x4_to_f16(a), y = i8x4_to_f16(b);
        return u32x4{x.x, x.y, y.x, y.y};
    };

    f32x4 o[RB][DT];
    float m[RB], l[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[b][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        m[b] = -INFINITY;
        l[b] = 0.0f;
    }
    bool bad = false;  // some V is not finite
    uint32_t most_vs = 0;  // int8: the lane's largest |V scale|
    auto process = [&](int j, Step &S, Rows &R, auto after_k, auto after_v) {
        if (SEL && S.seen == 0) return;  // uniform
        const int p0 = beg + kStep * j + 32 * w;
        f32x4 acc[RB][2];
        // (the wave's own reads of its V rows are ahead in its LDS queue, and these ahead of the next)
        constexpr int kPitch = HD * esz + 16;  // bytes of a K row
        uint8_t *const kl = reinterpret_cast<uint8_t *>(vl);
        if constexpr (TILE) {
            wave_lds_fence();
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int id = lane + 64 * j;
                if (32 * CH % 64 == 0 || id < 32 * CH) *reinterpret_cast<u32x4 *>(kl + (id / CH) * kPitch + 16 * (id % CH)) = R.k[0][j];
            }
            wave_lds_fence();
        }
#pragma unroll
        for (int st = 0; st < 2; ++st) {
#pragma unroll
            for (int b = 0; b < RB; ++b) acc[b][st] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            u32x4 kf[KL];
#pragma unroll
            for (int i = 0; i < KL; ++i) {
                if constexpr (TILE) kf[i] = *reinterpret_cast<const u32x4 *>(kl + (16 * st + r) * kPitch + 16 * (4 * i + g));
                else kf[i] = R.k[st][i];
            }
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                u32x4 k;
                if constexpr (I8) k = ks % 2 ? widen(kf[ks / 2].z, kf[ks / 2].w) : widen(kf[ks / 2].x, kf[ks / 2].y);
                else k = kf[ks];
                if (!I8 && !BIG && 4 * ks + 4 > n_ch && 4 * ks + g >= n_ch) k = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
                for (int b = 0; b < RB; ++b) acc[b][st] = mfma<RXQ4_DTYPE_F16>(k, qf[b][ks], acc[b][st]);
            }
        }
        if constexpr (TILE) wave_lds_fence();
        after_k();
        f32x4 vx[2], lg[2];
        if constexpr (I8) {
            // An infinite or NaN V scale: as an fp16 V below.  (Small pages: looked at after the
            // walk; a ballot here spills 27 registers.  Larger ones: the lanes' sizes spill 2.)
            const uint32_t size = __builtin_bit_cast(uint32_t, S.vs) & 0x7FFFFFFFu;
            const uint32_t here = (S.seen >> (lane & 31)) & 1u ? size : 0u;
            if constexpr (BIG) bad |= __builtin_amdgcn_ballot_w64(here >= 0x7F800000u) != 0;
            else most_vs = max(most_vs, here);
            S.vs = size < 0x7F800000u ? S.vs : 0.0f;
            if (lane < 32) {
                scl[w][0][lane] = S.ks;
                scl[w][1][lane] = S.vs;
                scl[w][2][lane] = log2_scale(S.vs);
            }
            wave_lds_fence();
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                const f32x4 kx = *reinterpret_cast<const f32x4 *>(&scl[w][0][16 * st + 4 * g]);
#pragma unroll
                for (int b = 0; b < RB; ++b) acc[b][st] *= kx;
                vx[st] = *reinterpret_cast<const f32x4 *>(&scl[w][1][16 * st + 4 * g]);
                lg[st] = *reinterpret_cast<const f32x4 *>(&scl[w][2][16 * st + 4 * g]);
            }
            wave_lds_fence();
        }
        const bool part = S.seen != ~0u;
        uint32_t ph[RB][4], pl[RB][4];
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            float sv[8], mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < 8; ++i) sv[i] = acc[b][i >> 2][i & 3] * p.sl2;
            if constexpr (TILE && !BIG) {
                if (!S.all[0]) {  // uniform
                    if (b == 0 && lane < 32) tokens_of[w][lane] = S.of[0];
                    wave_lds_fence();
#pragma unroll
                    for (int st = 0; st < 2; ++st) {
                        const i32x4 of = *reinterpret_cast<const i32x4 *>(&tokens_of[w][16 * st + 4 * g]);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (!(of[i] >> mine[b] & 1)) sv[4 * st + i] = -INFINITY;
                    }
                    wave_lds_fence();
                }
            } else if constexpr (TILE) {
#pragma unroll
                for (int st = 0; st < 2; ++st)
                    if (!S.all[st]) {  // uniform
                        // places of the operand that the row's token lists and sees
                        const int first = ((S.of[st] & 0xFFFFFF) << p.c.shift) + ((p0 + 16 * st) & ((1 << p.c.shift) - 1));
                        const int n = S.of[st] >> (24 + mine[b]) & 1 ? min(limit, qpos[b] + 1) - first : 0;
                        const int here = (S.seen >> (16 * st) & 0xFFFFu) != 0 ? n : 0;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (4 * g + i >= here) sv[4 * st + i] = -INFINITY;
                    }
            } else if (part || (!SEL && p0 + 31 > span.pos0)) {  // uniform: not every row sees all of them
                const uint32_t in = S.seen >> (4 * g);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (!((in >> (16 * (i >> 2) + (i & 3))) & 1u) || (!SEL && p0 + 16 * (i >> 2) + 4 * g + (i & 3) > qpos[b]))
                        sv[i] = -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) mx = fmaxf(mx, I8 ? sv[i] + lg[i >> 2][i & 3] : sv[i]);
            mx = max_xor_rows<16>(mx);
            mx = max_xor_rows<32>(mx);
            if (__builtin_amdgcn_ballot_w64(mx > m[b] + kLazy) != 0) {
                // (each row's by its own rule: no row depends on what others see)
                const float m_new = mx > m[b] + kLazy ? mx : m[b];
                const float corr = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[b] - m_new);
                m[b] = m_new;
                l[b] *= corr;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) o[b][dt] *= corr;
            }
            const float m_use = m[b] == -INFINITY ? 0.0f : m[b] - kShift;
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                float e0 = __builtin_amdgcn_exp2f(sv[i] - m_use), e1 = __builtin_amdgcn_exp2f(sv[i + 1] - m_use);
                l[b] += e0;
                l[b] += e1;
                if constexpr (I8) {
                    // (a position that the row does not see stays 0 whatever its scale)
                    e0 = sv[i] == -INFINITY ? 0.0f : e0 * vx[i >> 2][i & 3];
                    e1 = sv[i + 1] == -INFINITY ? 0.0f : e1 * vx[i >> 2][(i & 3) + 1];
                }
                ph[b][i >> 1] = pack2<RXQ4_DTYPE_F16>(e0, e1);
                pl[b][i >> 1] = low_halves(e0, e1, ph[b][i >> 1]);
            }
        }
        // Rows that are not there: zeros.  An infinity or NaN in V would reach the rows
        // that do not see it as 0 times it, and the others through the low half of P: such
        // values (int8: V scales) are staged as zeros, and the rows that see them get them
        // at the end.
        if constexpr (!I8) {
            if (!BIG && part)  // uniform
#pragma unroll
                for (int j = 0; j < NV; ++j)
                    if (!((S.seen >> ((lane + 64 * j) / CH)) & 1u)) R.v[j] = u32x4{0u, 0u, 0u, 0u};
            if (__builtin_amdgcn_ballot_w64(not_finite16<NV>(R.v)) != 0) {
                zero_not_finite16<NV>(R.v);
                bad = true;
            }
        }
        // (the wave's own earlier reads of its rows are ahead in its LDS queue)
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int id = lane + 64 * j;
            uint16_t *dst = &vl[(id / CH) * VROW + EC * (id % CH)];
            if constexpr (I8) {
                if (32 * CH % 64 == 0 || id < 32 * CH) {
                    *reinterpret_cast<u32x4 *>(dst) = widen(R.v[j].x, R.v[j].y);
                    *reinterpret_cast<u32x4 *>(dst + 8) = widen(R.v[j].z, R.v[j].w);
                }
            } else {
                *reinterpret_cast<u32x4 *>(dst) = R.v[j];
            }
        }
        after_v();
        // lane r of group g supplies dims 16 dt + 4 (r & 3) .. + 3 of positions 4 g + r / 4
        // and 16 + 4 g + r / 4 and receives dim 16 dt + r of positions 4 g .. + 3 and 16 + 4 g ..
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            const uint16_t *vp = &vl[(4 * g + (r >> 2)) * VROW + 16 * dt + 4 * (r & 3)];
            const u32x2 v0 = __builtin_bit_cast(
                u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4i16 *)vp));
            const u32x2 v1 = __builtin_bit_cast(
                u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                           (__attribute__((address_space(3))) v4i16 *)(vp + 16 * VROW)));
            const u32x4 a = u32x4{v0.x, v0.y, v1.x, v1.y};
#pragma unroll
            for (int b = 0; b < RB; ++b) {
                o[b][dt] = mfma<RXQ4_DTYPE_F16>(a, u32x4{ph[b][0], ph[b][1], ph[b][2], ph[b][3]}, o[b][dt]);
                o[b][dt] = mfma<RXQ4_DTYPE_F16>(a, u32x4{pl[b][0], pl[b][1], pl[b][2], pl[b][3]}, o[b][dt]);
            }
            if (TILE && dt % 2 == 1) __builtin_amdgcn_sched_barrier(0);  // (all reads at once: 32 registers)
        }
    };
    const int n_steps = (end - beg + kStep - 1) / kStep;
    const auto nothing = [] {};
    Step A, B;
    Operands next;
    if constexpr (TILE) {
        // The matrix and vector units bound it, not memory: K and V of one step in registers,
        // the next step's loaded where this one's products and stores are done with them, so
        // that another wave fits a SIMD.
        Rows R;
        for (int j0 = 0; j0 < n_steps; j0 += 32) {
            const int j1 = min(n_steps, j0 + 32);
            if (BIG && j0 > 0) ent = entries(j0);
            load_step(j0, ent, A, R, next);
            load_k(next, R);
            load_v(next, R);
            for (int j = j0; j < j1; ++j) {
                load_step(j + 1 < j1 ? j + 1 : kNoStep, ent, B, R, next);
                // (kept there: earlier they would need registers of their own)
                process(j, A, R, [&] {
                    __builtin_amdgcn_sched_barrier(0);
                    load_k(next, R);
                    __builtin_amdgcn_sched_barrier(0);
                }, [&] {
                    __builtin_amdgcn_sched_barrier(0);
                    load_v(next, R);
                    __builtin_amdgcn_sched_barrier(0);
                });
                A = B;
            }
        }
    } else {
        Rows RA, RB;
        for (int j0 = 0; j0 < n_steps; j0 += 32) {
            const int j1 = BIG ? min(n_steps, j0 + 32) : n_steps;
            if (j0 > 0) ent = entries(j0);
            load_step(j0, ent, A, RA, next);
            for (int j = j0;;) {
                if (!BIG) ent = next_entry(j + 2);
                load_step(j + 1 < j1 ? j + 1 : kNoStep, BIG ? ent : ent_next, B, RB, next);
                __builtin_amdgcn_sched_barrier(0);  // (the compiler would move them behind the products)
                process(j, A, RA, nothing, nothing);
                if (++j >= j1) break;
                if (!BIG) ent_next = next_entry(j + 2);
                load_step(j + 1 < j1 ? j + 1 : kNoStep, ent, A, RA, next);
                __builtin_amdgcn_sched_barrier(0);
                process(j, B, RB, nothing, nothing);
                if (++j >= j1) break;
            }
            if (!BIG) break;
        }
    }
    if constexpr (I8 && !BIG) bad = __builtin_amdgcn_ballot_w64(most_vs >= 0x7F800000u) != 0;
    // Merge: lane l of every wave holds row r, dims 16 dt + 4 g + i; wave w merges
    // the dims of tiles dt = w, w + 4, ...
    float (*const mg)[NM][64] = reinterpret_cast<float (*)[NM][64]>(smem);
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        __syncthreads();  // the V rows (the block before) are read
        l[b] = sum_xor_rows<16>(l[b]);
        l[b] = sum_xor_rows<32>(l[b]);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int i = 0; i < 4; ++i) mg[w][4 * dt + i][lane] = o[b][dt][i];
        mg[w][NM - 2][lane] = m[b];
        mg[w][NM - 1][lane] = l[b];
        if (bad) {  // uniform, rare: the wave's positions again (onto its part in LDS: no registers held for it)
            for (int pos = beg; pos < end; ++pos) {
                if (((pos - beg) / 32 & 3) != w || (LISTS == kNoLists && pos > qpos[b])) continue;
                int slot;
                if constexpr (TILE) {
                    const int k = pos >> p.c.shift, in = pos & ((1 << p.c.shift) - 1), of = work[p.tile * p.n_select + k];
                    const bool sees_it = of >> (24 + mine[b]) & 1 && ((of & 0xFFFFFF) << p.c.shift) + in < min(limit, qpos[b] + 1);
                    slot = sees_it ? (work[k] << p.c.shift) + in : -1;
                } else if constexpr (SEL) {
                    const int x = listed(pos);
                    slot = x >= 0 && seen_from(x, pos) > 0 ? slot_of(p.c, s, (x << p.c.shift) + (pos & ((1 << p.c.shift) - 1))) : -1;
                } else {
                    slot = slot_of(p.c, s, pos);
                }
                if (slot < 0) continue;
                const uint8_t *v = vb + slot_bytes(p.c, slot, row_bytes);
                const float vs = I8 ? vsp[(int64_t)slot * v_stride] : 1.0f;
                if (I8 && fabsf(vs) < INFINITY) continue;
                for (int dt = 0; dt < DT; ++dt) {
                    const int d = 16 * dt + 4 * g;
                    if (d >= hd) continue;
                    const u32x2 x = I8 ? u32x2{*reinterpret_cast<const uint32_t *>(v + d), 0u}
                                       : *reinterpret_cast<const u32x2 *>(v + 2 * d);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float y = I8 ? vs * (float)(int8_t)(x.x >> (8 * i))
                                           : f16_bits_to_f32((i < 2 ? x.x : x.y) >> (16 * (i & 1)) & 0xFFFFu);
                        if (!(fabsf(y) < INFINITY)) mg[w][4 * dt + i][lane] += y;
                    }
                }
            }
        }
        __syncthreads();
        float mw[4], M = -INFINITY;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            mw[v] = mg[v][NM - 2][lane];
            M = fmaxf(M, mw[v]);
        }
        float cw[4], L = 0.0f;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            cw[v] = M != -INFINITY ? __builtin_amdgcn_exp2f(mw[v] - M) : 0.0f;
            L += mg[v][NM - 1][lane] * cw[v];
        }
        if (16 * b + r >= rows) continue;
        const bool whole = unit.chunks <= 1;  // one chunk: no partials
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
        const int64_t at = (unit.slot * p.c.n_kv + kvh) * p.rows_blk + r;
#pragma unroll
        for (int dt = w; dt < DT; dt += 4) {
            f32x4 ov{};
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int v = 0; v < 4; ++v) ov[i] = __builtin_fmaf(cw[v], mg[v][4 * dt + i][lane], ov[i]);
            if (!(fabsf(ov[0]) + fabsf(ov[1]) + fabsf(ov[2]) + fabsf(ov[3]) < INFINITY)) {  // rare: the same sums
                ov = f32x4{};
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int v = 0; v < 4; ++v) ov[i] = add_weighed(ov[i], cw[v], mg[v][4 * dt + i][lane]);
            }
            const int d = 16 * dt + 4 * g;
            if (!whole) *reinterpret_cast<f32x4 *>(p.part + at * HD + d) = ov;
            else if (d < hd)
                *reinterpret_cast<u32x2 *>(p.out + orow[b] + d) = u32x2{pack2<RXQ4_DTYPE_F16>(ov[0] * inv, ov[1] * inv),
                                                                     pack2<RXQ4_DTYPE_F16>(ov[2] * inv, ov[3] * inv)};
        }
        if (!whole && w == 0 && g == 0) {
            p.stats[2 * at] = M;
            p.stats[2 * at + 1] = L;
        }
    }
}

// sum + w x of a row's chunk c.  The rounding is written out, as part of the results (left to
// the compiler, which of the sums it fuses changes with the code around them): fused; up to
// head_dim 64 product and sum are rounded each from the third chunk on.
template <int HD>
__device__ __forceinline__ float add_chunk(float sum, float w, float x, int c) {
    if (HD > 64 || c < 2) return __builtin_fmaf(w, x, sum);
    {
#pragma clang fp contract(off)
        return sum + w * x;
    }
}

// out = sum_c 2^(m_c - M) O_c / sum_c 2^(m_c - M) l_c over a row's n_c chunks in order,
// partials `at` and every `step` behind.  A wave takes a row: a lane's chunk for the
// weights, then a lane's dims.
template <int HD>
__device__ __forceinline__ void combine_row(const PagedParams &p, int64_t at, int64_t step, int n_c, uint16_t *out) {
    constexpr int VE = HD > 128 ? 4 : HD > 64 ? 2 : 1, U = 8;
    typedef float Piece __attribute__((ext_vector_type(VE)));
    const int lane = threadIdx.x & 63;
    const float *st = p.stats + 2 * (at + min(lane, n_c - 1) * step);
    const float mc = st[0], lc = st[1];
    const int d = min(lane * VE, HD - VE);
    const float *src = p.part + at * HD + d;
    Piece acc{};
    float e = 0.0f, L = 0.0f;
    for (int c0 = 0; c0 < n_c; c0 += U) {
        Piece x[U];
#pragma unroll
        for (int i = 0; i < U; ++i) x[i] = *reinterpret_cast<const Piece *>(src + min(c0 + i, n_c - 1) * step * HD);
        if (c0 == 0) {
            const float M = butterfly_max<64>(mc);
            e = M != -INFINITY && lane < n_c ? __builtin_amdgcn_exp2f(mc - M) : 0.0f;
            L = butterfly_sum<64>(e * lc);
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const float ec = __builtin_bit_cast(
                float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, e), min(c0 + i, 63)));
            if (c0 + i >= n_c) continue;  // uniform
            if (ec != 0.0f)
#pragma unroll
                for (int k = 0; k < VE; ++k) acc[k] = add_chunk<HD>(acc[k], ec, x[i][k], c0 + i);
            else
#pragma unroll
                for (int k = 0; k < VE; ++k) acc[k] = add_weighed(acc[k], 0.0f, x[i][k]);
        }
    }
    if (lane * VE >= p.c.hd) return;
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    out += d;
    if constexpr (VE == 1) {
        *out = f32_to_f16_bits(acc[0] * inv);
    } else {
#pragma unroll
        for (int i = 0; i < VE; i += 2)
            *reinterpret_cast<uint32_t *>(out + i) = pack2<RXQ4_DTYPE_F16>(acc[i] * inv, acc[i + 1] * inv);
    }
}

template <int HD>
__global__ __launch_bounds__(256) void attn_paged_combine_kernel(PagedParams p) {
    const int r = 4 * blockIdx.y + (threadIdx.x >> 6);
    const int kvh = blockIdx.x % p.c.n_kv, s = blockIdx.x / p.c.n_kv;
    const SeqSpan span = seq_span(p.b, s);
    const int first = p.firsts[2 * s], n_c = p.firsts[2 * s + 1];
    const int rows = min(span.n, p.b.max_new) * p.group;
    if (r >= rows || rows > kPagedRows || n_c <= 1 || n_c > p.n_chunks) return;  // not this kernel's, or written already
    const int64_t at = ((int64_t)first * p.c.n_kv + kvh) * p.rows_blk + r, step = (int64_t)p.c.n_kv * p.rows_blk;
    const int tok = r / p.group, head = kvh * p.group + r % p.group;
    combine_row<HD>(p, at, step, n_c, p.out + ((int64_t)(span.row0 + tok) * p.n_heads + head) * p.c.hd);
}

// Selected pages: a row is a token's head.
template <int HD>
__global__ __launch_bounds__(256) void attn_selected_combine_kernel(PagedParams p) {
    const int t = blockIdx.x, head = 4 * blockIdx.y + (threadIdx.x >> 6);
    if (head >= p.n_heads) return;
    SeqSpan span;
    const int s = seq_of_row(p.b, t, span);
    if (s >= p.b.n_seqs || t < span.row0 || t - span.row0 >= min(span.n, p.b.max_new)) return;
    const int kvh = head / p.group, j = head % p.group;
    const int64_t slot = (int64_t)t * p.n_chunks * p.head_blocks + j / kPagedRows;
    const int64_t at = (slot * p.c.n_kv + kvh) * p.rows_blk + j % kPagedRows;
    combine_row<HD>(p, at, (int64_t)p.head_blocks * p.c.n_kv * p.rows_blk, p.n_chunks,
                    p.out + ((int64_t)t * p.n_heads + head) * p.c.hd);
}

// The 16-row launch's chunks: their partials within `room` bytes.  Some six chunks of
// an fp16 and twelve of an int8 cache a CU (three to four of what runs at a time, for
// sequences of any lengths): 64 sequences of 64 to 8000 positions, 8 heads, fp16, 5 / 6
// / 8 / 12 a CU 98.7 / 91.7 / 94.6 / 103 us; 16 of 20000 to 40000, int8, 6 / 8 / 12 / 16
// 213 / 208 / 202 / 204.  Past kSeqs sequences the host cuts them from the limits: 299
// sequences of 500 positions and one of 13000 159 us, with max_len 131072 271; 255 and one
// on the device 125 and 134.
struct RowsPlan {
    int64_t slots;  // chunks of the batch at most, per KV head
    int64_t grid;   // workgroups
    size_t bytes;
};
RowsPlan plan_rows(PagedParams &p, int i8, size_t room) {
    const int cus = device_info().cu_count > 0 ? device_info().cu_count : 256;
    const int pad = p.c.hd <= 64 ? 64 : p.c.hd <= 96 ? 96 : p.c.hd <= 128 ? 128 : 256;
    p.rows_blk = (int)std::min<int64_t>((int64_t)std::min(p.b.max_new, p.b.n_tokens) * p.group, kPagedRows);
    const int64_t len = std::max<int64_t>(1, std::min<int64_t>(p.b.max_len, (int64_t)p.c.width << p.c.shift));
    const int64_t steps = (len + kStep - 1) / kStep, n = p.b.n_seqs;
    const size_t per = (size_t)p.c.n_kv * p.rows_blk * (pad + 2) * 4;  // bytes of a slot
    room -= std::min<size_t>(room, 8 * n + 256);
    int64_t most = std::min<int64_t>(steps, kMaxChunks);
    if (tuning().attn_split) most = std::min<int64_t>(most, tuning().attn_split);
    const int64_t units = std::min<int64_t>((i8 ? 12 : 6) * cus / p.c.n_kv, (int64_t)(room / per) - n);
    if (n > kSeqs) {
        most = std::min<int64_t>({most, std::max((4 * cus + n * p.c.n_kv - 1) / (n * p.c.n_kv), (len + 2047) / 2048), (int64_t)(room / per) / n});
    } else if (units < 1) {
        most = 1;
    }
    most = std::max<int64_t>(most, 1);
    const int64_t least = (steps + most - 1) / most;  // steps of a chunk
    p.min_tiles = (int)least;
    p.max_units = (int)std::max<int64_t>(units, 1);
    p.chunk = (int)least * kStep;
    p.n_chunks = (int)((steps + least - 1) / least);
    const int64_t slots = p.n_chunks == 1 || n > kSeqs ? n * p.n_chunks : std::min<int64_t>(units + n, n * p.n_chunks);
    return RowsPlan{slots, (slots + 7) / 8 * 8 * p.c.n_kv, p.n_chunks > 1 ? (per * slots + 8 * n + 255) / 256 * 256 : 0};
}

template <int HD>
hipError_t launch_rows(PagedParams &p, const RowsPlan &plan, float *ws, int i8, hipStream_t st) {
    const unsigned grid = (unsigned)plan.grid;
    p.part = ws;
    p.stats = ws + (size_t)plan.slots * p.c.n_kv * p.rows_blk * HD;
    p.firsts = reinterpret_cast<int *>(p.stats + (size_t)plan.slots * p.c.n_kv * p.rows_blk * 2);
    const bool big = p.c.shift >= 4;
    if (i8 && big) attn_paged_rows_kernel<HD, true, true, kNoLists><<<grid, 256, 0, st>>>(p);
    else if (i8) attn_paged_rows_kernel<HD, true, false, kNoLists><<<grid, 256, 0, st>>>(p);
    else if (big) attn_paged_rows_kernel<HD, false, true, kNoLists><<<grid, 256, 0, st>>>(p);
    else attn_paged_rows_kernel<HD, false, false, kNoLists><<<grid, 256, 0, st>>>(p);
    if (p.n_chunks > 1) {
        const dim3 rows((unsigned)(p.b.n_seqs * p.c.n_kv), (unsigned)(p.rows_blk + 3) / 4);
        attn_paged_combine_kernel<HD><<<rows, 256, 0, st>>>(p);
    }
    return hipGetLastError();
}

// The chunks of the listed places: steps enough for `want` workgroups, partials within the
// workspace.
struct SelectedPlan {
    int64_t grid;
    size_t bytes;
};
constexpr int kListEntries = 2048;  // of a tile's lists: 16 KB of LDS
SelectedPlan plan_selected(PagedParams &p, int i8) {
    const int cus = device_info().cu_count > 0 ? device_info().cu_count : 256;
    const int pad = p.c.hd <= 64 ? 64 : p.c.hd <= 96 ? 96 : p.c.hd <= 128 ? 128 : 256;
    p.rows_blk = std::min(p.group, kPagedRows);
    p.head_blocks = (p.group + kPagedRows - 1) / kPagedRows;
    // Tiles where the sequences have tokens to fill them and the tiles are enough for the CUs
    // (measured, us of tokens / narrow tiles, lists of 64 pages of 16, 32 / 8 heads, one sequence:
    // 4 new tokens 10 / 28, 32 16 / 30, 64 26 / 31, 128 45 / 32; 12 sequences of two or five 16 / 22, 25 /
    // 26, 32 of two to four 30 / 35, 35 / 40, 46 / 37, 64 of two to four 64 / 65, 86 / 74, 110 / 73).
    // Wide ones where they fill more than three quarters of the rounds that they take (at 28 / 4
    // heads a round is 512 tokens: 384 / 448 / 600 / 900 tokens wide 74 / 76 / 115 / 137 us, narrow
    // 67 / 86 / 99 / 157).
    if (p.b.max_new > 1 && p.b.n_tokens >= 4 * (int64_t)p.b.n_seqs)
        for (int blocks = pad <= 128 ? 2 : 1; blocks > 0; --blocks) {
            p.tile = (int)std::min<int64_t>({(int64_t)blocks * kPagedRows / p.group, 8, kListEntries / p.n_select});
            if (p.tile <= 1 || (blocks == 2 && p.tile * p.group <= kPagedRows)) continue;
            const int64_t whole = (int64_t)((p.b.n_tokens + p.tile - 1) / p.tile) * p.c.n_kv, starts = (int64_t)p.b.n_seqs * p.c.n_kv;
            if (blocks == 2) {
                const int64_t live = whole + starts - p.c.n_kv;  // (the first sequence starts a whole one)
                const int64_t slots = (int64_t)rows_waves(pad, i8, p.c.shift >= 4, kWideTileLists) * cus;
                if (4 * live <= 3 * slots * ((live + slots - 1) / slots)) continue;
            } else if (whole + starts < cus) {
                continue;
            }
            p.n_chunks = 1;
            return SelectedPlan{(whole + 7) / 8 * 8 + (starts + 7) / 8 * 8, 0};
        }
    p.tile = 1;
    const int64_t units = (int64_t)p.b.n_tokens * p.c.n_kv * p.head_blocks;
    const int64_t per = units * p.rows_blk * (pad + 2) * 4;  // bytes of one chunk of every unit
    const int64_t steps = std::min<int64_t>(p.b.max_len, (int64_t)p.c.width << p.c.shift) > 0
                              ? (((int64_t)p.n_select << p.c.shift) + kStep - 1) / kStep : 1;
    int64_t most = std::min<int64_t>({steps, kMaxChunks, cus / units, (int64_t)kWorkspaceBytes / per});
    if (tuning().attn_split) most = std::min<int64_t>(most, tuning().attn_split);
    most = std::max<int64_t>(most, 1);
    const int64_t least = (steps + most - 1) / most;
    p.chunk = (int)least * kStep;
    p.n_chunks = (int)((steps + least - 1) / least);
    return SelectedPlan{(units * p.n_chunks + 7) / 8 * 8, p.n_chunks > 1 ? (size_t)(per * p.n_chunks) : 0};
}

template <int HD>
hipError_t launch_selected(PagedParams &p, const SelectedPlan &plan, float *ws, int i8, hipStream_t st) {
    const unsigned grid = (unsigned)plan.grid;
    p.part = ws;
    p.stats = ws + (size_t)p.b.n_tokens * p.n_chunks * p.head_blocks * p.c.n_kv * p.rows_blk * HD;
    const bool big = p.c.shift >= 4;
    if (p.tile > 1) {
        const size_t lds = (size_t)2 * p.tile * p.n_select * 4;
        const auto launch = [&](auto i8_, auto big_) {
            constexpr bool I8 = decltype(i8_)::value, BIG = decltype(big_)::value;
            if constexpr (HD <= 128)
                if (p.tile * p.group > kPagedRows) {
                    attn_paged_rows_kernel<HD, I8, BIG, kWideTileLists><<<grid, 256, lds, st>>>(p);
                    return;
                }
            attn_paged_rows_kernel<HD, I8, BIG, kTileLists><<<grid, 256, lds, st>>>(p);
        };
        if (i8 && big) launch(std::true_type{}, std::true_type{});
        else if (i8) launch(std::true_type{}, std::false_type{});
        else if (big) launch(std::false_type{}, std::true_type{});
        else launch(std::false_type{}, std::false_type{});
        return hipGetLastError();
    }
    if (i8 && big) attn_paged_rows_kernel<HD, true, true, kTokenLists><<<grid, 256, 0, st>>>(p);
    else if (i8) attn_paged_rows_kernel<HD, true, false, kTokenLists><<<grid, 256, 0, st>>>(p);
    else if (big) attn_paged_rows_kernel<HD, false, true, kTokenLists><<<grid, 256, 0, st>>>(p);
    else attn_paged_rows_kernel<HD, false, false, kTokenLists><<<grid, 256, 0, st>>>(p);
    if (p.n_chunks > 1) {
        const dim3 rows((unsigned)p.b.n_tokens, (unsigned)(p.n_heads + 3) / 4);
        attn_selected_combine_kernel<HD><<<rows, 256, 0, st>>>(p);
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_attention_selected(uint16_t *out, const uint16_t *q, int n_heads, float scale,
                                     const int32_t *pages, int n_select, const SeqBatch &batch,
                                     const PagedCache &cache, int kv_int8, hipStream_t st) {
    PagedParams p{};
    p.out = out;
    p.q = q;
    p.b = batch;
    p.c = cache;
    p.n_heads = n_heads;
    p.group = n_heads / cache.n_kv;
    p.sl2 = scale * 1.4426950408889634f;
    p.lists = pages;
    p.n_select = n_select;
    const SelectedPlan plan = plan_selected(p, kv_int8);
    if (plan.grid > kPagedMostRows) return hipErrorInvalidValue;
    float *ws = nullptr;
    if (plan.bytes > 0) {
        const hipError_t e = Scratch{}.get(st, plan.bytes, &ws);
        if (e != hipSuccess) return e;
    }
    if (cache.hd <= 64) return launch_selected<64>(p, plan, ws, kv_int8, st);
    if (cache.hd <= 96) return launch_selected<96>(p, plan, ws, kv_int8, st);
    if (cache.hd <= 128) return launch_selected<128>(p, plan, ws, kv_int8, st);
    return launch_selected<256>(p, plan, ws, kv_int8, st);
}

hipError_t launch_attention_paged(uint16_t *out, const uint16_t *q, int n_heads, float scale,
                                  const SeqBatch &batch, const PagedCache &cache, int kv_int8,
                                  hipStream_t st) {
    PagedParams p{};
    p.out = out;
    p.q = q;
    p.b = batch;
    p.c = cache;
    p.n_heads = n_heads;
    p.group = n_heads / cache.n_kv;
    p.sl2 = scale * 1.4426950408889634f;
    // Sequences of up to 16 rows take the 16-row kernel; where the others of the batch
    // have more, on average half the most any has, the 128-row kernel takes them all.
    const int64_t most = (int64_t)std::min(batch.max_new, batch.n_tokens) * p.group;
    const bool blocks = most > kPagedRows;
    const bool rows = !blocks || (batch.n_seqs > 1 && (int64_t)batch.n_tokens * 2 < (int64_t)batch.n_seqs * batch.max_new);
    p.rows_limit = rows ? kPagedRows : 0;
    PagedParams pr = p;
    RowsPlan rp{};
    PagedBlockPlan bp{};
    if (rows) rp = plan_rows(pr, kv_int8, (blocks ? kWorkspaceBytes / 2 : kWorkspaceBytes) - 256);
    if (blocks) bp = plan_paged_blocks(p, kWorkspaceBytes - rp.bytes);
    // (before the first of the launches)
    if (rp.grid > kPagedMostRows || bp.grid > kPagedMostBlocks) return hipErrorInvalidValue;
    float *ws = nullptr;
    if (rp.bytes + bp.bytes > 0) {
        const hipError_t e = Scratch{}.get(st, rp.bytes + bp.bytes, &ws);
        if (e != hipSuccess) return e;
    }
    hipError_t e = hipSuccess;
    if (blocks) e = launch_paged_blocks(p, bp, ws ? ws + rp.bytes / 4 : nullptr, kv_int8, st);
    if (e != hipSuccess || !rows) return e;
    if (cache.hd <= 64) return launch_rows<64>(pr, rp, ws, kv_int8, st);
    if (cache.hd <= 96) return launch_rows<96>(pr, rp, ws, kv_int8, st);
    if (cache.hd <= 128) return launch_rows<128>(pr, rp, ws, kv_int8, st);
    return launch_rows<256>(pr, rp, ws, kv_int8, st);
}

}  // namespace rxq4
