// attn_paged_block.hip -- attention of prompt chunks over a paged KV cache: 128 query
// rows a workgroup, on the gfx950 matrix cores.
//
// The rows of a sequence and KV head are numbered t * group + j (new token t, j-th
// head of the group), cut into blocks of 128, the positions into tiles of 64 and
// those into chunks where there are few blocks.  The walk over the tiles, the
// products, the softmax, the LDS layout and the bounds are those of
// attn_prefill.hip; what is its own:
//   blocks   the batch's lengths are in device memory: a workgroup finds its
//            sequence and block by a sum over the sequences' block counts, a lane a
//            sequence;
//   pages    lane i of a wave looks up row i of the next tile (its page's table
//            entry is loaded a tile earlier).  Pages of 16 positions or more: what a
//            wave loads at once lies in one page, whose address it takes from the
//            lane that looked it up; smaller ones: each row's offset goes to the
//            lanes that load its chunks.  Scores in holes or past the block's sight
//            are -infinity;
//   splits   where the blocks leave CUs idle, every workgroup works out the same
//            chunk length from the batch's lengths: the shortest that leaves at most
//            a workgroup a CU (their 130 KB of LDS).  Chunks cut by the host from the
//            lengths' limit took 34.7 us on 12 drafts of 3 to 6 tokens after 500 to 6000
//            positions (28 / 4 heads), so 25.  A workgroup leaves (O, m, l) per query
//            row; attn_paged_block_combine adds a row's chunks in order.  The host
//            allows it (it launches the combine and lays the partials out by rows) where
//            the rows of the batch could not fill the CUs, decoding and padding rows
//            counted: 16 tokens of 64 / 8 heads after 30000 positions 51 us, with 584 rows
//            of padding or beside 512 decoding sequences, unsplit, 641 and 790.
// Bound: the chain of a tile in a wave (scores, maximum, exponentials, staging, P.V: 7000
// to 8500 cycles, 1536 of them its matrix instructions) between two barriers; the two
// waves of a SIMD are in the same part of it.
// Measured, 32 / 8 heads of 128, fp16: 512 tokens of 16 / 2 heads after 7000 positions
// 65 us (467 TFLOP/s), four prompts of 1254 to 3615 tokens 323 to 340 (519 to 546).
// The second wave group a phase later (V weighed an iteration after its scores, a third V
// buffer) made the prompts 341, a table load outside branches 356, raised priorities for
// the products or fences between the phases 332 to 336.
#include <math.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "attn_paged.h"
#include "attn_tile.h"
#include "launch.h"
#include "mfma_util.h"
#include "paged.h"
#include "q4k_device.h"

namespace rxq4 {
namespace {

constexpr int kMaxChunks = 64;  // chunks per block
constexpr int kSplitSeqs = 1024;  // sequences of a batch whose blocks are cut
// An int8 tile's floats in LDS: K scales, V scales, log2 |V scale|.
constexpr int kScl = 3 * kTile;

typedef const float __attribute__((address_space(1))) *GlobalFloat;
__device__ const float g_one = 1.0f;  // int8 caches without scales: read with stride 0

// Bytes of one K or V tile and of a wave group's LDS (two buffers of K, V).
template <int HD>
constexpr int tile_bytes() { return kTile * HD * 2; }
template <int HD, int G>
constexpr int block_lds() {
    return G * 4 * tile_bytes<HD>()      // K, V x 2 buffers
           + G * 2 * kScl * 4            // int8 scales
           + 2 * 256 * 4                 // (m, l) of the second group
           + G * 4 * 4;                  // a wave's flag: V not finite
}

template <typename Chunk>
__device__ __forceinline__ Chunk load_chunk(__amdgpu_buffer_rsrc_t r, int at, int down) {
    if constexpr (sizeof(Chunk) == 16) return __builtin_amdgcn_raw_buffer_load_b128(r, at, down, 0);
    else return __builtin_amdgcn_raw_buffer_load_b64(r, at, down, 0);
}

// Tiles that a block seeing positions [0, pos_end) walks (one where it sees
// nothing: its rows are zeros).
__device__ __forceinline__ int block_tiles(int pos_end) { return (max(pos_end, 1) + kTile - 1) / kTile; }

// Blocks of sequence s, and the tiles of its last.
__device__ __forceinline__ void seq_blocks(const PagedParams &p, int s, int &blocks, int &tiles) {
    blocks = 0;
    tiles = 0;
    if (s >= p.b.n_seqs) return;
    const SeqSpan span = seq_span(p.b, s);
    const int n = min(span.n, p.b.max_new), rows = n * p.group;
    if (rows <= p.rows_limit) return;
    blocks = (rows + kPagedBlock - 1) / kPagedBlock;
    tiles = block_tiles(min(span.pos0 + n, position_limit(p.b, p.c)));
}

// A workgroup's part of the batch: a block of a sequence and one of the chunks, of
// `chunk_tiles` tiles, that its tiles are cut into.
struct Unit {
    int seq, block, chunk, chunk_tiles;
};

// The idx-th unit of the batch, the same for a whole wave; false past the last one
// (chunk_tiles is set all the same).  The chunks are about as short as leaves at most
// p.max_units of them (a sequence's blocks counted as long as its last), or the
// blocks stay whole: every workgroup comes to the same length from the same sums.
__device__ __forceinline__ bool find_unit(const PagedParams &p, int idx, Unit &u) {
    const int lane = threadIdx.x & 63;
    int nb, nt;
    seq_blocks(p, lane, nb, nt);
    const auto sum = [&](auto f) {  // over the sequences
        float x = nb > 0 ? f(nb, nt) : 0.0f;
        for (int s0 = 64; s0 < p.b.n_seqs; s0 += 64) {
            int b, t;
            seq_blocks(p, s0 + lane, b, t);
            x += b > 0 ? f(b, t) : 0.0f;
        }
        return butterfly_sum<64>(x);
    };
    int ct = p.most_tiles;
    const float most = (float)p.max_units;
    const float blocks = p.n_chunks > 1 ? sum([](int b, int) { return (float)b; }) : most;
    if (blocks < most) {
        const float all = sum([](int b, int t) { return (float)b * (float)t; });
        ct = max(p.min_tiles, (int)(all / most));
        int tries = 6;
        while (sum([&](int b, int t) { return (float)b * (float)((t + ct - 1) / ct); }) > most) {
            // (a chunk a block more than their tiles' share at most: this many do)
            if (--tries == 0) {
                ct = max(ct, (int)fminf(all / (most - blocks), 0x1p24f) + 1);
                break;
            }
            ct += max(1, ct >> 4);
        }
        ct = min(ct, p.most_tiles);
    }
    u.chunk_tiles = ct = __builtin_amdgcn_readfirstlane(ct);
    for (int s0 = 0; s0 < p.b.n_seqs; s0 += 64) {
        if (s0 > 0) seq_blocks(p, s0 + lane, nb, nt);
        const int n_c = (nt + ct - 1) / ct, n = nb * n_c;
        int upto = n;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int x = __shfl_up(upto, d, 64);
            if (lane >= d) upto += x;
        }
        const uint64_t past = __builtin_amdgcn_ballot_w64(upto > idx);
        if (past != 0) {
            const int at = __builtin_ctzll(past);
            const int in = idx - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(n, at));
            const int chunks = __builtin_amdgcn_readlane(n_c, at);
            const int from_last = __builtin_amdgcn_readfirstlane(in / chunks);
            u.seq = s0 + at;
            u.block = __builtin_amdgcn_readlane(nb, at) - 1 - from_last;  // the latest tokens first
            u.chunk = in - from_last * chunks;
            return true;
        }
        idx -= __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

// BIG: pages of 16 positions or more.
template <int HD, bool I8, int G, bool BIG>
__global__ __launch_bounds__(256 * G) void attn_paged_block_kernel(PagedParams p) {
    constexpr int KS = HD / 16;             // k-steps of the scores
    constexpr int DT = HD / 32;             // 32-dim tiles of O
    constexpr int TB = tile_bytes<HD>();
    constexpr int CH = HD / 8;              // 16-byte chunks per row
    constexpr int NC = kTile * CH / 256;    // 8-dim chunks per thread and tile (K, V each)
    constexpr int esz = I8 ? 1 : 2;
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];

    const int gq = G == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
    const int tid = threadIdx.x & 255, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r32 = lane & 31, h = lane >> 5;
    uint8_t *const lds = smem + gq * 4 * TB;  // buffer b: K at 2 b TB, V at (2 b + 1) TB
    float *const scl = reinterpret_cast<float *>(smem + G * 4 * TB) + gq * 2 * kScl;
    float *const mgl = reinterpret_cast<float *>(smem + G * 4 * TB + G * 8 * kScl);
    int *const bad_v = reinterpret_cast<int *>(mgl + 512) + gq * 4;

    const int kvh = blockIdx.x % p.c.n_kv;
    Unit unit;
    const bool found = find_unit(p, blockIdx.x / p.c.n_kv, unit);
    if (p.n_chunks > 1 && blockIdx.x == 0 && threadIdx.x == 0) *p.chunk_tiles = unit.chunk_tiles;
    if (!found) return;  // uniform
    const int seq = unit.seq, block = unit.block, chunk = unit.chunk, chunk_tiles = unit.chunk_tiles;
    const SeqSpan span = seq_span(p.b, seq);
    const int hd = p.c.hd;
    const int n_rows = min(span.n, p.b.max_new) * p.group;
    const int blk_last = min(n_rows, (block + 1) * kPagedBlock) - 1;
    const int limit = position_limit(p.b, p.c);
    const int pos_end = min(span.pos0 + blk_last / p.group + 1, limit);  // positions the block sees
    const int n_tiles = block_tiles(pos_end);
    const int t_beg = chunk * chunk_tiles;
    const int t_end = min(n_tiles, t_beg + chunk_tiles);
    if (t_beg >= t_end) return;  // uniform

    // The lane's query row.
    const int row0 = block * kPagedBlock + 32 * w;
    const bool live_wave = row0 < n_rows;
    const RowMap rm = row_map(min(row0, n_rows - 1), p.group);
    int tok, hj, tok_last, unused;
    rm.at(min(r32, max(0, n_rows - 1 - row0)), tok, hj);
    rm.at(min(31, max(0, n_rows - 1 - row0)), tok_last, unused);
    const int qpos = span.pos0 + tok;  // last visible position
    const int wave_first = span.pos0 + rm.tok0;
    const int wave_end = live_wave ? span.pos0 + __builtin_amdgcn_readfirstlane(tok_last) + 1 : 0;
    const int row_bytes = p.c.n_kv * hd * esz;
    const uint8_t *kb = p.c.k + (int64_t)kvh * hd * esz;
    const uint8_t *vb = p.c.v + (int64_t)kvh * hd * esz;
    // (global pointers: a generic load would be waited for with the LDS reads)
    const GlobalFloat ksp = p.c.ks ? (GlobalFloat)(p.c.ks + kvh) : (GlobalFloat)&g_one;
    const GlobalFloat vsp = p.c.vs ? (GlobalFloat)(p.c.vs + kvh) : (GlobalFloat)&g_one;
    const int s_stride = p.c.ks ? p.c.n_kv : 0, v_stride = p.c.vs ? p.c.n_kv : 0;
    const int n_ch = hd >> 3;
    const bool negate = p.sl2 < 0.0f;
    // (a tiny positive scale for 0, so that masked scores stay -inf)
    const float sl2 = fmaxf(fabsf(p.sl2), 1e-30f);

    // Q^T fragments: dims 16 ks + 8 h .. + 7 of the row (zeros past hd).
    u32x4 qf[KS];
    {
        const uint16_t *qrow = p.q + ((int64_t)(span.row0 + tok) * p.n_heads + kvh * p.group + hj) * hd;
        const uint32_t flip = negate ? 0x80008000u : 0u;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int c = 2 * ks + h;
            u32x4 x = *reinterpret_cast<const u32x4 *>(qrow + 8 * min(c, n_ch - 1));
            x = u32x4{x.x ^ flip, x.y ^ flip, x.z ^ flip, x.w ^ flip};
            qf[ks] = c < n_ch ? x : u32x4{0u, 0u, 0u, 0u};
        }
    }

    // The thread's chunks of a tile: row, place in the row, LDS offsets.  Where a row
    // divides the 256 chunks, chunk j is kRows rows down and the places in a K row
    // repeat every kPerK chunks: only what differs is kept.
    constexpr bool kEven = 256 % CH == 0;
    constexpr int kRows = 256 / CH, kPer = kEven ? 1 : NC, kPerK = kEven && kRows % 16 ? 16 / kRows : kPer;
    static_assert(!kEven || kRows % 4 == 0, "the places in a V row repeat");
    int ik[kPerK], iv[kPer];
#pragma unroll
    for (int j = 0; j < kPerK; ++j) {
        const int id = tid + 256 * j, pr = id / CH, c = id % CH;
        ik[j] = pr * HD * 2 + 16 * k_pos<HD>(pr, c);
        if (j < kPer) iv[j] = pr * HD * 2 + 16 * v_pos<HD>(pr, c);
    }
    auto chunk_row = [&](int j) { return kEven ? tid / CH + j * kRows : (tid + 256 * j) / CH; };
    auto chunk_col = [&](int j) { return kEven ? tid % CH : (tid + 256 * j) % CH; };
    auto chunk_k = [&](int j) { return ik[j % kPerK] + (kEven ? j / kPerK * kPerK * kRows * HD * 2 : 0); };
    auto chunk_v = [&](int j) { return kEven ? iv[0] + j * kRows * HD * 2 : iv[j % kPer]; };
    using Chunk = typename std::conditional<I8, u32x2, u32x4>::type;
    struct Raw {
        Chunk c[NC];
        float s;
    };
    // Lane i of a wave looks up row i of a tile: the page's table entry one tile
    // before the tile's loads, then the row's offset, which the lanes of its chunks
    // get from it.
    const int32_t *const table = p.c.table ? p.c.table + (int64_t)seq * p.c.width : nullptr;
    auto entry = [&](int t) {
        const int i = min(t * kTile + lane, limit - 1) >> p.c.shift;
        return limit <= 0 ? -1 : table ? table[i] : i;
    };
    // Pages of 16 or more: the 64 chunks that a wave loads at once lie in one aligned
    // group of 16 rows, so in one page, and the wave takes its address from the lane
    // that looked it up: a resource over the 16 rows, of no bytes in a hole.
    int at_row[BIG ? kPer : 1];
    if constexpr (BIG) {
#pragma unroll
        for (int j = 0; j < kPer; ++j)
            at_row[j] = chunk_col(j) < n_ch ? chunk_row(j) % 16 * row_bytes + 8 * esz * chunk_col(j) : 0x7FFFFFFF - 15;
    }
    int ent = 0;
    uint64_t there = 0;  // the tile's positions in the block's sight and in the pool
    Raw K, V;
    auto load_tile = [&](int t) {
        const int pos = t * kTile + lane;
        const bool ok = pos < pos_end && (unsigned)ent < (unsigned)p.c.n_pages;
        there = __builtin_amdgcn_ballot_w64(ok);
        const int slot = ok ? (ent << p.c.shift) + (pos & ((1 << p.c.shift) - 1)) : 0;
        if constexpr (BIG) {
#pragma unroll
            for (int j = 0; j < NC; ++j) {
                const int g = (64 * w + 256 * j) / (16 * CH);
                const int page = __builtin_amdgcn_readlane(ent, 16 * g), p0 = t * kTile + 16 * g;
                const bool in_pool = p0 < pos_end && (unsigned)page < (unsigned)p.c.n_pages;
                const int64_t at = in_pool ? (int64_t)page * p.c.page_bytes + (p0 & ((1 << p.c.shift) - 1)) * row_bytes : 0;
                const int bytes = in_pool ? 16 * row_bytes - kvh * hd * esz : 0;
                const auto kr = make_rsrc(kb + at, bytes), vr = make_rsrc(vb + at, bytes);
                const int place = kEven ? at_row[0] : at_row[j % kPer], down = kEven ? j * kRows % 16 * row_bytes : 0;
                K.c[j] = load_chunk<Chunk>(kr, place, down);
                V.c[j] = load_chunk<Chunk>(vr, place, down);
            }
        } else {
            const int64_t off = ok ? slot_bytes(p.c, slot, row_bytes) : -1;
#pragma unroll
            for (int j = 0; j < NC; ++j) {
                const uint32_t lo = (uint32_t)__shfl((int)(uint32_t)off, chunk_row(j), 64);
                const int hi = __shfl((int)(off >> 32), chunk_row(j), 64);
                const int64_t at = (((int64_t)hi << 32) | lo) + 8 * esz * chunk_col(j);
                K.c[j] = Chunk{};
                V.c[j] = Chunk{};
                if (hi >= 0 && chunk_col(j) < n_ch) {
                    K.c[j] = *reinterpret_cast<const Chunk *>(kb + at);
                    V.c[j] = *reinterpret_cast<const Chunk *>(vb + at);
                }
            }
        }
        if (I8) {
            K.s = ksp[(int64_t)slot * s_stride];
            V.s = vsp[(int64_t)slot * v_stride];
            if (!ok) K.s = V.s = 0.0f;
        }
        ent = entry(t + G);
    };
    auto widen = [](Chunk c) {
        if constexpr (I8) {
            const u32x2 a = i8x4_to_f16(c.x), b = i8x4_to_f16(c.y);
            return u32x4{a.x, a.y, b.x, b.y};
        } else {
            return c;
        }
    };
    auto store_raw = [&](const Raw &R, int off, auto place, int s_off) {
#pragma unroll
        for (int j = 0; j < NC; ++j) *reinterpret_cast<u32x4 *>(lds + off + place(j)) = widen(R.c[j]);
        if (I8 && tid < kTile) scl[s_off + tid] = R.s;
    };
    // log2 |V scale| of the tile's positions, clamped, and a bound of theirs that
    // seldom moves (a maximum over the lanes for every tile costs 3%).  None for
    // the first tile, where the row's maximum is taken exactly in any case.
    float most_log = kMaxScale;
    auto store_log = [&](float vs, int s_off, bool first) {
        if constexpr (I8) {
            const float lg = fminf(fmaxf(__builtin_amdgcn_logf(fabsf(vs)), kMinScale), kMaxScale);
            if (!first && (__builtin_amdgcn_ballot_w64(lg > most_log) != 0 || most_log >= kMaxScale))
                most_log = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(
                               int, butterfly_max<64>(lg) + 0.125f)));
            if (tid < kTile) scl[s_off + tid] = lg;
        }
    };

    // An infinity or NaN in V would reach the rows that do not see it as 0 times it, and
    // the others through the low half of P: such values (int8: V scales) are staged
    // again as zeros, and the rows that see them get them at the end.
    if (lane == 0) bad_v[w] = 0;  // the wave's flag: some of its staging
    auto look_over = [&](Raw &R, int off, int s_off) {
        if constexpr (I8) {
            const bool bad = !(fabsf(R.s) < INFINITY);
            if (__builtin_amdgcn_ballot_w64(bad) == 0) return;
            if (bad && tid < kTile) scl[s_off + tid] = 0.0f;
        } else {
            if (__builtin_amdgcn_ballot_w64(not_finite16<NC>(R.c)) == 0) return;
            Raw Z = R;  // (copies: head_dim 80, 775 tokens, 20.2 us with the loaded registers changed in place, 19.5)
#pragma unroll
            for (int j = 0; j < NC; ++j) asm volatile("" : "+v"(Z.c[j]));
            zero_not_finite16<NC>(Z.c);
            store_raw(Z, off, chunk_v, s_off);
        }
        if (lane == 0) bad_v[w] = 1;
    };

    // Lane parts of the fragment addresses: K row 32 pt + r32, chunk
    // 2 ks + h; V row 16 kk + 8 x + 4 h + (r16 / 4), dims 32 dt + 16 (l / 16 % 2)
    // + 4 (r16 % 4) (the transposing read hands the lane dim 32 dt + r32).
    const int r16 = lane & 15;
    int ka[KS], va[DT];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) ka[ks] = r32 * HD * 2 + 16 * k_pos<HD>(r32, 2 * ks + h);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
        const int vr = 4 * h + (r16 >> 2), d = 32 * dt + 16 * ((lane >> 4) & 1) + 4 * (r16 & 3);
        va[dt] = vr * HD * 2 + 16 * v_pos<HD>(vr, d >> 3) + 2 * (d & 7);
    }

    f32x16 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = f32x16{};
    float m = -INFINITY, l = 0.0f;  // l: this lane's positions only

    u32x4 ph[4], pl[4];  // P^T hi / lo operands per 16-position k step
    auto softmax = [&](int t, int b, uint64_t in) {
        const int p0 = t * kTile;
        const uint8_t *kt = lds + b * 2 * TB;
        f32x16 s[2];
#pragma unroll
        for (int pt = 0; pt < 2; ++pt) {
            s[pt] = f32x16{};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
                s[pt] = mfma32h(*reinterpret_cast<const u32x4 *>(kt + ka[ks] + pt * 64 * HD), qf[ks], s[pt]);
        }
        if constexpr (I8) {
            const float *sk = scl + b * kScl;
#pragma unroll
            for (int pt = 0; pt < 2; ++pt)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const f32x4 x = *reinterpret_cast<const f32x4 *>(sk + 32 * pt + 8 * j + 4 * h);
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[pt][4 * j + i] *= x[i];
                }
        }
        if (p0 + kTile - 1 > wave_first || in != ~0ull) {  // uniform: the diagonal's tiles, holes
            const uint32_t in_h[2] = {(uint32_t)in >> (4 * h), (uint32_t)(in >> 32) >> (4 * h)};
#pragma unroll
            for (int pt = 0; pt < 2; ++pt)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (p0 + 32 * pt + 8 * (i >> 2) + 4 * h + (i & 3) > qpos ||
                        !((in_h[pt] >> (8 * (i >> 2) + (i & 3))) & 1u))
                        s[pt][i] = -INFINITY;
        }
        // the row's largest P in log2 units: the score, with V scales score +
        // log2 |scale|, at most the largest of each together
        float mx = -INFINITY;
#pragma unroll
        for (int pt = 0; pt < 2; ++pt)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[pt][i]);
        mx = max_xor_rows<32>(mx) * sl2;
        if constexpr (I8) {
            const float *sg = scl + b * kScl + 2 * kTile;
            if (__builtin_amdgcn_ballot_w64(mx + most_log > m + kLazy) != 0) {  // m may have to move: exactly
                mx = -INFINITY;
#pragma unroll
                for (int pt = 0; pt < 2; ++pt)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const f32x4 x = *reinterpret_cast<const f32x4 *>(sg + 32 * pt + 8 * j + 4 * h);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            mx = fmaxf(mx, __builtin_fmaf(s[pt][4 * j + i], sl2, x[i]));
                    }
                mx = max_xor_rows<32>(mx);
            } else {
                mx = -INFINITY;
            }
        }
        // m moves when the row's maximum has outgrown it by 2^kLazy (always
        // at a row's first visible position): |P| <= 2^(kLazy + kShift), and O
        // and l stay relative to the same m
        if (__builtin_amdgcn_ballot_w64(mx > m + kLazy) != 0) {
            // (each row's by its own rule: no row depends on what others see)
            const float m_new = mx > m + kLazy ? mx : m;
            const float corr = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - m_new);
            m = m_new;
            l *= corr;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[dt][i] *= corr;
        }
        const float m_use = m == -INFINITY ? 0.0f : m - kShift;  // rows with nothing visible yet: e = 0
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            f32x4 x0, x1;
            if constexpr (I8) {
                const float *sv = scl + b * kScl + kTile;
                x0 = *reinterpret_cast<const f32x4 *>(sv + 16 * kk + 4 * h);
                x1 = *reinterpret_cast<const f32x4 *>(sv + 16 * kk + 8 + 4 * h);
            }
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const int i = 8 * (kk & 1) + e;  // register of k = e
                float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kk >> 1][i], sl2, -m_use));
                float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kk >> 1][i + 1], sl2, -m_use));
                l += e0;
                l += e1;
                if constexpr (I8) {
                    e0 *= e < 4 ? x0[e] : x1[e - 4];
                    e1 *= e < 4 ? x0[e + 1] : x1[e - 3];
                }
                const uint32_t hi = pack2<RXQ4_DTYPE_F16>(e0, e1);
                ph[kk][e >> 1] = hi;
                pl[kk][e >> 1] = low_halves(e0, e1, hi);
            }
        }
    };
    auto weigh = [&](int b) {
        const uint8_t *vt = lds + (b * 2 + 1) * TB;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const uint8_t *vp = vt + va[dt] + kk * 32 * HD;
                const u32x2 v0 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                               (__attribute__((address_space(3))) v4i16 *)vp));
                const u32x2 v1 = __builtin_bit_cast(
                    u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                               (__attribute__((address_space(3))) v4i16 *)(vp + 16 * HD)));
                const u32x4 a = u32x4{v0.x, v0.y, v1.x, v1.y};
                o[dt] = mfma32h(a, ph[kk], o[dt]);
                o[dt] = mfma32h(a, pl[kk], o[dt]);
            }
    };

    // Tiles t_beg + gq, + G, ...: tile j of the group is in buffer j & 1
    // during iteration j, and tile j + 1 is written to the other one, which
    // every wave has left at the barrier.  A tile past the wave's visible
    // positions changes nothing and is skipped.
    const int n_j = (t_end - t_beg - gq + G - 1) / G;  // this group's tiles
    const int n_it = (t_end - t_beg + G - 1) / G;      // every group's iterations
    const int t_first = t_beg + gq;
    auto store_tile = [&](int t, int b, bool first) {
        store_raw(K, b * 2 * TB, chunk_k, b * kScl);
        store_raw(V, (b * 2 + 1) * TB, chunk_v, b * kScl + kTile);
        store_log(V.s, b * kScl + 2 * kTile, first);
        look_over(V, (b * 2 + 1) * TB, b * kScl + kTile);
    };
    uint64_t in = 0;
    if (n_j > 0) {
        ent = entry(t_first);
        load_tile(t_first);
        in = there;
        store_tile(t_first, 0, true);
    }
    for (int j = 0; j < n_it; ++j) {
        wait_lgkmcnt0();
        lds_barrier();
        const int t = t_first + G * j;
        const bool next = j + 1 < n_j;
        const bool live = j < n_j && t * kTile < wave_end;  // uniform
        if (next) load_tile(t + G);
        if (live) softmax(t, j & 1, in);
        if (next) store_tile(t + G, (j + 1) & 1, false);
        if (live) weigh(j & 1);
        in = there;
    }
    wait_lgkmcnt0();
    lds_barrier();
    if (__builtin_amdgcn_readfirstlane(bad_v[0] | bad_v[1] | bad_v[2] | bad_v[3]) != 0) {
        for (int t = t_beg; t < t_end; ++t) {
            if ((t - t_beg) % G != gq) continue;
            for (int pos = t * kTile; pos < min(wave_end, t * kTile + kTile); ++pos) {
                const int slot = pos < limit ? slot_of(p.c, seq, pos) : -1;
                if (slot < 0) continue;  // uniform
                const uint8_t *row = vb + slot_bytes(p.c, slot, row_bytes) + 4 * esz * h;
                const float vs = I8 ? vsp[(int64_t)slot * v_stride] : 1.0f;
                if (pos > qpos || (I8 && fabsf(vs) < INFINITY)) continue;
                int n = n_ch;
                asm volatile("" : "+s"(n));  // (compared here, not kept as CH conditions)
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    if (c >= n) continue;  // uniform
                    const u32x2 x = I8 ? u32x2{*reinterpret_cast<const uint32_t *>(row + 8 * c), 0u}
                                       : *reinterpret_cast<const u32x2 *>(row + 16 * c);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float v = I8 ? vs * (float)(int8_t)(x.x >> (8 * i))
                                           : f16_bits_to_f32((i < 2 ? x.x : x.y) >> (16 * (i & 1)) & 0xFFFFu);
                        if (!(fabsf(v) < INFINITY)) o[c / 4][4 * (c % 4) + i] += v;
                    }
                }
            }
        }
    }

    // Merge: the second group hands (O, m, l) over through its own buffers.
    l = sum_xor_rows<32>(l);
    if (G == 2) {
        float *mb = reinterpret_cast<float *>(smem + 4 * TB);  // HD / 2 x 256 floats
        if (gq == 1) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) mb[(16 * dt + i) * 256 + tid] = o[dt][i];
            mgl[tid] = m;
            mgl[256 + tid] = l;
        }
        wait_lgkmcnt0();
        lds_barrier();
        if (gq == 1) return;
        int bad = 0;  // either group's V
#pragma unroll
        for (int i = 0; i < 8; ++i) bad |= bad_v[i];
        bad = __builtin_amdgcn_readfirstlane(bad);
        const float m1 = mgl[tid], l1 = mgl[256 + tid];
        const float mm = fmaxf(m, m1);
        const bool any = mm != -INFINITY;
        const float c0 = any ? __builtin_amdgcn_exp2f(m - mm) : 0.0f;
        const float c1 = any ? __builtin_amdgcn_exp2f(m1 - mm) : 0.0f;
        l = l * c0 + l1 * c1;
        m = mm;
        if (bad != 0) {  // uniform, rare; the same sums
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    o[dt][i] = add_weighed(add_weighed(0.0f, c0, o[dt][i]), c1, mb[(16 * dt + i) * 256 + tid]);
        } else {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[dt][i] = __builtin_fmaf(c1, mb[(16 * dt + i) * 256 + tid], c0 * o[dt][i]);
        }
    }
    if (!live_wave) return;
    if (n_tiles > chunk_tiles) {  // the block has several chunks
        if (row0 + r32 >= n_rows) return;
        const int64_t at = ((int64_t)(span.row0 + tok) * p.n_heads + kvh * p.group + hj) * p.n_chunks + chunk;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *reinterpret_cast<f32x4 *>(p.part + at * HD + 32 * dt + 8 * j + 4 * h) =
                    f32x4{o[dt][4 * j], o[dt][4 * j + 1], o[dt][4 * j + 2], o[dt][4 * j + 3]};
        if (h == 0) {
            p.stats[2 * at] = m;
            p.stats[2 * at + 1] = l;
        }
        return;
    }
    // Output rows through the wave's own LDS rows: 16 bytes a lane, a row's
    // bytes together (straight from the registers: 8-byte pieces of 32 rows).
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    constexpr int OP = 2 * HD + 16;  // LDS pitch of a staged row
    static_assert(4 * 32 * OP <= 4 * TB, "the staged rows fit the group's buffers");
    uint8_t *ow = lds + w * 32 * OP;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t a = pack2<RXQ4_DTYPE_F16>(o[dt][4 * j] * inv, o[dt][4 * j + 1] * inv);
            const uint32_t c = pack2<RXQ4_DTYPE_F16>(o[dt][4 * j + 2] * inv, o[dt][4 * j + 3] * inv);
            *reinterpret_cast<u32x2 *>(ow + r32 * OP + 2 * (32 * dt + 8 * j + 4 * h)) = u32x2{a, c};
        }
    wait_lgkmcnt0();
#pragma unroll
    for (int i = 0; i < 32 * CH / 64; ++i) {
        const int id = lane + 64 * i, rr = id / CH, c = id % CH;
        const int orow = row0 + rr;
        if (orow < n_rows && c < n_ch) {
            int t, jj;
            rm.at(rr, t, jj);
            *reinterpret_cast<u32x4 *>(p.out + ((int64_t)(span.row0 + t) * p.n_heads + kvh * p.group + jj) * hd + 8 * c) =
                *reinterpret_cast<const u32x4 *>(ow + rr * OP + 16 * c);
        }
    }
}

// out = sum_c 2^(m_c - M) O_c / sum_c 2^(m_c - M) l_c over a row's chunks in order.  A
// wave takes a row: a lane's chunk for the weights, then a lane's dims.
template <int HD>
__global__ __launch_bounds__(256) void attn_paged_block_combine_kernel(PagedParams p) {
    constexpr int NE = (HD + 63) / 64;
    const int lane = threadIdx.x & 63;
    const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (id >= (int64_t)p.b.n_tokens * p.n_heads) return;
    const int t = (int)(id / p.n_heads), head = (int)(id % p.n_heads);
    SeqSpan span;
    const int seq = seq_of_row(p.b, t, span);
    if (seq >= p.b.n_seqs) return;
    const int n_rows = min(span.n, p.b.max_new) * p.group;
    const int row = (t - span.row0) * p.group + head % p.group;
    if (t < span.row0 || row >= n_rows || n_rows <= p.rows_limit) return;
    const int blk_last = min(n_rows, (row / kPagedBlock + 1) * kPagedBlock) - 1;
    const int tiles = block_tiles(min(span.pos0 + blk_last / p.group + 1, position_limit(p.b, p.c)));
    const int ct = *p.chunk_tiles, n_c = min((tiles + ct - 1) / ct, p.n_chunks);
    if (n_c <= 1) return;  // written already
    const int64_t at = id * p.n_chunks;
    const int c = min(lane, n_c - 1);
    const float mc = p.stats[2 * (at + c)], lc = p.stats[2 * (at + c) + 1];
    const float M = butterfly_max<64>(mc);
    const float e = M != -INFINITY && lane < n_c ? __builtin_amdgcn_exp2f(mc - M) : 0.0f;
    const float L = butterfly_sum<64>(e * lc);
    float acc[NE] = {};
    const float *src = p.part + at * HD;
    for (int i = 0; i < n_c; i += 4) {  // (four chunks' loads at once)
        float x[4][NE];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int k = 0; k < NE; ++k) x[j][k] = src[(int64_t)min(i + j, n_c - 1) * HD + min(lane + 64 * k, HD - 1)];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float ei = __shfl(e, (i + j) & 63, 64);  // (past the last chunk: that again, 0 times)
#pragma unroll
            for (int k = 0; k < NE; ++k) acc[k] = add_weighed(acc[k], ei, x[j][k]);
        }
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
    for (int k = 0; k < NE; ++k) {
        const int d = lane + 64 * k;
        if (d < p.c.hd) p.out[id * p.c.hd + d] = f32_to_f16_bits(acc[k] * inv);
    }
}

constexpr int kBigDim = 128;  // larger heads: one wave group, 512 registers a wave
int pad_dim(int hd) { return hd <= 64 ? 64 : hd <= 96 ? 96 : hd <= 128 ? 128 : 256; }
// Tiles per chunk at least, where a block is cut: one a wave group (27 drafts of 3 to 6
// tokens after up to 1181 positions 19.7 us with four, 17.7 so; head_dim 256, three
// chunks of 67 to 134 tokens 52.4 and 40.5).  Blocks of four tiles or less stay whole: the
// combine takes longer than their walk (5 drafts after up to 250 positions 10.5, cut 12.1).
constexpr int least_tiles(int pad) { return pad > kBigDim ? 1 : 2; }

// Blocks of the batch at most: every sequence's rows past the limit, each with a
// last block of its own.
int64_t most_blocks(const PagedParams &p) {
    const int64_t rows = (int64_t)p.b.n_tokens * p.group;
    return rows / kPagedBlock + std::min<int64_t>(p.b.n_seqs, rows / (p.rows_limit + 1));
}

template <int HD, bool I8, bool BIG>
hipError_t launch_t(const PagedParams &p, int64_t grid, hipStream_t st) {
    constexpr int G = HD > kBigDim ? 1 : 2;
    constexpr int lds = block_lds<HD, G>();
    // the dynamic LDS limit, raised once per device (devices 0..63)
    static std::atomic<uint64_t> raised{0};
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (!(raised.load(std::memory_order_acquire) & bit)) {
        e = hipFuncSetAttribute(reinterpret_cast<const void *>(&attn_paged_block_kernel<HD, I8, G, BIG>),
                                hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return e;
        raised.fetch_or(bit, std::memory_order_acq_rel);
    }
    attn_paged_block_kernel<HD, I8, G, BIG><<<(unsigned)grid, 256 * G, lds, st>>>(p);
    if (p.n_chunks > 1)
        attn_paged_block_combine_kernel<HD>
            <<<(unsigned)(((int64_t)p.b.n_tokens * p.n_heads + 3) / 4), 256, 0, st>>>(p);
    return hipGetLastError();
}

template <int HD>
hipError_t launch_hd(const PagedParams &p, int64_t grid, int i8, hipStream_t st) {
    const bool big = p.c.shift >= 4;
    if (i8) return big ? launch_t<HD, true, true>(p, grid, st) : launch_t<HD, true, false>(p, grid, st);
    return big ? launch_t<HD, false, true>(p, grid, st) : launch_t<HD, false, false>(p, grid, st);
}

}  // namespace

PagedBlockPlan plan_paged_blocks(const PagedParams &p, size_t room) {
    const int cus = device_info().cu_count > 0 ? device_info().cu_count : 256;
    const int64_t len = std::max<int64_t>(1, std::min<int64_t>(p.b.max_len, (int64_t)p.c.width << p.c.shift));
    const int tiles = (int)((len + kTile - 1) / kTile);
    const size_t per = (size_t)p.b.n_tokens * p.n_heads * (pad_dim(p.c.hd) + 2) * 4;
    const int64_t units = std::max(1, cus / p.c.n_kv);
    int64_t want = 1;
    if ((int64_t)p.b.n_tokens * p.group / kPagedBlock < units && p.b.n_seqs <= kSplitSeqs && tiles > 4 && room > 256)
        want = std::max<int64_t>(1, std::min<int64_t>({tiles / least_tiles(pad_dim(p.c.hd)), kMaxChunks, (int64_t)((room - 256) / per)}));
    if (tuning().attn_split) want = std::min<int64_t>(want, tuning().attn_split);
    const int64_t grid = (want > 1 ? std::max(units, most_blocks(p)) : most_blocks(p)) * p.c.n_kv;
    return PagedBlockPlan{(int)units, (int)want, tiles, grid, want > 1 ? per * want + 256 : 0};
}

hipError_t launch_paged_blocks(PagedParams p, const PagedBlockPlan &plan, float *ws, int i8, hipStream_t st) {
    p.max_units = plan.units;
    p.n_chunks = plan.n_chunks;
    p.most_tiles = plan.tiles;
    p.min_tiles = std::max((plan.tiles + plan.n_chunks - 1) / plan.n_chunks, least_tiles(pad_dim(p.c.hd)));
    p.chunk_tiles = reinterpret_cast<int *>(ws);
    p.part = ws ? ws + 64 : nullptr;
    p.stats = ws ? p.part + (size_t)p.b.n_tokens * p.n_heads * p.n_chunks * pad_dim(p.c.hd) : nullptr;
    switch (pad_dim(p.c.hd)) {
        case 64: return launch_hd<64>(p, plan.grid, i8, st);
        case 96: return launch_hd<96>(p, plan.grid, i8, st);
        case 128: return launch_hd<128>(p, plan.grid, i8, st);
        default: return launch_hd<256>(p, plan.grid, i8, st);
    }
}

}  // namespace rxq4
