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
// an int8 step holds half the bytes of an fp16 one.
constexpr int rows_waves(int hd, bool i8) { return hd > 128 ? 1 : hd == 64 ? 4 : i8 ? 3 : 2; }

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
template <int HD, bool I8, bool BIG>
__global__ __launch_bounds__(256, rows_waves(HD, I8)) void attn_paged_rows_kernel(PagedParams p) {
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

    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4;
    uint16_t *const vl = reinterpret_cast<uint16_t *>(smem) + w * 32 * VROW;
    // The KV heads of a sequence's chunk go to one XCD (workgroups are dealt to the eight in
    // turn): they read the same pages and scales (int8, 512 sequences of 1023 positions, 244
    // us with the heads on all, 216 so).  A sequence's chunks go to different ones.
    const int x8 = blockIdx.x / 8, kvh = x8 % p.c.n_kv;
    const RowsUnit unit = rows_unit(p, x8 / p.c.n_kv * 8 + blockIdx.x % 8);
    const int s = unit.s, c = unit.c, beg = c * unit.chunk;
    if (s < 0) return;  // uniform
    if (p.n_chunks > 1 && c == 0 && kvh == 0 && tid == 0) {
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
    auto entries = [&](int j) { return entry(beg + 32 * w + kStep * (j + (lane >> 1)) + 16 * (lane & 1)); };
    int ent = BIG ? entries(0) : entry(p_lane), ent_next = BIG ? 0 : entry(p_lane + kStep);
    const SeqSpan span = unit.span;
    const int rows = min(span.n, p.b.max_new) * p.group;
    const int end_seq = min(span.pos0 + (rows - 1) / p.group + 1, limit);
    const int end = min(end_seq, beg + unit.chunk);
    const int row = min(r, rows - 1);  // (columns past the last row repeat it)
    const int tok = row / p.group, head = kvh * p.group + row % p.group;
    const bool row_ok = r < rows;
    const int hd = p.c.hd, n_ch = hd / EC;
    const int64_t orow = ((int64_t)(span.row0 + tok) * p.n_heads + head) * hd;
    if (end <= beg) {  // uniform
        if (c == 0 && w == 0 && row_ok)  // the tokens see nothing
            for (int ch = g; ch < hd / 8; ch += 4) *reinterpret_cast<u32x4 *>(p.out + orow + 8 * ch) = u32x4{0u, 0u, 0u, 0u};
        return;
    }
    const int qpos = span.pos0 + tok;
    const int row_bytes = p.c.n_kv * hd * esz;
    const uint8_t *kb = p.c.k + (int64_t)kvh * hd * esz, *vb = p.c.v + (int64_t)kvh * hd * esz;

    u32x4 qf[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const int ch = I8 ? 2 * (4 * (ks / 2) + g) + ks % 2 : 4 * ks + g;  // of 8 dims
        qf[ks] = ch < hd / 8 ? load16(p.q + orow + 8 * ch) : u32x4{0u, 0u, 0u, 0u};
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
    struct Step {
        u32x4 k[2][KL], v[NV];
        float ks, vs;
        uint32_t seen;  // which of the wave's 32 positions there are
    };
    auto load_step = [&](int j, int e, Step &S) {
        const int mask = (1 << p.c.shift) - 1;
        if constexpr (BIG) {
            // an operand's rows: those of its positions that there are, from the first
            __amdgpu_buffer_rsrc_t kr[2], vr[2];
            S.seen = 0;
            int page[2], place[2];
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                const int pos = beg + 32 * w + kStep * j + 16 * st;
                page[st] = __builtin_amdgcn_readlane(e, (2 * j + st) & 63);
                const int n = (unsigned)page[st] < (unsigned)p.c.n_pages ? max(min(end - pos, 16), 0) : 0;
                S.seen |= ((1u << n) - 1) << (16 * st);
                page[st] = n > 0 ? page[st] : 0;
                place[st] = pos & mask;
                const int64_t base = (int64_t)page[st] * p.c.page_bytes + (int64_t)place[st] * row_bytes;
                const int bytes = n > 0 ? (n - 1) * row_bytes + hd * esz : 0;
                kr[st] = make_rsrc(kb + base, bytes);
                vr[st] = make_rsrc(vb + base, bytes);
            }
            if constexpr (I8) {
                const bool ok = (S.seen >> (lane & 31)) & 1;
                const int64_t at = ok ? ((int64_t)(lane & 16 ? page[1] : page[0]) << p.c.shift) +
                                            (lane & 16 ? place[1] : place[0]) + (lane & 15) : 0;
                S.ks = ksp[at * s_stride];
                S.vs = vsp[at * v_stride];
            }
#pragma unroll
            for (int st = 0; st < 2; ++st)
#pragma unroll
                for (int i = 0; i < KL; ++i) S.k[st][i] = buffer_load16(kr[st], ko[i]);
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                constexpr bool kSplit = 64 % CH != 0 || 64 / CH > 16;  // a load's rows may be in both operands
                if constexpr (kSplit) {
                    const bool first = (lane + 64 * j) / CH < 16;
                    S.v[j] = buffer_load16(vr[0], first ? vo[j] : kPast) | buffer_load16(vr[1], first ? kPast : vo[j]);
                } else {
                    S.v[j] = buffer_load16(vr[64 * j / CH / 16], vo[j]);
                }
            }
        } else {
            const int pos = p_lane + kStep * j;
            const bool ok = pos < end && (unsigned)e < (unsigned)p.c.n_pages;
            S.seen = (uint32_t)__builtin_amdgcn_ballot_w64(ok);
            const int place = pos & mask;
            if constexpr (I8) {
                const int64_t at = ok ? ((int64_t)e << p.c.shift) + place : 0;
                S.ks = ksp[at * s_stride];
                S.vs = vsp[at * v_stride];
            }
            if (lane < 32) rowoff[w][lane] = ok ? (int64_t)e * p.c.page_bytes + (int64_t)place * row_bytes : 0;
            wave_lds_fence();
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                const uint8_t *src = kb + rowoff[w][16 * st + r];
#pragma unroll
                for (int i = 0; i < KL; ++i) S.k[st][i] = load16(src + ko[i]);
            }
#pragma unroll
            for (int j = 0; j < NV; ++j) S.v[j] = load16(vb + rowoff[w][min((lane + 64 * j) / CH, 31)] + vo[j]);
            wave_lds_fence();
        }
    };
    auto widen = [](uint32_t a, uint32_t b) {  // 8 int8
        const u32x2 x = i8x4_to_f16(a), y = i8x4_to_f16(b);
        return u32x4{x.x, x.y, y.x, y.y};
    };

    f32x4 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;
    bool bad = false;  // some V is not finite
    uint32_t most_vs = 0;  // int8: the lane's largest |V scale|
    auto process = [&](int j, Step &S) {
        const int p0 = beg + kStep * j + 32 * w;
        f32x4 acc[2];
#pragma unroll
        for (int st = 0; st < 2; ++st) {
            acc[st] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                u32x4 k;
                if constexpr (I8) k = ks % 2 ? widen(S.k[st][ks / 2].z, S.k[st][ks / 2].w) : widen(S.k[st][ks / 2].x, S.k[st][ks / 2].y);
                else k = S.k[st][ks];
                if (!I8 && !BIG && 4 * ks + 4 > n_ch && 4 * ks + g >= n_ch) k = u32x4{0u, 0u, 0u, 0u};
                acc[st] = mfma<RXQ4_DTYPE_F16>(k, qf[ks], acc[st]);
            }
        }
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
                acc[st] *= *reinterpret_cast<const f32x4 *>(&scl[w][0][16 * st + 4 * g]);
                vx[st] = *reinterpret_cast<const f32x4 *>(&scl[w][1][16 * st + 4 * g]);
                lg[st] = *reinterpret_cast<const f32x4 *>(&scl[w][2][16 * st + 4 * g]);
            }
            wave_lds_fence();
        }
        const bool part = S.seen != ~0u;
        float sv[8], mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) sv[i] = acc[i >> 2][i & 3] * p.sl2;
        if (part || p0 + 31 > span.pos0) {  // uniform: not every row sees all of them
            const uint32_t in = S.seen >> (4 * g);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (!((in >> (16 * (i >> 2) + (i & 3))) & 1u) || p0 + 16 * (i >> 2) + 4 * g + (i & 3) > qpos)
                    sv[i] = -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) mx = fmaxf(mx, I8 ? sv[i] + lg[i >> 2][i & 3] : sv[i]);
        mx = max_xor_rows<16>(mx);
        mx = max_xor_rows<32>(mx);
        if (__builtin_amdgcn_ballot_w64(mx > m + kLazy) != 0) {
            // (each row's by its own rule: no row depends on what others see)
            const float m_new = mx > m + kLazy ? mx : m;
            const float corr = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - m_new);
            m = m_new;
            l *= corr;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[dt] *= corr;
        }
        const float m_use = m == -INFINITY ? 0.0f : m - kShift;
        uint32_t ph[4], pl[4];
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            float e0 = __builtin_amdgcn_exp2f(sv[i] - m_use), e1 = __builtin_amdgcn_exp2f(sv[i + 1] - m_use);
            l += e0;
            l += e1;
            if constexpr (I8) {
                // (a position that the row does not see stays 0 whatever its scale)
                e0 = sv[i] == -INFINITY ? 0.0f : e0 * vx[i >> 2][i & 3];
                e1 = sv[i + 1] == -INFINITY ? 0.0f : e1 * vx[i >> 2][(i & 3) + 1];
            }
            ph[i >> 1] = pack2<RXQ4_DTYPE_F16>(e0, e1);
            pl[i >> 1] = low_halves(e0, e1, ph[i >> 1]);
        }
        // Rows that are not there: zeros.  An infinity or NaN in V would reach the rows
        // that do not see it as 0 times it, and the others through the low half of P: such
        // values (int8: V scales) are staged as zeros, and the rows that see them get them
        // at the end.
        if constexpr (!I8) {
            if (!BIG && part)  // uniform
#pragma unroll
                for (int j = 0; j < NV; ++j)
                    if (!((S.seen >> ((lane + 64 * j) / CH)) & 1u)) S.v[j] = u32x4{0u, 0u, 0u, 0u};
            if (__builtin_amdgcn_ballot_w64(not_finite16<NV>(S.v)) != 0) {
                zero_not_finite16<NV>(S.v);
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
                    *reinterpret_cast<u32x4 *>(dst) = widen(S.v[j].x, S.v[j].y);
                    *reinterpret_cast<u32x4 *>(dst + 8) = widen(S.v[j].z, S.v[j].w);
                }
            } else {
                *reinterpret_cast<u32x4 *>(dst) = S.v[j];
            }
        }
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
            o[dt] = mfma<RXQ4_DTYPE_F16>(a, u32x4{ph[0], ph[1], ph[2], ph[3]}, o[dt]);
            o[dt] = mfma<RXQ4_DTYPE_F16>(a, u32x4{pl[0], pl[1], pl[2], pl[3]}, o[dt]);
        }
    };
    const int n_steps = (end - beg + kStep - 1) / kStep;
    Step A, B;
    for (int j0 = 0; j0 < n_steps; j0 += 32) {
        const int j1 = BIG ? min(n_steps, j0 + 32) : n_steps;
        if (j0 > 0) ent = entries(j0);
        load_step(j0, ent, A);
        for (int j = j0;;) {
            if (!BIG) ent = entry(p_lane + kStep * (j + 2));
            load_step(j + 1 < j1 ? j + 1 : kNoStep, BIG ? ent : ent_next, B);
            __builtin_amdgcn_sched_barrier(0);  // (the compiler would move them behind the products)
            process(j, A);
            if (++j >= j1) break;
            if (!BIG) ent_next = entry(p_lane + kStep * (j + 2));
            load_step(j + 1 < j1 ? j + 1 : kNoStep, ent, A);
            __builtin_amdgcn_sched_barrier(0);
            process(j, B);
            if (++j >= j1) break;
        }
        if (!BIG) break;
    }
    if constexpr (I8 && !BIG) bad = __builtin_amdgcn_ballot_w64(most_vs >= 0x7F800000u) != 0;
    l = sum_xor_rows<16>(l);
    l = sum_xor_rows<32>(l);

    // Merge: lane l of every wave holds row r, dims 16 dt + 4 g + i; wave w merges
    // the dims of tiles dt = w, w + 4, ...
    float (*const mg)[NM][64] = reinterpret_cast<float (*)[NM][64]>(smem);
    __syncthreads();  // the V rows are read
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) mg[w][4 * dt + i][lane] = o[dt][i];
    mg[w][NM - 2][lane] = m;
    mg[w][NM - 1][lane] = l;
    if (bad) {  // uniform, rare: the wave's positions again (onto its part in LDS: no registers held for it)
        for (int pos = beg; pos < end; ++pos) {
            if (((pos - beg) / 32 & 3) != w || pos > qpos) continue;
            const int slot = slot_of(p.c, s, pos);
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
    if (!row_ok) return;
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
            *reinterpret_cast<u32x2 *>(p.out + orow + d) = u32x2{pack2<RXQ4_DTYPE_F16>(ov[0] * inv, ov[1] * inv),
                                                                 pack2<RXQ4_DTYPE_F16>(ov[2] * inv, ov[3] * inv)};
    }
    if (!whole && w == 0 && g == 0) {
        p.stats[2 * at] = M;
        p.stats[2 * at + 1] = L;
    }
}

// out = sum_c 2^(m_c - M) O_c / sum_c 2^(m_c - M) l_c over a row's chunks in order.  A
// wave takes a row: a lane's chunk for the weights, then a lane's dims.
template <int HD>
__global__ __launch_bounds__(256) void attn_paged_combine_kernel(PagedParams p) {
    constexpr int VE = HD > 128 ? 4 : HD > 64 ? 2 : 1, U = 8;
    typedef float Piece __attribute__((ext_vector_type(VE)));
    const int lane = threadIdx.x & 63, r = 4 * blockIdx.y + (threadIdx.x >> 6);
    const int kvh = blockIdx.x % p.c.n_kv, s = blockIdx.x / p.c.n_kv;
    const SeqSpan span = seq_span(p.b, s);
    const int first = p.firsts[2 * s], n_c = p.firsts[2 * s + 1];
    const int rows = min(span.n, p.b.max_new) * p.group;
    if (r >= rows || rows > kPagedRows || n_c <= 1 || n_c > p.n_chunks) return;  // not this kernel's, or written already
    const int64_t at = ((int64_t)first * p.c.n_kv + kvh) * p.rows_blk + r, step = (int64_t)p.c.n_kv * p.rows_blk;
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
            if (ec != 0.0f) acc += ec * x[i];
            else
#pragma unroll
                for (int k = 0; k < VE; ++k) acc[k] = add_weighed(acc[k], 0.0f, x[i][k]);
        }
    }
    if (lane * VE >= p.c.hd) return;
    const int tok = r / p.group, head = kvh * p.group + r % p.group;
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    uint16_t *out = p.out + ((int64_t)(span.row0 + tok) * p.n_heads + head) * p.c.hd + d;
    if constexpr (VE == 1) {
        *out = f32_to_f16_bits(acc[0] * inv);
    } else {
#pragma unroll
        for (int i = 0; i < VE; i += 2)
            *reinterpret_cast<uint32_t *>(out + i) = pack2<RXQ4_DTYPE_F16>(acc[i] * inv, acc[i + 1] * inv);
    }
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
    if (i8 && big) attn_paged_rows_kernel<HD, true, true><<<grid, 256, 0, st>>>(p);
    else if (i8) attn_paged_rows_kernel<HD, true, false><<<grid, 256, 0, st>>>(p);
    else if (big) attn_paged_rows_kernel<HD, false, true><<<grid, 256, 0, st>>>(p);
    else attn_paged_rows_kernel<HD, false, false><<<grid, 256, 0, st>>>(p);
    if (p.n_chunks > 1) {
        const dim3 rows((unsigned)(p.b.n_seqs * p.c.n_kv), (unsigned)(p.rows_blk + 3) / 4);
        attn_paged_combine_kernel<HD><<<rows, 256, 0, st>>>(p);
    }
    return hipGetLastError();
}

}  // namespace

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
