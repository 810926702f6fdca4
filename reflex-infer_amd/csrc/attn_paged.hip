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
// for all of them, which is what bounds decoding (one to a few new tokens).
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

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

constexpr int kMaxChunks = 64;  // chunks of positions per sequence
__device__ __forceinline__ float log2_scale(float vs) {
    return fminf(fmaxf(__builtin_amdgcn_logf(fabsf(vs)), kMinScale), kMaxScale);
}

// 8 int8 (bytes of .x, .y) as 8 fp16 (exact).
__device__ __forceinline__ u32x4 i8_to_f16(u32x2 v) {
    uint32_t o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t wd = e < 2 ? v.x : v.y;
        const int sh = 16 * (e & 1);
        o[e] = pack2<RXQ4_DTYPE_F16>((float)(int8_t)(uint8_t)(wd >> sh), (float)(int8_t)(uint8_t)(wd >> (sh + 8)));
    }
    return u32x4{o[0], o[1], o[2], o[3]};
}

// Wave w takes positions 16 w .. + 15 of every 64-position tile of the chunk with
// its own online softmax; the four waves merge at the end.  Per tile, lane l =
// 16 g + r:
//   S^T = K . Q^T    v_mfma_f32_16x16x32_f16, src0 = 16 positions x 32 dims of K
//                    straight from memory (16 bytes a lane), src1 = Q^T; the lane
//                    gets positions 4 g + i of row r;
//   O^T += V^T P^T   v_mfma_f32_16x16x16_f16, src0 = 16 dims x 16 positions of V^T
//                    (ds_read_tr16_b64 of the wave's V rows in LDS), src1 = P^T as
//                    the score registers hold it, in fp16 hi + lo parts (22 bits).
// Lane r looks up the page of position r once; the V chunks' lanes get the row's
// offset from it.  int8: P holds the V scales, so the reference point of the
// exponentials follows the maximum of score + log2 |scale|, and neither end of
// fp16 is met whatever the scales.
// The loads of NB tiles go out before their arithmetic, the table entries of the
// next ones with them.
template <int HD, bool I8>
__global__ __launch_bounds__(256, HD <= 128 ? 2 : 1) void attn_paged_rows_kernel(PagedParams p) {
    constexpr int KS = HD / 32, DT = HD / 16, VROW = HD + 16, CH = HD / 8, NV = 16 * CH / 64;
    constexpr int NB = HD <= 128 ? 4 : 2;
    constexpr int esz = I8 ? 1 : 2;
    constexpr int NM = DT * 4 + 2;  // merge values per lane: O, m, l
    __shared__ __attribute__((aligned(16))) uint16_t vl[4][16 * VROW];
    __shared__ float mg[4][NM][64];

    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int kvh = blockIdx.x % p.c.n_kv, u = blockIdx.x / p.c.n_kv;
    const int s = u % p.b.n_seqs, c = u / p.b.n_seqs;
    const int beg = c * p.chunk;
    const int limit = position_limit(p.b, p.c);
    if (beg >= limit && c > 0) return;

    // Table entries of the first tiles, before the sequence's length is known.
    const int32_t *const table = p.c.table ? p.c.table + (int64_t)s * p.c.width : nullptr;
    auto entry = [&](int pos) {
        const int i = pos >> p.c.shift;
        return pos < limit ? (table ? table[i] : i) : -1;
    };
    int ent[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) ent[b] = entry(beg + kTile * b + 16 * w + r);
    const SeqSpan span = seq_span(p.b, s);
    const int rows = min(span.n, p.b.max_new) * p.group;
    if (rows == 0 || rows > kPagedRows) return;
    const int end_seq = min(span.pos0 + (rows - 1) / p.group + 1, limit);
    const int end = min(end_seq, beg + p.chunk);
    const int row = min(r, rows - 1);  // (columns past the last row repeat it)
    const int tok = row / p.group, head = kvh * p.group + row % p.group;
    const bool row_ok = r < rows;
    const int hd = p.c.hd, n_ch = hd >> 3;
    const int64_t orow = ((int64_t)(span.row0 + tok) * p.n_heads + head) * hd;
    if (end <= beg) {  // uniform
        if (c == 0 && w == 0 && row_ok)  // the tokens see nothing
            for (int ch = g; ch < n_ch; ch += 4) *reinterpret_cast<u32x4 *>(p.out + orow + 8 * ch) = u32x4{0u, 0u, 0u, 0u};
        return;
    }
    const int qpos = span.pos0 + tok;
    const int row_bytes = p.c.n_kv * hd * esz;
    const uint8_t *kb = p.c.k + (int64_t)kvh * hd * esz, *vb = p.c.v + (int64_t)kvh * hd * esz;

    u32x4 qf[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
        qf[ks] = 4 * ks + g < n_ch ? load16(p.q + orow + 8 * (4 * ks + g)) : u32x4{0u, 0u, 0u, 0u};

    f32x4 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;
    bool bad = false;  // some V is not finite
    const int n_tiles = (end - beg + kTile - 1) / kTile;

    for (int j0 = 0; j0 < n_tiles; j0 += NB) {
        u32x4 kf[NB][KS], vr[NB][NV];
        float ksc[NB], vsc[NB];
        uint32_t seen[NB];  // which of the wave's 16 positions there are
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int pos = beg + kTile * (j0 + b) + 16 * w + r;
            const bool ok = pos < end && (unsigned)ent[b] < (unsigned)p.c.n_pages;
            const int slot = ok ? (ent[b] << p.c.shift) + (pos & ((1 << p.c.shift) - 1)) : -1;
            seen[b] = (uint32_t)__builtin_amdgcn_ballot_w64(ok) & 0xFFFFu;
            const int64_t off = ok ? slot_bytes(p.c, slot, row_bytes) : -1;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                kf[b][ks] = u32x4{0u, 0u, 0u, 0u};
                if (ok && 4 * ks + g < n_ch) {
                    const uint8_t *src = kb + off + 8 * esz * (4 * ks + g);
                    if constexpr (I8) kf[b][ks] = u32x4{reinterpret_cast<const uint32_t *>(src)[0], reinterpret_cast<const uint32_t *>(src)[1], 0u, 0u};
                    else kf[b][ks] = load16(src);
                }
            }
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int id = lane + 64 * j;
                const uint32_t lo = (uint32_t)__shfl((int)(uint32_t)off, id / CH, 64);
                const int hi = __shfl((int)(off >> 32), id / CH, 64);
                vr[b][j] = u32x4{0u, 0u, 0u, 0u};
                if (hi >= 0 && id % CH < n_ch) {
                    const uint8_t *src = vb + (((int64_t)hi << 32) | lo) + 8 * esz * (id % CH);
                    if constexpr (I8) vr[b][j] = u32x4{reinterpret_cast<const uint32_t *>(src)[0], reinterpret_cast<const uint32_t *>(src)[1], 0u, 0u};
                    else vr[b][j] = load16(src);
                }
            }
            if constexpr (I8) {
                const int64_t at = (int64_t)max(slot, 0) * p.c.n_kv + kvh;
                ksc[b] = p.c.ks ? p.c.ks[at] : 1.0f;
                vsc[b] = p.c.vs ? p.c.vs[at] : 1.0f;
            }
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) ent[b] = entry(beg + kTile * (j0 + NB + b) + 16 * w + r);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            if (j0 + b >= n_tiles) break;  // uniform
            const int p0 = beg + kTile * (j0 + b) + 16 * w;
            if (seen[b] == 0) continue;    // uniform
            f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const u32x4 k = I8 ? i8_to_f16(u32x2{kf[b][ks].x, kf[b][ks].y}) : kf[b][ks];
                acc = mfma<RXQ4_DTYPE_F16>(k, qf[ks], acc);
            }
            float sv[4], vx[4], lg[4];
            bool vis[4];
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                vis[i] = ((seen[b] >> (4 * g + i)) & 1) && p0 + 4 * g + i <= qpos;
                float x = acc[i] * p.sl2;
                vx[i] = 1.0f;
                lg[i] = 0.0f;
                if constexpr (I8) {
                    x *= __shfl(ksc[b], 4 * g + i, 64);
                    vx[i] = __shfl(vsc[b], 4 * g + i, 64);
                    lg[i] = log2_scale(vx[i]);
                }
                sv[i] = vis[i] ? x : -INFINITY;
                mx = fmaxf(mx, sv[i] + lg[i]);
            }
            mx = max_xor_rows<16>(mx);
            mx = max_xor_rows<32>(mx);
            const float m_new = fmaxf(m, mx);
            const bool any = m_new != -INFINITY;
            const float corr = any ? __builtin_amdgcn_exp2f(m - m_new) : 1.0f;
            const float m_use = any ? m_new - kShift : 0.0f;
            float e[4], sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                e[i] = __builtin_amdgcn_exp2f(sv[i] - m_use);
                sum += e[i];
                if (I8) e[i] = vis[i] ? e[i] * vx[i] : 0.0f;
            }
            l = l * corr + sum;  // this lane's positions
            m = m_new;
            const uint32_t h01 = pack2<RXQ4_DTYPE_F16>(e[0], e[1]), h23 = pack2<RXQ4_DTYPE_F16>(e[2], e[3]);
            const f16x4 ph = __builtin_bit_cast(f16x4, u32x2{h01, h23});
            const f16x4 pl = __builtin_bit_cast(f16x4, u32x2{low_halves(e[0], e[1], h01), low_halves(e[2], e[3], h23)});
            // An infinity or NaN in V would reach the rows that do not see it as 0 times
            // it, and the others through the low half of P: such values are staged as
            // zeros, and the rows that see them get them at the end.
            if constexpr (!I8) {
                if (__builtin_amdgcn_ballot_w64(not_finite16<NV>(vr[b])) != 0) {
                    zero_not_finite16<NV>(vr[b]);
                    bad = true;
                }
            }
            // (the wave's own earlier reads of its rows are ahead in its LDS queue)
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int id = lane + 64 * j;
                *reinterpret_cast<u32x4 *>(&vl[w][(id / CH) * VROW + 8 * (id % CH)]) =
                    I8 ? i8_to_f16(u32x2{vr[b][j].x, vr[b][j].y}) : vr[b][j];
            }
            // lane r of group g supplies dims 16 dt + 4 (r & 3) .. + 3 of position
            // 4 g + r / 4 and receives dim 16 dt + r of positions 4 g .. + 3
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const f16x4 a = __builtin_bit_cast(
                    f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4i16 *)
                                                                   &vl[w][(4 * g + (r >> 2)) * VROW + 16 * dt + 4 * (r & 3)]));
                o[dt] *= corr;
                o[dt] = __builtin_amdgcn_mfma_f32_16x16x16f16(a, ph, o[dt], 0, 0, 0);
                o[dt] = __builtin_amdgcn_mfma_f32_16x16x16f16(a, pl, o[dt], 0, 0, 0);
            }
        }
    }
    if (bad) {  // uniform, rare: the wave's positions again
        for (int pos = beg; pos < end; ++pos) {
            if (((pos - beg) >> 4 & 3) != w || pos > qpos) continue;
            const int slot = slot_of(p.c, s, pos);
            if (slot < 0) continue;
            const uint16_t *v = reinterpret_cast<const uint16_t *>(vb + slot_bytes(p.c, slot, row_bytes));
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int d = 16 * dt + 4 * g + i;
                    const float x = d < hd ? f16_bits_to_f32(v[d]) : 0.0f;
                    if (!(fabsf(x) < INFINITY)) o[dt][i] += x;
                }
        }
    }
    l = sum_xor_rows<16>(l);
    l = sum_xor_rows<32>(l);

    // Merge: lane l of every wave holds row r, dims 16 dt + 4 g + i; wave w merges
    // the dims of tiles dt = w, w + 4, ...
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) mg[w][4 * dt + i][lane] = o[dt][i];
    mg[w][NM - 2][lane] = m;
    mg[w][NM - 1][lane] = l;
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
    const bool whole = end_seq <= p.chunk;  // one chunk: no partials
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    const int64_t at = ((int64_t)(s * p.c.n_kv + kvh) * p.n_chunks + c) * p.rows_blk + r;
#pragma unroll
    for (int dt = w; dt < DT; dt += 4) {
        f32x4 ov;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float x = 0.0f;
#pragma unroll
            for (int v = 0; v < 4; ++v) x += mg[v][4 * dt + i][lane] * cw[v];
            ov[i] = x;
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

// out = sum_c 2^(m_c - M) O_c / sum_c 2^(m_c - M) l_c over a row's chunks in a fixed
// order.  Workgroup: a row and 64 of its dims; wave v sums the chunks v, v + 4, ..,
// the waves add up in order.
template <int HD>
__global__ __launch_bounds__(256) void attn_paged_combine_kernel(PagedParams p) {
    constexpr int NS = (HD + 63) / 64;
    __shared__ float part[4][64];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int d = blockIdx.x % NS * 64 + lane;
    const int r = blockIdx.x / NS % p.rows_blk, u = blockIdx.x / NS / p.rows_blk;
    const int kvh = u % p.c.n_kv, s = u / p.c.n_kv;
    const int64_t at = (int64_t)u * p.n_chunks * p.rows_blk + r;
    const float *st = p.stats + 2 * at, *src = p.part + at * HD + min(d, HD - 1);
    const int64_t step = p.rows_blk;
    // (the first loads before the sequence's length: what is past it is not used)
    const int cl = min(lane, p.n_chunks - 1);
    float mc = st[2 * cl * step], lc = st[2 * cl * step + 1];
    constexpr int U = 4;
    float x[U];
#pragma unroll
    for (int i = 0; i < U; ++i) x[i] = src[(int64_t)min(w + 4 * i, p.n_chunks - 1) * step * HD];
    const SeqSpan span = seq_span(p.b, s);
    const int rows = min(span.n, p.b.max_new) * p.group;
    if (r >= rows || rows > kPagedRows) return;  // uniform
    const int end = min(span.pos0 + (rows - 1) / p.group + 1, position_limit(p.b, p.c));
    const int n_c = (max(end, 0) + p.chunk - 1) / p.chunk;
    if (n_c <= 1) return;  // written already
    if (lane >= n_c) {
        mc = -INFINITY;
        lc = 0.0f;
    }
    const float M = butterfly_max<64>(mc);
    const float e = M != -INFINITY && lane < n_c ? __builtin_amdgcn_exp2f(mc - M) : 0.0f;
    const float L = butterfly_sum<64>(e * lc);
    float acc = 0.0f;
    for (int c0 = 0; c0 < n_c; c0 += 4 * U) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int c = c0 + w + 4 * i;
            const float ec = __shfl(e, min(c, 63), 64);
            if (c < n_c && ec != 0.0f) acc += ec * x[i];
        }
        if (c0 + 4 * U < n_c)
#pragma unroll
            for (int i = 0; i < U; ++i) x[i] = src[(int64_t)min(c0 + 4 * U + w + 4 * i, n_c - 1) * step * HD];
    }
    part[w][lane] = acc;
    __syncthreads();
    if (w == 0 && d < p.c.hd) {
        const float sum = part[0][lane] + part[1][lane] + part[2][lane] + part[3][lane];
        const int tok = r / p.group, head = kvh * p.group + r % p.group;
        p.out[((int64_t)(span.row0 + tok) * p.n_heads + head) * p.c.hd + d] =
            f32_to_f16_bits(L == 0.0f ? 0.0f : sum * (1.0f / L));
    }
}

// The 16-row launch's split: its partials within `room` bytes.
struct RowsPlan {
    int64_t units;
    size_t bytes;
};
RowsPlan plan_rows(PagedParams &p, size_t room) {
    const int cus = device_info().cu_count > 0 ? device_info().cu_count : 256;
    const int pad = p.c.hd <= 64 ? 64 : p.c.hd <= 96 ? 96 : p.c.hd <= 128 ? 128 : 256;
    p.rows_blk = (int)std::min<int64_t>((int64_t)std::min(p.b.max_new, p.b.n_tokens) * p.group, kPagedRows);
    const int64_t units = (int64_t)p.b.n_seqs * p.c.n_kv;
    const int64_t len = std::max<int64_t>(1, std::min<int64_t>(p.b.max_len, (int64_t)p.c.width << p.c.shift));
    int64_t want = std::max((4 * cus + units - 1) / units, (len + 1023) / 1024);
    want = std::min<int64_t>({want, kMaxChunks, (len + 2 * kTile - 1) / (2 * kTile)});
    const size_t per = (size_t)units * p.rows_blk * (pad + 2) * 4;
    want = std::max<int64_t>(1, std::min<int64_t>(want, (int64_t)(room / per)));
    if (tuning().attn_split) want = std::min<int64_t>(want, tuning().attn_split);
    p.chunk = (int)(((len + want - 1) / want + kTile - 1) / kTile * kTile);
    p.n_chunks = (int)((len + p.chunk - 1) / p.chunk);
    return RowsPlan{units, p.n_chunks > 1 ? (per * p.n_chunks + 255) / 256 * 256 : 0};
}

template <int HD>
hipError_t launch_rows(PagedParams &p, const RowsPlan &plan, float *ws, int i8, hipStream_t st) {
    if (plan.units * p.n_chunks > 0x7FFFFF) return hipErrorInvalidValue;
    p.part = ws;
    p.stats = ws + (size_t)plan.units * p.n_chunks * p.rows_blk * HD;
    const unsigned grid = (unsigned)(plan.units * p.n_chunks);
    if (i8) attn_paged_rows_kernel<HD, true><<<grid, 256, 0, st>>>(p);
    else attn_paged_rows_kernel<HD, false><<<grid, 256, 0, st>>>(p);
    if (p.n_chunks > 1)
        attn_paged_combine_kernel<HD><<<(unsigned)(plan.units * p.rows_blk * ((HD + 63) / 64)), 256, 0, st>>>(p);
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
    if (rows) rp = plan_rows(pr, (blocks ? kWorkspaceBytes / 2 : kWorkspaceBytes) - 256);
    if (blocks) bp = plan_paged_blocks(p, kWorkspaceBytes - rp.bytes);
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
