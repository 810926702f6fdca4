// attn_paged.hip -- attention of a batch's new tokens over a paged KV cache.
//
// Token at position p, head h: out = sum_j e^(s_j) v_j / sum_j e^(s_j) over the
// positions j <= p whose page is in the pool, s_j = scale q.k_j, KV head h /
// group; the sums relative to a running maximum, in fp32.
//
// A wave per token and head: a lane's score per position, 64 positions a step,
// then a lane's dims of the output.
#include <math.h>

#include "launch.h"
#include "paged.h"
#include "q4k_device.h"

namespace rxq4 {
namespace {

struct PagedParams {
    uint16_t *out;
    const uint16_t *q;
    SeqBatch b;
    PagedCache c;
    int n_heads, group;
    float scale;
};

template <bool I8>
__global__ __launch_bounds__(64) void attn_paged_row_kernel(PagedParams p) {
    constexpr int esz = I8 ? 1 : 2;
    __shared__ float qs[256];
    const int lane = threadIdx.x;
    const int t = blockIdx.x / p.n_heads, h = blockIdx.x % p.n_heads;
    const int s = seq_of_row(p.b, t);
    if (s >= p.b.n_seqs) return;
    const SeqSpan q = seq_span(p.b, s);
    if (t < q.row0 || t - q.row0 >= min(q.n, p.b.max_new)) return;
    const int hd = p.c.hd, kvh = h / p.group;
    const int row_bytes = p.c.n_kv * hd * esz;
    const int end = min(q.pos0 + (t - q.row0) + 1, position_limit(p.b, p.c));
    const uint16_t *qrow = p.q + ((int64_t)t * p.n_heads + h) * hd;
    for (int i = lane; i < hd; i += 64) qs[i] = f16_bits_to_f32(qrow[i]);
    __syncthreads();
    float m = -INFINITY, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int p0 = 0; p0 < end; p0 += 64) {
        const int pos = p0 + lane;
        const int slot = pos < end ? slot_of(p.c, s, pos) : -1;
        float sc = -INFINITY;
        if (slot >= 0) {
            const uint8_t *k = p.c.k + slot_bytes(p.c, slot, row_bytes) + (int64_t)kvh * hd * esz;
            float d = 0.0f;
            for (int i = 0; i < hd; ++i)
                d += qs[i] * (I8 ? (float)reinterpret_cast<const int8_t *>(k)[i]
                                 : f16_bits_to_f32(reinterpret_cast<const uint16_t *>(k)[i]));
            if (I8 && p.c.ks) d *= p.c.ks[(int64_t)slot * p.c.n_kv + kvh];
            sc = d * p.scale;
        }
        const uint64_t seen = __builtin_amdgcn_ballot_w64(slot >= 0);
        if (seen == 0) continue;
        const float m_new = fmaxf(m, butterfly_max<64>(sc));
        const float m_use = m_new == -INFINITY ? 0.0f : m_new;
        const float corr = expf(m - m_use);
        const float e = slot >= 0 ? expf(sc - m_use) : 0.0f;
        l = l * corr + butterfly_sum<64>(e);
        m = m_new;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] *= corr;
        const float ve = I8 && p.c.vs && slot >= 0 ? p.c.vs[(int64_t)slot * p.c.n_kv + kvh] : 1.0f;
        for (int j = 0; j < 64; ++j) {
            if (!((seen >> j) & 1)) continue;  // uniform
            const uint8_t *v = p.c.v + slot_bytes(p.c, __shfl(slot, j, 64), row_bytes) + (int64_t)kvh * hd * esz;
            const float w = __shfl(e, j, 64), x = __shfl(ve, j, 64);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = lane + 64 * i;
                if (d < hd)
                    o[i] += w * (I8 ? x * (float)reinterpret_cast<const int8_t *>(v)[d]
                                    : f16_bits_to_f32(reinterpret_cast<const uint16_t *>(v)[d]));
            }
        }
    }
    const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;  // (NaN stays)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int d = lane + 64 * i;
        if (d < hd) p.out[((int64_t)t * p.n_heads + h) * hd + d] = f32_to_f16_bits(o[i] * inv);
    }
}

}  // namespace

hipError_t launch_attention_paged(uint16_t *out, const uint16_t *q, int n_heads, float scale,
                                  const SeqBatch &batch, const PagedCache &cache, int kv_int8,
                                  hipStream_t st) {
    const PagedParams p{out, q, batch, cache, n_heads, n_heads / cache.n_kv, scale};
    const unsigned grid = (unsigned)batch.n_tokens * (unsigned)n_heads;
    if (kv_int8) attn_paged_row_kernel<true><<<grid, 64, 0, st>>>(p);
    else attn_paged_row_kernel<false><<<grid, 64, 0, st>>>(p);
    return hipGetLastError();
}

}  // namespace rxq4
