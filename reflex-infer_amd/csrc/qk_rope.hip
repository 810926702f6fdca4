// qk_rope.hip -- between a layer's Q/K/V projection and its attention: RMS norm of
// each query and key head, rotation by position, and the store of the new keys
// and values into a paged cache (fp16, or int8 with a scale per position and
// head), in one pass over the projection's output.
//
//   norm      x w / sqrt(mean x^2 + eps)
//   rotation  (a, b) -> (a cos - b sin, b cos + a sin) of the pairs (i, i + n_rot / 2)
//             or (2 i, 2 i + 1), the angle position * inv_freq[i]: its product and
//             its remainder to whole turns in 64 bits (a product of 32 bits is off by up to
//             2^-8 radians at positions 65536 to 131071), sine and cosine in 32 of the
//             remainder's nearest fp32 number of half turns, turned on by what that
//             rounds off (up to 2^-25 half turns, 9e-8 of the sine: next to a half
//             turn more than all of its other errors)
//   int8      scale = max |x| / 127, rint(x / scale), both divisions IEEE, so that
//             the bytes follow from the 32-bit row alone
// A workgroup takes one token and its heads, or a part of them: its threads form
// the token's sines and cosines once, in LDS, while the first heads' rows are on
// their way; then each head belongs to L lanes of a wave, 8 dims a lane (16-byte
// loads and stores, the next head's loads ahead of this one's arithmetic), the
// sums over the L lanes by lane swaps and the pair's other half through the wave's
// own LDS.
// Bound: for many tokens the rows' bytes, in and out; for a few the chain of lengths,
// table entry, sine and store.  So a few tokens' heads are spread over workgroups, a pass
// each; many tokens keep all heads in one, which shares the sines.
// With coordinates on several axes (a pair's angle from its axis's) the token's n_axes
// values and the pairs' axes are loads beside the first rows': 3595 tokens from bf16 on three
// axes 24.7 us, one token of 16 / 2 heads 4.5.
// Measured, 32 / 8 heads of 128: 3595 tokens from bf16 24.4 us (3.6 TB/s; a copy of the
// bytes 17; 31 with each row's loads after the sines), 64 tokens into int8 4.9, one token
// of 16 / 2 heads 4.1.
#include <math.h>

#include "launch.h"
#include "mfma_util.h"
#include "paged.h"
#include "q4k_device.h"

namespace rxq4 {
namespace {

constexpr int kWaves = 4;

struct RopeParams {
    uint16_t *q_out;
    const void *q, *k, *v;
    int64_t q_stride, kv_stride;
    const float *qw, *kw, *inv_freq;
    float eps;
    int n_heads, n_rot, interleaved;
    int heads_wg;  // heads (queries, keys, values in order) of a workgroup
    SeqBatch b;
    PagedCache c;
    RopeAxes a;
};

// Eight values of a row as they are stored, and widened.
template <int DT>
struct Raw {
    u32x4 a[DT == RXQ4_DTYPE_F32 ? 2 : 1];
};

template <int DT>
__device__ __forceinline__ Raw<DT> load8(const void *base, int64_t at) {
    Raw<DT> r;
    const uint8_t *s = static_cast<const uint8_t *>(base) + at * (DT == RXQ4_DTYPE_F32 ? 4 : 2);
    r.a[0] = load16(s);
    if constexpr (DT == RXQ4_DTYPE_F32) r.a[1] = load16(s + 16);
    return r;
}

template <int DT>
__device__ __forceinline__ void widen8(const Raw<DT> &r, float *x) {
    if constexpr (DT == RXQ4_DTYPE_F32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __builtin_bit_cast(f32x4, r.a[i >> 2])[i & 3];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t u = i & 1 ? r.a[0][i >> 1] >> 16 : r.a[0][i >> 1] & 0xFFFFu;
            x[i] = DT == RXQ4_DTYPE_F16 ? f16_bits_to_f32(u) : bf16_bits_to_f32(u);
        }
    }
}

__device__ __forceinline__ void lds8(const float *s, float *x) {
    const f32x4 a = reinterpret_cast<const f32x4 *>(s)[0], b = reinterpret_cast<const f32x4 *>(s)[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[i] = a[i];
        x[4 + i] = b[i];
    }
}

// A head of the token: queries, keys and values in order.
struct Head {
    bool q, v;
    int hk;  // its number among its kind
};
__device__ __forceinline__ Head head_of(const RopeParams &p, int h) {
    const bool q = h < p.n_heads, v = h >= p.n_heads + p.c.n_kv;
    return Head{q, v, q ? h : v ? h - p.n_heads - p.c.n_kv : h - p.n_heads};
}

// DT: type of q, k, v; L: lanes a head (8 L >= head_dim); AX: the angles from p.a's
// coordinates, their loads beside the first rows' (the slot follows from the lengths).
template <int DT, int L, bool I8, bool AX>
__global__ __launch_bounds__(64 * kWaves, DT == RXQ4_DTYPE_F32 ? 7 : 8) void qk_rope_kernel(RopeParams p) {
    constexpr int HPW = 64 / L;  // heads of a wave at a time
    __shared__ float cs[128], sn[128];
    __shared__ __attribute__((aligned(16))) float wts[2][256], xl[kWaves][64 * 8];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int t = blockIdx.x;
    const int hd = p.c.hd, half = p.n_rot >> 1;
    const int sub = lane % L;
    const bool dims = 8 * sub < hd;
    const int d0 = dims ? 8 * sub : 0;
    const int h_end = min(p.n_heads + 2 * p.c.n_kv, ((int)blockIdx.y + 1) * p.heads_wg);
    // (lanes past the last head repeat it)
    const auto load = [&](int h0) {
        const Head h = head_of(p, min(h0 + lane / L, h_end - 1));
        return load8<DT>(h.q ? p.q : h.v ? p.v : p.k, (int64_t)t * (h.q ? p.q_stride : p.kv_stride) + (int64_t)h.hk * hd + d0);
    };
    int h0 = blockIdx.y * p.heads_wg + w * HPW;
    Raw<DT> next = load(h0);
    const float freq = tid < half ? p.inv_freq[tid] : 0.0f;
    int coord = 0;
    if constexpr (AX) {
        const int axis = tid < half && p.a.axis_of ? p.a.axis_of[tid] : 0;
        if (tid < half && (unsigned)axis < (unsigned)p.a.n) coord = p.a.at[axis * p.a.stride + t];
    }
    if (tid < hd) {
        if (p.qw) wts[0][tid] = p.qw[tid];
        if (p.kw) wts[1][tid] = p.kw[tid];
    }
    SeqSpan span;
    const int seq = seq_of_row(p.b, t, span);
    if (seq >= p.b.n_seqs) return;  // uniform
    if (t < span.row0 || t - span.row0 >= min(span.n, p.b.max_new)) return;
    const int pos = span.pos0 + (t - span.row0);
    const int slot = pos >= 0 && pos < position_limit(p.b, p.c) ? slot_of(p.c, seq, pos) : -1;
    if (tid < half) {
        const double turns = (double)(AX ? coord : pos) * (double)freq * 0.15915494309189533577;
        const double halves = 2.0 * (turns - rint(turns));
        const float near = (float)halves, rest = (float)((halves - (double)near) * 3.14159265358979323846);
        float s, c;
        sincospif(near, &s, &c);
        cs[tid] = __builtin_fmaf(-s, rest, c);
        sn[tid] = __builtin_fmaf(c, rest, s);
    }
    __syncthreads();
    // This lane's part of the rotation, the same for every head: x c + y s with the
    // pair's other half y; the sine's sign is in s.
    float c[8], s[8];
    uint32_t turn = 0;  // bit i: dim 8 sub + i is rotated
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int d = 8 * sub + i;
        const bool first = p.interleaved ? !(i & 1) : d < half;
        const int j = p.interleaved ? d >> 1 : first ? d : d - half;
        const bool on = d < p.n_rot;
        turn |= (uint32_t)on << i;
        c[i] = on ? cs[j] : 1.0f;
        s[i] = on ? first ? -sn[j] : sn[j] : 0.0f;
    }
    const bool whole = half % 8 == 0;  // a lane's eight dims are all of one half
    float *const mine = xl[w] + lane * 8;
    const float *const head = xl[w] + (lane - sub) * 8;
    const float *const other = head + (8 * sub < half ? 8 * sub + half : 8 * sub < p.n_rot ? 8 * sub - half : 0);
    for (; h0 < h_end; h0 += kWaves * HPW) {
        const bool live = h0 + lane / L < h_end && dims;
        const Head h = head_of(p, min(h0 + lane / L, h_end - 1));
        float x[8];
        widen8<DT>(next, x);
        next = load(h0 + kWaves * HPW);
        if (p.qw || p.kw) {  // uniform; lanes whose head has no weight leave theirs
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss += dims ? x[i] * x[i] : 0.0f;
            ss = group_sum<L>(ss);
            if (!h.v && (h.q ? p.qw : p.kw)) {
                const float r = 1.0f / sqrtf(ss / (float)hd + p.eps);
                float wt[8];
                lds8(wts[h.q ? 0 : 1] + d0, wt);
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = x[i] * r * wt[i];
            }
        }
        if (half > 0) {  // uniform
            float y[8];
            if (p.interleaved) {
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = x[i ^ 1];
            } else {
                wave_lds_fence();  // the reads of the heads before are done
                reinterpret_cast<f32x4 *>(mine)[0] = f32x4{x[0], x[1], x[2], x[3]};
                reinterpret_cast<f32x4 *>(mine)[1] = f32x4{x[4], x[5], x[6], x[7]};
                wave_lds_fence();
                if (whole) {
                    lds8(other, y);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int d = 8 * sub + i;
                        y[i] = head[d < half ? d + half : d < p.n_rot ? d - half : 0];
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (!h.v && (turn >> i & 1)) x[i] = x[i] * c[i] + y[i] * s[i];
        }
        if (h.q) {
            const bool none = pos < 0;
            u32x4 r;
#pragma unroll
            for (int i = 0; i < 4; ++i) r[i] = none ? 0u : pack2<RXQ4_DTYPE_F16>(x[2 * i], x[2 * i + 1]);
            if (live) *reinterpret_cast<u32x4 *>(p.q_out + ((int64_t)t * p.n_heads + h.hk) * hd + d0) = r;
        } else if constexpr (!I8) {
            u32x4 r;
#pragma unroll
            for (int i = 0; i < 4; ++i) r[i] = pack2<RXQ4_DTYPE_F16>(x[2 * i], x[2 * i + 1]);
            uint8_t *dst = (h.v ? p.c.v : p.c.k) + slot_bytes(p.c, max(slot, 0), p.c.n_kv * hd * 2) + (h.hk * hd + d0) * 2;
            if (live && slot >= 0) *reinterpret_cast<u32x4 *>(dst) = r;
        }
        if constexpr (I8) {
            // the largest |x| as bits: an infinity or NaN is larger than any number
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (dims) top = max(top, __builtin_bit_cast(uint32_t, x[i]) & 0x7FFFFFFFu);
#pragma unroll
            for (int off = L / 2; off > 0; off >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off, 64));
            const float scale = __builtin_bit_cast(float, top) / 127.0f;
            uint32_t b[2] = {0u, 0u};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float z = scale > 0.0f && scale < INFINITY ? rintf(x[i] / scale) : 0.0f;
                const int n = (int)fminf(fmaxf(z, -127.0f), 127.0f);
                b[i >> 2] |= ((uint32_t)n & 0xFFu) << (8 * (i & 3));
            }
            if (!h.q && live && slot >= 0) {
                uint8_t *dst = (h.v ? p.c.v : p.c.k) + slot_bytes(p.c, slot, p.c.n_kv * hd) + h.hk * hd + d0;
                *reinterpret_cast<u32x2 *>(dst) = u32x2{b[0], b[1]};
                if (sub == 0) (h.v ? p.c.vs : p.c.ks)[(int64_t)slot * p.c.n_kv + h.hk] = scale;
            }
        }
    }
}

template <int DT, int L>
void launch_l(const RopeParams &p, dim3 grid, int i8, hipStream_t st) {
    if (p.a.at) {
        if (i8) qk_rope_kernel<DT, L, true, true><<<grid, 64 * kWaves, 0, st>>>(p);
        else qk_rope_kernel<DT, L, false, true><<<grid, 64 * kWaves, 0, st>>>(p);
    } else {
        if (i8) qk_rope_kernel<DT, L, true, false><<<grid, 64 * kWaves, 0, st>>>(p);
        else qk_rope_kernel<DT, L, false, false><<<grid, 64 * kWaves, 0, st>>>(p);
    }
}

template <int DT>
void launch_dt(RopeParams &p, int i8, hipStream_t st) {
    const int L = p.c.hd <= 64 ? 8 : p.c.hd <= 128 ? 16 : 32;
    const int n_all = p.n_heads + 2 * p.c.n_kv, at_once = kWaves * (64 / L);
    const int cus = device_info().cu_count > 0 ? device_info().cu_count : 256;
    p.heads_wg = p.b.n_tokens < cus ? at_once : n_all;
    const dim3 grid(p.b.n_tokens, (n_all + p.heads_wg - 1) / p.heads_wg);
    if (L == 8) launch_l<DT, 8>(p, grid, i8, st);
    else if (L == 16) launch_l<DT, 16>(p, grid, i8, st);
    else launch_l<DT, 32>(p, grid, i8, st);
}

}  // namespace

hipError_t launch_qk_norm_rope(uint16_t *q_out, const void *q, const void *k, const void *v, int x_dtype,
                               int64_t q_stride, int64_t kv_stride, int n_heads, const float *q_weight,
                               const float *k_weight, float eps, const float *inv_freq, int n_rot,
                               int interleaved, const RopeAxes &axes, const SeqBatch &batch,
                               const PagedCache &cache, int kv_int8, hipStream_t st) {
    RopeParams p{q_out, q, k, v, q_stride, kv_stride, q_weight, k_weight, inv_freq, eps,
                 n_heads, n_rot, interleaved, 0, batch, cache, axes};
    if (x_dtype == RXQ4_DTYPE_F32) launch_dt<RXQ4_DTYPE_F32>(p, kv_int8, st);
    else if (x_dtype == RXQ4_DTYPE_F16) launch_dt<RXQ4_DTYPE_F16>(p, kv_int8, st);
    else launch_dt<RXQ4_DTYPE_BF16>(p, kv_int8, st);
    return hipGetLastError();
}

}  // namespace rxq4
