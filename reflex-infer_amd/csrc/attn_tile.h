// attn_tile.h -- what the attention kernels with 128 query rows a workgroup share:
// their MFMA, the places of K and V chunks in LDS, the row numbering, and the
// constants of their softmax.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mfma_util.h"
#include "q4k_device.h"

namespace rxq4 {
namespace {

typedef short v4i16 __attribute__((ext_vector_type(4)));

constexpr int kTile = 64;  // positions per tile
// The reference point m of a row's exponentials moves when the row's maximum has
// outgrown it by 2^kLazy, and P holds 2^kShift times them, up to 2^(kLazy +
// kShift) = 2^15: fp16's range is used from its top (65504) and the low half of
// P ends at 2^-24 = 2^-35 of the reference point.
constexpr float kLazy = 4.0f;
constexpr float kShift = 11.0f;
// V scales below 2^kMinScale count as that where the reference point is chosen
// (what they weigh is 0 in an fp16 output) and those above 2^kMaxScale as that.
constexpr float kMinScale = -40.0f, kMaxScale = 127.0f;

__device__ __forceinline__ f32x16 mfma32h(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// lo = RNE_f16(e - f32(hi)) for a pair: the difference is exact in fp32.  (Not in
// inline asm: an MFMA may read a VALU result two wait states later at the earliest,
// which the compiler keeps only for instructions that it knows.)
__device__ __forceinline__ uint32_t low_halves(float e0, float e1, uint32_t hi) {
    return pack2<RXQ4_DTYPE_F16>(e0 - f16_bits_to_f32(hi & 0xFFFFu), e1 - f16_bits_to_f32(hi >> 16));
}

// Infinities and NaN among N x 8 fp16: whether there are any (times 0 they are
// NaN), and zeros in their place (a half with all exponent bits set carries into
// its top bit).
template <int N>
__device__ __forceinline__ bool not_finite16(const u32x4 *x) {
    f16x2 sum[4] = {};
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t v = x[j][i];  // (a bit cast of the vector's element itself takes element 0)
            sum[i] = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, v), f16x2{0, 0}, sum[i]);
        }
    const f16x2 all = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    return !(all.x == 0) || !(all.y == 0);
}
template <int N>
__device__ __forceinline__ void zero_not_finite16(u32x4 *x) {
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t all = (((x[j][i] & 0x7C007C00u) + 0x04000400u) >> 15) & 0x00010001u;
            x[j][i] &= ~(all * 0xFFFFu);
        }
}

// Token and head of query row row0 + r (r < 32), from the uniform division of
// row0: the quotient of rem0 + r < group + 32 by the group from a reciprocal
// ((x + 0.5) / group is at least 0.5 / group from an integer, far more than
// the reciprocal's error).
struct RowMap {
    int tok0, rem0, group;
    float rcp;
    __device__ void at(int r, int &tok, int &head) const {
        const int x = rem0 + r;
        const int q = (int)(((float)x + 0.5f) * rcp);
        tok = tok0 + q;
        head = x - q * group;
    }
};
__device__ __forceinline__ RowMap row_map(int row0, int group) {
    const int t = row0 / group;
    return RowMap{t, row0 - t * group, group, __builtin_amdgcn_rcpf((float)group)};
}

// Place of 16-byte chunk c of row p in the LDS row (HD fp16).
template <int HD>
__device__ __forceinline__ int k_pos(int p, int c) {
    if (HD == 64) return c ^ ((p >> 1) & 7);            // two rows cover the banks
    if (HD == 96) return (c & ~3) | ((c ^ (p >> 2)) & 3);  // rows p, p + 4, .. share a bank window
    return c ^ (p & 15);                                // a row (or half of it) covers them
}
template <int HD>
__device__ __forceinline__ int v_pos(int p, int c) {
    if (HD == 64) return c ^ (((p >> 1) & 1) << 2);
    if (HD == 96) return c;
    return c ^ ((p & 3) << 2);
}

// 4 int8 of w (xor 0x80 gives x + 128) as fp16: 0x6400 | byte = 1024 + byte
// exactly, and the subtraction is exact.
__device__ __forceinline__ u32x2 i8x4_to_f16(uint32_t w) {
    const uint32_t u = w ^ 0x80808080u;
    const half2_t off = as_half2(0x64806480u);  // 1152
    const half2_t a = as_half2(__builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - off;
    const half2_t b = as_half2(__builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - off;
    return u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
}

}  // namespace
}  // namespace rxq4
