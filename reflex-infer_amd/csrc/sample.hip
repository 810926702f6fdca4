// sample.hip -- the next token of each row of logits: temperature, top-k, top-p,
// min-p and a given random number.
//
// The order is logits descending, equal ones by index.  Every step is a place in
// it: top-k a rank, top-p and the draw a sum of weights, min-p a weight.  So the row
// need not be sorted: counts and sums of weights over bins of the logits say in
// which bin a place lies, and only that bin's logits (or, where the kept ones are
// few, all down to there at once) are sorted.
// Weights exp((l - max) / T) are formed in 64 bits and summed as whole numbers, so
// the sums depend on no order: off by half a unit (2^-49 of a slice's largest weight) a
// logit, and by 2^-(63 - log2 n_vocab) of the row's largest for each block of a slice.
// Within a block the unit is as small as the row's sum leaves room for (2^-61 of it):
// with 2^-(62 - log2 n_vocab) of the largest weight a draw among a million equal weights
// of 2^-23 went a token wide.
//
//   sample_slices_kernel  a workgroup per slice of a row (in registers): its largest
//       logit, the count and weight of 512 bins of 1/16 in (l / T) on a grid that all
//       slices share (the last bin: all further down) and of blocks of 16 bins, and
//       its indices in the order of the bins (a counting sort in LDS);
//   sample_pick_kernel    a workgroup per row: the slices' blocks together, the bins
//       of a block where they are asked for, then the places, in a window of up to
//       512 sorted logits.  A bin with more is narrowed by the logits' ordered bit
//       patterns, 256 parts at a time, down to a window or to equal logits.
// Bound: two launches, the 64-bit arithmetic of a slice (some 40 instructions a
// logit), and the pick's chain of dependent steps in one workgroup.
// Measured, 151936 logits a row: one row 17 us (slices 5, pick 11), 128 rows of mixed
// settings 78 to 83 (slices 45, pick 35: a row whose nucleus ends among thousands of
// equally likely logits takes 35, the others 8 to 12).
#include <math.h>

#include <algorithm>

#include "launch.h"
#include "paged.h"
#include "q4k_device.h"

namespace rxq4 {
namespace {

typedef unsigned long long u64;

constexpr int kThreads = 512;                 // of the pick
constexpr int kBins = 512, kBlock = 16, kBlocks = kBins / kBlock;
constexpr double kBinsPerUnit = 16.0;
constexpr int kSlices = kThreads;             // of a row, at most
constexpr int kWindow = kThreads;               // logits sorted at once
constexpr int kParts = 256;                   // of a bin that holds more
constexpr double kSliceUnit = 0x1p48;         // weight units of a slice

// Larger patterns are larger logits; NaN is least, -0 is 0.
__device__ __forceinline__ uint32_t order_key(float l) {
    const uint32_t u = __builtin_bit_cast(uint32_t, l == 0.0f ? 0.0f : l);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return 0u;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// A slice's part of the workspace.
struct Slice {
    u64 mass[kBins];           // weights relative to the slice's largest logit
    u64 block_mass[kBlocks];
    int top_bin;               // the last place of its first block on the grid
    uint32_t top;              // the largest logit's pattern (0: no token)
    uint32_t first, unused;    // its lowest index in the slice (temperature 0)
    uint16_t end[kBins];       // indices before the end of each bin
    uint16_t block_end[kBlocks];
};

struct SampleParams {
    SampleRows a;
    Slice *slices;      // [row][slice]
    uint16_t *index;    // [row][slice][per]: indices in the slice, by bin
    int row0, n_slices, per;
    double unit;        // weight units of a row's blocks
};

// e^-d for d >= 0 (0 from 100 on): 2^-n of the nearest whole n = d / ln 2, and the
// Taylor series of the rest to the 12th power (|r| <= ln 2 / 2: off by 2^-52).
__device__ __forceinline__ double exp_neg(double d) {
    d = fmin(d, 100.0);
    const double n = rint(d * 1.4426950408889634);
    double r = __builtin_fma(n, 0.69314718055994529, -d);   // ln 2 in two parts
    r = __builtin_fma(n, 2.3190468138462996e-17, r);
    double e = 1.0 / 479001600.0;
    e = __builtin_fma(e, r, 1.0 / 39916800.0);
    e = __builtin_fma(e, r, 1.0 / 3628800.0);
    e = __builtin_fma(e, r, 1.0 / 362880.0);
    e = __builtin_fma(e, r, 1.0 / 40320.0);
    e = __builtin_fma(e, r, 1.0 / 5040.0);
    e = __builtin_fma(e, r, 1.0 / 720.0);
    e = __builtin_fma(e, r, 1.0 / 120.0);
    e = __builtin_fma(e, r, 1.0 / 24.0);
    e = __builtin_fma(e, r, 1.0 / 6.0);
    e = __builtin_fma(e, r, 0.5);
    e = __builtin_fma(e, r, 1.0);
    e = __builtin_fma(e, r, 1.0);
    return ldexp(e, -(int)n);
}
// The weight of a logit beside the largest (a finite one beside an infinity: 0; NaN
// from 0 times infinity goes the same way).
__device__ __forceinline__ double weight_of(float l, float top, double inv_t) {
    return l == top ? 1.0 : exp_neg(((double)top - (double)l) * inv_t);
}
// ... rounded to whole units, at most 2^51 of them: the low bits of 2^52 + w.
__device__ __forceinline__ u64 whole(double w) {
    return __builtin_bit_cast(u64, w + 0x1p52) & 0xFFFFFFFFFFFFFull;
}

__device__ __forceinline__ u64 shfl_xor64(u64 v, int d) {
    const uint32_t lo = __shfl_xor((int)(uint32_t)v, d, 64), hi = __shfl_xor((int)(v >> 32), d, 64);
    return (u64)hi << 32 | lo;
}

// Sums over a wave's lanes up to each one, and the largest of its values, on the VALU.
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 dpp_add_from64(u64 x) {
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, CTRL, ROWS, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(x >> 32), CTRL, ROWS, 0xF, false);
    return x + ((u64)hi << 32 | lo);
}
__device__ __forceinline__ u64 wave_prefix64(u64 x) {
    x = dpp_add_from64<0x111, 0xF>(x);  // as in wave_prefix
    x = dpp_add_from64<0x112, 0xF>(x);
    x = dpp_add_from64<0x114, 0xF>(x);
    x = dpp_add_from64<0x118, 0xF>(x);
    x = dpp_add_from64<0x142, 0xA>(x);
    return dpp_add_from64<0x143, 0xC>(x);
}
__device__ __forceinline__ u64 lane_63(u64 x) {
    return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, 63) |
           (u64)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), 63) << 32;
}
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t x) {
    return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
    float a, b;
    swap_rows<32>(__builtin_bit_cast(float, x), a, b);
    x = max(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b));
    swap_rows<16>(__builtin_bit_cast(float, x), a, b);
    x = max(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b));
    x = dpp_max<0x128>(x);  // row_ror:8, 4, 2, 1
    x = dpp_max<0x124>(x);
    x = dpp_max<0x122>(x);
    return dpp_max<0x121>(x);
}

// Sums over the T threads up to each one (inclusive); `wave`: T / 64 values of LDS.
// Every thread of the workgroup takes part.
template <int T>
__device__ __forceinline__ u64 scan64(u64 v, u64 *wave) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    v = wave_prefix64(v);
    __syncthreads();
    if (lane == 63) wave[w] = v;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < T / 64 - 1; ++i) v += i < w ? wave[i] : 0;
    return v;
}
template <int T>
__device__ __forceinline__ uint32_t scan32(uint32_t v, u64 *wave) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    v = (uint32_t)wave_prefix((int)v);
    __syncthreads();
    if (lane == 63) wave[w] = v;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < T / 64 - 1; ++i) v += i < w ? (uint32_t)wave[i] : 0u;
    return v;
}

// The place of a logit on the bins' grid: in fp32 and saturated, the same in every
// slice, and no smaller for a larger logit, which is all the bins need.
__device__ __forceinline__ int grid_place(float l, float grid) {
    return (int)floorf(__builtin_amdgcn_fmed3f(l * grid, -0x1.fffffep30f, 0x1.fffffep30f));
}

// T threads, PER logits each.
// A logit's weight e^-d, d = (top - l) / T: two tables for the nearest n / 16 and the
// series of the rest (|r| <= 1 / 32: its 7th power is below 2^-47 of the weight); from
// d = 40 on less than half a unit.
template <int T, int PER>
__global__ __launch_bounds__(T) void sample_slices_kernel(SampleParams p) {
    constexpr int kEach = kBins > T ? kBins / T : 1;  // bins of a thread, of the first kBins / kEach
    __shared__ uint32_t count[kBins];
    __shared__ u64 mass[kBins], wave[T / 64];
    __shared__ double ones[41], parts[16];  // e^-i in units, e^-(i / 16)
    __shared__ uint16_t sorted[T * PER];
    __shared__ uint32_t top_first;
    __shared__ float tops[T / 64];
    const int tid = threadIdx.x;
    const int s = blockIdx.x % p.n_slices, r = blockIdx.x / p.n_slices, row = p.row0 + r;
    const int n = min(p.per, p.a.n_vocab - s * p.per);
    const float *l = p.a.logits + (int64_t)row * p.a.stride + (int64_t)s * p.per;
    float x[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) x[i] = l[min(i * T + tid, n - 1)];
    const float t = p.a.temperature ? p.a.temperature[row] : 1.0f;
    if (tid == 0) top_first = ~0u;
#pragma unroll
    for (int i = tid; i < kBins; i += T) {
        count[i] = 0;
        mass[i] = 0;
    }
    if (tid < 41 + 16) {
        const double e = exp_neg(tid < 41 ? (double)tid : (tid - 41) * 0.0625);
        if (tid < 41) ones[tid] = e * kSliceUnit;
        else parts[tid - 41] = e;
    }
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if (i * T + tid >= n) x[i] = -INFINITY;
        top = fmaxf(top, x[i]);  // (NaN is not taken)
    }
    top = butterfly_max<64>(top);
    if ((tid & 63) == 0) tops[tid >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < T / 64; ++i) top = fmaxf(top, tops[i]);
    Slice &out = p.slices[(int64_t)r * p.n_slices + s];
    const bool none = top == -INFINITY;
    if (none || !(t > 0.0f)) {  // uniform: no token, or the largest logit alone is asked for
        if (!none) {
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (x[i] == top) atomicMin(&top_first, (uint32_t)(i * T + tid));
        }
#pragma unroll
        for (int i = tid; i < kBins; i += T) {
            out.mass[i] = 0;
            out.end[i] = 0;
        }
        if (tid < kBlocks) {
            out.block_mass[tid] = 0;
            out.block_end[tid] = 0;
        }
        __syncthreads();
        if (tid == 0) {
            out.top = none ? 0u : order_key(top);
            out.first = top_first;
            out.top_bin = 0;
        }
        return;
    }
    if (tid == 0) {
        out.top = order_key(top);
        out.first = ~0u;
    }
    if (top == INFINITY) {  // uniform, rare: beside infinities the others weigh nothing
        top = 0x1.fffffep127f;
#pragma unroll
        for (int i = 0; i < PER; ++i) x[i] = x[i] == INFINITY ? top : -INFINITY;
    }
    const double inv_t = 1.0 / (double)t;
    const float grid = fminf((float)(kBinsPerUnit * inv_t), 0x1.fffffep127f);
    // blocks are those of the grid, so that the slices' blocks match
    const int top_bin = grid_place(top, grid) | (kBlock - 1);
    uint32_t place[PER];  // bin, and number in it
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        place[i] = ~0u;
        if (x[i] > -INFINITY) {
            const uint32_t b = min((uint32_t)top_bin - (uint32_t)grid_place(x[i], grid), (uint32_t)(kBins - 1));
            const double d = ((double)top - (double)x[i]) * inv_t;
            const double at = rint(fmin(d * 16.0, 640.0));
            const int n16 = (int)at;
            const double q = at * 0.0625 - d;
            double e = 1.0 / 720.0;
            e = __builtin_fma(e, q, 1.0 / 120.0);
            e = __builtin_fma(e, q, 1.0 / 24.0);
            e = __builtin_fma(e, q, 1.0 / 6.0);
            e = __builtin_fma(e, q, 0.5);
            e = __builtin_fma(e, q, 1.0);
            e = __builtin_fma(e, q, 1.0);
            const u64 w = n16 < 640 ? whole(ones[n16 >> 4] * parts[n16 & 15] * e) : 0;
            place[i] = b << 16 | atomicAdd(&count[b], 1u);
            if (w) atomicAdd(&mass[b], w);
        }
    }
    __syncthreads();
    uint32_t mine = 0;
    const bool has = tid * kEach < kBins;
    if (has)
#pragma unroll
        for (int i = 0; i < kEach; ++i) mine += count[tid * kEach + i];
    uint32_t at = scan32<T>(mine, wave) - mine;
    if (has) {
        u64 m = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int b = tid * kEach + i;
            const uint32_t c = count[b];
            count[b] = at;
            at += c;
            out.end[b] = (uint16_t)at;
            out.mass[b] = mass[b];
            m += mass[b];
        }
        constexpr int kHold = kBlock / kEach;  // threads of a block
#pragma unroll
        for (int d = 1; d < kHold; d <<= 1) m += shfl_xor64(m, d);
        if (tid % kHold == kHold - 1) {
            out.block_mass[tid / kHold] = m;
            out.block_end[tid / kHold] = (uint16_t)at;
        }
    }
    if (tid == 0) out.top_bin = top_bin;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i)
        if (place[i] != ~0u) sorted[count[place[i] >> 16] + (place[i] & 0xFFFFu)] = (uint16_t)(i * T + tid);
    __syncthreads();
    uint32_t *dst = reinterpret_cast<uint32_t *>(p.index + ((int64_t)r * p.n_slices + s) * p.per);
    for (int i = tid; i < (n + 1) / 2; i += T) dst[i] = reinterpret_cast<const uint32_t *>(sorted)[i];
}

// A place in the order.
struct Found {
    uint32_t rank;    // logits before it
    u64 before, w;    // their weight, its own
    uint32_t key;
    uint32_t nth;     // of the logits equal to it, where `index` is not known
    int index;        // -1: not known
};

struct Pick {
    // up to the end of each block of the row's bins, and of each bin of one block
    u64 block_mass[kBlocks], bin_mass[kBlock];
    uint32_t block_count[kBlocks], bin_count[kBlock];
    int shift[kSlices];     // bins of a slice below the row's top, kBins: it is all past the bins
    double scale[kSlices];  // a slice's weight unit in the row's
    // the logits of some bins: where they begin in a slice's indices, and how many there
    // are up to the end of each slice
    int from[kSlices];
    uint32_t upto[kSlices];
    // the window: sorted (~pattern, index), weights up to the end of each
    u64 item[kWindow], mass[kWindow];
    uint32_t place[256];
    u64 part_mass[kParts];
    uint32_t part_count[kParts];
    u64 wave[kThreads / 64];
    u64 u[4];
    uint32_t v[4];
};

struct Picker {
    const SampleParams &p;
    Pick &sh;
    int r, row;
    float top;
    double inv_t, unit;
    // the window: n places from rank base_rank on
    int n;
    uint32_t base_rank;
    u64 base_mass, end_mass;
    int block;           // whose bins are in sh
    uint32_t logits;     // of the bins last gathered

    __device__ u64 weight(uint32_t key) const {
        return (u64)rint(weight_of(key_value(key), top, inv_t) * unit);
    }
    __device__ const Slice &slice(int s) const { return p.slices[(int64_t)r * p.n_slices + s]; }
    __device__ float logit(int s, uint32_t i) const {
        return p.a.logits[(int64_t)row * p.a.stride + (int64_t)s * p.per + i];
    }

    // Gathers the bins [b0, b1]: their part of every slice's indices.
    __device__ __forceinline__ void gather(int b0, int b1) {
        const int tid = threadIdx.x;
        uint32_t c = 0;
        if (tid < p.n_slices) {
            const int sf = sh.shift[tid], j0 = max(b0 - sf, 0), j1 = b1 == kBins - 1 ? kBins - 1 : b1 - sf;
            int beg = 0;
            if (j1 >= j0) {
                const Slice &sl = slice(tid);
                const int end = sl.end[j1];
                beg = j0 > 0 ? sl.end[j0 - 1] : 0;
                c = end - beg;
            }
            sh.from[tid] = beg;
        }
        const uint32_t to = scan32<kThreads>(c, sh.wave);
        if (tid < p.n_slices) sh.upto[tid] = to;
        __syncthreads();
        logits = sh.upto[p.n_slices - 1];
    }
    // f(index in the row, pattern) for the gathered logits.
    template <class F>
    __device__ __forceinline__ void each(F f) const {
        load<4>([&](int, uint32_t index, uint32_t key) { f(index, key); });
    }
    // Q of a thread at a time.
    template <int Q, class F>
    __device__ __forceinline__ void load(F f) const {
        for (uint32_t i0 = threadIdx.x; i0 < logits; i0 += Q * kThreads) {
            int s[Q];
            uint32_t at[Q];
            float x[Q];
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                const uint32_t i = min(i0 + q * kThreads, logits - 1);
                int a = 0, b = p.n_slices - 1;  // the first slice with upto > i
                while (a < b) {
                    const int m = (a + b) >> 1;
                    if (sh.upto[m] > i) b = m;
                    else a = m + 1;
                }
                s[q] = a;
                at[q] = p.index[((int64_t)r * p.n_slices + a) * p.per + sh.from[a] + (i - (a > 0 ? sh.upto[a - 1] : 0))];
            }
#pragma unroll
            for (int q = 0; q < Q; ++q) x[q] = logit(s[q], at[q]);
#pragma unroll
            for (int q = 0; q < Q; ++q)
                if (i0 + q * kThreads < logits) f(q, (uint32_t)(s[q] * p.per) + at[q], order_key(x[q]));
        }
    }

    // Sorts the gathered logits with patterns in [lo, hi], `count` <= kWindow of them, into
    // the window.
    __device__ __forceinline__ void window(uint32_t lo, uint32_t hi, uint32_t count, uint32_t rank, u64 before) {
        window(lo, hi, count, rank, before, [&](auto f) { each(f); });
    }
    template <class Each>
    __device__ __forceinline__ void window(uint32_t lo, uint32_t hi, uint32_t count, uint32_t rank, u64 before,
                                           Each each_item) {
        const int tid = threadIdx.x;
        __syncthreads();
        if (tid == 0) sh.v[0] = 0;
        sh.item[tid] = ~0ull;
        __syncthreads();
        each_item([&](uint32_t index, uint32_t key) {
            if (key < lo || key > hi) return;
            const uint32_t i = atomicAdd(&sh.v[0], 1u);
            if (i < kWindow) sh.item[i] = (u64)~key << 32 | index;
        });
        __syncthreads();
        // ascending (the empty places last)
        int size = 64;
        while (size < (int)count) size <<= 1;
        u64 x = sh.item[tid];
        const bool live = tid < size;  // the same for a wave
        if (size <= 256) {
            // an item's place is the number of smaller ones: kThreads / size threads an item
            const int i = tid & (size - 1), each = size * size / kThreads, j0 = tid / size * each;
            const u64 y = sh.item[i];
            uint32_t smaller = 0;
            for (int j = 0; j < each; ++j) smaller += sh.item[j0 + j] < y;
            if (live) sh.place[tid] = 0;
            __syncthreads();
            atomicAdd(&sh.place[i], smaller);
            __syncthreads();
            if (tid < (int)count) sh.item[sh.place[tid]] = x;
            __syncthreads();
            x = sh.item[tid];
        } else {
            // bitonic; partners of the same wave need no barrier, and waves without items
            // only take part in those
            for (int k = 2; k <= size; k <<= 1)
                for (int j = k >> 1; j > 0; j >>= 1) {
                    u64 y = x;
                    if (j >= 64) {
                        __syncthreads();
                        if (live) sh.item[tid] = x;
                        __syncthreads();
                        if (live) y = sh.item[tid ^ j];
                    } else if (live) {
                        y = shfl_xor64(x, j);
                    }
                    const bool up = (tid & k) == 0, low = (tid & j) == 0;
                    if ((y < x) == (up == low)) x = y;
                }
        }
        u64 to = tid < (int)count ? weight(~(uint32_t)(x >> 32)) : 0;
        if (live) to = wave_prefix64(to);
        __syncthreads();
        if ((tid & 63) == 63) sh.wave[tid >> 6] = to;
        sh.item[tid] = x;
        __syncthreads();
        if (live)
            for (int i = 0; i < tid >> 6; ++i) to += sh.wave[i];
        sh.mass[tid] = to;
        __syncthreads();
        n = (int)count;
        base_rank = rank;
        base_mass = before;
        end_mass = before + sh.mass[n - 1];
    }

    __device__ __forceinline__ Found at_window(int i) const {
        const u64 x = sh.item[i], to = sh.mass[i], from = i > 0 ? sh.mass[i - 1] : 0;
        return Found{base_rank + i, base_mass + from, to - from, ~(uint32_t)(x >> 32), 0, (int)(uint32_t)x};
    }

    // The first of `m` <= 64 ends (counts or masses up to there, on top of rank and
    // before) past the target, or the last with a logit: every wave by itself.
    __device__ __forceinline__ int first_past(const uint32_t *count, const u64 *mass, int m, uint32_t rank, u64 before, bool by_count,
                              double target) const {
        const int lane = threadIdx.x & 63, i = min(lane, m - 1);
        const bool some = lane < m && count[i] > (lane > 0 ? count[i - 1] : 0);
        const bool past = some && (by_count ? (double)(rank + count[i]) > target : (double)(before + mass[i]) > target);
        const u64 a = __builtin_amdgcn_ballot_w64(past), b = __builtin_amdgcn_ballot_w64(some);
        return a ? __builtin_ctzll(a) : 63 - __builtin_clzll(b);
    }

    // The counts and masses of the bins of block `b`, up to the end of each, on top of
    // those before the block.
    __device__ __forceinline__ void open_block(int b) {
        const int tid = threadIdx.x;
        if (b == block) return;  // uniform
        block = b;
        __syncthreads();
        if (tid < kBlock) {
            sh.bin_count[tid] = 0;
            sh.bin_mass[tid] = 0;
        }
        __syncthreads();
        if (b < kBlocks - 1) {  // 16 bins of a slice
            for (int i = tid; i < p.n_slices * kBlock; i += kThreads)
                add_bin(i / kBlock, b * kBlock - sh.shift[i / kBlock] + i % kBlock, i % kBlock);
        } else {                // any past the other blocks
            for (int i = tid; i < p.n_slices * kBins; i += kThreads) {
                const int to = min(i % kBins + sh.shift[i / kBins], kBins - 1) - b * kBlock;
                if (to >= 0) add_bin(i / kBins, i % kBins, to);
            }
        }
        __syncthreads();
        if (tid < 64) {
            uint32_t c = tid < kBlock ? sh.bin_count[tid] : 0;
            u64 m = tid < kBlock ? sh.bin_mass[tid] : 0;
            c = (uint32_t)wave_prefix((int)c);
            m = wave_prefix64(m);
            if (tid < kBlock) {
                sh.bin_count[tid] = c;
                sh.bin_mass[tid] = m;
            }
        }
        __syncthreads();
    }
    __device__ __forceinline__ void add_bin(int s, int j, int to) {
        if (j < 0) return;
        const Slice &sl = slice(s);
        const uint32_t c = sl.end[j] - (j > 0 ? sl.end[j - 1] : 0);
        if (c == 0) return;
        atomicAdd(&sh.bin_count[to], c);
        atomicAdd(&sh.bin_mass[to], (u64)rint((double)sl.mass[j] * sh.scale[s]));
    }

    // The first place at which the number (by_count) or the weight of the logits down to
    // it exceeds `target`; the last one if none does.
    __device__ __forceinline__ Found find(bool by_count, double target) {
        const int tid = threadIdx.x;
        if (n > 0 && by_count && target >= base_rank && target < base_rank + n) return at_window((int)target - (int)base_rank);
        if (n > 0 && !by_count && target >= (double)base_mass && target < (double)end_mass) return search(target);
        const int b = first_past(sh.block_count, sh.block_mass, kBlocks, 0, 0, by_count, target);
        uint32_t rank = b > 0 ? sh.block_count[b - 1] : 0;
        u64 before = b > 0 ? sh.block_mass[b - 1] : 0;
        open_block(b);
        const int bin = first_past(sh.bin_count, sh.bin_mass, kBlock, rank, before, by_count, target);
        uint32_t count = sh.bin_count[bin];
        if (bin > 0) {
            count -= sh.bin_count[bin - 1];
            rank += sh.bin_count[bin - 1];
            before += sh.bin_mass[bin - 1];
        }
        gather(b * kBlock + bin, b * kBlock + bin);
        uint32_t lo = 0, hi = ~0u;
        // the thread's logits, where eight a thread hold them (pattern 0: none)
        constexpr int kHeld = 8;
        uint32_t key[kHeld] = {}, index[kHeld];
        const bool held = count > kWindow && logits <= kHeld * kThreads;
        if (held)
            load<kHeld>([&](int q, uint32_t i, uint32_t x) {
                key[q] = x;
                index[q] = i;
            });
        const auto each_item = [&](auto f) {
            if (held) {
#pragma unroll
                for (int q = 0; q < kHeld; ++q)
                    if (key[q] != 0) f(index[q], key[q]);
            } else {
                each(f);
            }
        };
        const auto each_key = [&](auto f) {
            each_item([&](uint32_t, uint32_t x) { f(x); });
        };
        while (count > kWindow) {  // narrow it
            __syncthreads();
            if (tid == 0) {
                sh.v[1] = ~0u;
                sh.v[2] = 0;
            }
            if (tid < kParts) {
                sh.part_count[tid] = 0;
                sh.part_mass[tid] = 0;
            }
            __syncthreads();
            uint32_t least = ~0u, most = 0;
            each_key([&](uint32_t key) {
                if (key >= lo && key <= hi) {
                    least = min(least, key);
                    most = max(most, key);
                }
            });
            least = ~wave_max(~least);
            most = wave_max(most);
            if ((tid & 63) == 0) {
                atomicMin(&sh.v[1], least);
                atomicMax(&sh.v[2], most);
            }
            __syncthreads();
            lo = sh.v[1];
            hi = sh.v[2];
            if (lo == hi) {  // equal logits
                const u64 w = weight(lo);
                double nth = by_count ? target - (double)rank : w > 0 ? floor((target - (double)before) / (double)w) : 0.0;
                nth = fmin(fmax(nth, 0.0), (double)(count - 1));
                return Found{rank + (uint32_t)nth, before + (u64)nth * w, w, lo, (uint32_t)nth, -1};
            }
            const int shift = max(24 - (int)__builtin_clz(hi - lo), 0);  // to at most kParts
            each_key([&](uint32_t key) {
                if (key >= lo && key <= hi) {
                    const uint32_t part = (hi - key) >> shift;
                    atomicAdd(&sh.part_count[part], 1u);
                    atomicAdd(&sh.part_mass[part], weight(key));
                }
            });
            __syncthreads();
            // every wave for itself: its lanes' four parts each
            const int lane = tid & 63;
            uint32_t c[kParts / 64], c_to = 0;
            u64 m[kParts / 64], m_to = 0;
#pragma unroll
            for (int i = 0; i < kParts / 64; ++i) {
                c_to += c[i] = sh.part_count[kParts / 64 * lane + i];
                m_to += m[i] = sh.part_mass[kParts / 64 * lane + i];
            }
            c_to = (uint32_t)wave_prefix((int)c_to);
            m_to = wave_prefix64(m_to);
            // from the lane's last part back to its first: the first part past the target, or
            // the last with a logit
            uint32_t first = kParts, last_of = 0, c_before = 0, c_last = 0;
            u64 m_before = 0, m_last = 0;
#pragma unroll
            for (int i = kParts / 64 - 1; i >= 0; --i) {
                if (c[i] > 0) {
                    if (last_of == 0) {
                        last_of = kParts / 64 * lane + i + 1;
                        c_last = c_to - c[i];
                        m_last = m_to - m[i];
                    }
                    if (by_count ? (double)(rank + c_to) > target : (double)(before + m_to) > target) {
                        first = kParts / 64 * lane + i;
                        c_before = c_to - c[i];
                        m_before = m_to - m[i];
                    }
                }
                c_to -= c[i];
                m_to -= m[i];
            }
            const u64 past = __builtin_amdgcn_ballot_w64(first < kParts), some = __builtin_amdgcn_ballot_w64(last_of > 0);
            const int from_lane = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
            const uint32_t part = (uint32_t)__builtin_amdgcn_readlane((int)(past ? first : last_of - 1), from_lane);
            const u64 mass = past ? m_before : m_last;
            rank += (uint32_t)__builtin_amdgcn_readlane((int)(past ? c_before : c_last), from_lane);
            before += (u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)mass, from_lane) |
                      (u64)(uint32_t)__builtin_amdgcn_readlane((int)(mass >> 32), from_lane) << 32;
            count = sh.part_count[part];
            // the patterns of the part: (hi - key) >> shift == part
            const uint32_t top_of = hi - (part << shift), width = (1u << shift) - 1;
            lo = top_of - lo > width ? top_of - width : lo;
            hi = top_of;
        }
        window(lo, hi, count, rank, before, each_item);
        if (by_count) return at_window(min(max((int)(target - (double)rank), 0), n - 1));
        return search(target);
    }

    // How many of the window's first places f holds for, up to where it ends (f(i) for i
    // < n; every wave by itself).
    template <class F>
    __device__ __forceinline__ int prefix(F f) const {
        const int lane = threadIdx.x & 63;
        for (int i0 = 0; i0 < n; i0 += 64) {
            const u64 no = __builtin_amdgcn_ballot_w64(i0 + lane >= n || !f(min(i0 + lane, n - 1)));
            if (no) return i0 + __builtin_ctzll(no);
        }
        return n;
    }
    // The window's first place whose weights exceed the target, or its last.
    __device__ __forceinline__ Found search(double target) const {
        return at_window(min(prefix([&](int i) { return (double)(base_mass + sh.mass[i]) <= target; }), n - 1));
    }
};

__global__ __launch_bounds__(kThreads) void sample_pick_kernel(SampleParams p) {
    __shared__ Pick sh;
    __shared__ int top_bin, finer;
    __shared__ uint32_t top_key;
    const int tid = threadIdx.x, r = blockIdx.x, row = p.row0 + r;
    const SampleRows &a = p.a;
    const float t = a.temperature ? a.temperature[row] : 1.0f;
    const int k = a.top_k ? a.top_k[row] : 0;
    const float top_p = a.top_p ? a.top_p[row] : 1.0f, min_p = a.min_p ? a.min_p[row] : 0.0f;
    const float u = fminf(fmaxf(a.u[row], 0.0f), 0x1.fffffep-1f);
    const Slice *slices = p.slices + (int64_t)r * p.n_slices;
    // the blocks of the first slices, a thread's one each, before what they are relative to
    const int s_mine = tid / kBlocks, b_mine = tid % kBlocks;
    uint32_t c_mine = 0;
    u64 m_mine = 0;
    if (s_mine < p.n_slices) {
        c_mine = slices[s_mine].block_end[b_mine];
        m_mine = slices[s_mine].block_mass[b_mine];
    }
    if (tid == 0) {
        top_key = 0;
        sh.v[0] = ~0u;
    }
    if (tid < kBlocks) {
        sh.block_count[tid] = 0;
        sh.block_mass[tid] = 0;
    }
    __syncthreads();
    uint32_t mine = 0;
    int bin = 0;
    if (tid < p.n_slices) {
        mine = slices[tid].top;
        bin = slices[tid].top_bin;
    }
    {
        const uint32_t most = wave_max(mine);
        if ((tid & 63) == 0) atomicMax(&top_key, most);
    }
    __syncthreads();
    const uint32_t tk = top_key;
    if (tk == 0) {  // uniform: no token
        if (tid == 0) a.ids[row] = -1;
        return;
    }
    if (!(t > 0.0f)) {  // uniform: the largest logit, lowest index
        if (tid < p.n_slices && mine == tk) atomicMin(&sh.v[0], (uint32_t)(tid * p.per) + slices[tid].first);
        __syncthreads();
        if (tid == 0) a.ids[row] = (int)sh.v[0];
        return;
    }
    const float top = key_value(tk);
    const double inv_t = 1.0 / (double)t;
    if (tid < p.n_slices && mine == tk) top_bin = bin;  // (all that write it write the same)
    __syncthreads();
    if (tid < p.n_slices) {
        sh.shift[tid] = mine != 0 ? (int)min((uint32_t)top_bin - (uint32_t)bin, (uint32_t)kBins) : kBins;
        sh.scale[tid] = mine != 0 ? weight_of(key_value(mine), top, inv_t) * (p.unit / kSliceUnit) : 0.0;
    }
    __syncthreads();
    for (int s = s_mine; s < p.n_slices; s += kThreads / kBlocks) {
        if (s != s_mine) {
            c_mine = slices[s].block_end[b_mine];
            m_mine = slices[s].block_mass[b_mine];
        }
        const int to = min(b_mine + sh.shift[s] / kBlock, kBlocks - 1);
        const uint32_t prev = b_mine > 0 ? slices[s].block_end[b_mine - 1] : 0;
        if (c_mine == prev) continue;
        atomicAdd(&sh.block_count[to], c_mine - prev);
        atomicAdd(&sh.block_mass[to], (u64)rint((double)m_mine * sh.scale[s]));
    }
    __syncthreads();
    if (tid < 64) {
        uint32_t c = tid < kBlocks ? sh.block_count[tid] : 0;
        u64 m = tid < kBlocks ? sh.block_mass[tid] : 0;
        c = (uint32_t)wave_prefix((int)c);
        m = wave_prefix64(m);
        // the row's sum to 2^61 up to 2^62: room for the roundings of its parts
        const int up = max(__builtin_clzll(lane_63(m)) - 2, 0);
        if (tid < kBlocks) {
            sh.block_count[tid] = c;
            sh.block_mass[tid] = m << up;
        }
        if (tid == 0) finer = up;
    }
    __syncthreads();
    const double fine = ldexp(1.0, finer);
    if (tid < p.n_slices) sh.scale[tid] *= fine;
    Picker pick{p, sh, r, row, top, inv_t, p.unit * fine, 0, 0, 0, 0, -1, 0};
    uint32_t keep = sh.block_count[kBlocks - 1];
    u64 kept = sh.block_mass[kBlocks - 1];
    const bool by_k = k > 0 && (uint32_t)k < keep;

    // The block that the kept logits cannot go past: all down to there in one window, if
    // they fit it.  (Top-p's share is one of what top-k keeps, so that with both the
    // window goes down to top-k's border.)
    int last = kBlocks - 1;
    if (by_k) last = pick.first_past(sh.block_count, sh.block_mass, kBlocks, 0, 0, true, (double)k - 1.0);
    if (top_p < 1.0f && !(by_k && sh.block_count[last] <= kWindow))
        last = min(last, pick.first_past(sh.block_count, sh.block_mass, kBlocks, 0, 0, false,
                                         nextafter((double)top_p * (double)sh.block_mass[last], -INFINITY)));
    // (a weight of min_p lies -log(min_p) below the top: a block more for the grid's
    // place and roundings)
    const int min_p_block =
        min_p > 0.0f ? (int)fmin(fmax(-log((double)min_p) * (kBinsPerUnit / kBlock), 0.0) + 2.0, (double)(kBlocks - 1)) : 0;
    if (min_p > 0.0f && !by_k && !(top_p < 1.0f)) last = min(last, min_p_block);
    if (last < kBlocks - 1 && sh.block_count[last] <= kWindow) {
        pick.gather(0, last * kBlock + kBlock - 1);
        pick.window(0u, ~0u, sh.block_count[last], 0, 0);
    }
    // Top-k's, top-p's and min-p's borders, then the draw: places of the order, one
    // after the other.
    Found f{};
    for (int step = 0; step < 5; ++step) {
        bool by_count = true;
        double target = 0.0;
        if (step == 0) {
            if (!by_k) continue;
            target = (double)k - 1.0;
        } else if (step == 1) {
            // the shortest prefix that reaches the share (0: the first logit)
            if (!(top_p < 1.0f)) continue;
            by_count = false;
            target = fmax(nextafter((double)top_p * (double)kept, -INFINITY), 0.0);
        } else if (step == 2) {
            // how many logits weigh enough: those of the window, if it ends below them, else
            // down to the kept ones' border or to where none can
            if (!(min_p > 0.0f)) continue;
            const auto enough = [&](uint32_t key) { return weight_of(key_value(key), top, inv_t) >= (double)min_p; };
            uint32_t most = 0;
            const bool from_top = pick.n > 0 && pick.base_rank == 0;
            if (from_top) most = pick.prefix([&](int i) { return enough(~(uint32_t)(sh.item[i] >> 32)); });
            if (!from_top || (most == (uint32_t)pick.n && most < keep)) {  // uniform
                __syncthreads();
                if (tid == 0) sh.v[0] = 0;
                uint32_t c = 0;
                pick.gather(0, min(last, min_p_block) * kBlock + kBlock - 1);
                pick.each([&](uint32_t, uint32_t key) { c += enough(key); });
#pragma unroll
                for (int d = 32; d > 0; d >>= 1) c += __shfl_xor((int)c, d, 64);
                if ((tid & 63) == 0) atomicAdd(&sh.v[0], c);
                __syncthreads();
                most = sh.v[0];
            }
            most = max(most, 1u);
            if (most >= keep) continue;
            target = (double)most - 1.0;
        } else if (step == 3) {
            by_count = false;
            target = (double)u * (double)kept;
        } else {
            if (f.rank < keep) continue;
            target = (double)keep - 1.0;
        }
        f = pick.find(by_count, target);
        if (step < 3 && f.rank + 1 < keep) {
            keep = f.rank + 1;
            kept = f.before + f.w;
        }
    }
    if (f.index >= 0) {  // uniform
        if (tid == 0) a.ids[row] = f.index;
        return;
    }
    // the nth logit of its pattern by index: its slice, then through it in order
    uint32_t before = 0;
    for (int s = 0; s < p.n_slices; ++s) {
        const int n = min(p.per, a.n_vocab - s * p.per);
        uint32_t c = 0;
        for (int i = tid; i < n; i += kThreads) c += order_key(pick.logit(s, i)) == f.key;
        const uint32_t to = scan32<kThreads>(c, sh.wave);
        __syncthreads();
        if (tid == kThreads - 1) sh.v[0] = to;
        __syncthreads();
        const uint32_t all = sh.v[0];
        if (before + all <= f.nth) {
            before += all;
            continue;
        }
        for (int i0 = 0; i0 < n; i0 += kThreads) {
            const bool is = i0 + tid < n && order_key(pick.logit(s, i0 + tid)) == f.key;
            const uint32_t upto = before + scan32<kThreads>(is, sh.wave);
            if (is && upto == f.nth + 1) a.ids[row] = s * p.per + i0 + tid;
            __syncthreads();
            if (tid == kThreads - 1) sh.v[0] = upto;
            __syncthreads();
            before = sh.v[0];
            if (before > f.nth) return;  // uniform
        }
    }
}

}  // namespace

hipError_t launch_sample(const SampleRows &rows, int n_rows, hipStream_t st) {
    SampleParams p{};
    p.a = rows;
    // Slices of 2048 logits for a few rows, which leave CUs free, of 8192 for some, of
    // 16384 for many: fewer bins to put together.
    const int cus = device_info().cu_count > 0 ? device_info().cu_count : 256;
    int most = 2048;
    if ((int64_t)((rows.n_vocab + most - 1) / most) * n_rows > 2 * cus || rows.n_vocab > kSlices * most) most = 8192;
    if ((int64_t)((rows.n_vocab + most - 1) / most) * n_rows > 2 * cus || rows.n_vocab > kSlices * most) most = 16384;
    p.n_slices = (rows.n_vocab + most - 1) / most;
    p.per = ((rows.n_vocab + p.n_slices - 1) / p.n_slices + 1) & ~1;
    int bits = 62;
    for (int n = 1; n < rows.n_vocab; n <<= 1) --bits;
    p.unit = ldexp(1.0, std::min(bits, 52));
    const size_t row_bytes = (size_t)p.n_slices * (sizeof(Slice) + 2 * (size_t)p.per);
    const int group = (int)std::max<size_t>(1, std::min<size_t>(n_rows, kWorkspaceBytes / row_bytes));
    float *ws = nullptr;
    hipError_t e = Scratch{}.get(st, (size_t)group * row_bytes, &ws);
    if (e != hipSuccess) return e;
    p.slices = reinterpret_cast<Slice *>(ws);
    p.index = reinterpret_cast<uint16_t *>(p.slices + (size_t)group * p.n_slices);
    for (p.row0 = 0; p.row0 < n_rows; p.row0 += group) {
        const int n = std::min(group, n_rows - p.row0);
        if (most == 2048) sample_slices_kernel<256, 8><<<n * p.n_slices, 256, 0, st>>>(p);
        else if (most == 8192) sample_slices_kernel<1024, 8><<<n * p.n_slices, 1024, 0, st>>>(p);
        else sample_slices_kernel<1024, 16><<<n * p.n_slices, 1024, 0, st>>>(p);
        sample_pick_kernel<<<n, kThreads, 0, st>>>(p);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace rxq4
