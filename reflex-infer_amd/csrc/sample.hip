// sample.hip -- the next token of each row of logits: temperature, top-k, top-p,
// min-p and a given random number.
//
// The order is logits descending, equal ones by index.  Every step is a place in
// it: top-k a rank, top-p and the draw a sum of weights, min-p a weight.  So the row
// need not be sorted: counts and sums of weights over bins of the logits say in
// which bin a place lies, and only that bin's logits (or, where the kept ones are
// few, all bins down to there at once) are sorted.
// Weights exp((l - max) / T) are formed in 64 bits and summed as whole numbers, so
// the sums depend on no order: off by half a unit (2^-49 of a slice's largest weight,
// and 2^-(63 - log2 n_vocab) of the row's) a logit.
//
//   sample_slices_kernel  a workgroup per slice of a row (up to 16384 logits, in
//       registers): its largest logit, the count and weight of 512 bins of 1/16 in
//       (l / T) on a grid that all slices share (the last bin: all further down), and
//       its indices in the order of the bins (a counting sort in LDS);
//   sample_pick_kernel    a workgroup per row: the slices' bins together, then the
//       places; a window of up to 1024 logits of some bins sorted in LDS.  A bin with
//       more logits is narrowed by their ordered bit patterns, 256 parts at a time,
//       down to a window or to equal logits.
// Bound: two launches, the reads of the row (the slices) and the chain of dependent
// steps of one workgroup (the pick).
#include <math.h>

#include <algorithm>

#include "launch.h"
#include "paged.h"
#include "q4k_device.h"

namespace rxq4 {
namespace {

typedef unsigned long long u64;

constexpr int kThreads = 1024;
constexpr int kPer = 16;                      // logits of a thread
constexpr int kSlice = kThreads * kPer;       // of a slice, at most
constexpr int kBins = 512;
constexpr double kBinsPerUnit = 16.0;
constexpr int kWindow = 1024;                 // logits sorted at once
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
constexpr uint32_t kMinusInf = 0x007FFFFFu;  // order_key(-inf): it and NaN are no tokens

// A slice's part of the workspace.
struct Slice {
    u64 mass[kBins];          // weight relative to the slice's largest logit
    uint32_t top;             // its pattern (0: no token)
    uint32_t first;           // its lowest index in the slice
    double top_bin;           // its place on the grid
    uint16_t end[kBins];      // indices before the end of each bin
};

struct SampleParams {
    SampleRows a;
    Slice *slices;      // [row][slice]
    uint16_t *index;    // [row][slice][per]: indices in the slice, by bin
    int row0, n_slices, per;
    double unit;        // weight units of a row
};

__device__ __forceinline__ double weight_of(float l, float top, double inv_t) {
    return l == top ? 1.0 : top == INFINITY ? 0.0 : exp(((double)l - (double)top) * inv_t);
}

__device__ __forceinline__ u64 shfl_up64(u64 v, int d) {
    const uint32_t lo = __shfl_up((int)(uint32_t)v, d, 64), hi = __shfl_up((int)(v >> 32), d, 64);
    return (u64)hi << 32 | lo;
}

// Sums over the threads up to each one (inclusive); `wave`: 16 values of LDS.
// Every thread of the workgroup takes part.
__device__ u64 scan64(u64 v, u64 *wave) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const u64 x = shfl_up64(v, d);
        if (lane >= d) v += x;
    }
    __syncthreads();
    if (lane == 63) wave[w] = v;
    __syncthreads();
    for (int i = 0; i < w; ++i) v += wave[i];
    return v;
}
__device__ uint32_t scan32(uint32_t v, u64 *wave) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t x = __shfl_up((int)v, d, 64);
        if (lane >= d) v += x;
    }
    __syncthreads();
    if (lane == 63) wave[w] = v;
    __syncthreads();
    for (int i = 0; i < w; ++i) v += (uint32_t)wave[i];
    return v;
}

__global__ __launch_bounds__(kThreads) void sample_slices_kernel(SampleParams p) {
    __shared__ uint32_t count[kBins];
    __shared__ u64 mass[kBins], wave[kThreads / 64];
    __shared__ uint16_t sorted[kSlice];
    __shared__ uint32_t top_key, top_first;
    const int tid = threadIdx.x;
    const int s = blockIdx.x % p.n_slices, r = blockIdx.x / p.n_slices, row = p.row0 + r;
    const int n = min(p.per, p.a.n_vocab - s * p.per);
    const float *l = p.a.logits + (int64_t)row * p.a.stride + (int64_t)s * p.per;
    uint32_t key[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int at = i * kThreads + tid;
        const float x = l[min(at, n - 1)];
        key[i] = at < n ? order_key(x) : 0u;
    }
    const float t = p.a.temperature ? p.a.temperature[row] : 1.0f;
    if (tid == 0) {
        top_key = 0;
        top_first = ~0u;
    }
    if (tid < kBins) {
        count[tid] = 0;
        mass[tid] = 0;
    }
    __syncthreads();
    uint32_t best = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) best = max(best, key[i]);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) best = max(best, (uint32_t)__shfl_xor((int)best, d, 64));
    if ((tid & 63) == 0) atomicMax(&top_key, best);
    __syncthreads();
    const uint32_t tk = top_key;
    Slice &out = p.slices[(int64_t)r * p.n_slices + s];
    if (tk <= kMinusInf || !(t > 0.0f)) {  // uniform: no token, or the largest logit alone is asked for
        if (tk > kMinusInf) {
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                if (key[i] == tk) atomicMin(&top_first, (uint32_t)(i * kThreads + tid));
        }
        if (tid < kBins) {
            out.mass[tid] = 0;
            out.end[tid] = 0;
        }
        __syncthreads();
        if (tid == 0) {
            out.top = tk <= kMinusInf ? 0u : tk;
            out.first = top_first;
            out.top_bin = -INFINITY;
        }
        return;
    }
    const float top = key_value(tk);
    const double inv_t = 1.0 / (double)t, grid = kBinsPerUnit * inv_t;
    const double top_bin = top == INFINITY ? INFINITY : floor((double)top * grid);
    uint32_t place[kPer];  // bin, and number in it
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        place[i] = ~0u;
        if (key[i] > kMinusInf) {
            const float x = key_value(key[i]);
            const double below = x == top ? 0.0 : top_bin - floor((double)x * grid);
            const int b = below < (double)(kBins - 1) ? (int)below : kBins - 1;
            const u64 w = (u64)rint(weight_of(x, top, inv_t) * kSliceUnit);
            place[i] = (uint32_t)b << 16 | atomicAdd(&count[b], 1u);
            if (w) atomicAdd(&mass[b], w);
        }
    }
    __syncthreads();
    const uint32_t mine = tid < kBins ? count[tid] : 0u;
    const uint32_t end = scan32(mine, wave);
    if (tid < kBins) {
        count[tid] = end - mine;
        out.end[tid] = (uint16_t)end;
        out.mass[tid] = mass[tid];
    }
    if (tid == 0) {
        out.top = tk;
        out.first = ~0u;
        out.top_bin = top_bin;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPer; ++i)
        if (place[i] != ~0u) sorted[count[place[i] >> 16] + (place[i] & 0xFFFFu)] = (uint16_t)(i * kThreads + tid);
    __syncthreads();
    uint32_t *dst = reinterpret_cast<uint32_t *>(p.index + ((int64_t)r * p.n_slices + s) * p.per);
    for (int i = tid; i < (n + 1) / 2; i += kThreads) dst[i] = reinterpret_cast<const uint32_t *>(sorted)[i];
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
    // the row's bins: counts and weights up to the end of each
    u64 mass_to[kBins];
    uint32_t count_to[kBins];
    uint16_t shift[512];    // bins of a slice below the row's top
    double scale[512];      // a slice's weight unit in the row's
    // the window: sorted (~pattern, index), weights up to the end of each
    u64 item[kWindow], mass[kWindow];
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
    double inv_t;
    // the window: n places from rank base_rank on
    int n;
    uint32_t base_rank;
    u64 base_mass, end_mass;

    __device__ u64 weight(uint32_t key) const {
        return (u64)rint(weight_of(key_value(key), top, inv_t) * p.unit);
    }
    __device__ const Slice &slice(int s) const { return p.slices[(int64_t)r * p.n_slices + s]; }
    __device__ float logit(int s, uint32_t i) const {
        return p.a.logits[(int64_t)row * p.a.stride + (int64_t)s * p.per + i];
    }

    // f(slice, index in it, pattern) for the logits of the bins [b0, b1]: 32 threads a
    // slice.
    template <class F>
    __device__ void each(int b0, int b1, F f) const {
        for (int s = threadIdx.x >> 5; s < p.n_slices; s += kThreads / 32) {
            const int sf = sh.shift[s], j0 = max(b0 - sf, 0), j1 = b1 == kBins - 1 ? kBins - 1 : b1 - sf;
            if (j1 < j0) continue;
            const Slice &sl = slice(s);
            const int beg = j0 > 0 ? sl.end[j0 - 1] : 0, end = sl.end[j1];
            const uint16_t *index = p.index + ((int64_t)r * p.n_slices + s) * p.per;
            for (int i = beg + (threadIdx.x & 31); i < end; i += 32) {
                const uint32_t at = index[i];
                f(s, at, order_key(logit(s, at)));
            }
        }
    }

    // Sorts the logits of the bins [b0, b1] with patterns in [lo, hi], `count` <=
    // kWindow of them, into the window.
    __device__ void window(int b0, int b1, uint32_t lo, uint32_t hi, uint32_t count, uint32_t rank, u64 before) {
        const int tid = threadIdx.x;
        __syncthreads();
        if (tid == 0) sh.v[0] = 0;
        sh.item[tid] = ~0ull;
        __syncthreads();
        each(b0, b1, [&](int s, uint32_t at, uint32_t key) {
            if (key < lo || key > hi) return;
            const uint32_t i = atomicAdd(&sh.v[0], 1u);
            if (i < kWindow) sh.item[i] = (u64)~key << 32 | (uint32_t)(s * p.per + at);
        });
        __syncthreads();
        // bitonic, ascending (the empty places last); partners of the same wave need no
        // barrier
        int size = 64;
        while (size < (int)count) size <<= 1;
        u64 x = sh.item[tid];
        for (int k = 2; k <= size; k <<= 1)
            for (int j = k >> 1; j > 0; j >>= 1) {
                u64 y;
                if (j >= 64) {
                    __syncthreads();
                    sh.item[tid] = x;
                    __syncthreads();
                    y = sh.item[tid ^ j];
                } else {
                    const uint32_t a = __shfl_xor((int)(uint32_t)x, j, 64), b = __shfl_xor((int)(x >> 32), j, 64);
                    y = (u64)b << 32 | a;
                }
                const bool up = (tid & k) == 0 || k == size, low = (tid & j) == 0;
                if ((y < x) == (up == low)) x = y;
            }
        __syncthreads();
        sh.item[tid] = x;
        const u64 w = tid < (int)count ? weight(~(uint32_t)(x >> 32)) : 0;
        const u64 to = scan64(w, sh.wave);
        sh.mass[tid] = to;
        __syncthreads();
        n = (int)count;
        base_rank = rank;
        base_mass = before;
        end_mass = before + sh.mass[n - 1];
    }

    __device__ Found at_window(int i) const {
        const u64 x = sh.item[i], to = sh.mass[i], from = i > 0 ? sh.mass[i - 1] : 0;
        return Found{base_rank + i, base_mass + from, to - from, ~(uint32_t)(x >> 32), 0, (int)(uint32_t)x};
    }

    // The first place at which the number (by_count) or the weight of the logits down to
    // it exceeds `target`; the last one if none does.
    __device__ Found find(bool by_count, double target) {
        const int tid = threadIdx.x;
        if (n > 0 && by_count && target >= base_rank && target < base_rank + n) return at_window((int)target - (int)base_rank);
        if (n > 0 && !by_count && target >= (double)base_mass && target < (double)end_mass) return search(target);
        // its bin: the first whose end exceeds the target, else the last with a logit
        __syncthreads();
        if (tid == 0) {
            sh.v[1] = kBins;
            sh.v[2] = 0;
        }
        __syncthreads();
        if (tid < kBins) {
            const bool some = sh.count_to[tid] > (tid > 0 ? sh.count_to[tid - 1] : 0);
            if (some && (by_count ? (double)sh.count_to[tid] > target : (double)sh.mass_to[tid] > target)) atomicMin(&sh.v[1], (uint32_t)tid);
            if (some) atomicMax(&sh.v[2], (uint32_t)tid);
        }
        __syncthreads();
        const int b = sh.v[1] < kBins ? (int)sh.v[1] : (int)sh.v[2];
        uint32_t rank = b > 0 ? sh.count_to[b - 1] : 0, count = sh.count_to[b] - rank;
        u64 before = b > 0 ? sh.mass_to[b - 1] : 0;
        uint32_t lo = 0, hi = ~0u;
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
            each(b, b, [&](int, uint32_t, uint32_t key) {
                if (key >= lo && key <= hi) {
                    least = min(least, key);
                    most = max(most, key);
                }
            });
            atomicMin(&sh.v[1], least);
            atomicMax(&sh.v[2], most);
            __syncthreads();
            lo = sh.v[1];
            hi = sh.v[2];
            if (lo == hi) {  // equal logits
                const u64 w = weight(lo);
                double nth = by_count ? target - (double)rank : w > 0 ? floor((target - (double)before) / (double)w) : 0.0;
                nth = fmin(fmax(nth, 0.0), (double)(count - 1));
                return Found{rank + (uint32_t)nth, before + (u64)nth * w, w, lo, (uint32_t)nth, -1};
            }
            const u64 range = (u64)(hi - lo) + 1;
            each(b, b, [&](int, uint32_t, uint32_t key) {
                if (key >= lo && key <= hi) {
                    const int part = (int)((u64)(hi - key) * kParts / range);
                    atomicAdd(&sh.part_count[part], 1u);
                    atomicAdd(&sh.part_mass[part], weight(key));
                }
            });
            __syncthreads();
            const uint32_t c = tid < kParts ? sh.part_count[tid] : 0;
            const u64 m = tid < kParts ? sh.part_mass[tid] : 0;
            const uint32_t c_to = scan32(c, sh.wave);
            const u64 m_to = scan64(m, sh.wave);
            __syncthreads();
            if (tid == 0) {
                sh.v[1] = kParts;
                sh.v[2] = 0;
            }
            __syncthreads();
            if (c > 0) {
                if (by_count ? (double)(rank + c_to) > target : (double)(before + m_to) > target) atomicMin(&sh.v[1], (uint32_t)tid);
                atomicMax(&sh.v[2], (uint32_t)tid);
            }
            __syncthreads();
            const uint32_t part = sh.v[1] < kParts ? sh.v[1] : sh.v[2];
            if (tid == (int)part) {
                sh.v[3] = c_to - c;
                sh.u[0] = m_to - m;
                sh.v[0] = c;
            }
            __syncthreads();
            rank += sh.v[3];
            before += sh.u[0];
            count = sh.v[0];
            // the patterns of the part: (hi - key) * kParts / range == part
            const uint32_t from = (uint32_t)(((u64)part * range + kParts - 1) / kParts);
            const uint32_t to = (uint32_t)((((u64)part + 1) * range + kParts - 1) / kParts - 1);
            lo = hi - to;
            hi = hi - from;
        }
        window(b, b, lo, hi, count, rank, before);
        if (by_count) return at_window(min(max((int)(target - (double)rank), 0), n - 1));
        return search(target);
    }

    // The window's first place whose weights exceed the target, or its last.
    __device__ Found search(double target) {
        const int tid = threadIdx.x;
        __syncthreads();
        if (tid == 0) sh.v[1] = n - 1;
        __syncthreads();
        if (tid < n && (double)(base_mass + sh.mass[tid]) > target) atomicMin(&sh.v[1], (uint32_t)tid);
        __syncthreads();
        return at_window((int)sh.v[1]);
    }
};

__global__ __launch_bounds__(kThreads) void sample_pick_kernel(SampleParams p) {
    __shared__ Pick sh;
    __shared__ double top_bin;
    __shared__ uint32_t top_key;
    const int tid = threadIdx.x, r = blockIdx.x, row = p.row0 + r;
    const SampleRows &a = p.a;
    const float t = a.temperature ? a.temperature[row] : 1.0f;
    const int k = a.top_k ? a.top_k[row] : 0;
    const float top_p = a.top_p ? a.top_p[row] : 1.0f, min_p = a.min_p ? a.min_p[row] : 0.0f;
    const float u = fminf(fmaxf(a.u[row], 0.0f), 0x1.fffffep-1f);
    const Slice *slices = p.slices + (int64_t)r * p.n_slices;
    if (tid == 0) {
        top_key = 0;
        sh.v[0] = ~0u;
    }
    if (tid < kBins) {
        sh.count_to[tid] = 0;
        sh.mass_to[tid] = 0;
    }
    __syncthreads();
    uint32_t mine = 0;
    double bin = 0.0;
    if (tid < p.n_slices) {
        mine = slices[tid].top;
        bin = slices[tid].top_bin;
        atomicMax(&top_key, mine);
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
        const double below = mine == tk ? 0.0 : top_bin - bin;
        sh.shift[tid] = mine != 0 && below < (double)(kBins - 1) ? (uint16_t)below : kBins - 1;
        sh.scale[tid] = mine != 0 ? weight_of(key_value(mine), top, inv_t) * (p.unit / kSliceUnit) : 0.0;
    }
    __syncthreads();
    for (int i = tid; i < p.n_slices * kBins; i += kThreads) {
        const int s = i / kBins, j = i % kBins;
        const uint32_t c = slices[s].end[j] - (j > 0 ? slices[s].end[j - 1] : 0);
        if (c == 0) continue;
        const int b = min(j + sh.shift[s], kBins - 1);
        atomicAdd(&sh.count_to[b], c);
        atomicAdd(&sh.mass_to[b], (u64)rint((double)slices[s].mass[j] * sh.scale[s]));
    }
    __syncthreads();
    {
        const uint32_t c = scan32(tid < kBins ? sh.count_to[tid] : 0, sh.wave);
        const u64 m = scan64(tid < kBins ? sh.mass_to[tid] : 0, sh.wave);
        __syncthreads();
        if (tid < kBins) {
            sh.count_to[tid] = c;
            sh.mass_to[tid] = m;
        }
        __syncthreads();
    }
    Picker pick{p, sh, r, row, top, inv_t, 0, 0, 0, 0};
    uint32_t keep = sh.count_to[kBins - 1];
    u64 kept = sh.mass_to[kBins - 1];

    // Bins that the kept logits cannot go past: all down to there in one window, if
    // they fit it.
    int last = kBins - 1;
    {
        const uint32_t want = k > 0 && (uint32_t)k < keep ? (uint32_t)k : keep;
        if (tid == 0) {
            sh.v[0] = kBins - 1;
            sh.v[1] = kBins - 1;
        }
        __syncthreads();
        if (tid < kBins && sh.count_to[tid] >= want) atomicMin(&sh.v[0], (uint32_t)tid);
        __syncthreads();
        last = (int)sh.v[0];
        const double most = (double)top_p * (double)sh.mass_to[last];
        if (top_p < 1.0f && tid < kBins && (double)sh.mass_to[tid] >= most && sh.count_to[tid] > 0) atomicMin(&sh.v[1], (uint32_t)tid);
        __syncthreads();
        if (top_p < 1.0f) last = min(last, (int)sh.v[1]);
        // (a weight of min_p lies -log(min_p) below the top: one bin more for the grid's
        // place and one for roundings)
        if (min_p > 0.0f) last = min(last, (int)fmin(fmax(-log((double)min_p) * kBinsPerUnit, 0.0) + 2.0, (double)(kBins - 1)));
        const bool filtered = want < keep || top_p < 1.0f || min_p > 0.0f;
        if (filtered && sh.count_to[last] <= kWindow) pick.window(0, last, 0u, ~0u, sh.count_to[last], 0, 0);
    }
    if (k > 0 && (uint32_t)k < keep) {
        const Found f = pick.find(true, (double)k - 1.0);
        keep = f.rank + 1;
        kept = f.before + f.w;
    }
    if (top_p < 1.0f) {
        // the shortest prefix that reaches the target
        const Found f = pick.find(false, nextafter((double)top_p * (double)kept, -INFINITY));
        if (f.rank + 1 < keep) {
            keep = f.rank + 1;
            kept = f.before + f.w;
        }
    }
    if (min_p > 0.0f) {
        // how many logits weigh enough: those of the window, if it ends below them
        __syncthreads();
        if (tid == 0) sh.v[0] = 0;
        __syncthreads();
        uint32_t c = 0;
        const auto enough = [&](uint32_t key) { return weight_of(key_value(key), top, inv_t) >= (double)min_p; };
        const bool in_window = pick.n > 0 && pick.base_rank == 0 &&
                               ((uint32_t)pick.n >= keep || !enough(~(uint32_t)(sh.item[pick.n - 1] >> 32)));
        if (in_window) {
            if (tid < pick.n) c = enough(~(uint32_t)(sh.item[tid] >> 32));
        } else {
            pick.each(0, last, [&](int, uint32_t, uint32_t key) { c += enough(key); });
        }
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) c += __shfl_xor((int)c, d, 64);
        if ((tid & 63) == 0) atomicAdd(&sh.v[0], c);
        __syncthreads();
        const uint32_t most = max(1u, sh.v[0]);
        if (most < keep) {
            const Found f = pick.find(true, (double)most - 1.0);
            keep = f.rank + 1;
            kept = f.before + f.w;
        }
    }
    Found f = pick.find(false, (double)u * (double)kept);
    if (f.rank >= keep) f = pick.find(true, (double)keep - 1.0);
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
        const uint32_t to = scan32(c, sh.wave);
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
            const uint32_t upto = before + scan32(is, sh.wave);
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
    p.n_slices = (rows.n_vocab + kSlice - 1) / kSlice;
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
        sample_slices_kernel<<<n * p.n_slices, kThreads, 0, st>>>(p);
        sample_pick_kernel<<<n, kThreads, 0, st>>>(p);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace rxq4
