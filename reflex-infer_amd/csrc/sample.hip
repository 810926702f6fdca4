// sample.hip -- the next token of each row of logits: temperature, top-k, top-p,
// min-p and a given random number.
//
// The order is logits descending, equal ones by index.  Every step is a place in
// it: top-k a count, top-p and the draw a sum of weights, min-p a weight.  A
// place is found by descending through the logits' ordered 32-bit patterns, eight
// bits at a time: counts and sums of weights of the 256 patterns below what is
// known, then the one where the place lies.  Equal logits weigh the same, so only
// the draw's last step needs their indices.
// Weights exp((l - max) / T) are formed in 64 bits and summed as whole numbers in
// units of 2^-kBits (of the largest weight), so the sums depend on no order:
// off by 2^-(kBits + 1) a logit at most.
//
// A workgroup takes a row.
#include <math.h>

#include "launch.h"
#include "q4k_device.h"

namespace rxq4 {
namespace {

constexpr int kThreads = 1024;

// Larger patterns are larger logits; NaN is least, -0 is 0.
__device__ __forceinline__ uint32_t order_key(float l) {
    const uint32_t u = __builtin_bit_cast(uint32_t, l == 0.0f ? 0.0f : l);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return 0u;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}
constexpr uint32_t kMinusInf = 0x007FFFFFu;  // order_key(-inf)

struct Row {
    const float *l;
    int n;
    float top;       // the largest logit, finite or +inf
    double inv_t;
    double unit;     // 2^kBits
    __device__ unsigned long long weight(uint32_t key) const {
        if (key <= kMinusInf) return 0;
        const float x = key_value(key);
        if (x == top) return (unsigned long long)unit;
        if (top == INFINITY) return 0;
        return (unsigned long long)rint(exp(((double)x - (double)top) * inv_t) * unit);
    }
};

struct Shared {
    unsigned long long mass[256];
    unsigned int count[256];
    unsigned long long pick_mass;
    unsigned int pick, pick_count;
};

// A place: the pattern `key`, the logits above it (their number and weight) and
// its own number.
struct Place {
    uint32_t key;
    unsigned int above, equal;
    unsigned long long above_mass;
};

// The first pattern, descending, at which the count (by_count) or the mass of the
// logits down to it exceeds `target`; the last one there is if none does.
__device__ Place find(const Row &r, Shared &sh, bool by_count, double target) {
    const int tid = threadIdx.x;
    Place p{0, 0, 0, 0};
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        if (tid < 256) {
            sh.mass[tid] = 0;
            sh.count[tid] = 0;
        }
        __syncthreads();
        const uint32_t known = shift == 24 ? 0u : ~0u << (shift + 8);
        for (int i = tid; i < r.n; i += kThreads) {
            const uint32_t key = order_key(r.l[i]);
            if (key <= kMinusInf || (key & known) != p.key) continue;
            const int b = (key >> shift) & 255;
            atomicAdd(&sh.count[b], 1u);
            atomicAdd(&sh.mass[b], r.weight(key));
        }
        __syncthreads();
        if (tid == 0) {
            unsigned int n = p.above;
            unsigned long long m = p.above_mass;
            int last = -1;
            unsigned int last_n = n;
            unsigned long long last_m = m;
            for (int b = 255; b >= 0; --b) {
                if (sh.count[b] == 0) continue;
                last = b;
                last_n = n;
                last_m = m;
                n += sh.count[b];
                m += sh.mass[b];
                if (by_count ? (double)n > target : (double)m > target) break;
            }
            sh.pick = last;
            sh.pick_count = last_n;
            sh.pick_mass = last_m;
        }
        __syncthreads();
        p.key |= sh.pick << shift;
        p.above = sh.pick_count;
        p.above_mass = sh.pick_mass;
        p.equal = sh.count[sh.pick];
    }
    return p;
}

__global__ __launch_bounds__(kThreads) void sample_row_kernel(SampleRows a, double unit) {
    __shared__ Shared sh;
    __shared__ uint32_t top_key;
    const int tid = threadIdx.x, row = blockIdx.x;
    Row r{a.logits + (int64_t)row * a.stride, a.n_vocab, 0.0f, 0.0, unit};
    if (tid == 0) top_key = 0;
    __syncthreads();
    uint32_t best = 0;
    for (int i = tid; i < r.n; i += kThreads) best = max(best, order_key(r.l[i]));
    atomicMax(&top_key, best);
    __syncthreads();
    const uint32_t top = top_key;
    if (top <= kMinusInf) {  // uniform
        if (tid == 0) a.ids[row] = -1;
        return;
    }
    const float t = a.temperature ? a.temperature[row] : 1.0f;
    r.top = key_value(top);
    uint32_t key = top;
    unsigned int nth = 0;  // of the logits equal to it
    if (t > 0.0f) {
        r.inv_t = 1.0 / (double)t;
        // the kept prefix: the logits above `cut.key` and `n_equal` equal to it
        Place cut = find(r, sh, false, INFINITY);  // everything
        unsigned int n_equal = cut.equal;
        const int k = a.top_k ? a.top_k[row] : 0;
        if (k > 0 && (unsigned)k < cut.above + cut.equal) {
            cut = find(r, sh, true, (double)k - 1.0);
            n_equal = k - cut.above;
        }
        auto total = [&]() { return (double)cut.above_mass + (double)n_equal * (double)r.weight(cut.key); };
        const float top_p = a.top_p ? a.top_p[row] : 1.0f;
        if (top_p < 1.0f) {
            // the shortest prefix whose weight reaches the target: its last logit is the
            // first at which the sum does not stay below
            const double target = (double)top_p * total();
            const Place c = find(r, sh, false, nextafter(target, -INFINITY));
            const double w = (double)r.weight(c.key);
            const double more = w > 0 ? ceil((target - (double)c.above_mass) / w) : 1.0;
            const unsigned int n = (unsigned)fmin(fmax(more, 1.0), (double)c.equal);
            if (c.key > cut.key || (c.key == cut.key && n < n_equal)) {
                cut = c;
                n_equal = n;
            }
        }
        const float min_p = a.min_p ? a.min_p[row] : 0.0f;
        if (min_p > 0.0f) {
            // how many logits weigh enough: a count over the row
            __syncthreads();
            if (tid == 0) sh.pick = 0;
            __syncthreads();
            unsigned int n = 0;
            for (int i = tid; i < r.n; i += kThreads) {
                const uint32_t x = order_key(r.l[i]);
                if (x > kMinusInf)
                    n += (x == top ? 1.0 : exp(((double)key_value(x) - (double)r.top) * r.inv_t)) >= (double)min_p;
            }
            atomicAdd(&sh.pick, n);
            __syncthreads();
            const unsigned int keep = max(1u, sh.pick);
            if (keep < cut.above + n_equal) {
                cut = find(r, sh, true, (double)keep - 1.0);
                n_equal = keep - cut.above;
            }
        }
        const float u = fminf(fmaxf(a.u[row], 0.0f), 0x1.fffffep-1f);
        const double target = (double)u * total();
        const Place c = find(r, sh, false, target);
        key = max(c.key, cut.key);
        if (c.key >= cut.key) {
            const double w = (double)r.weight(key);
            nth = w > 0 ? (unsigned)fmax(0.0, floor((target - (double)c.above_mass) / w)) : 0;
            nth = min(nth, (c.key == cut.key ? n_equal : c.equal) - 1);
        } else {
            nth = n_equal - 1;
        }
    }
    // the nth logit of pattern `key` by index
    __shared__ unsigned int seen[kThreads / 64];
    unsigned int before = 0;
    for (int i0 = 0; i0 < r.n; i0 += kThreads) {
        const bool is = i0 + tid < r.n && order_key(r.l[i0 + tid]) == key;
        const uint64_t m = __builtin_amdgcn_ballot_w64(is);
        __syncthreads();
        if ((tid & 63) == 0) seen[tid >> 6] = __builtin_popcountll(m);
        __syncthreads();
        unsigned int n = before, all = before;
        for (int j = 0; j < kThreads / 64; ++j) {
            n += j < (tid >> 6) ? seen[j] : 0;
            all += seen[j];
        }
        n += __builtin_popcountll(m & ((1ull << (tid & 63)) - 1));
        if (is && n == nth) a.ids[row] = i0 + tid;
        before = all;
        if (before > nth) break;  // uniform
    }
}

}  // namespace

hipError_t launch_sample(const SampleRows &rows, int n_rows, hipStream_t st) {
    int bits = 62;
    for (int n = 1; n < rows.n_vocab; n <<= 1) --bits;
    sample_row_kernel<<<n_rows, kThreads, 0, st>>>(rows, ldexp(1.0, bits < 52 ? bits : 52));
    return hipGetLastError();
}

}  // namespace rxq4
