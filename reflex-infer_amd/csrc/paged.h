// paged.h -- where the tokens of a batch and the positions of a paged cache lie:
// device helpers shared by the serving kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "launch.h"

namespace rxq4 {

// A wave's LDS accesses stay in order between its lanes.
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// One sequence of a batch: rows [row0, row0 + n) of q, the first at position
// pos0 (negative where seq_lens is below the new tokens).  Whatever the device
// arrays hold, the rows lie within [0, n_tokens) and no sum of theirs overflows.
struct SeqSpan {
    int row0, n, pos0;
};
__device__ __forceinline__ SeqSpan seq_span(const SeqBatch &b, int start, int end, int len) {
    const int a = min(max(start, 0), b.n_tokens);
    const int e = min(max(end, a), b.n_tokens);
    return SeqSpan{a, e - a, max(len, -(1 << 30)) - (e - a)};
}
__device__ __forceinline__ SeqSpan seq_span(const SeqBatch &b, int s) {
    return seq_span(b, b.starts[s], b.starts[s + 1], b.lens[s]);
}

// x summed over the lanes up to this one, on the VALU: shifts within rows of 16
// lanes, then each row's last lane added to the rows behind it.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add_from(int x) {
    return x + __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int wave_prefix(int x) {
    x = dpp_add_from<0x111, 0xF>(x);  // row_shr:1
    x = dpp_add_from<0x112, 0xF>(x);
    x = dpp_add_from<0x114, 0xF>(x);
    x = dpp_add_from<0x118, 0xF>(x);
    x = dpp_add_from<0x142, 0xA>(x);  // row_bcast:15 into rows 1 and 3
    return dpp_add_from<0x143, 0xC>(x);  // row_bcast:31 into rows 2 and 3
}

// The sequence that row t belongs to (n_seqs: none) and its rows, the same for a
// whole wave: the number of sequences that end at or before t, 64 parts at a time.
// Of the last 64 a lane loads all of one at once: a round trip to memory for up to 64
// sequences, two for up to 4096.
__device__ __forceinline__ int seq_of_row(const SeqBatch &b, int t, SeqSpan &span) {
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int part = b.n_seqs > 4096 ? 4096 : b.n_seqs > 64 ? 64 : 1; part > 1; part >>= 6) {
        const int end = base + (lane + 1) * part;
        const bool ends = end <= b.n_seqs && b.starts[end] <= t;
        base += part * __builtin_popcountll(__builtin_amdgcn_ballot_w64(ends));
    }
    const int j = min(base + lane, b.n_seqs - 1);
    const int start = b.starts[j], end = b.starts[j + 1], len = b.lens[j];
    const int n = __builtin_popcountll(__builtin_amdgcn_ballot_w64(base + lane < b.n_seqs && end <= t));
    if (n == 64 || base + n >= b.n_seqs) return b.n_seqs;
    span = seq_span(b, __builtin_amdgcn_readlane(start, n), __builtin_amdgcn_readlane(end, n),
                    __builtin_amdgcn_readlane(len, n));
    return __builtin_amdgcn_readfirstlane(base + n);
}

// Positions that the batch's tokens may see or store: below the table's end.
__device__ __forceinline__ int position_limit(const SeqBatch &b, const PagedCache &c) {
    return (int)min((int64_t)b.max_len, (int64_t)c.width << c.shift);
}

// The slot (page * page_size + place) of position pos < position_limit of
// sequence s, -1 in a hole.  Slots are below 2^31.
__device__ __forceinline__ int slot_of(const PagedCache &c, int s, int pos) {
    const int i = pos >> c.shift;
    const int page = c.table ? c.table[(int64_t)s * c.width + i] : i;
    return (unsigned)page < (unsigned)c.n_pages ? (page << c.shift) + (pos & ((1 << c.shift) - 1)) : -1;
}

// Bytes from the cache's base to a slot's row of `row_bytes`.
__device__ __forceinline__ int64_t slot_bytes(const PagedCache &c, int slot, int row_bytes) {
    return (int64_t)(slot >> c.shift) * c.page_bytes + (int64_t)(slot & ((1 << c.shift) - 1)) * row_bytes;
}

}  // namespace rxq4
