// attn_paged.h -- the arguments of the paged attention kernels: 16 query rows a
// workgroup (attn_paged.hip) and 128 (attn_paged_block.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "launch.h"

namespace rxq4 {

struct PagedParams {
    uint16_t *out;
    const uint16_t *q;
    float *part, *stats;  // partials: O pieces; (maximum in log2 units, sum)
    SeqBatch b;
    PagedCache c;
    int n_heads, group;
    float sl2;            // scale * log2(e)
    int rows_limit;       // sequences of at most this many rows are the 16-row kernel's (0: none)
    int rows_blk;         // 16 rows: rows of a sequence that the partials hold
    int n_chunks;         // chunks of a sequence's or block's positions at most
    int max_units;        // chunks of the batch per KV head, about (16 rows) or at most
    int min_tiles;        // steps (16 rows) or tiles of a chunk at least
    int *firsts;          // 16 rows: a sequence's first slot and its chunks, for the combine
    int chunk;            // 16 rows: positions per chunk where the host cuts them
    int most_tiles;       // 128 rows: tiles of a block at most
    int *chunk_tiles;     // 128 rows: tiles of a chunk, left for the combine
};

// sum + w x, x a part relative to its own maximum and w its weight beside the other
// parts.  Infinities and NaN (a V that is none, seen by the row) stay what they are where
// w is below fp32's range: their weight is never 0.
__device__ __forceinline__ float add_weighed(float sum, float w, float x) {
    return __builtin_fmaf(fabsf(x) < INFINITY ? w : 1.0f, x, sum);
}

// Query rows of a workgroup of the smaller and of the larger kernel.
constexpr int kPagedRows = 16, kPagedBlock = 128;

// Sequences of more than rows_limit rows (new tokens x group), 128 rows a
// workgroup; partials within `room` bytes at `ws` (null: no split).
struct PagedBlockPlan {
    int units, n_chunks, tiles;
    int64_t grid;  // workgroups
    size_t bytes;  // of partials
};
PagedBlockPlan plan_paged_blocks(const PagedParams &p, size_t room);
// (more workgroups than this are refused)
constexpr int64_t kPagedMostRows = 0x7FFFFF, kPagedMostBlocks = 0x3FFFFF;
hipError_t launch_paged_blocks(PagedParams p, const PagedBlockPlan &plan, float *ws, int kv_int8, hipStream_t st);

}  // namespace rxq4
