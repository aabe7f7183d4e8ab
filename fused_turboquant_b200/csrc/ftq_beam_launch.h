// Host-side launchers of beam search and parallel sampling on the paged cache (ftq_beam.cuh, ftq_select.cuh): rows of a
// page table that become copies of others, blocks that are moved and copied, the best continuations of beams.
#pragma once

#include "ftq_common.cuh"

namespace ftq {

constexpr int kBeamMax = 64;        // beams of a request, continuations that are selected
constexpr int kBeamMaxEnds = 16;    // tokens that end an answer
constexpr int kForkWarps = 128;     // warps of a fork or compaction: 8 CTAs of 16

struct ForkParams {
    int32_t* table;         // [R, max_blocks]
    int32_t* lens;          // [R]
    int32_t* free_blocks;   // [num_blocks], the first *n_free are free
    int32_t* n_free;
    int32_t* shares;        // [num_blocks]: rows that hold a block besides the first of them
    const int32_t *parents, *keep;   // [R], [R] or NULL
    int R, max_blocks, num_blocks, group;
    int32_t* copies;        // [R, 2]
    int32_t* done;          // [1]
    // scratch: the new table; counts of the warps and the rows that need a block; ranks of those; two marks per block
    int32_t *next, *counts, *ranks, *part_count, *part_first;
};

struct CompactParams {
    int32_t *table, *free_blocks, *n_free, *shares;   // shares NULL: no block has several holders
    const int32_t* lens;
    int R, max_blocks, num_blocks;
    int32_t* copies;        // [num_blocks / 2, 2]
    int32_t *map, *counts;  // scratch: [num_blocks], [2 * 8]
};

struct SharedLensParams {
    const int32_t *table, *lens;
    int32_t* out;           // [groups]
    int groups, group, max_blocks;
};

struct CopyPagesParams {
    uint8_t* pool;
    const int32_t* copies;  // [n, 2]
    int64_t layer_stride, block_bytes, num_blocks;
    int n, n_layers;
};

struct SelectParams {
    const void* logits;     // rows [requests * beams], row_stride elements apart
    int64_t row_stride;
    const float* scores;    // [requests, beams]
    const int32_t* ends;    // [n_ends]
    float* out_scores;      // [requests, n]
    int32_t *parents, *tokens;
    float* end_scores;      // [requests, beams, n_ends]
    float2* sums;           // scratch [rows, chunks]: (maximum, sum of exponentials) of a chunk
    unsigned long long* keys;   // scratch [rows, chunks, keep]: the chunk's largest, in order
    int R, K, V, n, n_ends, keep, chunks, chunk;
};

// chunks of a row, and the size of one in tokens
struct SelectPlan { int chunks, chunk; };
SelectPlan select_plan(int dtype, int requests, int beams, int vocab, int keep);

cudaError_t launch_pages_fork(const ForkParams& p, cudaStream_t stream);
cudaError_t launch_pages_compact(const CompactParams& p, cudaStream_t stream);
cudaError_t launch_shared_lens(const SharedLensParams& p, cudaStream_t stream);
cudaError_t launch_copy_pages(const CopyPagesParams& p, cudaStream_t stream);
cudaError_t launch_select(int dtype, const SelectParams& p, cudaStream_t stream);

}  // namespace ftq
