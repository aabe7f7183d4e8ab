// Host-side launchers of attention with common leading blocks (ftq_shared_attn.cuh), one translation unit per head_dim and key
// width; one more for the kernels before and behind it.
#pragma once

#include "ftq_common.cuh"

namespace ftq {

constexpr int kSharedWarps = 8;         // of a CTA
constexpr int kSharedMaxRows = 1024;    // rows of one launch (more are several)
constexpr int kSharedPiece = 40;        // places of a unit besides those of its pages
// tiles of eight columns of a product: what the registers hold of O
constexpr int shared_tiles(int head_dim) { return head_dim == 256 ? 2 : 4; }

struct SharedAttnParams {
    const void* q;               // [R * K, Hq, D]
    const uint8_t* pool;         // of the layer
    int64_t num_blocks;
    const int32_t *block_table, *seq_lens, *shared_lens;   // [R * K, max_blocks], [R * K], [R]
    int max_blocks, max_seq, R, K, Hq, Hkv, q_dtype;
    void* out;
    // units of a KV head and head block, their columns' rows in the workspace, places of a page
    int units_group, units_row, rows_group, rows_row, cost_group, cost_row, cols;
    int warps, least_pages;      // of the grid; of a piece
    int *plan, *plan_tokens, *plan_leader;
    uint8_t* q_rows;             // fp16 [R, Hkv, K * G, D]
    float* rows;                 // (O, m, l) [D + 4]: the groups' pieces, from base_row on those of single rows
    int64_t base_row;
    int* status;
    int first;                   // the call's first launch: the status starts with it
    Codebook lk, lv;
    float inv_v_scale, q_scale, rsqrt_d;
    SignBits signs;
};

#define FTQ_DECLARE_SHARED(DD, KB) \
    cudaError_t launch_shared_attn_d##DD##_k##KB(int bits_v, const SharedAttnParams& p, int grid, cudaStream_t stream);
FTQ_DECLARE_SHARED(64, 2) FTQ_DECLARE_SHARED(64, 3) FTQ_DECLARE_SHARED(64, 4)
FTQ_DECLARE_SHARED(128, 2) FTQ_DECLARE_SHARED(128, 3) FTQ_DECLARE_SHARED(128, 4)
FTQ_DECLARE_SHARED(256, 2) FTQ_DECLARE_SHARED(256, 3) FTQ_DECLARE_SHARED(256, 4)
cudaError_t launch_shared_prepare(int head_dim, const SharedAttnParams& p, cudaStream_t stream);
cudaError_t launch_shared_merge(int head_dim, int out_dtype, const SharedAttnParams& p, cudaStream_t stream);

}  // namespace ftq
