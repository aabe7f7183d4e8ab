// Host-side launchers of what a serving step needs beside the attention: pages of the requests, ancestor masks, the
// acceptance of a drafted tree (ftq_spec.cuh) and the processing of logits (ftq_logits.cuh).
#pragma once

#include "ftq_common.cuh"

namespace ftq {

constexpr int kTreeMaxNodes = 256;      // nodes of a tree
constexpr int kPagesMaxRequests = 8192; // requests of a page table
constexpr int kLogitSegment = 2048;     // tokens of the vocabulary a CTA takes

struct PagesParams {
    int32_t* table;         // [R, max_blocks]
    int32_t* lens;          // [R]
    int32_t* free_blocks;   // [num_blocks], the first *n_free are free
    int32_t* n_free;
    const int32_t* arg;     // [R] new tokens (extend) or tokens that stay (trim)
    int R, max_blocks, num_blocks;
    // extend
    int64_t* slots;         // [R, width] or, packed, [width]
    int32_t *granted, *starts;   // [R], [R + 1]
    int width;
    bool packed;
};

struct MaskParams {
    const int32_t *parents, *tree_lens, *context_lens;   // [B, T], [B] or NULL, [B] or NULL
    int32_t *masks, *positions;                          // [B, T, W], [B, T]
    int B, T;
};

struct CommitParams {
    const int32_t *block_table, *seq_lens, *tree_lens;    // [B, max_blocks], [B] with the tree, [B] or NULL
    const int32_t *tokens, *parents, *next;               // [B, T]
    int32_t *path, *n_accepted, *out_tokens, *new_lens;   // [B, T], [B], [B, T], [B]
    uint8_t* pool;
    int64_t layer_stride, num_blocks;
    int B, T, max_blocks, Hkv, n_layers, pdk, pdv, page_bytes;
};

struct LogitParams {
    const void* logits;                    // [R * T] rows, row_stride elements apart
    int64_t row_stride;
    const int32_t *history, *history_lens, *prompt_lens;   // [R, H], [R], [R] or NULL (no prompt)
    const float *repetition, *frequency, *presence;        // [R] or NULL
    const int32_t* bias_ids;               // [R, K], negative: none
    const float* bias;
    const uint8_t* allowed;                // [R * T, allowed_stride bytes], bit v % 8 of byte v / 8
    int64_t allowed_stride;
    const int32_t *tree_tokens, *tree_masks;   // [R, T], [R, T, W]
    float* out;                            // [R * T, V] or NULL
    unsigned long long* keys;              // [R * T, segments] or NULL
    int R, T, V, H, K, segments, rows_per_cta;
};

cudaError_t launch_pages_extend(const PagesParams& p, cudaStream_t stream);
cudaError_t launch_pages_trim(const PagesParams& p, cudaStream_t stream);
cudaError_t launch_tree_masks(const MaskParams& p, cudaStream_t stream);
cudaError_t launch_tree_commit(const CommitParams& p, cudaStream_t stream);
cudaError_t launch_logits(int dtype, LogitParams p, int32_t* best, cudaStream_t stream);

}  // namespace ftq
