// Host-side launchers of attention with common leading blocks (ftq_shared_attn.cuh), one translation unit per head_dim and key
// width; one more for the kernels before and behind it.
#pragma once

#include "ftq_common.cuh"

namespace ftq {

constexpr int kSharedMaxRows = 1024;    // rows of one launch (more are several)
constexpr int kSharedPiece = 40;        // places of a unit besides those of its pages
constexpr int kSharedMaxWarps = 16;     // of a CTA
// Tiles of eight columns that a warp keeps O of: at most 128 registers of it.
constexpr int shared_most_tiles(int head_dim) { return head_dim == 256 ? 2 : 4; }
constexpr int shared_least_tiles(int head_dim) { return head_dim == 64 ? 2 : 1; }

// Shared memory of a CTA from `base` on: the 64 KB window of the tables on a boundary of its size; before and behind it, first-fit,
// the warps' rings and queries, then the plan.
constexpr int kSharedPlanBytes = (2 * kSharedMaxRows + 8) * 4, kSharedSmemLimit = 226 * 1024;
constexpr int shared_ring_bytes(int page_bytes, int ring) { return (ring * page_bytes + 127) / 128 * 128; }
constexpr int shared_smem_from(int base, int warps, int ring_bytes, int q_bytes) {
    int free0 = base, free1 = (base + 65535) / 65536 * 65536;
    const int end0 = free1;
    free1 += 65536;
    for (int i = 0; i < 2 * warps + 1; i++) {
        const int bytes = i < warps ? ring_bytes : i < 2 * warps ? q_bytes : kSharedPlanBytes;
        const int a0 = (free0 + 127) / 128 * 128;
        if (a0 + bytes <= end0) free0 = a0 + bytes;
        else free1 = (free1 + 127) / 128 * 128 + bytes;
    }
    return (free1 > free0 ? free1 : free0) - base;
}
// (wherever the dynamic part starts in the first 4 KB)
constexpr int shared_smem(int warps, int ring_bytes, int q_bytes) {
    int worst = shared_smem_from(0, warps, ring_bytes, q_bytes);
    for (int base = 16; base <= 4096; base += 128) {
        const int n = shared_smem_from(base, warps, ring_bytes, q_bytes);
        worst = n > worst ? n : worst;
    }
    return worst;
}
// Warps of a CTA: as many as the registers of O leave room for (8 of 255, 12 of 168, 16 of 128) and shared memory with two pages
// on their way each.
struct SharedShape { int warps, ring, smem; };
constexpr SharedShape shared_shape(int head_dim, int page_bytes, int tiles) {
    const int o = tiles * head_dim / 4, q_bytes = 8 * tiles * head_dim * 2;
    int warps = o > 64 ? 8 : o > 32 ? 12 : 16;
    while (shared_smem(warps, shared_ring_bytes(page_bytes, 2), q_bytes) > kSharedSmemLimit) warps -= 2;
    const int ring = shared_smem(warps, shared_ring_bytes(page_bytes, 4), q_bytes) <= kSharedSmemLimit ? 4 : 2;
    return {warps, ring, shared_smem(warps, shared_ring_bytes(page_bytes, ring), q_bytes)};
}

struct SharedAttnParams {
    const void* q;               // [R * K, Hq, D]
    const uint8_t* pool;         // of the layer
    int64_t num_blocks;
    const int32_t *block_table, *seq_lens, *shared_lens;   // [R * K, max_blocks], [R * K], [R]
    int max_blocks, max_seq, R, K, Hq, Hkv, q_dtype;
    void* out;
    // units of an entry, of a KV head; their columns' rows in the workspace; places of a page; columns of a unit
    int units_group, units_row, blocks_group, blocks_row, rows_group, rows_row, cost_group, cost_row, cols;
    int warps;                   // of the grid
    int *plan, *plan_unit, *plan_tokens, *plan_leader;
    FastDiv by_hq, by_group, by_rows, by_cols, by_cost_group, by_cost_row;      // Hq, Hq / Hkv, K, cols, places of a page
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
    cudaError_t launch_shared_attn_d##DD##_k##KB(int bits_v, int tiles, const SharedAttnParams& p, int grid, cudaStream_t stream);
FTQ_DECLARE_SHARED(64, 2) FTQ_DECLARE_SHARED(64, 3) FTQ_DECLARE_SHARED(64, 4)
FTQ_DECLARE_SHARED(128, 2) FTQ_DECLARE_SHARED(128, 3) FTQ_DECLARE_SHARED(128, 4)
FTQ_DECLARE_SHARED(256, 2) FTQ_DECLARE_SHARED(256, 3) FTQ_DECLARE_SHARED(256, 4)
cudaError_t launch_shared_prepare(int head_dim, const SharedAttnParams& p, cudaStream_t stream);
cudaError_t launch_shared_merge(int head_dim, int out_dtype, const SharedAttnParams& p, cudaStream_t stream);

}  // namespace ftq
