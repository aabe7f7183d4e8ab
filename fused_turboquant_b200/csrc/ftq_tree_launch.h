// Host-side launchers of tree attention, one translation unit per head_dim and key width (ftq_tree_attn_inst.cu).
#pragma once

#include "ftq_launch.h"
#include "ftq_tree_attn.cuh"

namespace ftq {

// Rows of a product: the node x head rows of a KV head in the narrowest of 16, 32, 64, 128 that holds them (64 is the most
// at head_dim 256, whose O takes twice the TMEM); more than that in row tiles.
inline int tree_rows(int head_dim, int rows) {
    return rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 || head_dim == 256 ? 64 : 128;
}

// (TreeCfg::HALVES)
inline int tree_halves(int head_dim, int n) { return head_dim == 256 || n == 128 ? 1 : 2; }

#define FTQ_DECLARE_TREE(DD, KB) \
    cudaError_t launch_tree_attn_d##DD##_k##KB(int bits_v, int n, const TreeAttnParams& p, int grid, cudaStream_t stream);
FTQ_DECLARE_TREE(64, 2) FTQ_DECLARE_TREE(64, 3) FTQ_DECLARE_TREE(64, 4)
FTQ_DECLARE_TREE(128, 2) FTQ_DECLARE_TREE(128, 3) FTQ_DECLARE_TREE(128, 4)
FTQ_DECLARE_TREE(256, 2) FTQ_DECLARE_TREE(256, 3) FTQ_DECLARE_TREE(256, 4)
cudaError_t launch_tree_merge(int head_dim, int out_dtype, const TreeMergeParams& p, cudaStream_t stream);

}  // namespace ftq
