// Instantiates tree attention for one head_dim (FTQ_D) and key width (FTQ_BK); FTQ_D = 0: the merge kernels.
#include "ftq_tree_launch.h"

#if !defined(FTQ_D)
#error "compile with -DFTQ_D=64, 128 or 256 and -DFTQ_BK=2, 3 or 4, or with -DFTQ_D=0"
#endif
#define FTQ_CAT4(a, b, c, d) a##b##c##d
#define FTQ_CAT(a, b, c, d) FTQ_CAT4(a, b, c, d)

namespace ftq {

#if FTQ_D > 0
template <int BV, int N>
static cudaError_t run_tree(const TreeAttnParams& p, int grid, cudaStream_t stream) {
    using C = TreeCfg<FTQ_D, FTQ_BK, BV, N>;
    constexpr auto kern = tree_attn_kernel<FTQ_D, FTQ_BK, BV, N>;
    const cudaError_t e = allow_smem<kern>(C::SMEM_BYTES);
    return e != cudaSuccess ? e : launch_dependent(kern, dim3(grid), C::THREADS, C::SMEM_BYTES, stream, p);
}

template <int BV>
static cudaError_t tree_by_rows(int n, const TreeAttnParams& p, int grid, cudaStream_t stream) {
    switch (n) {
        case 16: return run_tree<BV, 16>(p, grid, stream);
        case 32: return run_tree<BV, 32>(p, grid, stream);
        case 64: return run_tree<BV, 64>(p, grid, stream);
#if FTQ_D != 256
        case 128: return run_tree<BV, 128>(p, grid, stream);
#endif
    }
    return cudaErrorInvalidValue;
}

// FTQ_ONLY_BITS=<b>: bits_v = b only (the wait-expiry test library)
cudaError_t FTQ_CAT(launch_tree_attn_d, FTQ_D, _k, FTQ_BK)(int bits_v, int n, const TreeAttnParams& p, int grid, cudaStream_t stream) {
#ifdef FTQ_ONLY_BITS
    if (bits_v == FTQ_ONLY_BITS) return tree_by_rows<FTQ_ONLY_BITS>(n, p, grid, stream);
#else
    switch (bits_v) {
        case 2: return tree_by_rows<2>(n, p, grid, stream);
        case 3: return tree_by_rows<3>(n, p, grid, stream);
        case 4: return tree_by_rows<4>(n, p, grid, stream);
    }
#endif
    return cudaErrorInvalidValue;
}
#else
template <int D, typename OT>
static cudaError_t run_merge(const TreeMergeParams& p, cudaStream_t stream) {
    const int64_t rows = static_cast<int64_t>(p.B) * p.T * p.Hq;
    // (a warp per row where there are few, an octet where there are many)
    if (rows <= static_cast<int64_t>(kWideMerge) * sm_count())
        return launch_dependent(tree_merge_kernel<D, OT, 4>, dim3(static_cast<unsigned>((rows + 3) / 4)), 128, 0, stream, p);
    return launch_dependent(tree_merge_kernel<D, OT, 1>, dim3(static_cast<unsigned>((rows + 15) / 16)), 128, 0, stream, p);
}
template <int D>
static cudaError_t merge_by_type(int out_dtype, const TreeMergeParams& p, cudaStream_t stream) {
    switch (out_dtype) {
        case kF32: return run_merge<D, float>(p, stream);
        case kF16: return run_merge<D, __half>(p, stream);
        case kBF16: return run_merge<D, __nv_bfloat16>(p, stream);
    }
    return cudaErrorInvalidValue;
}
cudaError_t launch_tree_merge(int head_dim, int out_dtype, const TreeMergeParams& p, cudaStream_t stream) {
    return head_dim == 64 ? merge_by_type<64>(out_dtype, p, stream) : head_dim == 128 ? merge_by_type<128>(out_dtype, p, stream)
                                                                                     : merge_by_type<256>(out_dtype, p, stream);
}
#endif

}  // namespace ftq
