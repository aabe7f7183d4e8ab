// Kernels and launchers of ftq_spec.cuh and ftq_logits.cuh.
#include <algorithm>

#include "ftq_launch.h"
#include "ftq_logits.cuh"
#include "ftq_spec.cuh"

namespace ftq {
namespace {

// `ctas` CTAs as one cluster (1: none)
template <auto kern>
cudaError_t run_pages(const PagesParams& p, int64_t writes, int smem, cudaStream_t stream) {
    const cudaError_t e = allow_smem<kern>(4 * 4 * kPagesMaxRequests);
    if (e != cudaSuccess) return e;
    int ctas = 1;
    while (ctas < kPagesCluster && writes > static_cast<int64_t>(ctas) * 4 * kPagesThreads) ctas *= 2;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(kPagesThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attrs[2]{};
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = ctas;
    attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
    cfg.attrs = attrs;
    cfg.numAttrs = ctas > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, p);
}

template <typename T>
cudaError_t run_logits(const LogitParams& p, bool vec, dim3 grid, int smem, cudaStream_t stream) {
    const cudaError_t e = vec ? allow_smem<logits_kernel<T, true>>(kLogitSegment * 13) : allow_smem<logits_kernel<T, false>>(kLogitSegment * 13);
    if (e != cudaSuccess) return e;
    return vec ? launch_dependent(logits_kernel<T, true>, grid, kLogitThreads, smem, stream, p)
               : launch_dependent(logits_kernel<T, false>, grid, kLogitThreads, smem, stream, p);
}

}  // namespace

cudaError_t launch_pages_extend(const PagesParams& p, cudaStream_t stream) {
    return run_pages<pages_extend_kernel>(p, p.packed ? p.width : static_cast<int64_t>(p.R) * p.width, 4 * 4 * p.R, stream);
}
cudaError_t launch_pages_trim(const PagesParams& p, cudaStream_t stream) {
    return run_pages<pages_trim_kernel>(p, p.R, 2 * 4 * p.R, stream);
}

cudaError_t launch_tree_masks(const MaskParams& p, cudaStream_t stream) {
    return launch_dependent(tree_masks_kernel, dim3(p.B), (p.T + 31) / 32 * 32, 0, stream, p);
}

cudaError_t launch_tree_commit(const CommitParams& p, cudaStream_t stream) {
    // (a warp per layer and head, fewer where there are more than fill the device several times)
    const int items = (p.n_layers * p.Hkv + kCommitWarps - 1) / kCommitWarps, most = std::max(1, 64 * sm_count() / p.B);
    return launch_dependent(tree_commit_kernel, dim3(std::min(items, most), p.B), 32 * kCommitWarps, 0, stream, p);
}

cudaError_t launch_logits(int dtype, LogitParams p, int32_t* best, cudaStream_t stream) {
    const int es = dtype == kF32 ? 4 : 2;
    auto aligned16 = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; };
    // eight tokens a load where every row begins on 16 bytes and ends with a whole load; else a token a load, coalesced
    const bool vec = p.V % 8 == 0 && aligned16(p.logits) && p.row_stride * es % 16 == 0 && (!p.out || aligned16(p.out));
    // rows of a request that share a count: as few as fill the device (five CTAs an SM) once, and no more than a CTA has room for
    const int64_t ctas = static_cast<int64_t>(p.segments) * p.R, want = 5 * sm_count();
    int chunks = static_cast<int>(ctas >= want ? 1 : std::min<int64_t>(p.T, (want + ctas - 1) / ctas));
    chunks = std::max(chunks, (p.T + kTreeMaxNodes - 1) / kTreeMaxNodes);
    p.rows_per_cta = (p.T + chunks - 1) / chunks;
    chunks = (p.T + p.rows_per_cta - 1) / p.rows_per_cta;
    const dim3 grid(p.segments, p.R, chunks);
    const int smem = kLogitSegment * (p.K > 0 ? 13 : 9);
    cudaError_t e = dtype == kF32 ? run_logits<float>(p, vec, grid, smem, stream)
                    : dtype == kF16 ? run_logits<__half>(p, vec, grid, smem, stream)
                                    : run_logits<__nv_bfloat16>(p, vec, grid, smem, stream);
    if (e != cudaSuccess || !p.keys) return e;
    const int64_t rows = static_cast<int64_t>(p.R) * p.T;
    return launch_dependent(logits_best_kernel, dim3(static_cast<unsigned>((rows + 3) / 4)), 128, 0, stream, p.keys, best, rows, p.segments);
}

}  // namespace ftq
