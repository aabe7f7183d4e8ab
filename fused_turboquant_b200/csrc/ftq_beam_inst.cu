// Kernels and launchers of ftq_beam.cuh and ftq_select.cuh.
#include <algorithm>

#include "ftq_beam.cuh"
#include "ftq_launch.h"
#include "ftq_serve_launch.h"
#include "ftq_select.cuh"

namespace ftq {
namespace {

template <typename T>
cudaError_t run_select(const SelectParams& p, cudaStream_t stream) {
    // what the sorts need (the tokens that are ranked by counting are fewer)
    const int rounds = ((p.chunk * static_cast<int>(sizeof(T)) + 15) / 16 + 1 + kSelectThreads - 1) / kSelectThreads;
    const int rows_smem = 8 * select_pow2(std::max({kSelectRoom, p.keep * rounds, p.keep * 16 / static_cast<int>(sizeof(T))}));
    const int join_smem = 16 * std::max(kSelectRoom, select_join_size(p.K, p.chunks, p.keep, p.n));
    cudaError_t e = allow_smem<beam_join_kernel<T>>(16 * kSelectJoin);
    if (e != cudaSuccess) return e;
    const int64_t ctas = static_cast<int64_t>(p.R) * p.K * p.chunks;
    e = launch_dependent(beam_rows_kernel<T>, dim3(static_cast<unsigned>(ctas)), kSelectThreads, rows_smem, stream, p);
    if (e != cudaSuccess) return e;
    return launch_dependent(beam_join_kernel<T>, dim3(p.R), kSelectThreads, join_smem, stream, p);
}
static_assert(8 * select_pow2(kSelectMaxKeep * kSelectVectors) <= 48 * 1024, "shared memory of beam_rows_kernel");

}  // namespace

// A CTA's part of a row is as long as its threads' vectors can be looked at again, and as short as fills the device where there are
// few rows, but at least a vector a thread (shorter ones leave more to be joined than they save).
SelectPlan select_plan(int dtype, int requests, int beams, int vocab, int keep) {
    const int n = dtype == kF32 ? 4 : 8, most = (kSelectVectors * kSelectThreads - 1) * n, least = kSelectThreads * n;
    const int64_t rows = static_cast<int64_t>(requests) * beams, want = 12 * sm_count();
    int64_t chunks = std::max<int64_t>((static_cast<int64_t>(vocab) + most - 1) / most, rows > 0 ? (want + rows - 1) / rows : 1);
    int64_t chunk = std::max<int64_t>((vocab + chunks - 1) / chunks, std::min(least, vocab));
    chunk = std::min<int64_t>((chunk + n - 1) / n * n, most);
    chunks = (vocab + chunk - 1) / chunk;
    return {static_cast<int>(chunks), static_cast<int>(chunk)};
}

cudaError_t launch_select(int dtype, const SelectParams& p, cudaStream_t stream) {
    return dtype == kF32 ? run_select<float>(p, stream) : dtype == kF16 ? run_select<__half>(p, stream) : run_select<__nv_bfloat16>(p, stream);
}

namespace {
// a cluster of all CTAs, or a single one
template <auto kern, typename P>
cudaError_t run_fork(const P& p, bool little, int smem, int most_smem, cudaStream_t stream) {
    if (most_smem > 48 * 1024) {
        const cudaError_t e = allow_smem<kern>(most_smem);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(little ? 1 : kForkCtas);
    cfg.blockDim = dim3(kForkThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attrs[2]{};
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = kForkCtas;
    attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
    cfg.attrs = attrs;
    cfg.numAttrs = little ? 1 : 2;
    return cudaLaunchKernelEx(&cfg, kern, p);
}
}  // namespace

// One CTA where its warps keep all entries in shared memory; a few thousand blocks.
cudaError_t launch_pages_fork(const ForkParams& p, cudaStream_t stream) {
    const int64_t items = static_cast<int64_t>(p.R) * ((p.max_blocks + kForkSpan - 1) / kForkSpan);
    return run_fork<pages_fork_kernel>(p, items <= kForkThreads / 32 * kForkKept, fork_smem(p.R), fork_smem(kPagesMaxRequests), stream);
}
cudaError_t launch_pages_compact(const CompactParams& p, cudaStream_t stream) {
    return run_fork<pages_compact_kernel>(p, p.num_blocks <= 4 * kForkThreads && static_cast<int64_t>(p.R) * p.max_blocks <= 16 * kForkThreads, 0, 0, stream);
}
cudaError_t launch_shared_lens(const SharedLensParams& p, cudaStream_t stream) {
    return launch_dependent(shared_lens_kernel, dim3(p.groups), 256, 0, stream, p);
}

cudaError_t launch_copy_pages(const CopyPagesParams& p, cudaStream_t stream) {
    // eight CTAs an SM, by pairs first, then by parts of a block (2 KB at least, a load of each half of the threads)
    const int64_t want = 8 * sm_count();
    const int x = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(p.n, (want + p.n_layers - 1) / p.n_layers)));
    const int64_t parts = std::min<int64_t>(want / (static_cast<int64_t>(x) * p.n_layers), p.block_bytes / 2048);
    return launch_dependent(copy_pages_kernel, dim3(x, p.n_layers, static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>(parts, 64)))),
                            kCopyThreads, 0, stream, p);
}

}  // namespace ftq
