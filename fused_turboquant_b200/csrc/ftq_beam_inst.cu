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
    const int rounds = ((p.chunk * static_cast<int>(sizeof(T)) + 15) / 16 + kSelectThreads - 1) / kSelectThreads;
    const int rows_smem = 8 * select_pow2(std::max({kSelectRoom, p.keep * rounds, p.keep * 16 / static_cast<int>(sizeof(T))}));
    const int join_smem = 16 * std::max(kSelectRoom, select_join_size(p.K, p.chunks, p.keep, p.n));
    cudaError_t e = allow_smem<beam_join_kernel<T, 512>>(16 * kSelectJoin);
    if (e != cudaSuccess) return e;
    const int64_t ctas = static_cast<int64_t>(p.R) * p.K * p.chunks;
    e = launch_dependent(beam_rows_kernel<T>, dim3(static_cast<unsigned>(ctas)), kSelectThreads, rows_smem, stream, p);
    if (e != cudaSuccess) return e;
    // (8 requests of eight beams, 2300 tokens each: 20 us with 256 threads, 15 with 512; 64 requests of 576 42 and 44)
    if (static_cast<int64_t>(p.K) * p.chunks * p.keep > kJoinFew)
        return launch_dependent(beam_join_kernel<T, 512>, dim3(p.R), 512, join_smem, stream, p);
    return launch_dependent(beam_join_kernel<T, 256>, dim3(p.R), 256, join_smem, stream, p);
}
static_assert(8 * select_pow2(kSelectMaxKeep * kSelectVectors) <= 48 * 1024, "shared memory of beam_rows_kernel");

}  // namespace

// A CTA's part of a row is as long as its threads' vectors can be sorted, at most, and a vector a thread at least (shorter ones leave more
// to be joined than they save).  In between, the number of parts that gives the shortest schedule: rounds of five CTAs an SM, of which
// each costs its vectors and, for the threshold and the tokens that reach it, as much as 1024 more; and the request's CTA of
// beam_join_kernel about one for each token that it gets.  (Eight beams of 131072 bf16 logits, in a graph: 2, 8, 16 and 64 requests 49,
// 35, 29 and 42 us in parts that fill 12 CTAs an SM; 12, 15, 18 and 42 now.)
SelectPlan select_plan(int dtype, int requests, int beams, int vocab, int keep) {
    const int n = dtype == kF32 ? 4 : 8;
    const int64_t most = (kSelectVectors * kSelectThreads - 1) * n, least = std::min<int64_t>(kSelectThreads * n, vocab);
    const int64_t rows = std::max<int64_t>(1, static_cast<int64_t>(requests) * beams), slots = 5 * sm_count();
    auto chunk_of = [&](int64_t chunks) { return std::min(most, (std::max((vocab + chunks - 1) / chunks, least) + n - 1) / n * n); };
    int64_t chunk = 0, cost = 0;
    const int64_t lo = (vocab + most - 1) / most, hi = std::max<int64_t>(lo, (vocab + least - 1) / least);
    for (int64_t chunks = lo; chunks <= std::min(hi, lo + 64); chunks++) {
        const int64_t c = chunk_of(chunks), all = rows * ((vocab + c - 1) / c), t = (all + slots - 1) / slots * (c / n + 1024) + beams * ((vocab + c - 1) / c) * keep;
        if (chunk == 0 || t < cost) {
            cost = t;
            chunk = c;
        }
    }
    return {static_cast<int>((vocab + chunk - 1) / chunk), static_cast<int>(chunk)};
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
