// Instantiates attention with common leading blocks for one head_dim (FTQ_D) and key width (FTQ_BK); FTQ_D = 0: the kernels before
// and behind it.
#include <algorithm>

#include "ftq_launch.h"
#include "ftq_shared_attn.cuh"

#if !defined(FTQ_D)
#error "compile with -DFTQ_D=64, 128 or 256 and -DFTQ_BK=2, 3 or 4, or with -DFTQ_D=0"
#endif
#define FTQ_CAT4(a, b, c, d) a##b##c##d
#define FTQ_CAT(a, b, c, d) FTQ_CAT4(a, b, c, d)

namespace ftq {

#if FTQ_D > 0
template <int BV, int NT>
static cudaError_t run_shared(const SharedAttnParams& p, int grid, cudaStream_t stream) {
    using C = SharedCfg<FTQ_D, FTQ_BK, BV, NT>;
    constexpr auto kern = shared_attn_kernel<FTQ_D, FTQ_BK, BV, NT>;
    const cudaError_t e = allow_smem<kern>(C::SMEM_BYTES);
    return e != cudaSuccess ? e : launch_dependent(kern, dim3(grid), C::THREADS, C::SMEM_BYTES, stream, p);
}

template <int BV>
static cudaError_t shared_by_tiles(int tiles, const SharedAttnParams& p, int grid, cudaStream_t stream) {
    constexpr int LEAST = shared_least_tiles(FTQ_D), MOST = shared_most_tiles(FTQ_D);
    if (tiles == LEAST) return run_shared<BV, LEAST>(p, grid, stream);
    if (tiles == MOST) return run_shared<BV, MOST>(p, grid, stream);
    if constexpr (2 * LEAST < MOST)
        if (tiles == 2 * LEAST) return run_shared<BV, 2 * LEAST>(p, grid, stream);
    return cudaErrorInvalidValue;
}

// FTQ_ONLY_BITS=<b>: bits_v = b only (the wait-expiry test library)
cudaError_t FTQ_CAT(launch_shared_attn_d, FTQ_D, _k, FTQ_BK)(int bits_v, int tiles, const SharedAttnParams& p, int grid, cudaStream_t stream) {
#ifdef FTQ_ONLY_BITS
    if (bits_v == FTQ_ONLY_BITS) return shared_by_tiles<FTQ_ONLY_BITS>(tiles, p, grid, stream);
#else
    switch (bits_v) {
        case 2: return shared_by_tiles<2>(tiles, p, grid, stream);
        case 3: return shared_by_tiles<3>(tiles, p, grid, stream);
        case 4: return shared_by_tiles<4>(tiles, p, grid, stream);
    }
#endif
    return cudaErrorInvalidValue;
}
#else
template <int D>
static cudaError_t run_prepare(const SharedAttnParams& p, cudaStream_t stream) {
    const int64_t rows = static_cast<int64_t>(p.R) * p.K * p.Hq;
    const int ctas = static_cast<int>(std::min<int64_t>((rows + 31) / 32, 2 * sm_count()));
    return launch_dependent(shared_prepare_kernel<D>, dim3(1 + ctas), 256, 0, stream, p);
}
cudaError_t launch_shared_prepare(int head_dim, const SharedAttnParams& p, cudaStream_t stream) {
    return head_dim == 64 ? run_prepare<64>(p, stream) : head_dim == 128 ? run_prepare<128>(p, stream) : run_prepare<256>(p, stream);
}

template <int D, typename OT>
static cudaError_t run_merge(const SharedAttnParams& p, cudaStream_t stream) {
    const int64_t rows = static_cast<int64_t>(p.R) * p.K * p.Hq;
    if (rows <= 2 * static_cast<int64_t>(kWideMerge) * sm_count())
        return launch_dependent(shared_merge_kernel<D, OT, 4>, dim3(static_cast<unsigned>(rows)), 128, 0, stream, p);
    return launch_dependent(shared_merge_kernel<D, OT, 1>, dim3(static_cast<unsigned>((rows + 3) / 4)), 128, 0, stream, p);
}
template <int D>
static cudaError_t merge_by_type(int out_dtype, const SharedAttnParams& p, cudaStream_t stream) {
    switch (out_dtype) {
        case kF32: return run_merge<D, float>(p, stream);
        case kF16: return run_merge<D, __half>(p, stream);
        case kBF16: return run_merge<D, __nv_bfloat16>(p, stream);
    }
    return cudaErrorInvalidValue;
}
cudaError_t launch_shared_merge(int head_dim, int out_dtype, const SharedAttnParams& p, cudaStream_t stream) {
    return head_dim == 64 ? merge_by_type<64>(out_dtype, p, stream) : head_dim == 128 ? merge_by_type<128>(out_dtype, p, stream)
                                                                                     : merge_by_type<256>(out_dtype, p, stream);
}
#endif

}  // namespace ftq
