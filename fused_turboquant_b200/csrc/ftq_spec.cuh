// Speculative serving around the paged cache: pages of the requests, ancestor masks of drafted token trees, and the
// move of the accepted tokens' compressed keys and values.  Integers and bytes only.  All of it is bound by latency
// (launch, dependent loads, the walk down a tree), so every operator is one launch and keeps its state on the device.
// Measured: giving back, taking and the masks together 16.5 us, for one request of 8 nodes as for 256 of 16 or whole prompts of new
// ones, which is what three calls from Python take: in a graph 5.8, 10.2 and 15.2 us.  Accepting and moving 9.0 us for one request of 32
// layers (in a graph 4.8), 11.4 us for 32 (0.6 us of HBM).
#pragma once

#include "ftq_serve_launch.h"

namespace ftq {

// ------------------------------------------------------------------ pages of requests
// State: block table, lengths, a stack of free block ids.  A request of n tokens that gets m more needs
// ceil((n + m) / 16) - ceil(n / 16) further blocks; the running sum of the needs (an exclusive scan over the requests)
// says which entries of the stack are whose.  Trimming is the reverse: the same scan says where the blocks go back, so
// that blocks taken and given back at once leave the stack as it was.
//
// One cluster of up to kPagesCluster CTAs: every CTA makes the scan of all requests for itself (a few loads a thread), the
// slots and table entries are dealt out to all threads, and the state that everybody has read is changed behind a
// cluster barrier.  One CTA where there is little to write.
constexpr int kPagesThreads = 512, kPagesCluster = 8;


// Exclusive scan over the CTA's threads, and the sum of all.
template <typename T>
__device__ __forceinline__ T block_scan(T v, int64_t* warp_sums, T& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    T x = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const T y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
    }
    __syncthreads();        // (the sums of the scan before have been read)
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    T before = 0, all = 0;
    for (int w = 0; w < kPagesThreads / 32; w++) {
        const T s = static_cast<T>(warp_sums[w]);
        before += w < warp ? s : 0;
        all += s;
    }
    total = all;
    return before + x - v;
}

// the last of the n ascending entries that is not above x
__device__ __forceinline__ int last_not_above(const int* a, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ int pages_of(int tokens) { return (tokens + kPageTokens - 1) / kPageTokens; }

__device__ __forceinline__ void cluster_barrier(int ctas) {
    if (ctas > 1) {
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
    } else {
        __syncthreads();
    }
}

__global__ void __launch_bounds__(kPagesThreads) pages_extend_kernel(const PagesParams p) {
    extern __shared__ int s_requests[];
    __shared__ int64_t warp_sums[kPagesThreads / 32];
    __shared__ int s_taken;
    int* const s_off = s_requests;                 // blocks wanted by the requests before
    int* const s_len = s_requests + p.R;           // tokens so far
    int* const s_get = s_requests + 2 * p.R;       // tokens granted, -1: refused
    int* const s_start = s_requests + 3 * p.R;     // packed: first token
    const int tid = threadIdx.x, cta = blockIdx.x, ctas = gridDim.x;
    after_previous_kernel();
    let_next_kernel_start();
    const int room = kPageTokens * p.max_blocks;
    const int avail = min(max(*p.n_free, 0), p.num_blocks);
    if (tid == 0) s_taken = 0;
    int base_off = 0;
    int64_t base_start = 0;     // (of refused requests too, and those may have asked for anything)
    for (int r0 = 0; r0 < p.R; r0 += kPagesThreads) {
        const int r = r0 + tid;
        const bool live = r < p.R;
        const int n = live ? min(max(p.lens[r], 0), room) : 0, m = live ? p.arg[r] : 0;
        int64_t start = 0;
        if (p.packed) {
            int64_t sum;
            start = base_start + block_scan<int64_t>(max(m, 0), warp_sums, sum);
            base_start += sum;
        }
        const bool fits = live && m >= 0 && m <= room - n && m <= p.width - start;
        const int want = fits ? pages_of(n + m) - pages_of(n) : 0;
        int total;
        const int off = base_off + block_scan(want, warp_sums, total);
        base_off += total;
        const bool ok = fits && (want == 0 || off + want <= avail);
        if (live) {
            s_off[r] = off;
            s_len[r] = n;
            s_get[r] = ok ? m : -1;
            if (p.packed) s_start[r] = static_cast<int>(min(start, static_cast<int64_t>(INT32_MAX)));
            if (ok && want > 0) atomicMax(&s_taken, off + want);
        }
    }
    __syncthreads();
    const int taken = s_taken;
    // table entries of the blocks taken, in the order of the requests
    for (int x = cta * kPagesThreads + tid; x < taken; x += ctas * kPagesThreads) {
        const int r = last_not_above(s_off, p.R, x);
        p.table[static_cast<int64_t>(r) * p.max_blocks + pages_of(s_len[r]) + x - s_off[r]] = p.free_blocks[avail - 1 - x];
    }
    const int64_t tokens = p.packed ? p.width : static_cast<int64_t>(p.R) * p.width;
    for (int64_t i = static_cast<int64_t>(cta) * kPagesThreads + tid; i < tokens; i += ctas * kPagesThreads) {
        int r, j;
        if (p.packed) {
            r = last_not_above(s_start, p.R, static_cast<int>(i));
            j = static_cast<int>(i) - s_start[r];
        } else {
            r = tokens <= INT32_MAX ? static_cast<int>(static_cast<uint32_t>(i) / static_cast<uint32_t>(p.width)) : static_cast<int>(i / p.width);
            j = static_cast<int>(i - static_cast<int64_t>(r) * p.width);
        }
        int64_t slot = -1;
        if (j < s_get[r]) {
            const int pos = s_len[r] + j, page = pos / kPageTokens, held = pages_of(s_len[r]);
            const int id = page < held ? p.table[static_cast<int64_t>(r) * p.max_blocks + page] : p.free_blocks[avail - 1 - (s_off[r] + page - held)];
            slot = id < 0 ? -1 : static_cast<int64_t>(id) * kPageTokens + (pos & (kPageTokens - 1));
        }
        p.slots[i] = slot;
    }
    cluster_barrier(ctas);
    if (cta == 0) {     // (granted and starts may lie where the other CTAs found new_lens)
        for (int r = tid; r <= p.R; r += kPagesThreads) {
            p.starts[r] = !p.packed ? r * p.width : r < p.R ? s_start[r] : static_cast<int>(min(base_start, static_cast<int64_t>(INT32_MAX)));
            if (r == p.R) continue;
            p.granted[r] = max(s_get[r], 0);
            p.lens[r] = s_len[r] + max(s_get[r], 0);
        }
        if (tid == 0) *p.n_free = avail - taken;
    }
}

__global__ void __launch_bounds__(kPagesThreads) pages_trim_kernel(const PagesParams p) {
    extern __shared__ int s_requests[];
    __shared__ int64_t warp_sums[kPagesThreads / 32];
    int* const s_off = s_requests;                 // blocks given back by the requests before
    int* const s_keep = s_requests + p.R;          // tokens that stay
    const int tid = threadIdx.x, cta = blockIdx.x, ctas = gridDim.x;
    after_previous_kernel();
    let_next_kernel_start();
    const int room = kPageTokens * p.max_blocks;
    const int avail = min(max(*p.n_free, 0), p.num_blocks);
    int gone = 0;
    for (int r0 = 0; r0 < p.R; r0 += kPagesThreads) {
        const int r = r0 + tid;
        const bool live = r < p.R;
        const int n = live ? min(max(p.lens[r], 0), room) : 0, keep = live ? min(max(p.arg[r], 0), n) : 0;
        int total;
        const int off = gone + block_scan(pages_of(n) - pages_of(keep), warp_sums, total);
        gone += total;
        if (live) {
            s_off[r] = off;
            s_keep[r] = keep;
        }
    }
    __syncthreads();
    for (int x = cta * kPagesThreads + tid; x < gone; x += ctas * kPagesThreads) {
        const int r = last_not_above(s_off, p.R, x);
        int32_t* entry = p.table + static_cast<int64_t>(r) * p.max_blocks + pages_of(s_keep[r]) + x - s_off[r];
        const int to = avail + gone - 1 - x;   // (the first block that goes back lies on top)
        if (to < p.num_blocks) p.free_blocks[to] = *entry;
        *entry = -1;
    }
    cluster_barrier(ctas);
    if (cta == 0) {
        for (int r = tid; r < p.R; r += kPagesThreads) p.lens[r] = s_keep[r];
        if (tid == 0) *p.n_free = min(avail + gone, p.num_blocks);
    }
}

// ------------------------------------------------------------------ ancestor masks
// A thread per node walks up to the root; a parent that is not in [0, node) ends the walk, so that every walk ends.
// Bit j of a node's words: j is the node or one of its ancestors.  Its position is the context's length + its depth.

__global__ void __launch_bounds__(kTreeMaxNodes) tree_masks_kernel(const MaskParams p) {
    __shared__ int s_parent[kTreeMaxNodes];
    __shared__ uint32_t s_mask[kTreeMaxNodes * (kTreeMaxNodes / 32 + 1)];   // (rows an odd number of words apart)
    const int b = blockIdx.x, i = threadIdx.x, W = (p.T + 31) / 32, row = W | 1;
    after_previous_kernel();
    let_next_kernel_start();
    const int nodes = p.tree_lens ? min(max(p.tree_lens[b], 0), p.T) : p.T;
    if (i < p.T) s_parent[i] = p.parents[static_cast<int64_t>(b) * p.T + i];
    for (int k = i; k < p.T * row; k += blockDim.x) s_mask[k] = 0;
    __syncthreads();
    if (i < p.T) {
        int depth = -1;
        for (int j = i, next; i < nodes; j = next) {
            s_mask[i * row + (j >> 5)] |= 1u << (j & 31);
            depth++;
            next = s_parent[j];
            if (next < 0 || next >= j) break;
        }
        p.positions[static_cast<int64_t>(b) * p.T + i] = (p.context_lens ? p.context_lens[b] : 0) + max(depth, 0);
    }
    __syncthreads();
    for (int k = i; k < p.T * W; k += blockDim.x)
        p.masks[static_cast<int64_t>(b) * p.T * W + k] = static_cast<int32_t>(s_mask[k / W * row + k % W]);
}

// ------------------------------------------------------------------ acceptance of a tree
// The walk: node 0 is accepted; after node c comes its lowest child whose token is the target model's next one after
// c.  Path token k moves from position context + path[k] to context + k in every layer and head.  A CTA has one
// sequence; each of its warps walks the tree for itself (a node or a few per lane, a ballot per step: no barrier), then
// its warps move (layer, head) pairs.  path[k] >= k and the path ascends, so a place is written only after it has been
// read, if a warp goes up in batches: it loads a batch's rows, then stores them.
constexpr int kCommitWarps = 4, kCommitBatch = 8;

__global__ void __launch_bounds__(32 * kCommitWarps) tree_commit_kernel(const CommitParams p) {
    __shared__ int s_path[kCommitWarps][kTreeMaxNodes];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, b = blockIdx.y;
    const int64_t row = static_cast<int64_t>(b) * p.T;
    int* const path = s_path[warp];
    after_previous_kernel();
    let_next_kernel_start();
    const int len = max(p.seq_lens[b], 0);
    const int nodes = min(min(p.tree_lens ? max(p.tree_lens[b], 0) : p.T, p.T), len), ctx = len - nodes;
    constexpr int PER = kTreeMaxNodes / 32;
    int tok[PER], par[PER], nxt[PER];
#pragma unroll
    for (int k = 0; k < PER; k++) {
        const int j = 32 * k + lane;
        tok[k] = j < nodes ? p.tokens[row + j] : 0;
        nxt[k] = j < nodes ? p.next[row + j] : 0;
        const int up = j < nodes ? p.parents[row + j] : -1;
        par[k] = up < j ? up : -1;
    }
    int n = 0, moved = 0;
    for (int cur = nodes > 0 ? 0 : -1; cur >= 0; n++) {
        if (lane == 0) path[n] = cur;
        moved += cur != n;
        int mine = nxt[0];
#pragma unroll
        for (int k = 1; k < PER; k++) mine = cur >> 5 == k ? nxt[k] : mine;
        const int want = __shfl_sync(0xffffffffu, mine, cur & 31);
        int found = -1;
#pragma unroll
        for (int k = PER - 1; k >= 0; k--) {
            if (32 * k >= nodes) continue;
            const uint32_t hit = __ballot_sync(0xffffffffu, par[k] == cur && tok[k] == want);
            if (hit) found = 32 * k + __ffs(hit) - 1;
        }
        cur = found;
    }
    __syncwarp();
    if (blockIdx.x == 0 && warp == 0) {
        for (int k = lane; k < p.T; k += 32) {
            p.path[row + k] = k < n ? path[k] : -1;
            p.out_tokens[row + k] = k < n ? p.next[row + path[k]] : -1;
        }
        if (lane == 0) {
            p.n_accepted[b] = n;
            p.new_lens[b] = ctx + n;
        }
    }
    if (moved == 0) return;
    const int32_t* bt = p.block_table + static_cast<int64_t>(b) * p.max_blocks;
    const int first = n - moved;   // (the path's head is in place: path[k] == k up to here and nowhere later)
    const int kw = p.pdk / 4, words = kw + p.pdv / 4, half = p.pdv / 8;   // 32-bit words: K row, both rows, half a V row
    const int off_kn = kPageTokens * p.pdk, off_vc = off_kn + 2 * kPageTokens, off_vn = off_vc + kPageTokens * p.pdv;
    auto page_of = [&](int pos) -> int64_t {   // start of the page's first head, -1: none
        const int id = pos / kPageTokens < p.max_blocks ? bt[pos / kPageTokens] : -1;
        return id >= 0 && id < p.num_blocks ? static_cast<int64_t>(id) * p.Hkv * p.page_bytes : -1;
    };
    // byte of word w of the two rows of a page's token
    auto word_at = [&](int w, int tok16) {
        const int i = w - kw, v = (tok16 & 2) ? (i < half ? i + half : i - half) : i;
        return w < kw ? tok16 * p.pdk + 4 * w : off_vc + tok16 * p.pdv + 4 * v;
    };
    for (int it = blockIdx.x * kCommitWarps + warp; it < p.n_layers * p.Hkv; it += gridDim.x * kCommitWarps) {
        uint8_t* const base = p.pool + (it / p.Hkv) * p.layer_stride + static_cast<int64_t>(it % p.Hkv) * p.page_bytes;
        for (int k0 = first; k0 < n; k0 += kCommitBatch) {
            uint32_t x[kCommitBatch][2];
            uint16_t norm[kCommitBatch];
#pragma unroll
            for (int k = 0; k < kCommitBatch; k++) {
                const int pos = k0 + k < n ? ctx + path[k0 + k] : -1, t = pos & (kPageTokens - 1);
                const int64_t page = pos >= 0 ? page_of(pos) : -1;
                x[k][0] = x[k][1] = 0;
                norm[k] = 0;
                if (page < 0) continue;
                if (lane < words) x[k][0] = *reinterpret_cast<const uint32_t*>(base + page + word_at(lane, t));
                if (lane + 32 < words) x[k][1] = *reinterpret_cast<const uint32_t*>(base + page + word_at(lane + 32, t));
                if (lane < 2) norm[k] = *reinterpret_cast<const uint16_t*>(base + page + (lane ? off_vn : off_kn) + 2 * t);
            }
            __syncwarp();
#pragma unroll
            for (int k = 0; k < kCommitBatch; k++) {
                if (k0 + k >= n) continue;
                const int pos = ctx + k0 + k, t = pos & (kPageTokens - 1);
                const int64_t page = page_of(pos);
                if (page < 0 || page_of(ctx + path[k0 + k]) < 0) continue;
                if (lane < words) *reinterpret_cast<uint32_t*>(base + page + word_at(lane, t)) = x[k][0];
                if (lane + 32 < words) *reinterpret_cast<uint32_t*>(base + page + word_at(lane + 32, t)) = x[k][1];
                if (lane < 2) *reinterpret_cast<uint16_t*>(base + page + (lane ? off_vn : off_kn) + 2 * t) = norm[k];
            }
            __syncwarp();
        }
    }
}

}  // namespace ftq
