// Rows of a page table that share blocks: forking, compaction, and the copies of pages that go with them.  Integers and
// bytes only.
//
// shares[b] counts the rows that hold block b besides the first of them, so that blocks of one holder, and free ones, have 0:
// taking blocks (pages_extend_kernel) does not know of it.  Two rows never hold one block that either of them will write to,
// i.e. their partly filled last one.
#pragma once

#include "ftq_beam_launch.h"

namespace ftq {

constexpr int kForkCtas = 8, kForkThreads = 32 * kForkWarps / kForkCtas;
constexpr int kForkSpan = 256;      // table entries of a row that a warp takes at a time

// Exclusive scan over the CTA's threads, and the sum of all.
__device__ __forceinline__ int fork_scan(int v, int* warp_sums, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
    }
    __syncthreads();        // (the sums of the scan before have been read)
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kForkThreads / 32; w++) {
        const int s = warp_sums[w];
        before += w < warp ? s : 0;
        all += s;
    }
    total = all;
    return before + x - v;
}

// (what one CTA wrote before it, the others read after it: past L1, by __ldcg)
__device__ __forceinline__ void fork_barrier() {
    __threadfence();
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}

__device__ __forceinline__ int fork_pages(int tokens) { return (tokens + kPageTokens - 1) / kPageTokens; }

// ------------------------------------------------------------------ fork
// Row r becomes the first keep[r] tokens of what row parents[r] was.  All rows change at once:
//
//   new[r][j] = old[parent(r)][j]           for the blocks that its tokens fill
//   a block whose last holder goes is free  (in the order of the rows and their entries, the first of them on top)
//   a partly filled last block stays with the first row that has it as such, if no row has it as a whole one; every other
//   row takes a block from the stack, in the order of the rows, and a copy is listed
//
// or, where the stack has too few, nothing does.  The new table is made beside the old one.  Only entries that differ change a
// count (beams differ in their last few blocks).  A block that nobody holds any more is claimed by its first entry in the old
// table: an atomic minimum on its count, which is below zero then.  Six phases between the barriers of a cluster of 8 CTAs;
// a warp has a contiguous part of the entries, so that the sums of the warps' counts give the order.
__global__ void __cluster_dims__(kForkCtas) __launch_bounds__(kForkThreads) pages_fork_kernel(const ForkParams p) {
    __shared__ int warp_sums[kForkThreads / 32];
    const int tid = threadIdx.x, lane = tid & 31, cta = blockIdx.x, warp = cta * (kForkThreads / 32) + (tid >> 5);
    after_previous_kernel();
    let_next_kernel_start();
    const int room = kPageTokens * p.max_blocks;
    const int avail = min(max(*p.n_free, 0), p.num_blocks);
    struct Row { int parent, len, old; };       // the row that it becomes (-1: none), tokens it will have, tokens it has
    auto tokens_of = [&](int r) { return min(max(p.lens[r], 0), room); };
    auto row_of = [&](int r) {
        const int first = p.group > 0 ? r / p.group * p.group : 0, n = p.group > 0 ? p.group : p.R, x = p.parents[r];
        Row row{x >= 0 && x < n ? first + x : -1, 0, tokens_of(r)};
        if (row.parent >= 0) row.len = min(tokens_of(row.parent), p.keep ? max(p.keep[r], 0) : INT32_MAX);
        return row;
    };
    auto valid = [&](int id) { return static_cast<uint32_t>(id) < static_cast<uint32_t>(p.num_blocks); };
    // the partly filled last block of row r, before anybody takes one; -1: it has none
    auto last_of = [&](const Row& row) {
        if (row.len % kPageTokens == 0) return -1;
        const int id = p.table[static_cast<int64_t>(row.parent) * p.max_blocks + fork_pages(row.len) - 1];
        return valid(id) ? id : -1;
    };
    // the warp's entries, by spans of a row: f(index of the entry in the table, old block, new block)
    const int spans = (p.max_blocks + kForkSpan - 1) / kForkSpan;
    const int64_t items = static_cast<int64_t>(p.R) * spans, per = (items + kForkWarps - 1) / kForkWarps;
    auto each_entry = [&](bool made, auto&& f) {
        const int64_t end = min(items, (warp + 1) * per);
        for (int64_t it = warp * per; it < end; it++) {
            const int r = static_cast<int>(it / spans), j0 = static_cast<int>(it - static_cast<int64_t>(r) * spans) * kForkSpan;
            const Row row = row_of(r);
            const int old_pages = fork_pages(row.old), new_pages = fork_pages(row.len), n = min(max(old_pages, new_pages) - j0, kForkSpan);
            if (n <= 0) continue;
            const int64_t at = static_cast<int64_t>(r) * p.max_blocks + j0;
            const int32_t* from = p.table + static_cast<int64_t>(max(row.parent, 0)) * p.max_blocks + j0;
            int x[kForkSpan / 32], y[kForkSpan / 32];
#pragma unroll
            for (int k = 0; k < kForkSpan / 32; k++) {
                const int j = 32 * k + lane;
                x[k] = j0 + j < old_pages && j < n ? p.table[at + j] : -1;
                y[k] = j0 + j >= new_pages || j >= n ? -1 : made ? __ldcg(p.next + at + j) : from[j];
            }
#pragma unroll
            for (int k = 0; k < kForkSpan / 32; k++)
                if (32 * k < n) f(at + 32 * k + lane, 32 * k + lane < n, x[k], y[k]);
        }
    };
    // ---- the new table; counts of what differs
    for (int r = cta * kForkThreads + tid; r < p.R; r += kForkCtas * kForkThreads) {
        const int b = last_of(row_of(r));
        if (b >= 0) {
            __stcg(p.part_count + b, 0);
            __stcg(p.part_first + b, INT32_MAX);
        }
    }
    for (int i = cta * kForkThreads + tid; i < 2 * p.R; i += kForkCtas * kForkThreads) p.copies[i] = -1;
    each_entry(false, [&](int64_t at, bool live, int x, int y) {
        if (!live) return;
        __stcg(p.next + at, y);
        if (x == y) return;
        if (valid(y)) atomicAdd(p.shares + y, 1);
        if (valid(x)) atomicAdd(p.shares + x, -1);
    });
    fork_barrier();
    // ---- who claims the blocks that nobody holds, and who has a partly filled last block
    each_entry(true, [&](int64_t at, bool live, int x, int y) {
        if (live && x != y && valid(x) && __ldcg(p.shares + x) < 0) atomicMin(p.shares + x, INT32_MIN + static_cast<int>(at));
    });
    for (int r = cta * kForkThreads + tid; r < p.R; r += kForkCtas * kForkThreads) {
        const int b = last_of(row_of(r));
        if (b >= 0) {
            atomicAdd(p.part_count + b, 1);
            atomicMin(p.part_first + b, r);
        }
    }
    fork_barrier();
    // ---- how many there are of both
    auto claims = [&](int64_t at, bool live, int x, int y) {
        return live && x != y && valid(x) && __ldcg(p.shares + x) == INT32_MIN + static_cast<int>(at);
    };
    {
        int mine = 0;
        each_entry(true, [&](int64_t at, bool live, int x, int y) { mine += __popc(__ballot_sync(0xffffffffu, claims(at, live, x, y))); });
        if (lane == 0) __stcg(p.counts + warp, mine);
    }
    if (cta == 0) {
        int base = 0;
        for (int r0 = 0; r0 < p.R; r0 += kForkThreads) {
            const int r = r0 + tid, b = r < p.R ? last_of(row_of(r)) : -1;
            const int held = b >= 0 ? __ldcg(p.shares + b) + 1 : 0;
            const int need = held > 1 && !(held == __ldcg(p.part_count + b) && __ldcg(p.part_first + b) == r);
            int total;
            const int rank = base + fork_scan(need, warp_sums, total);
            if (r < p.R) p.ranks[r] = need ? rank : -1;     // (read by this CTA's same thread only)
            base += total;
        }
        if (tid == 0) __stcg(p.counts + kForkWarps, base);
    }
    fork_barrier();
    // ---- give back, or take all of it back
    int freed = 0, before = 0;
    {
        int c[kForkWarps / 32];
#pragma unroll
        for (int k = 0; k < kForkWarps / 32; k++) c[k] = __ldcg(p.counts + 32 * k + lane);
#pragma unroll
        for (int k = 0; k < kForkWarps / 32; k++) {
            freed += __reduce_add_sync(0xffffffffu, c[k]);
            before += __reduce_add_sync(0xffffffffu, 32 * k + lane < warp ? c[k] : 0);
        }
    }
    const int wanted = __ldcg(p.counts + kForkWarps), top = min(avail + freed, p.num_blocks);
    const bool ok = wanted <= top;
    each_entry(true, [&](int64_t at, bool live, int x, int y) {
        const bool mine = claims(at, live, x, y);
        const uint32_t all = __ballot_sync(0xffffffffu, mine);
        if (mine) {
            const int to = avail + freed - 1 - (before + __popc(all & ((1u << lane) - 1)));
            if (ok && to < p.num_blocks) __stcg(p.free_blocks + to, x);
        }
        before += __popc(all);
    });
    fork_barrier();     // (the claims have been read)
    each_entry(true, [&](int64_t at, bool live, int x, int y) {
        if (claims(at, live, x, y)) atomicExch(p.shares + x, ok ? 0 : -1);
    });
    if (!ok) {
        fork_barrier();
        each_entry(true, [&](int64_t, bool live, int x, int y) {
            if (!live || x == y) return;
            if (valid(y)) atomicAdd(p.shares + y, -1);
            if (valid(x)) atomicAdd(p.shares + x, 1);
        });
        if (cta == 0 && tid == 0) *p.done = 0;
        return;
    }
    // ---- take: the rows' own last blocks, then the table
    if (cta == 0) {
        for (int r0 = 0; r0 < p.R; r0 += kForkThreads) {
            const int r = r0 + tid, rank = r < p.R ? p.ranks[r] : -1;
            if (rank < 0) continue;
            const Row row = row_of(r);
            const int b = last_of(row), to = __ldcg(p.free_blocks + top - 1 - rank);
            p.copies[2 * rank] = b;
            p.copies[2 * rank + 1] = to;
            atomicAdd(p.shares + b, -1);
            __stcg(p.next + static_cast<int64_t>(r) * p.max_blocks + fork_pages(row.len) - 1, to);
        }
    }
    fork_barrier();
    // (the old table goes row by row; what others still need of it is in the new one, but for the lengths)
    const int64_t end = min(items, (warp + 1) * per);
    for (int64_t it = warp * per; it < end; it++) {
        const int r = static_cast<int>(it / spans), j0 = static_cast<int>(it - static_cast<int64_t>(r) * spans) * kForkSpan;
        const Row row = row_of(r);
        const int old_pages = fork_pages(row.old), new_pages = fork_pages(row.len), n = min(max(old_pages, new_pages), j0 + kForkSpan);
        for (int j = j0 + lane; j < n; j += 32) {
            const int64_t at = static_cast<int64_t>(r) * p.max_blocks + j;
            p.table[at] = j < new_pages ? __ldcg(p.next + at) : -1;
        }
    }
    // (a length is somebody else's parent's until everybody is done with it)
    constexpr int MOST = 8192 / kForkThreads;
    int len[MOST];
    if (cta == 0) {
#pragma unroll
        for (int k = 0; k < MOST; k++) {
            const int r = k * kForkThreads + tid;
            len[k] = r < p.R ? row_of(r).len : 0;
        }
    }
    fork_barrier();
    if (cta == 0) {
#pragma unroll
        for (int k = 0; k < MOST; k++) {
            const int r = k * kForkThreads + tid;
            if (r < p.R) p.lens[r] = len[k];
        }
        if (tid == 0) {
            *p.n_free = top - wanted;
            *p.done = 1;
        }
    }
}

// ------------------------------------------------------------------ compaction
// Of num_blocks - n blocks in use those beyond the first num_blocks - n places move down: the k-th of them, by its id, into
// the k-th hole.  Every other block stays where it is, so that this is the least that has to move, and no block that is
// written is read.  The free ones are then the last n, the lowest of them on top of the stack.
__global__ void __cluster_dims__(kForkCtas) __launch_bounds__(kForkThreads) pages_compact_kernel(const CompactParams p) {
    __shared__ int warp_sums[kForkThreads / 32];
    const int tid = threadIdx.x, cta = blockIdx.x, first = cta * kForkThreads + tid;
    constexpr int ALL = kForkCtas * kForkThreads;
    after_previous_kernel();
    let_next_kernel_start();
    const int nb = p.num_blocks, n = min(max(*p.n_free, 0), nb), used = nb - n;
    auto valid = [&](int id) { return static_cast<uint32_t>(id) < static_cast<uint32_t>(nb); };
    for (int i = first; i < nb; i += ALL) __stcg(p.map + i, INT32_MAX);
    for (int i = first; i < nb / 2 * 2; i += ALL) __stcg(p.copies + i, -1);
    fork_barrier();
    for (int i = first; i < n; i += ALL) {
        const int id = p.free_blocks[i];
        if (valid(id)) __stcg(p.map + id, -1);
    }
    fork_barrier();
    // ---- holes below `used` and blocks beyond it, counted and then numbered by id
    const int per = (nb + kForkCtas - 1) / kForkCtas, from = min(nb, cta * per), to = min(nb, from + per);
    int holes = 0, movers = 0;
    for (int i0 = from; i0 < to; i0 += kForkThreads) {
        const int i = i0 + tid;
        const bool in_use = i < to && __ldcg(p.map + i) >= 0;
        holes += __syncthreads_count(i < to && i < used && !in_use);
        movers += __syncthreads_count(i < to && i >= used && in_use);
    }
    if (tid == 0) {
        __stcg(p.counts + cta, holes);
        __stcg(p.counts + kForkCtas + cta, movers);
    }
    fork_barrier();
    int at_hole = 0, at_mover = 0, all_holes = 0, all_movers = 0;
    for (int c = 0; c < kForkCtas; c++) {
        const int h = __ldcg(p.counts + c), m = __ldcg(p.counts + kForkCtas + c);
        at_hole += c < cta ? h : 0;
        at_mover += c < cta ? m : 0;
        all_holes += h;
        all_movers += m;
    }
    // (as many of either, unless the stack holds a block twice: then nothing beyond the fewer is written)
    const int moved = min(min(all_holes, all_movers), nb / 2);
    for (int i0 = from; i0 < to; i0 += kForkThreads) {
        const int i = i0 + tid;
        const bool in_use = i < to && __ldcg(p.map + i) >= 0;
        const bool hole = i < to && i < used && !in_use, mover = i < to && i >= used && in_use;
        int total;
        const int k = fork_scan(hole ? 1 : mover ? 1 << 16 : 0, warp_sums, total);
        const int rank = hole ? at_hole + (k & 0xffff) : at_mover + (k >> 16);
        if ((hole || mover) && rank < moved) __stcg(p.copies + 2 * rank + (hole ? 1 : 0), i);
        at_hole += total & 0xffff;
        at_mover += total >> 16;
    }
    fork_barrier();
    for (int k = first; k < moved; k += ALL) {
        const int2 c = __ldcg(reinterpret_cast<const int2*>(p.copies) + k);
        __stcg(p.map + c.x, c.y);
        if (p.shares) {
            p.shares[c.y] = p.shares[c.x];
            p.shares[c.x] = 0;
        }
    }
    for (int i = first; i < n; i += ALL) p.free_blocks[i] = nb - 1 - i;
    fork_barrier();
    const int room = kPageTokens * p.max_blocks;
    const int warps = ALL / 32, lane = tid & 31, warp = first >> 5, spans = (p.max_blocks + kForkSpan - 1) / kForkSpan;
    for (int64_t it = warp; it < static_cast<int64_t>(p.R) * spans; it += warps) {
        const int r = static_cast<int>(it / spans), j0 = static_cast<int>(it - static_cast<int64_t>(r) * spans) * kForkSpan;
        const int m = min(fork_pages(min(max(p.lens[r], 0), room)) - j0, kForkSpan);
        int32_t* row = p.table + static_cast<int64_t>(r) * p.max_blocks + j0;
#pragma unroll
        for (int k = 0; k < kForkSpan / 32; k++) {
            const int j = 32 * k + lane, id = j < m ? row[j] : -1;
            if (id >= used && valid(id)) {
                const int now = __ldcg(p.map + id);
                if (now >= 0 && now < used) row[j] = now;
            }
        }
    }
}

// ------------------------------------------------------------------ leading blocks in common
// A CTA per group of rows: tokens in leading blocks that are whole, and the same, in all rows that have tokens.
__global__ void __launch_bounds__(256) shared_lens_kernel(const SharedLensParams p) {
    __shared__ int s_whole, s_first, s_cut;
    const int tid = threadIdx.x;
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * p.group;
    after_previous_kernel();
    let_next_kernel_start();
    if (tid == 0) {
        s_whole = p.max_blocks;
        s_first = INT32_MAX;
    }
    __syncthreads();
    for (int k = tid; k < p.group; k += blockDim.x) {
        const int n = p.lens[row0 + k];
        if (n > 0) {
            atomicMin(&s_whole, n / kPageTokens);
            atomicMin(&s_first, k);
        }
    }
    __syncthreads();
    const int whole = s_first == INT32_MAX ? 0 : s_whole, first = s_first;
    if (tid == 0) s_cut = whole;
    __syncthreads();
    for (int j0 = 0; j0 < whole; j0 += blockDim.x) {
        const int j = j0 + tid;
        if (j < whole) {
            const int id = p.table[(row0 + first) * p.max_blocks + j];
            bool same = true;
#pragma unroll 4
            for (int k = 0; k < p.group; k++)
                if (k > first && p.lens[row0 + k] > 0) same &= p.table[(row0 + k) * p.max_blocks + j] == id;
            if (!same) atomicMin(&s_cut, j);
        }
        __syncthreads();
        if (s_cut < j0 + static_cast<int>(blockDim.x)) break;
    }
    if (tid == 0) p.out[blockIdx.x] = kPageTokens * s_cut;
}

// ------------------------------------------------------------------ copies of pages
// A CTA has a layer, every gridDim.x-th pair and a part of a block's bytes (blockIdx.z of gridDim.z); it looks at 256 pairs at
// a time, and pairs with an id outside the pool are passed over.
constexpr int kCopyThreads = 256;
__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const CopyPagesParams p) {
    __shared__ int2 s_pair[kCopyThreads];
    __shared__ int s_n;
    const int tid = threadIdx.x;
    after_previous_kernel();
    let_next_kernel_start();
    uint8_t* const base = p.pool + static_cast<int64_t>(blockIdx.y) * p.layer_stride;
    const int units = static_cast<int>(p.block_bytes / 16), per = (units + gridDim.z - 1) / gridDim.z;
    const int u0 = per * blockIdx.z, u1 = min(units, u0 + per);
    for (int64_t k0 = blockIdx.x; k0 < p.n; k0 += static_cast<int64_t>(kCopyThreads) * gridDim.x) {
        const int64_t k = k0 + static_cast<int64_t>(tid) * gridDim.x;
        int2 c = make_int2(-1, -1);
        if (k < p.n) c = make_int2(p.copies[2 * k], p.copies[2 * k + 1]);
        __syncthreads();        // (the list before has been read)
        if (tid == 0) s_n = 0;
        __syncthreads();
        if (c.x >= 0 && c.y >= 0 && c.x < p.num_blocks && c.y < p.num_blocks) s_pair[atomicAdd(&s_n, 1)] = c;
        __syncthreads();
        for (int i = 0; i < s_n; i++) {
            const uint4* from = reinterpret_cast<const uint4*>(base + s_pair[i].x * p.block_bytes);
            uint4* to = reinterpret_cast<uint4*>(base + s_pair[i].y * p.block_bytes);
            for (int u = u0 + tid; u < u1; u += 4 * kCopyThreads) {
                uint4 x[4];
#pragma unroll
                for (int w = 0; w < 4; w++)
                    if (u + w * kCopyThreads < u1) x[w] = from[u + w * kCopyThreads];
#pragma unroll
                for (int w = 0; w < 4; w++)
                    if (u + w * kCopyThreads < u1) to[u + w * kCopyThreads] = x[w];
            }
        }
    }
}

}  // namespace ftq
