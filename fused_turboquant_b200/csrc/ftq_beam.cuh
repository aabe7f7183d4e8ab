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

// of the cluster, or of the only CTA (what one CTA wrote before it, the others read after it: past L1, by __ldcg)
__device__ __forceinline__ void fork_barrier() {
    if (gridDim.x > 1) {
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
    } else {
        __syncthreads();
    }
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
// table: an atomic minimum on its count, which is below zero then.
//
// One cluster of 8 CTAs, or one CTA where there is little; four barriers.  A warp has a contiguous part of the entries, so that the
// sums of the warps' counts give the order, and keeps its first ones in shared memory from phase to phase; CTA 0 has the
// rows' last blocks besides.  Bound by the chain parents -> lengths -> entries -> counts -> claims -> stack, each a round trip to L2:
// 14 us for 256 rows of 47 blocks (entries read anew in each of seven phases: 30), 6 for four rows.
constexpr int kForkKept = 2;        // spans of entries that a warp keeps
struct ForkSpan { int n, pages; int64_t at; };      // entries (old or new ones), new ones of them, the first one's place
constexpr int fork_smem(int R) { return kForkThreads / 32 * kForkKept * (kForkSpan * 8 + static_cast<int>(sizeof(ForkSpan))) + 8 * R; }

__global__ void __launch_bounds__(kForkThreads) pages_fork_kernel(const ForkParams p) {
    extern __shared__ __align__(16) uint8_t s_raw[];
    __shared__ int warp_sums[kForkThreads / 32];
    constexpr int WARPS = kForkThreads / 32, PER = kForkSpan / 32;
    const int tid = threadIdx.x, lane = tid & 31, cta = blockIdx.x, warp = cta * WARPS + (tid >> 5), warps = gridDim.x * WARPS;
    int2* const s_entry = reinterpret_cast<int2*>(s_raw) + (tid >> 5) * kForkKept * kForkSpan;        // the warp's: (old, new)
    ForkSpan* const s_span = reinterpret_cast<ForkSpan*>(s_raw + WARPS * kForkKept * kForkSpan * 8) + (tid >> 5) * kForkKept;
    int* const s_last = reinterpret_cast<int*>(s_raw + fork_smem(0));     // CTA 0: rows' partly filled last blocks, -1: none
    int* const s_len = s_last + p.R;                                      // ... and lengths
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
    // the warp's entries, by spans of a row: f(place in the table, it is one, old block, new block, it stays)
    const int spans = (p.max_blocks + kForkSpan - 1) / kForkSpan;
    const int64_t items = static_cast<int64_t>(p.R) * spans, per = (items + warps - 1) / warps, item0 = warp * per, item1 = min(items, (warp + 1) * per);
    auto each_entry = [&](bool made, auto&& f) {
        for (int64_t it = item0; it < item1; it++) {
            const int kept = it - item0 < kForkKept ? static_cast<int>(it - item0) : -1;
            ForkSpan span;
            int x[PER], y[PER];
            if (made && kept >= 0) {
                span = s_span[kept];
#pragma unroll
                for (int k = 0; k < PER; k++) {
                    const int2 e = s_entry[kept * kForkSpan + 32 * k + lane];
                    x[k] = e.x;
                    y[k] = e.y;
                }
            } else {
                const int r = static_cast<int>(it / spans), j0 = static_cast<int>(it - static_cast<int64_t>(r) * spans) * kForkSpan;
                const Row row = row_of(r);
                const int old_pages = fork_pages(row.old), new_pages = fork_pages(row.len);
                span.n = min(max(old_pages, new_pages) - j0, kForkSpan);
                span.pages = min(max(new_pages - j0, 0), kForkSpan);
                span.at = static_cast<int64_t>(r) * p.max_blocks + j0;
                const int32_t* from = p.table + static_cast<int64_t>(max(row.parent, 0)) * p.max_blocks + j0;
#pragma unroll
                for (int k = 0; k < PER; k++) {
                    const int j = 32 * k + lane;
                    x[k] = j0 + j < old_pages && j < span.n ? p.table[span.at + j] : -1;
                    y[k] = j >= span.pages ? -1 : made ? __ldcg(p.next + span.at + j) : from[j];
                }
                if (kept >= 0) {
                    if (lane == 0) s_span[kept] = span;
#pragma unroll
                    for (int k = 0; k < PER; k++) s_entry[kept * kForkSpan + 32 * k + lane] = make_int2(x[k], y[k]);
                }
            }
#pragma unroll
            for (int k = 0; k < PER; k++)
                if (32 * k < span.n) f(span.at + 32 * k + lane, 32 * k + lane < span.n, x[k], y[k], kept >= 0);
            __syncwarp();
        }
    };
    // ---- the new table; counts of what differs; who has which partly filled last block
    each_entry(false, [&](int64_t at, bool live, int x, int y, bool kept) {
        if (!live) return;
        if (!kept) __stcg(p.next + at, y);
        if (x == y) return;
        if (valid(y)) atomicAdd(p.shares + y, 1);
        if (valid(x)) atomicAdd(p.shares + x, -1);
    });
    for (int i = cta * kForkThreads + tid; i < 2 * p.R; i += gridDim.x * kForkThreads) p.copies[i] = -1;
    if (cta == 0) {
        for (int r = tid; r < p.R; r += kForkThreads) {
            const Row row = row_of(r);
            int b = -1;
            if (row.len % kPageTokens != 0) b = p.table[static_cast<int64_t>(row.parent) * p.max_blocks + fork_pages(row.len) - 1];
            if (!valid(b)) b = -1;
            s_len[r] = row.len;
            s_last[r] = b;
            if (b >= 0) {
                __stcg(p.part_count + b, 0);
                __stcg(p.part_first + b, INT32_MAX);
            }
        }
        __syncthreads();
        for (int r = tid; r < p.R; r += kForkThreads) {
            const int b = s_last[r];
            if (b < 0) continue;
            atomicAdd(p.part_count + b, 1);
            atomicMin(p.part_first + b, r);
        }
    }
    fork_barrier();
    // ---- who claims the blocks that nobody holds
    each_entry(true, [&](int64_t at, bool live, int x, int y, bool) {
        if (live && x != y && valid(x) && __ldcg(p.shares + x) < 0) atomicMin(p.shares + x, INT32_MIN + static_cast<int>(at));
    });
    fork_barrier();
    // ---- how many there are, and how many rows need a block
    auto claims = [&](int64_t at, bool live, int x, int y) {
        return live && x != y && valid(x) && __ldcg(p.shares + x) == INT32_MIN + static_cast<int>(at);
    };
    {
        int mine = 0;
        each_entry(true, [&](int64_t at, bool live, int x, int y, bool) { mine += __popc(__ballot_sync(0xffffffffu, claims(at, live, x, y))); });
        if (lane == 0) __stcg(p.counts + warp, mine);
    }
    if (cta == 0) {
        int base = 0;
        for (int r0 = 0; r0 < p.R; r0 += kForkThreads) {
            const int r = r0 + tid, b = r < p.R ? s_last[r] : -1;
            const int held = b >= 0 ? __ldcg(p.shares + b) + 1 : 0;
            const int need = held > 1 && !(held == __ldcg(p.part_count + b) && __ldcg(p.part_first + b) == r);
            int total;
            const int rank = base + fork_scan(need, warp_sums, total);
            if (r < p.R) p.ranks[r] = need ? rank : -1;     // (read by the same thread only)
            base += total;
        }
        if (tid == 0) __stcg(p.counts + kForkWarps, base);
    }
    fork_barrier();
    // ---- give back and write the table, or take all of it back
    int freed = 0, before = 0;
    {
        int c[kForkWarps / 32];
#pragma unroll
        for (int k = 0; k < kForkWarps / 32; k++) c[k] = 32 * k + lane < warps ? __ldcg(p.counts + 32 * k + lane) : 0;
#pragma unroll
        for (int k = 0; k < kForkWarps / 32; k++) {
            freed += __reduce_add_sync(0xffffffffu, c[k]);
            before += __reduce_add_sync(0xffffffffu, 32 * k + lane < warp ? c[k] : 0);
        }
    }
    const int wanted = __ldcg(p.counts + kForkWarps), top = min(avail + freed, p.num_blocks);
    const bool ok = wanted <= top;
    each_entry(true, [&](int64_t at, bool live, int x, int y, bool) {
        // (a claim that somebody else has cleared by now was not this entry's)
        const bool mine = claims(at, live, x, y);
        const uint32_t all = __ballot_sync(0xffffffffu, mine);
        if (mine) {
            const int to = avail + freed - 1 - (before + __popc(all & ((1u << lane) - 1)));
            if (ok && to < p.num_blocks) __stcg(p.free_blocks + to, x);
            atomicExch(p.shares + x, ok ? 0 : -1);
        }
        before += __popc(all);
        // (what others need of the old table is in the new one, and its lengths stay until they are done)
        if (ok && live && x != y) p.table[at] = y;
    });
    fork_barrier();
    if (!ok) {
        each_entry(true, [&](int64_t, bool live, int x, int y, bool) {
            if (!live || x == y) return;
            if (valid(y)) atomicAdd(p.shares + y, -1);
            if (valid(x)) atomicAdd(p.shares + x, 1);
        });
        if (cta == 0 && tid == 0) *p.done = 0;
        return;
    }
    // ---- take: the rows' own last blocks, and the lengths
    if (cta == 0) {
        for (int r = tid; r < p.R; r += kForkThreads) {
            const int rank = p.ranks[r], len = s_len[r];
            if (rank >= 0) {
                const int b = s_last[r], to = __ldcg(p.free_blocks + top - 1 - rank);
                p.copies[2 * rank] = b;
                p.copies[2 * rank + 1] = to;
                atomicAdd(p.shares + b, -1);
                p.table[static_cast<int64_t>(r) * p.max_blocks + fork_pages(len) - 1] = to;
            }
            p.lens[r] = len;
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
// written is read.  The free ones are then the last n, the lowest of them on top of the stack.  Six phases, each a pass over the
// blocks, the stack or the table: 8 to 10 us.
__global__ void __launch_bounds__(kForkThreads) pages_compact_kernel(const CompactParams p) {
    __shared__ int warp_sums[kForkThreads / 32];
    const int tid = threadIdx.x, cta = blockIdx.x, first = cta * kForkThreads + tid;
    const int ctas = gridDim.x, ALL = ctas * kForkThreads;
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
    const int per = (nb + ctas - 1) / ctas, from = min(nb, cta * per), to = min(nb, from + per);
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
    for (int c = 0; c < ctas; c++) {
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
    // a part of the columns at a time, a (row, column) a thread: an entry of a row that has tokens against the first such row's
    constexpr int COLUMNS = 1024;
    for (int j0 = 0; j0 < whole; j0 += COLUMNS) {
        const int n = min(COLUMNS, whole - j0);
        for (int64_t i = tid; i < static_cast<int64_t>(p.group - first - 1) * n; i += blockDim.x) {
            const int k = first + 1 + static_cast<int>(i / n), j = j0 + static_cast<int>(i % n);
            if (p.table[(row0 + k) * p.max_blocks + j] != p.table[(row0 + first) * p.max_blocks + j] && p.lens[row0 + k] > 0) atomicMin(&s_cut, j);
        }
        __syncthreads();
        if (s_cut < j0 + n) break;
    }
    if (tid == 0) p.out[blockIdx.x] = kPageTokens * s_cut;
}

// ------------------------------------------------------------------ copies of pages
// A CTA has a layer, every gridDim.x-th pair and a part of a block's bytes (blockIdx.z of gridDim.z); it looks at 256 pairs at
// a time, and pairs with an id outside the pool are passed over.  Bound by HBM: 678 MB there and back in 113 us, 6.0 TB/s, 92 % of a plain
// copy's rate; 95 MB in 14 us.
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
