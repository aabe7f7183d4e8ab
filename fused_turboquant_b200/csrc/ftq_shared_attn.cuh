// Paged decode attention of rows that share their leading blocks (beams, samples of a prompt): one new token of every row.
//
//   o_b = sum_j softmax_j(q_b . k_j scale) v_j     over the row's tokens, k_j = |k_j| levels[code] in the rotated space
//
// A page of common tokens is fetched and dequantised once for all rows of a group; look-ups and byte work, which bound the
// decode kernel (ftq_attn_flow.cuh), are the same for one row as for eight, and only the products and the softmax grow.
//
// Units.  The common tokens of a group and one KV head, with the group's rows x heads as the columns of the products, in
// blocks of 8 NT; and the tokens that a row has to itself, with its heads as columns.  All units lie on one line of places: so
// many for a unit on its own, and so many more for each of its pages, by what they cost; warp w of the grid takes the places
// [w share, (w + 1) share).  A warp works for itself: its pages come by bulk copies to a ring of its own, it keeps
// (O, m, l) of all columns in registers and leaves them in the workspace, a piece of a unit at a time.  No barrier, no atomic.
// shared_merge_kernel joins a row's pieces by their maxima, rotates back (core/hadamard.py:93-100) and stores.
// shared_prepare_kernel, before both, rotates the queries and makes the prefix sums of the places.
//
// A page of 16 tokens, 128 coordinates and 4-bit codes takes a warp 315, 373 and 474 instructions for one, two and four tiles of
// columns, and an SM 115, 160 and 262 cycles: look-ups alone are 64 shared-memory wavefronts, products 16 a tile, 8 cycles each.
// With four tiles the registers hold eight warps, two a scheduler, and the latencies of the chain look-up -> product -> softmax ->
// product show (issue 0.43 a cycle; 0.55 and 0.63 with twelve and sixteen warps); narrower kernels would look everything up twice.
//   32 requests of 8 beams, 8192 common tokens and 128 of their own, 32 / 8 heads, K4V4: 168 us (decode_attention on the 256 rows, of which
//   each reads all: 423); floor 48 us (316 MB), of which prepare 4 and merge 14 us.
// On the way (us, the same case): four tiles with a branch a tile 268; tiles known to the compiler, each lane's tokens of S in the order
// of its values' registers 202; a slack of 2^10 for the maximum 191; block ids in the requesting lanes, scores and weights in the same
// registers 175.  Without gain: the next page's scores beside this one's values (188), two pages a stage with the queries read once for
// both (178; 190), queries in registers and 16 columns a warp, two warps to a page (223), the queries' loads free to be moved (187).
//
// Rounded to fp16, which the products take: queries in the rotated space, centroids, weights times norms (all else is fp32; error against 64
// bits 3.9e-4 of the output's size with fp16 outputs, of which the output's own rounding is 2.1e-4).
// Tables, page layout and fragment maps are those of ftq_attn_mma.cuh with the columns as heads (NH = 2).  Weights carry the
// values' norms into fp16: they are scaled by a power of two that goes with the largest norm so far (lazily, as the maximum).
#pragma once

#include "ftq_attn_mma.cuh"
#include "ftq_shared_launch.h"

namespace ftq {

template <int D, int BK, int BV, int NT>
struct SharedCfg : MmaCfg<D, BK, BV, 2> {
    using M = MmaCfg<D, BK, BV, 2>;
    static constexpr SharedShape SHAPE = shared_shape(D, M::PAGE_BYTES, NT);
    static constexpr int WARPS = SHAPE.warps, THREADS = 32 * WARPS, COLS = 8 * NT;
    static constexpr int RING = SHAPE.ring, RING_BYTES = shared_ring_bytes(M::PAGE_BYTES, RING);     // pages on their way, per warp
    static constexpr int Q_BYTES = COLS * D * 2, PLAN_BYTES = kSharedPlanBytes, SMEM_BYTES = SHAPE.smem;
    static constexpr bool ROT = !(BV == 3 && D <= 128);     // (see FlowCfg)
};

// ------------------------------------------------------------------ plan
// first page of a unit's piece that starts `at` places into it
__device__ __forceinline__ int shared_page_of(int at, const FastDiv& cost, int pages) {
    const int x = at - kSharedPiece;
    return x <= 0 ? 0 : min(static_cast<int>(fast_div(x + cost.d - 1, cost)), pages);
}
__device__ __forceinline__ int shared_len(const SharedAttnParams& p, int b) { return max(0, min(p.seq_lens[b], p.max_seq)); }
// tokens of group r that are taken as common (whole blocks, as far as its longest row goes), and that row
__device__ __forceinline__ int shared_common(const SharedAttnParams& p, int r, int& leader) {
    int most = 0;
    leader = r * p.K;
    for (int k = 0; k < p.K; k++) {
        const int n = shared_len(p, r * p.K + k);
        if (n > most) {
            most = n;
            leader = r * p.K + k;
        }
    }
    return max(0, min(p.shared_lens[r], most)) / kPageTokens * kPageTokens;
}

// plan: [e] first place of entry e (groups, then rows), [entries] the end, then the share of a warp as a divisor; plan_unit: places
// of a unit of an entry (0: it has no pages); plan_tokens, plan_leader: the common tokens, and the row that they are read through.
template <int D>
__global__ void __launch_bounds__(256) shared_prepare_kernel(const __grid_constant__ SharedAttnParams p) {
    constexpr int E = D / kOctet;
    __shared__ int s_sum[8];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    let_next_kernel_start();
    after_previous_kernel();
    if (blockIdx.x == 0) {
        const int entries = p.R + p.R * p.K;
        int base = 0, longest = 0;
        for (int e0 = 0; e0 < entries; e0 += 256) {
            const int e = e0 + tid;
            int places = 0;
            if (e < entries) {
                int leader;
                const bool group = e < p.R;
                const int common = shared_common(p, group ? e : (e - p.R) / p.K, leader);
                const int pages = (group ? common : max(0, shared_len(p, e - p.R) - common) + kPageTokens - 1) / kPageTokens;
                const int unit = pages == 0 ? 0 : kSharedPiece + pages * (group ? p.cost_group : p.cost_row);
                places = unit * (group ? p.units_group : p.units_row);
                p.plan_unit[e] = unit;
                longest = max(longest, pages);
                p.plan_tokens[e] = common;
                p.plan_leader[e] = leader;
            }
            int x = places;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, x, d);
                if (lane >= d) x += y;
            }
            __syncthreads();
            if (lane == 31) s_sum[warp] = x;
            __syncthreads();
            int before = base;
            for (int w = 0; w < 8; w++) {
                before += w < warp ? s_sum[w] : 0;
                base += s_sum[w];
            }
            if (e < entries) p.plan[e] = before + x - places;
        }
        // A unit's pieces are walked side by side but joined one after the other: the longest one has at most so many that the two balance.
        longest = __reduce_max_sync(0xffffffffu, longest);
        __syncthreads();
        if (lane == 0) s_sum[warp] = longest;
        __syncthreads();
        if (tid == 0) {
            for (int w = 0; w < 8; w++) longest = max(longest, s_sum[w]);
            const int least = max(2, static_cast<int>(0.4f * sqrtf(static_cast<float>(longest))));
            p.plan[entries] = base;
            const uint32_t share = max((base + p.warps - 1) / p.warps, kSharedPiece + least * p.cost_group), bits = 32 - __clz(share - 1);
            p.plan[entries + 1] = share;        // (make_fastdiv)
            p.plan[entries + 2] = static_cast<int>(static_cast<uint32_t>(((1ull << (31 + bits)) + share - 1) / share));
            p.plan[entries + 3] = 31 + bits;
            if (p.first) *p.status = 0;
        }
        return;
    }
    // a row's head per octet; a row's 16-byte chunks lie in the order in which the lanes of a product take them, those of odd
    // rows with each four exchanged
    const int t8 = lane & 7, G = p.Hq / p.Hkv;
    const int64_t rows = static_cast<int64_t>(p.R) * p.K * p.Hq;
    for (int64_t i0 = (static_cast<int64_t>(blockIdx.x - 1) * 8 + warp) * 4; i0 < rows; i0 += static_cast<int64_t>(gridDim.x - 1) * 32) {
        const int64_t i = i0 + (lane >> 3);
        const bool live = i < rows;
        const uint8_t* src = static_cast<const uint8_t*>(p.q) + (live ? i : 0) * (D * 2);
        float a[E];
#pragma unroll
        for (int k = 0; k < E / 8; k++) {
            float tmp[8];
            const uint8_t* at = src + 16 * (t8 + 8 * k);
            if (p.q_dtype == kBF16) load8<__nv_bfloat16>(reinterpret_cast<const __nv_bfloat16*>(at), tmp);
            else load8<__half>(reinterpret_cast<const __half*>(at), tmp);
#pragma unroll
            for (int c = 0; c < 8; c++)
                a[8 * k + c] = __uint_as_float(__float_as_uint(tmp[c]) ^ sign_mask(p.signs, load_coord(t8, 8 * k + c)));
        }
        octet_fwht<E>(a, lane);
        if (!live) continue;
        const int hq = static_cast<int>(i % p.Hq), h = hq / G;
        const int64_t b = i / p.Hq, r = b / p.K;
        const int n = static_cast<int>(b - r * p.K) * G + hq - h * G;      // row of the (group, KV head)
        __half* dst = reinterpret_cast<__half*>(p.q_rows) + ((r * p.Hkv + h) * p.K * G + n) * D;
#pragma unroll
        for (int k = 0; k < E; k++) {
            const int coord = t8 + 8 * k, tg = coord / (D / 4), chunk = coord % (D / 4) / 8;
            dst[8 * ((4 * chunk + tg) ^ ((n & 1) * 4)) + coord % 8] = __ushort_as_half(static_cast<unsigned short>(f2h_sat(a[k] * p.q_scale)));
        }
    }
}

// ------------------------------------------------------------------ attention
// The reference maximum of a column is renewed when a score exceeds it by 2^kSharedSlack, the values' scale when a norm
// exceeds the one that it goes with by kSharedNorms: a weight stays below 2^10 * 2 * 16 = 2^15, which fp16 holds, and one that is
// 2^-14 of a column's largest still has all its bits.  (One for all columns of a warp: with the decode kernel's slack of 3
// every third page of the serving batch below did it, 512 scores of which one in fifty has three times the others' size.)
constexpr float kSharedSlack = 10.f, kSharedNorms = 16.f;
__device__ __forceinline__ uint32_t pack_weights(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

struct SharedPiece {
    int next;            // where the next piece starts
    int row;             // row of the block table
    int page0, n_pages;  // of the row's pages
    int tokens;          // from page0 on
    int cols;            // columns
    int col0;            // first column's row in its (group, KV head)
    int qh;              // group x Hkv + KV head
    int hkv;
    int limit0;          // tokens before page0
    bool group, ragged;  // common tokens; columns of a group with fewer of them
    int64_t out;         // rows in the workspace
};

// What a warp does with a piece: pages from its ring, TILES tiles of eight columns.
template <int D, int BK, int BV, int TILES>
struct SharedState {
    using M = MmaCfg<D, BK, BV, 2>;
    float o[TILES][2 * M::NMT][4], m[TILES][2], l[TILES][2];
    float vlimit, vscale;       // the largest norm of a value that needs no other scale, and the power of two that goes with it
};

template <int D, int BK, int BV, int NT>
__global__ void __launch_bounds__(SharedCfg<D, BK, BV, NT>::THREADS, 1) shared_attn_kernel(const __grid_constant__ SharedAttnParams p) {
    using C = SharedCfg<D, BK, BV, NT>;
    using WK = Window<BK, false>;
    using WV = Window<BV, false>;
    constexpr int NKB = C::NKB, NMT = C::NMT, ROW = D + 4;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    const uint32_t sbase = static_cast<uint32_t>(__cvta_generic_to_shared(smem_raw));
    const uint32_t window = (sbase + 65535u) & ~65535u, end0 = window;
    uint32_t free0 = sbase, free1 = window + 65536u;
    auto take = [&](uint32_t bytes) {
        uint32_t a = (free0 + 127u) & ~127u;
        if (a + bytes <= end0) { free0 = a + bytes; return a; }
        a = (free1 + 127u) & ~127u;
        free1 = a + bytes;
        return a;
    };
    auto gptr = [&](uint32_t saddr) { return smem_raw + (saddr - sbase); };
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, tg = lane & 3;
    uint32_t my_ring = 0, my_q = 0;
#pragma unroll
    for (int w = 0; w < C::WARPS; w++) { const uint32_t a = take(C::RING_BYTES); if (w == warp) my_ring = a; }
#pragma unroll
    for (int w = 0; w < C::WARPS; w++) { const uint32_t a = take(C::Q_BYTES); if (w == warp) my_q = a; }
    int* const s_plan = reinterpret_cast<int*>(gptr(take(C::PLAN_BYTES)));
    __shared__ __align__(8) unsigned long long s_bars[C::WARPS][C::RING + 1];
    const uint32_t my_bars = static_cast<uint32_t>(__cvta_generic_to_shared(&s_bars[warp][0])), q_bar = my_bars + 8 * C::RING;

    let_next_kernel_start();
    // ---- tables: a row of 32 copies of an entry is two shuffles, a conversion and one store
    {
        const float lev_k = p.lk.v[lane & 15], lev_v = p.lv.v[lane & 15];
        auto pair = [&](float lev, int lo, int hi) {
            const __half2 h = __floats2half2_rn(__shfl_sync(0xffffffffu, lev, lo), __shfl_sync(0xffffffffu, lev, hi));
            return *reinterpret_cast<const uint32_t*>(&h);
        };
        auto entry = [&](float lev, int bits, int e) {
            if (bits == 4) return pair(lev, e & 15, e >> 4);
            if (bits == 3) return pair(lev, e & 7, e >> 3 & 7);
            const uint32_t x = pair(lev, e & 3, (e >> 2) & 3), y = pair(lev, (e >> 4) & 3, e >> 6);
            return (lane & 1) ? y : x;
        };
        uint32_t* tb = reinterpret_cast<uint32_t*>(gptr(window));
#pragma unroll 4
        for (int e = warp; e < 256; e += C::WARPS) {
            tb[e * 64 + lane] = entry(lev_k, BK, e);
            tb[e * 64 + 32 + lane] = entry(lev_v, BV, e);
        }
        // (columns that a unit does not have are computed too: from zeros, or from what an earlier unit left)
        for (int i = lane; i < C::Q_BYTES / 16; i += 32) reinterpret_cast<uint4*>(gptr(my_q))[i] = make_uint4(0, 0, 0, 0);
    }
    if (lane == 0) {
#pragma unroll
        for (int r = 0; r <= C::RING; r++) mbar_init(my_bars + 8 * r, 1);
    }
    mbar_fence_init();
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
    after_previous_kernel();
    const int entries = p.R + p.R * p.K;
    for (int i = tid; i < entries + 2; i += C::THREADS) s_plan[i] = p.plan[i];
    __syncthreads();

    const int total = s_plan[entries], share = s_plan[entries + 1], G = p.Hq / p.Hkv;
    // (neighbours on the line are on different SMs, so that a short line has them all)
    const int me = warp * gridDim.x + blockIdx.x;
    const int64_t from = static_cast<int64_t>(me) * share;
    if (from >= total) return;
    const int end = static_cast<int>(min(from + share, static_cast<int64_t>(total)));

    auto locate = [&](int pos) {
        SharedPiece it{};
        int lo = 0, hi = entries;     // plan[lo] <= pos < plan[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (s_plan[mid] <= pos) lo = mid; else hi = mid;
        }
        const bool group = it.group = lo < p.R;
        const int units = group ? p.units_group : p.units_row, unit_places = p.plan_unit[lo];
        const FastDiv cost = group ? p.by_cost_group : p.by_cost_row;
        const int pages = fast_div(unit_places - kSharedPiece, cost);
        const int u = (pos - s_plan[lo]) / unit_places, at = pos - s_plan[lo] - u * unit_places;
        const int to = min(unit_places, at + end - pos);
        const int blocks = units / p.Hkv, all = group ? p.K * G : G, blk = u % blocks;
        it.hkv = u / blocks;
        const int r = group ? lo : static_cast<int>(fast_div(lo - p.R, p.by_rows)), common = p.plan_tokens[lo], leader = p.plan_leader[lo];
        it.cols = min(C::COLS, all - blk * C::COLS);
        it.qh = r * p.Hkv + it.hkv;
        it.row = group ? leader : lo - p.R;
        it.col0 = (group ? 0 : (lo - p.R - r * p.K) * G) + blk * C::COLS;
        const int page0 = shared_page_of(at, cost, pages);
        it.n_pages = shared_page_of(to, cost, pages) - page0;
        it.page0 = page0 + (group ? 0 : common / kPageTokens);
        it.limit0 = it.page0 * kPageTokens;
        it.tokens = min((group ? common : shared_len(p, it.row)) - it.limit0, it.n_pages * kPageTokens);
        // rows of a group that end before the common tokens do
        it.ragged = false;
        if (group) {
            bool shorter = false;
            for (int k = lane; k < p.K; k += 32) {
                const int n = shared_len(p, r * p.K + k);
                shorter |= n > 0 && n < it.limit0 + it.tokens;      // (rows without tokens are left out at the end)
            }
            it.ragged = __any_sync(0xffffffffu, shorter);
        }
        const int64_t slot = me + static_cast<int64_t>(group ? lo : lo - p.R) * units + u;
        it.out = group ? slot * p.rows_group : p.base_row + slot * p.rows_row;
        it.next = pos + to - at;
        return it;
    };

    const uint32_t blk_stride = static_cast<uint32_t>(p.Hkv) * C::PAGE_BYTES;
    const uint64_t policy = l2_evict_first_policy();
    // A lane's rows of S: the page tokens whose weights the transposition then hands to the lanes that have those tokens'
    // values, in the order of their registers (register j of lane tg: token 4 tg + (j + tg) % 4 where ROT is set)
    const int q4 = g >> 1, turn = C::ROT ? q4 : 0, tokA = 4 * q4 + (((g & 1) + turn) & 3), tokB = 4 * q4 + (((g & 1) + 2 + turn) & 3);
    const uint32_t koffA = tokA * C::PDK + slice_word<C::KSB>(tg), koffB = tokB * C::PDK + slice_word<C::KSB>(tg), ksh = slice_shift<C::KSB>(tg);
    const uint32_t noff = C::OFF_KN + 8 * q4, vsh = slice_shift<C::VSB>(g);
    const uint32_t sel_norms = (2 * (tokA & 3)) * 0x11u + 0x10u + ((2 * (tokB & 3)) * 0x11u + 0x10u) * 0x100u;     // the two tokens' of a quad's fp16 norms
    const uint32_t lk_lane = window | (BK == 2 ? (lane & 15) * 8 : lane * 4);
    const uint32_t lv_lane = window | 128u | (BV == 2 ? (lane & 15) * 8 : lane * 4);
    uint32_t taken = 0, q_parity = 0;     // pages that the warp has taken from its ring: buffer taken % RING, its parity (taken / RING) % 2
    bool lost = false;        // a wait ran out: nothing is requested any more, and the warp's pieces are NaN
    bool bad_any = false;
#ifdef FTQ_TEST_WAIT_EXPIRY
    // a page, or where a group has five rows the queries
    bool test_drop = blockIdx.x == 0 && warp == 5 && p.K != 5, test_drop_q = blockIdx.x == 0 && warp == 5 && p.K == 5;
#endif

    auto walk = [&](auto tiles_tag, const SharedPiece& it) {
        constexpr int TILES = decltype(tiles_tag)::value;
        const uint8_t* const base = p.pool + static_cast<int64_t>(it.hkv) * C::PAGE_BYTES;
        int bad = INT32_MAX;
        // block ids of pages k0 .. k0 + 31 of the piece; an id outside the pool is replaced by 0, and the first such page remembered
        auto load_ids = [&](int k0) {
            const int k = k0 + lane;
            int id = 0;
            if (k < it.n_pages) {
                id = p.block_table[static_cast<int64_t>(it.row) * p.max_blocks + it.page0 + k];
                if (static_cast<uint32_t>(id) >= static_cast<uint64_t>(p.num_blocks)) {
                    id = 0;
                    bad = min(bad, k);
                }
            }
            return id;
        };
        // page k of the piece to the ring, by the lane that has its id
        const uint32_t first_page = taken;
        auto request = [&](int ids, uint32_t k) {
            const uint32_t rb = (first_page + k) % C::RING;
            if (lane == (k & 31)) {
                mbar_expect_tx(my_bars + 8 * rb, C::PAGE_BYTES);
#ifdef FTQ_TEST_WAIT_EXPIRY
                const bool drop = test_drop && k == 0;    // (see kMbarSpinLimit)
                test_drop = false;
                if (!drop)
#endif
                bulk_g2s_hint(my_ring + rb * C::PAGE_BYTES, base + static_cast<uint64_t>(static_cast<uint32_t>(ids)) * blk_stride, C::PAGE_BYTES, my_bars + 8 * rb, policy);
            }
            __syncwarp();
        };
        int ids = load_ids(0), ids_next = load_ids(32);
        const bool requested = !lost;
        if (requested) {
            if (lane == 0) {
                mbar_expect_tx(q_bar, it.cols * D * 2);
#ifdef FTQ_TEST_WAIT_EXPIRY
                const bool drop = test_drop_q;
                test_drop_q = false;
                if (!drop)
#endif
                bulk_g2s_hint(my_q, p.q_rows + (static_cast<int64_t>(it.qh) * p.K * G + it.col0) * (D * 2), it.cols * D * 2, q_bar, policy);
            }
            __syncwarp();
#pragma unroll
            for (int k = 0; k < C::RING; k++)
                if (k < it.n_pages) request(ids, static_cast<uint32_t>(k));
        }
        SharedState<D, BK, BV, TILES> st;
#pragma unroll
        for (int nt = 0; nt < TILES; nt++) {
#pragma unroll
            for (int mt = 0; mt < 2 * NMT; mt++)
#pragma unroll
                for (int i = 0; i < 4; i++) st.o[nt][mt][i] = 0.f;
            st.m[nt][0] = st.m[nt][1] = 0.f;
            st.l[nt][0] = st.l[nt][1] = 0.f;
        }
        st.vlimit = 0.f;
        st.vscale = 1.f;
        const uint32_t q_lane = my_q + g * (D * 2), q_odd = (((it.col0 + g) & 1) * 64) ^ (tg * 16);
        if (!lost) lost = !__all_sync(0xffffffffu, mbar_wait(q_bar, q_parity));
        const bool no_queries = lost;
        q_parity ^= 1;

        auto row_len = [&](int col) { return shared_len(p, it.group ? it.qh / p.Hkv * p.K + (it.col0 + col) / G : it.row); };
        // tokens of a column from page k on
        auto tokens_of = [&](int col, int k) {
            const int left = it.tokens - k * kPageTokens;
            return it.ragged && col < it.cols ? min(left, row_len(col) - it.limit0 - k * kPageTokens) : left;
        };
        int k = 0;
        for (; k < it.n_pages; k++) {
            const uint32_t rb = taken % C::RING;
            // (every lane polls; the vote makes one answer of theirs)
            if (!lost) lost = !__all_sync(0xffffffffu, mbar_wait(my_bars + 8 * rb, taken / C::RING & 1));
            if (lost) break;
            taken++;
            const uint32_t page = my_ring + rb * C::PAGE_BYTES;
            uint32_t kw[2][C::KW], vw[4][C::VW];
            lds_slice<C::KSB>(page + koffA, ksh, kw[0]);
            lds_slice<C::KSB>(page + koffB, ksh, kw[1]);
            const uint2 kn2 = lds64(page + noff), vn2 = lds64(page + noff + (C::OFF_VN - C::OFF_KN));
            // ---- S = K Q^T
            float x[TILES][4];          // scores, then less the maximum, then weights
            {
                typename WK::template Run<C::KW> run[2];
#pragma unroll
                for (int r = 0; r < 2; r++) {
#pragma unroll
                    for (int j = 0; j < C::KW; j++) run[r].w[j] = kw[r][j];
                    WK::shift(run[r]);
                }
#pragma unroll
                for (int kb = 0; kb < NKB; kb += 2) {
                    uint32_t a[2][4];
#pragma unroll
                    for (int s = 0; s < 2; s++) {
                        WK::pairs(run[0], kb + s, lk_lane, a[s][0], a[s][2]);
                        WK::pairs(run[1], kb + s, lk_lane, a[s][1], a[s][3]);
                    }
#pragma unroll
                    for (int nt = 0; nt < TILES; nt++) {
                        const uint4 q = lds128(q_lane + nt * 8 * (D * 2) + ((kb / 2 * 64) ^ q_odd));
                        if (kb == 0) mma_16816_z(x[nt], a[0][0], a[0][1], a[0][2], a[0][3], q.x, q.y);
                        else mma_16816(x[nt], a[0][0], a[0][1], a[0][2], a[0][3], q.x, q.y);
                        mma_16816(x[nt], a[1][0], a[1][1], a[1][2], a[1][3], q.z, q.w);
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int u = C::ROT ? (j + tg) & 3 : j, slice = g ^ ((u & 2) << 1);
                lds_slice<C::VSB>(page + C::OFF_VC + (4 * tg + u) * C::PDV + slice_word<C::VSB>(slice), vsh, vw[j]);
            }
            // the buffer is free for the page RING further on
            __syncwarp();
            const int next = k + C::RING;
            if (next < it.n_pages) {
                if ((next & 31) == 0) {     // (a batch of ids ahead)
                    ids = ids_next;
                    ids_next = load_ids(next + 32);
                }
                request(ids, next);
            }

            // ---- softmax (base 2), per column; lanes of a column: the eight that differ in g
            const uint32_t knab = __byte_perm(kn2.x, kn2.y, sel_norms), vnab = __byte_perm(vn2.x, vn2.y, sel_norms);
            // A value whose norm is infinite, or none, makes no number of the columns that attend it: by its score, so that it is nothing
            // to those that it is masked for (0 times it would be no number either), nor to the scale of the others
            const __half2 vn_half = *reinterpret_cast<const __half2*>(&vnab), none = __hsub2(vn_half, vn_half);
            const uint32_t vn_fine = vnab & __hlt2_mask(vn_half, __half2half2(__ushort_as_half(0x7c00)));
            const float2 kn = __half22float2(__hadd2(*reinterpret_cast<const __half2*>(&knab), none));
            float2 vn = __half22float2(*reinterpret_cast<const __half2*>(&vn_fine));
            const int left = it.tokens - k * kPageTokens;
            const bool whole = left >= kPageTokens && !it.ragged;
            float most = -INFINITY;
#pragma unroll
            for (int nt = 0; nt < TILES; nt++)
#pragma unroll
                for (int i = 0; i < 4; i++) x[nt][i] = fmaf(x[nt][i], i < 2 ? kn.x : kn.y, -st.m[nt][i & 1]);
            if (!whole) {
                if (tokA >= left) vn.x = 0.f;
                if (tokB >= left) vn.y = 0.f;
#pragma unroll
                for (int nt = 0; nt < TILES; nt++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int mine = tokens_of(8 * nt + 2 * tg + h, k);
                        if (tokA >= mine) x[nt][h] = -INFINITY;
                        if (tokB >= mine) x[nt][2 + h] = -INFINITY;
                    }
            }
#pragma unroll
            for (int nt = 0; nt < TILES; nt++)
#pragma unroll
                for (int i = 0; i < 4; i++) most = fmaxf(most, x[nt][i]);
            if (__any_sync(0xffffffffu, k == 0 || most > kSharedSlack || fmaxf(vn.x, vn.y) > st.vlimit)) {
                float v = fmaxf(vn.x, vn.y), change = 1.f;
#pragma unroll
                for (int d = 4; d <= 16; d <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
                if (v > st.vlimit) {        // (norms are not negative, nor infinite here)
                    // 2^-e with the norm in [2^e, 2^(e + 1))
                    const float now = __uint_as_float((254u << 23) - (__float_as_uint(v) & 0x7f800000u));
                    change = now / st.vscale;
                    st.vscale = now;
                    st.vlimit = v * kSharedNorms;
                }
#pragma unroll
                for (int nt = 0; nt < TILES; nt++) {
                    float corr[2];
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        float m = fmaxf(x[nt][h], x[nt][2 + h]);
#pragma unroll
                        for (int d = 4; d <= 16; d <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
                        // (of a column that has no token in its first page there are none, see below)
                        const float up = k == 0 ? (m == -INFINITY ? 0.f : m) : fmaxf(m, 0.f);
                        corr[h] = k == 0 ? 0.f : fast_exp2(-up);
                        st.l[nt][h] *= corr[h];
                        corr[h] *= change;
                        st.m[nt][h] += up;
                        x[nt][h] -= up;
                        x[nt][2 + h] -= up;
                    }
#pragma unroll
                    for (int mt = 0; mt < 2 * NMT; mt++)
#pragma unroll
                        for (int i = 0; i < 4; i++) st.o[nt][mt][i] *= corr[i & 1];
                }
            }
            vn.x *= st.vscale;
            vn.y *= st.vscale;
            uint32_t pb[TILES][2];
#pragma unroll
            for (int nt = 0; nt < TILES; nt++) {
#pragma unroll
                for (int i = 0; i < 4; i++) x[nt][i] = fast_exp2(x[nt][i]);
                st.l[nt][0] += x[nt][0] + x[nt][2];
                st.l[nt][1] += x[nt][1] + x[nt][3];
                pb[nt][0] = movmatrix_trans(pack_weights(x[nt][0] * vn.x, x[nt][1] * vn.x));
                pb[nt][1] = movmatrix_trans(pack_weights(x[nt][2] * vn.y, x[nt][3] * vn.y));
            }
            // ---- O^T += V^T P^T
            {
                typename WV::template Run<C::VW> run[4];
                WV::merge(vw[0], vw[1], run[0], run[1]);
                WV::merge(vw[2], vw[3], run[2], run[3]);
#pragma unroll
                for (int j = 0; j < 4; j++) WV::shift(run[j]);
#pragma unroll
                for (int m2 = 0; m2 < NMT; m2++) {
                    uint32_t e[4], f[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) WV::pairs(run[j], m2, lv_lane, e[j], f[j]);
#pragma unroll
                    for (int nt = 0; nt < TILES; nt++) {
                        mma_16816(st.o[nt][2 * m2], e[0], e[1], e[2], e[3], pb[nt][0], pb[nt][1]);
                        mma_16816(st.o[nt][2 * m2 + 1], f[0], f[1], f[2], f[3], pb[nt][0], pb[nt][1]);
                    }
                }
            }
        }
        // (a warp that gives up waits once more for each copy that is on its way, so that none comes after the CTA has left; as long as
        // a wait may take)
        if (lost && requested) {
            if (no_queries) mbar_wait(q_bar, q_parity ^ 1);
            for (const int last = min(k + C::RING, it.n_pages); k < last; k++, taken++) mbar_wait(my_bars + 8 * (taken % C::RING), taken / C::RING & 1);
        }
        // ---- the piece's rows: O in coordinates (D/8) g .. + D/8 of columns 2 tg, 2 tg + 1, (m, l) behind them
        bad = __reduce_min_sync(0xffffffffu, bad);
        bad_any |= bad != INT32_MAX;
        // (rows that end before the piece, or the first bad page of it, have lost nothing)
        const bool spoilt = lost || bad != INT32_MAX;
        const int sound = it.limit0 + (lost || !spoilt ? 0 : bad * kPageTokens);
#pragma unroll
        for (int nt = 0; nt < TILES; nt++) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int col = 8 * nt + 2 * tg + h;
                float l = st.l[nt][h];
#pragma unroll
                for (int d = 4; d <= 16; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
                if (col >= it.cols) continue;
                const bool none = spoilt && row_len(col) > sound;
                const float scale = none ? __int_as_float(0x7fc00000) : p.inv_v_scale / st.vscale;
                float* const to = p.rows + (it.out + col) * ROW;
#pragma unroll
                for (int f = 0; f < NMT; f++)
                    *reinterpret_cast<float4*>(to + (D / 8) * g + 4 * f) =
                        make_float4(st.o[nt][2 * f][h] * scale, st.o[nt][2 * f][2 + h] * scale, st.o[nt][2 * f + 1][h] * scale, st.o[nt][2 * f + 1][2 + h] * scale);
                if (g == 0)
                    *reinterpret_cast<float2*>(to + D) =
                        make_float2(none ? __int_as_float(0x7fc00000) : l == 0.f ? -INFINITY : st.m[nt][h], l);
            }
        }
        __syncwarp();       // (the next piece's queries come to where these were read)
    };

    for (int pos = static_cast<int>(from); pos < end;) {
        const SharedPiece it = locate(pos);
        pos = it.next;
        if (it.n_pages == 0) continue;      // (a share that ends among a unit's places on its own)
        if (NT > 1 && it.cols <= 8) walk(std::integral_constant<int, 1>{}, it);
        else walk(std::integral_constant<int, NT>{}, it);
    }
    if (lane == 0 && (lost || bad_any)) atomicOr(p.status, (lost ? kStatusWaitExpired : 0) | (bad_any ? kStatusBadBlock : 0));
}

// ------------------------------------------------------------------ merge
// A warp per row, or WARPS = 4 where rows are few: each takes a piece at a time, a lane D / 32 coordinates of it, so that the loads of
// several pieces are on their way together (1536 rows of heads of 256 with up to 50 pieces: an octet a piece, a warp a row 40 us, as long as the
// attention; 15 now.  8192 rows of a few pieces: an octet a row 15 us).
template <int D, typename OT, int WARPS>
__global__ void __launch_bounds__(128) shared_merge_kernel(const __grid_constant__ SharedAttnParams p) {
    constexpr int E = D / kOctet, ROW = D + 4, PL = D / 32;
    __shared__ float s_max[4], s_sum[4];
    __shared__ __align__(16) float s_all[4 * D];
    const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % WARPS, t = lane & 7;
    float* const s_acc = s_all + (threadIdx.x >> 5) / WARPS * WARPS * D;      // the row's warps'
    let_next_kernel_start();
    after_previous_kernel();
    const int64_t n_rows = static_cast<int64_t>(p.R) * p.K * p.Hq;
    const int64_t mine = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / (32 * WARPS);
    const int64_t v = mine < n_rows ? mine : n_rows - 1;
    const int b = fast_div(static_cast<uint32_t>(v), p.by_hq), hq = static_cast<int>(v) - b * p.Hq, G = p.by_group.d, h = fast_div(hq, p.by_group), r = fast_div(b, p.by_rows);
    const int* const tail = p.plan + p.R + p.R * p.K;
    const FastDiv share{static_cast<uint32_t>(tail[1]), static_cast<uint32_t>(tail[2]), static_cast<uint32_t>(tail[3])};
    // the row's pieces of its group's unit, and of its own: rows `step` floats apart
    struct Parts { const float* first; int n, step; };
    auto parts_of = [&](bool group) {
        const int e = group ? r : p.R + b, units = group ? p.units_group : p.units_row;
        const int i = (group ? (b - r * p.K) * G : 0) + hq - h * G, blk = fast_div(i, p.by_cols), u = h * (group ? p.blocks_group : p.blocks_row) + blk;
        const int e0 = p.plan[e], places = p.plan_unit[e];
        const FastDiv cost = group ? p.by_cost_group : p.by_cost_row;
        Parts x{nullptr, 0, (group ? p.rows_group : p.rows_row) * ROW};
        if (places == 0) return x;
        const int pages = fast_div(places - kSharedPiece, cost), pos = e0 + u * places;
        int c0 = fast_div(pos, share), c1 = fast_div(pos + places - 1, share);
        // (a share that ends among the unit's places on its own has none of its pages, nor has one that begins behind its last page's first place)
        if (shared_page_of(static_cast<int>(min(static_cast<int64_t>(c0 + 1) * share.d - pos, static_cast<int64_t>(places))), cost, pages) == 0) c0++;
        if (c1 > c0 && shared_page_of(static_cast<int>(c1 * share.d) - pos, cost, pages) == pages) c1--;
        x.n = c1 - c0 + 1;
        const int64_t slot = c0 + static_cast<int64_t>(group ? e : e - p.R) * units + u;
        x.first = p.rows + ((group ? 0 : p.base_row) * ROW + slot * x.step + static_cast<int64_t>(i - blk * p.cols) * ROW);
        return x;
    };
    const bool any = shared_len(p, b) > 0;
    const Parts a = parts_of(true), z = parts_of(false);
    auto row_of = [&](int k) { return k < a.n ? a.first + static_cast<int64_t>(k) * a.step : z.first + static_cast<int64_t>(k - a.n) * z.step; };
    const int n = any ? a.n + z.n : 0;
    float M = -INFINITY, L = 0.f, acc[E];
    // (0 of a piece without a token of this row, a group's common ones that lie behind its end; not a number where the piece's
    // rows are none)
    auto weight = [&](float m) { return m == -INFINITY ? 0.f : fast_exp2(m - M); };
    for (int k = 32 * warp + lane; k < n; k += 32 * WARPS) M = fmaxf(M, row_of(k)[D]);
    __syncwarp();
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
    if constexpr (WARPS > 1) {
        if (lane == 0) s_max[warp] = M;
        __syncthreads();
        M = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
    }
    float mine_acc[PL];
#pragma unroll
    for (int i = 0; i < PL; i++) mine_acc[i] = 0.f;
#pragma unroll 4
    for (int k = warp; k < n; k += WARPS) {
        const float* const row = row_of(k);
        const float m = row[D], l = row[D + 1];
        float x[PL];
        if constexpr (PL == 2) {
            *reinterpret_cast<float2*>(x) = *reinterpret_cast<const float2*>(row + 2 * lane);
        } else {
#pragma unroll
            for (int i = 0; i < PL; i += 4) *reinterpret_cast<float4*>(x + i) = *reinterpret_cast<const float4*>(row + PL * lane + i);
        }
        const float f = weight(m);
        L = fmaf(l, f, L);
#pragma unroll
        for (int i = 0; i < PL; i++) mine_acc[i] = fmaf(x[i], f, mine_acc[i]);
    }
#pragma unroll
    for (int i = 0; i < PL; i++) s_acc[warp * D + PL * lane + i] = mine_acc[i];
    if constexpr (WARPS > 1) {      // each warp's sums, then the first warp's of all
        if (lane == 0) s_sum[warp] = L;
        __syncthreads();
        if (warp > 0) return;
        L = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
    } else {
        __syncwarp();
    }
#pragma unroll
    for (int x = 0; x < E / 8; x++)
#pragma unroll
        for (int c = 0; c < 8; c++) {
            const float* const at = s_acc + 8 * (t + 8 * x) + c;
            acc[8 * x + c] = WARPS > 1 ? (at[0] + at[D]) + (at[2 * D] + at[3 * D]) : at[0];
        }
    const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int k = 0; k < E; k++) acc[k] *= inv;
    octet_fwht<E>(acc, lane);
#pragma unroll
    for (int k = 0; k < E; k++) {
        if (mine >= n_rows || (k & 3) != (lane >> 3)) continue;
        const float x = acc[k] * p.rsqrt_d;
        reinterpret_cast<OT*>(p.out)[v * D + t + 8 * k] = from_float<OT>(__uint_as_float(__float_as_uint(x) ^ sign_mask(p.signs, t + 8 * k)));
    }
}

}  // namespace ftq
