// Attention of drafted token trees over the paged cache: every node attends the context and the nodes in its mask.
//
// The nodes of a tree are few queries over one context.  With the queries on the M side of the products (as in the chunk
// kernel, ftq_attn_chunk.cuh) a tile of 128 rows is full from 32 nodes of a GQA group of 4 on only, and all of a smaller
// tree's products are padding.  Here the tokens are the M side, so that a product is as wide as the tree:
//
//   S^T = K.Q^T    tcgen05.mma, M = 128 tokens, N = rows (node x head of the group, padded to 16), K = D; the dequantised
//                  keys go straight from registers to TMEM (A operand), the queries lie in shared memory (K-major)
//   softmax        a thread per token: the norms of its key and value are two registers, and whether a row attends it is a
//                  bit; the maxima that the weights refer to are lazy (below), so that no value crosses lanes in a tile
//   O^T += V^T.P^T  M = coordinates, N = rows, K = tokens; V (A operand, MN-major) and the weights p * |v| (B operand,
//                  MN-major: a thread stores its token's row) in shared memory; O stays in TMEM
//
// The order of the coordinates inside K's products is free, so is that of V's coordinates on the lanes: both are chosen so
// that a quad of lanes reads a token's codes as they lie (16 bytes a lane, whole half pages a warp) and no value is
// moved between lanes: a 16x256b store to TMEM puts lane 4g + t's codes into row g, columns 8j + 2t.
//
// Lazy maxima: a row's weights refer to the largest score of an earlier tile (m); while no score is above m + 13 (base 2) a
// tile costs one vote per 32 rows.  Otherwise the warpgroup finds the new maxima and rescales O and the sums.
// (With a slack of 3, as in the decode kernels, half of the tiles did: of 32 rows there is always one that has found a
// larger score.)  Weights are fp16: |v| is scaled by a power of two, so that the largest so far is 1 to 2, and again when
// one of 4 or more comes; p * |v| is then at most 2^15, and a weight of 2^-14 of the largest still has all its bits.
// Queries are scaled the same way.  Scores, sums and O are fp32.
//
// Work: units (sequence, KV head, row tile) in a line of places, a place per tile of 128 tokens and kTreePiece more per
// unit, cut into equal shares, one per CTA (one CTA per SM).  Every piece leaves its rows (O, m, l) in the
// workspace; tree_merge_kernel joins the pieces of a unit, rotates back and stores.
//
// Every wait is bounded.  After one has run out nothing waits any more, the CTA's rows become NaN and the status word says
// so.  Block ids outside the pool are not followed: the rows that attend a token of such a page are NaN.
#pragma once

#include "ftq_attn_chunk.cuh"
#include "ftq_serve_launch.h"

namespace ftq {

constexpr int kTreeTile = 128;         // tokens of a tile
constexpr int kTreePiece = 3;          // places that a unit costs besides its tiles
constexpr int kTreeMaxSeqs = 1024;     // sequences of a launch
constexpr float kTreeSlack = 13.f, kTreeGrowth = 4.f;

struct TreeAttnParams {
    const void* q;              // [B, T, Hq, D]
    const uint8_t* pool;        // one layer: [num_blocks, Hkv, page_bytes]
    const int32_t* block_table; // [B, max_blocks]
    const int32_t* seq_lens;    // [B], the tree included
    const int32_t* tree_lens;   // [B] or NULL (= T)
    const int32_t* masks;       // [B, T, W]
    int64_t num_blocks;
    int max_blocks, max_seq, T, W, Hq, Hkv, q_dtype, B, row_tiles;
    FastDiv group;              // Hq / Hkv
    float q_scale;              // softmax scale / (key table's scale) * log2(e) / sqrt(D)
    float inv_v_scale;
    int* plan;                  // [B + 2]: first place of every sequence, all places, places of a share
    float* whole;               // rows of units that one CTA has: [B][Hkv * row_tiles][N][D + 4]
    float* cut;                 // rows of the others: [grid][2][N][D + 4]
    unsigned long long* errors; // expired waits, bad block ids (see ChunkAttnParams)
    unsigned long long epoch;
    Codebook lk, lv;            // scaled for their fp16 rounding
    SignBits signs;
};

// The part of a unit that a CTA has: places [off, off_end) of its tiles + kTreePiece.
__host__ __device__ __forceinline__ int tree_tile_of(int off) { return off > kTreePiece ? off - kTreePiece : 0; }

template <int D, int BK, int BV, int N>
struct TreeCfg {
    static constexpr int WG = N > 32 ? 2 : 1;              // softmax warpgroups
    static constexpr int CW = N / WG;                      // rows of one
    static constexpr int CH = CW < 32 ? CW : 32, NCH = CW / CH;
    // warps: softmax; keys; values; the products; addresses and norms; queries and masks
    static constexpr int SM_WARPS = 4 * WG, W_K = SM_WARPS, W_V = W_K + 4, W_MMA = W_K + 8, W_FEED = W_MMA + 1, W_Q = W_MMA + 2;
    static constexpr int Q_WARPS = 2, WARPS = W_Q + Q_WARPS, THREADS = 32 * WARPS;
    // Registers: 16 warps have 128 each; of the 96 that 20 start with, the softmax warps get some of the others'
    // (the sum stays what the block was launched with)
    static constexpr bool SPLIT = WARPS == 20;
    static constexpr int REGS = SPLIT ? 96 : 128, R_SM = N == 128 ? 152 : 112, R_DQ = N == 128 ? 56 : 80, R_Q = N == 128 ? 64 : 96;
    static_assert(!SPLIT || SM_WARPS * R_SM + 8 * R_DQ + 4 * R_Q <= WARPS * REGS, "");
    static constexpr int AHEAD = N == 128 || D == 256 ? 1 : 2;   // tiles whose codes are under way in registers
    static constexpr int PDK = packed_dim(D, BK), PDV = packed_dim(D, BV);
    static constexpr int OFF_KN = kPageTokens * PDK;
    static constexpr int OFF_VC = OFF_KN + 2 * kPageTokens;
    static constexpr int OFF_VN = OFF_VC + kPageTokens * PDV;
    static constexpr int PAGE_BYTES = OFF_VN + 2 * kPageTokens;
    static constexpr int ATOMS = D / 64, MB = D == 256 ? 2 : 1;   // 64-coordinate atoms of a row; M blocks of O^T
    // V in slots of 64 tokens; P in one or two buffers of 128 tokens, 64 rows to an atom
    static constexpr int VS = D == 256 ? 3 : 4, V_SLOT = 64 * D * 2;
    static constexpr int PST = D == 256 || (D == 128 && N == 128) ? 1 : 2, P_ATOM = kTreeTile * 128, P_BUF = P_ATOM * ((N + 63) / 64);
    static constexpr int Q_BYTES = N * D * 2, MW = (N + 31) / 32, MASK_BYTES = kTreeMaxNodes * MW * 4;
    // shared-memory addresses: the dynamic part (the only one) starts in the first 4 KB; the look-up window takes 64 KB at
    // 64 KB, V follows it (at head_dim 64 a product reads an atom beyond its slot, into the next or P: unused rows)
    static constexpr int WINDOW = 65536, LOW = 4096, A_V = 131072;
    static constexpr bool P_HIGH = VS * V_SLOT + PST * P_BUF <= 99 * 1024;
    static constexpr int A_P = P_HIGH ? A_V + VS * V_SLOT : LOW;
    static constexpr int A_Q = P_HIGH ? LOW : LOW + PST * P_BUF;
    // queries and masks of two pieces where they fit
    static constexpr int QB = A_Q + 2 * (Q_BYTES + MASK_BYTES) + 8 * 1024 <= WINDOW ? 2 : 1;
    static constexpr int A_MASK = A_Q + QB * Q_BYTES;
    static constexpr int A_NM = A_MASK + QB * MASK_BYTES;  // - reference maximum; factors of l and O
    static constexpr int A_LC = A_NM + N * 4, A_CORR = A_LC + N * 4;
    static constexpr int A_RED = A_CORR + N * 4;           // [SM_WARPS][32], [SM_WARPS]
    static constexpr int A_FIRST = A_RED + SM_WARPS * 33 * 4;   // [kTreeMaxSeqs + 1]
    static constexpr int A_MISC = (A_FIRST + (kTreeMaxSeqs + 1) * 4 + 15) / 16 * 16;
    // rings: pieces (struct TreePiece); block ids of a tile's pages; where they lie (64 bits each); the norms of a tile's
    // keys and of its values
    static constexpr int PIECES = 8, PAGES = 8, NORMS = D == 256 ? 4 : 8;
    static constexpr int A_PIECE = A_MISC + 256, A_ID = A_PIECE + PIECES * 48, A_PAGE = A_ID + PAGES * 32, A_NORM = A_PAGE + PAGES * 64;
    static constexpr int A_BAR = A_NORM + NORMS * 4 * kTreeTile;
    static constexpr int END_LOW = A_BAR + 592;
    static constexpr int SMEM_BYTES = A_V + VS * V_SLOT + (P_HIGH ? PST * P_BUF : 0);
    static_assert(END_LOW <= WINDOW && SMEM_BYTES <= 227 * 1024 && THREADS <= 1024, "");
    // TMEM columns
    static constexpr int COL_K = 0, COL_S = D, COL_O = D + 2 * N;
    static_assert(COL_O + MB * N <= 512, "");
};

__device__ __forceinline__ float warp_max(float x) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;\n" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ void tc_st_16x256b_x4(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::
            "r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
            "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
// The products are issued by one elected lane inside a branch: 32 cycles a product of 64 columns, what the tensor core
// takes.  (The form of the chunk kernel, a whole warp with a predicate on each instruction, takes 66, whatever the width.)
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
    return r != 0;
}
__device__ __forceinline__ void one_mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t hi, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n.reg .pred p;\n.reg .b64 da, db;\nmov.b64 da, {%1, %3};\nmov.b64 db, {%2, %3};\nsetp.ne.b32 p, %5, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n}\n" ::"r"(d), "r"(a), "r"(b), "r"(hi), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void one_mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t hi, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n.reg .pred p;\n.reg .b64 db;\nmov.b64 db, {%2, %3};\nsetp.ne.b32 p, %5, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n}\n" ::"r"(d), "r"(a), "r"(b), "r"(hi), "r"(idesc), "r"(acc) : "memory");
}
// 32 lanes x NC columns, one row per lane, complete
template <int NC>
__device__ __forceinline__ void tc_load(uint32_t addr, uint32_t (&r)[NC]) {
    if constexpr (NC == 32) {
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,"
            "%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\ntcgen05.wait::ld.sync.aligned;\n"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
              "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
              "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
              "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
            : "r"(addr) : "memory");
    } else {
        tc_ld16(addr, r);
        tc_wait_ld(r);
    }
}
__device__ __forceinline__ uint32_t f2h2(float lo, float hi) {
    uint32_t h;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(h) : "f"(hi), "f"(lo));
    return h;
}
// barrier of some warps; true if any of their threads says so
template <int THREADS = 128>
__device__ __forceinline__ bool group_any(int id, bool mine) {
    uint32_t r;
    __syncwarp();
    asm volatile("{\n.reg .pred p, q;\nsetp.ne.u32 p, %1, 0;\nbarrier.cta.red.or.pred q, %2, %3, p;\nselp.u32 %0, 1, 0, q;\n}\n"
                 : "=r"(r) : "r"(static_cast<uint32_t>(mine)), "r"(id), "n"(THREADS) : "memory");
    return r != 0;
}

// A piece of a CTA's share: some tiles of one unit.
struct TreePiece {
    int b, hkv, row0, rows;     // sequence, KV head, first row and rows of the row tile
    int tile0, n_tiles;         // (n_tiles = 0: there is none any more)
    int seq, ctx;               // tokens, tokens before the tree
    float* out;                 // [rows][D + 4]
    int64_t spare;
};
static_assert(sizeof(TreePiece) == 48, "");

// Asynchronous copies of a few bytes to shared memory (coherent: through L1, like an ordinary load).
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;\n" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}

// A lane's codes of a tile: its runs in two rows of two pages.
template <int XW>
struct TreeCodes {
    uint32_t w[2][2][XW];
};
// SB bytes into words, on the widest loads that their alignment allows (a run starts at a multiple of its size).
template <int SB, int XW>
__device__ __forceinline__ void tree_fetch(const uint8_t* src, uint32_t (&w)[XW]) {
    if constexpr (SB % 16 == 0) {
#pragma unroll
        for (int i = 0; i < SB / 16; i++) {
            const uint4 x = reinterpret_cast<const uint4*>(src)[i];
            w[4 * i] = x.x; w[4 * i + 1] = x.y; w[4 * i + 2] = x.z; w[4 * i + 3] = x.w;
        }
    } else if constexpr (SB % 8 == 0) {
#pragma unroll
        for (int i = 0; i < SB / 8; i++) {
            const uint2 x = reinterpret_cast<const uint2*>(src)[i];
            w[2 * i] = x.x; w[2 * i + 1] = x.y;
        }
    } else if constexpr (SB % 4 == 0) {
#pragma unroll
        for (int i = 0; i < SB / 4; i++) w[i] = reinterpret_cast<const uint32_t*>(src)[i];
    } else {   // six bytes on a two-byte boundary
        static_assert(SB == 6, "");
        const uint16_t* h = reinterpret_cast<const uint16_t*>(src);
        w[0] = h[0] | static_cast<uint32_t>(h[1]) << 16;
        w[1] = h[2];
    }
}

template <int D, int BK, int BV, int N>
__global__ void __launch_bounds__(TreeCfg<D, BK, BV, N>::THREADS, 1)
tree_attn_kernel(const __grid_constant__ TreeAttnParams p) {
    using C = TreeCfg<D, BK, BV, N>;
    constexpr int E = D / kOctet, ROW = D + 4, CH = C::CH, NCH = C::NCH;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    const uint32_t raw = static_cast<uint32_t>(__cvta_generic_to_shared(smem_raw));
    auto at = [&](uint32_t a) { return smem_raw + (a - raw); };
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    uint32_t* const misc = reinterpret_cast<uint32_t*>(at(C::A_MISC));   // 0: TMEM, 1: a wait ran out, 2, 3: largest |q|, 8..: scan, 40..: heads
    volatile uint32_t* const gave_up = misc + 1;
    constexpr uint32_t BAR = C::A_BAR;
    constexpr uint32_t k_full = BAR, k_empty = BAR + 16, s_full = BAR + 32, s_free = BAR + 48, p_full = BAR + 64, o_done = BAR + 80,
                       v_full = BAR + 96, v_empty = BAR + 128, drained = BAR + 160;
    constexpr uint32_t q_full = BAR + 168, q_empty = BAR + 184, o_free = BAR + 200, page_full = BAR + 208, page_empty = BAR + 272,
                       norm_full = BAR + 336, norm_empty = BAR + 400,
                       piece_full = BAR + 464, piece_empty = BAR + 528;
    constexpr int W_V = C::W_V, W_MMA = C::W_MMA;

    // ---- look-up window (struct Window): 256 rows of 256 bytes, keys in the first half of a row, values in the second
    {
        auto build = [&](int off, auto bits, const Codebook& cb) {
            constexpr int NB = decltype(bits)::value;
            const float lev = cb.v[lane & 15];
            for (int e = warp; e < 256; e += C::WARPS) {
                auto pair = [&](int lo, int hi) {
                    const __half2 h = __floats2half2_rn(__shfl_sync(0xffffffffu, lev, lo), __shfl_sync(0xffffffffu, lev, hi));
                    return *reinterpret_cast<const uint32_t*>(&h);
                };
                uint32_t x;
                if constexpr (NB == 4) {
                    x = pair(e & 15, e >> 4);
                } else if constexpr (NB == 3) {
                    x = pair(e & 7, (e >> 3) & 7);
                } else {
                    const uint32_t a = pair(e & 3, (e >> 2) & 3), b = pair((e >> 4) & 3, e >> 6);
                    x = (lane & 1) ? b : a;
                }
                *reinterpret_cast<uint32_t*>(at(C::WINDOW + e * 256 + off + lane * 4)) = x;
            }
        };
        build(0, std::integral_constant<int, BK>{}, p.lk);
        build(128, std::integral_constant<int, BV>{}, p.lv);
    }
    if (warp == W_MMA) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(static_cast<uint32_t>(C::A_MISC)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n");
        if (lane == 0) {
            for (int i = 0; i < 2; i++) {
                mbar_init(k_full + 8 * i, 4);
                mbar_init(k_empty + 8 * i, 1);
                mbar_init(s_full + 8 * i, 1);
                mbar_init(s_free + 8 * i, C::SM_WARPS);
                mbar_init(p_full + 8 * i, C::SM_WARPS);
                mbar_init(o_done + 8 * i, 1);
            }
            for (int i = 0; i < 4; i++) {
                mbar_init(v_full + 8 * i, 4);
                mbar_init(v_empty + 8 * i, 1);
            }
            for (int i = 0; i < C::QB; i++) {
                mbar_init(q_full + 8 * i, C::Q_WARPS);
                mbar_init(q_empty + 8 * i, 1 + C::SM_WARPS);
            }
            for (int i = 0; i < C::PAGES; i++) {
                mbar_init(page_full + 8 * i, 1);
                mbar_init(page_empty + 8 * i, 8);
            }
            for (int i = 0; i < C::NORMS; i++) {
                mbar_init(norm_full + 8 * i, 1);
                mbar_init(norm_empty + 8 * i, C::SM_WARPS);
            }
            for (int i = 0; i < C::PIECES; i++) {
                mbar_init(piece_full + 8 * i, 1);
                mbar_init(piece_empty + 8 * i, C::SM_WARPS + 1 + C::Q_WARPS);
            }
            mbar_init(o_free, C::SM_WARPS);
            mbar_init(drained, 1);
            mbar_fence_init();
        }
        tc_fence_before();
    }
    if (tid == 0) misc[1] = misc[2] = misc[3] = 0;
    after_previous_kernel();    // (nothing in global memory was touched so far)

    // ---- the line of places
    const int U = p.Hkv * p.row_tiles, G = gridDim.x, cta = blockIdx.x;
    int* const first = reinterpret_cast<int*>(at(C::A_FIRST));
    {
        int base = 0;
        for (int b0 = 0; b0 < p.B; b0 += C::THREADS) {
            const int b = b0 + tid;
            const int len = b < p.B ? max(0, min(p.seq_lens[b], p.max_seq)) : 0;
            const int v = b < p.B ? U * ((len + kTreeTile - 1) / kTreeTile + kTreePiece) : 0;
            int x = v;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, x, d);
                if (lane >= d) x += y;
            }
            __syncthreads();
            if (lane == 31) misc[8 + warp] = x;
            __syncthreads();
            int sum = 0, before = 0;
            for (int w = 0; w < C::WARPS; w++) {
                before += w < warp ? static_cast<int>(misc[8 + w]) : 0;
                sum += misc[8 + w];
            }
            if (b < p.B) first[b] = base + before + x - v;
            base += sum;
        }
        if (tid == 0) first[p.B] = base;
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, misc[0], 0);
    const int total = first[p.B], share = (total + G - 1) / G;
    const int end = static_cast<int>(min(static_cast<int64_t>(total), static_cast<int64_t>(cta + 1) * share));
    if (cta == 0) {
        for (int b = tid; b <= p.B; b += C::THREADS) p.plan[b] = first[b];
        if (tid == 0) p.plan[p.B + 1] = share;
    }
    // bounded wait; once one has run out nobody waits any more
    auto wait = [&](uint32_t bar, uint32_t parity) {
#pragma unroll 1
        for (int i = 0; i < kChunkSpinLimit; i++) {
            if (mbar_try_wait(bar, parity & 1u)) return;
            if ((i & 63) == 63 && *gave_up) return;
        }
        *gave_up = 1;
    };

    // the first piece with tiles from a place on; moves on to the place behind it
    auto next_piece = [&](int& pos) {
        TreePiece pc{};
#pragma unroll 1
        while (pos < end && pc.n_tiles == 0) {
            int lo = 0, hi = p.B;
#pragma unroll 1
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (first[mid] <= pos) lo = mid; else hi = mid;
            }
            const int len = (first[lo + 1] - first[lo]) / U, rel = pos - first[lo], u = rel / len, off = rel - u * len;
            const int off_end = min(len, off + end - pos), t0 = tree_tile_of(off), t1 = tree_tile_of(off_end);
            pos += off_end - off;
            if (t1 <= t0) continue;
            pc.b = lo;
            pc.hkv = u / p.row_tiles;
            pc.row0 = (u - pc.hkv * p.row_tiles) * N;
            pc.rows = min(N, p.T * static_cast<int>(p.group.d) - pc.row0);
            pc.tile0 = t0;
            pc.n_tiles = t1 - t0;
            pc.seq = max(0, min(p.seq_lens[lo], p.max_seq));
            pc.ctx = pc.seq - min(p.tree_lens ? max(p.tree_lens[lo], 0) : p.T, min(p.T, pc.seq));
            pc.out = off == 0 && off_end == len ? p.whole + (static_cast<int64_t>(lo) * U + u) * N * ROW
                                                : p.cut + (2 * static_cast<int64_t>(cta) + (off == 0 ? 1 : 0)) * N * ROW;
        }
        return pc;
    };
    // piece n, and its slot back
    auto piece_at = [&](int n) {
        wait(piece_full + 8 * (n % C::PIECES), n / C::PIECES);
        __syncwarp();
        TreePiece pc = *reinterpret_cast<const TreePiece*>(at(C::A_PIECE + n % C::PIECES * 48));
        if (__any_sync(0xffffffffu, *gave_up != 0)) pc.n_tiles = 0;   // (what stands there may be no piece)
        if (lane == 0) mbar_arrive(piece_empty + 8 * (n % C::PIECES));
        return pc;
    };
    // the power of two that brings every query of a piece below 2^15: |rotated| <= D * largest |q|
    auto query_exponent = [&](int qb) {
        const float top = __uint_as_float(misc[2 + qb]) * (fabsf(p.q_scale) * D);
        return top > 0.f ? max(-120, min(120, 14 - ilogbf(top))) : 0;
    };

    // A piece's queries (rotated, scaled, fp16, K-major with 128-byte swizzle) and masks, by NW warps (thread `me` of them); the
    // first piece's by all warps, before they part.
    auto prepare_piece = [&](const TreePiece& pc, int qb, auto warps, int me) {
        constexpr int NW = decltype(warps)::value, OCTETS = 4 * NW;
        const int t8 = lane & 7, octet = me >> 3, group = static_cast<int>(p.group.d), rows = pc.rows, row0 = pc.row0;
        auto meet = [&] { group_any<32 * NW>(NW == C::WARPS ? 0 : 3, false); };
        auto query = [&](int r) {   // row r's 16-byte pieces: eight coordinates each
            const int i = fast_div(row0 + r, p.group), h = row0 + r - i * group;
            return static_cast<const uint4*>(p.q) + (((static_cast<int64_t>(pc.b) * p.T + i) * p.Hq + pc.hkv * group + h) * D) / 8;
        };
        auto widen = [&](const uint4& x, float (&o)[8]) {
            if (p.q_dtype == kBF16) load8<__nv_bfloat16>(reinterpret_cast<const __nv_bfloat16*>(&x), o);
            else load8<__half>(reinterpret_cast<const __half*>(&x), o);
        };
        // the largest query, for their common scale
        float top = 0.f;
#pragma unroll 4
        for (int k = me; k < rows * (D / 8); k += 32 * NW) {
            float v[8];
            widen(query(k / (D / 8))[k % (D / 8)], v);
#pragma unroll
            for (int c = 0; c < 8; c++) top = fabsf(v[c]) <= FLT_MAX ? fmaxf(top, fabsf(v[c])) : top;
        }
        __syncwarp();
        top = warp_max(top);
        if (me == 0) misc[2 + qb] = 0;
        meet();
        if (lane == 0) atomicMax(misc + 2 + qb, __float_as_uint(top));
        meet();
        const float up = p.q_scale * ldexpf(1.f, query_exponent(qb));
        uint4 x[D / 64];
        auto load = [&](int r) {
#pragma unroll
            for (int k = 0; k < D / 64; k++) x[k] = r < rows ? query(r)[t8 + 8 * k] : make_uint4(0, 0, 0, 0);
        };
        load(octet);
#pragma unroll 1
        for (int r = octet; r - octet < N; r += OCTETS) {
            float a[E];
#pragma unroll
            for (int k = 0; k < D / 64; k++) {
                float v[8];
                widen(x[k], v);
#pragma unroll
                for (int c = 0; c < 8; c++)
                    a[8 * k + c] = __uint_as_float(__float_as_uint(v[c] * up) ^ sign_mask(p.signs, load_coord(t8, 8 * k + c)));
            }
            load(r + OCTETS);
            octet_fwht<E>(a, lane);
            // Coordinate c = t8 + 8 k is code 4 jj + (c & 3) of lane t's run: place 16 jj + 4 t + (c & 3).  Two lanes have two
            // neighbours: of two k's the even lane stores the first, the odd lane the second.
            uint8_t* dst = at(C::A_Q + qb * C::Q_BYTES) + r * 128;
#pragma unroll
            for (int k = 0; k < E; k += 2) {
                const float other = __shfl_xor_sync(0xffffffffu, (t8 & 1) ? a[k] : a[k + 1], 1);
                const int c = (t8 & 6) + 8 * (k + (t8 & 1)), t = c / (D / 4), jj = (c % (D / 4)) / 4, place = 16 * jj + 4 * t + (c & 3);
                const uint32_t h = (t8 & 1) ? f2h2(other, a[k + 1]) : f2h2(a[k], other);
                if (r < N) *reinterpret_cast<uint32_t*>(dst + (place >> 6) * (N * 128) + ((((place & 63) >> 3) ^ (r & 7)) << 4) + (place & 7) * 2) = h;
            }
        }
        // which rows attend a node: bit r of its words
        if ((pc.tile0 + pc.n_tiles) * kTreeTile > pc.ctx) {
            uint32_t* const cm = reinterpret_cast<uint32_t*>(at(C::A_MASK)) + qb * (C::MASK_BYTES / 4);
            for (int k = me; k < (pc.seq - pc.ctx) * C::MW; k += 32 * NW) {
                const int node = k / C::MW, w = k % C::MW;
                uint32_t bits = 0;
                // (a node's heads are neighbours: a run of bits)
                const int r1 = min(rows, 32 * w + 32);
#pragma unroll 1
                for (int r = 32 * w; r < r1;) {
                    const int i = fast_div(row0 + r, p.group), stop = min(r1, (i + 1) * group - row0);
                    if ((static_cast<uint32_t>(p.masks[(static_cast<int64_t>(pc.b) * p.T + i) * p.W + (node >> 5)]) >> (node & 31)) & 1u)
                        bits |= (0xffffffffu >> (32 - (stop - r))) << (r & 31);
                    r = stop;
                }
                cm[k] = bits;
            }
        }
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
    };
    const int begin = static_cast<int>(min(static_cast<int64_t>(cta) * share, static_cast<int64_t>(end)));
    if (begin < end) {
        int pos = begin;
        const TreePiece pc = next_piece(pos);
        if (pc.n_tiles > 0) prepare_piece(pc, 0, std::integral_constant<int, C::WARPS>{}, tid);
    }
    __syncthreads();

    // (a warpgroup runs one and the same instruction)
    if constexpr (C::SPLIT && C::R_Q < C::REGS) {
        if (warp >= W_MMA) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(C::R_Q));
    }
    if (warp < C::SM_WARPS) {
        if constexpr (C::SPLIT) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(C::R_SM));
        // ================= softmax: a thread per token of the tile
        for (int n = 0, g0 = 0;; n++) {
            const TreePiece pc = piece_at(n);
            if (group_any(1 + (warp >> 2), pc.n_tiles == 0)) break;      // (all warps of the group, or none)
            const int qb = n % C::QB, rows = pc.rows, seq = pc.seq, ctx = pc.ctx, n_tiles = pc.n_tiles;
            const int wg = warp >> 2, quarter = warp & 3, my_tok = quarter * 32 + lane, bar_id = 1 + wg;
            const uint32_t tl = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
            const float* const s_nm = reinterpret_cast<const float*>(at(C::A_NM)) + wg * C::CW;
            float* const s_lc = reinterpret_cast<float*>(at(C::A_LC)) + wg * C::CW;
            float* const s_corr = reinterpret_cast<float*>(at(C::A_CORR)) + wg * C::CW;
            float* const red = reinterpret_cast<float*>(at(C::A_RED));
            float* const red_v = red + C::SM_WARPS * 32;
            float l[NCH][CH], m_run[NCH], vs[NCH];     // sums of the thread's tokens; lane c: maximum of row c; scale of |v|
#pragma unroll
            for (int ch = 0; ch < NCH; ch++) {
                m_run[ch] = -INFINITY;
                vs[ch] = 0.f;
#pragma unroll
                for (int c = 0; c < CH; c++) l[ch][c] = 0.f;
            }
            if (quarter == 0 && lane < 32) {
#pragma unroll
                for (int c = 0; c < C::CW; c += 32)
                    if (c + lane < C::CW) const_cast<float*>(s_nm)[c + lane] = INFINITY;
            }
            group_any(bar_id, false);
            wait(q_full + 8 * qb, n / C::QB);
            __syncwarp();
            const float q_down = ldexpf(1.f, -query_exponent(qb));
            const uint32_t* const cm = reinterpret_cast<const uint32_t*>(at(C::A_MASK)) + qb * (C::MASK_BYTES / 4);
#pragma unroll 1
            for (int it = 0; it < n_tiles; it++) {
                const int g = g0 + it, sb = g & 1, pb = g % C::PST;
                wait(norm_full + 8 * (g % C::NORMS), g / C::NORMS);
                __syncwarp();
                const __half* const norms = reinterpret_cast<const __half*>(at(C::A_NORM + (g % C::NORMS) * 4 * kTreeTile));
                const float kn = __half2float(norms[my_tok]) * q_down, vn = __half2float(norms[kTreeTile + my_tok]);
                const int pos = (pc.tile0 + it) * kTreeTile + my_tok, node = pos - ctx;
                const bool boundary = (pc.tile0 + it + 1) * kTreeTile > ctx;     // (uniform: the tile reaches the tree or the end)
                wait(s_full + 8 * sb, g >> 1);
                __syncwarp();
                tc_fence_after();
                bool p_free = false;
#pragma unroll
                for (int ch = 0; ch < NCH; ch++) {
                    const int col = wg * C::CW + ch * CH;
                    const uint32_t s_at = tl + C::COL_S + sb * N + col;
                    uint32_t bits = 0xffffffffu;
                    if (boundary) bits = pos >= seq ? 0u : node < 0 ? 0xffffffffu : cm[node * C::MW + col / 32] >> (col & 31);
                    float x[CH];
                    // x = score - maximum (base 2), -inf where the row does not attend the token
                    auto scores = [&](bool masked) {
                        uint32_t s[CH];
                        tc_load(s_at, s);
                        const u64 kn2 = pk2(kn, kn);
#pragma unroll
                        for (int c = 0; c < CH; c += 4) {
                            const float4 nm = *reinterpret_cast<const float4*>(s_nm + ch * CH + c);
                            upk2(fma2(pk2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), kn2, pk2(nm.x, nm.y)), x[c], x[c + 1]);
                            upk2(fma2(pk2(__uint_as_float(s[c + 2]), __uint_as_float(s[c + 3])), kn2, pk2(nm.z, nm.w)), x[c + 2], x[c + 3]);
                        }
                        if (masked) {
#pragma unroll
                            for (int c = 0; c < CH; c++) x[c] = (bits >> c) & 1u ? x[c] : -INFINITY;
                        }
                    };
                    scores(boundary);
                    float top = x[0];
#pragma unroll
                    for (int c = 1; c + 1 < CH; c += 2) top = fmaxf(fmaxf(top, x[c]), x[c + 1]);
                    top = fmaxf(top, x[CH - 1]);
                    const float av = fabsf(vn);
                    const bool grow = av <= FLT_MAX && (vs[ch] == 0.f ? av > 0.f : av * vs[ch] > kTreeGrowth);
                    if (group_any(bar_id, top > kTreeSlack || grow)) {
                        // ---- new maxima of these rows
                        float mine = -INFINITY;
#pragma unroll 1
                        for (int c = 0; c < CH; c += 16) {
                            uint32_t s[16];
                            tc_ld16(s_at + c, s);
                            tc_wait_ld(s);
#pragma unroll
                            for (int j = 0; j < 16; j++) {
                                const float r = warp_max((bits >> (c + j)) & 1u ? __uint_as_float(s[j]) * kn : -INFINITY);
                                if (lane == c + j) mine = r;
                            }
                        }
                        const float wv = warp_max(av <= FLT_MAX ? av : 0.f);
                        red[warp * 32 + lane] = mine;
                        if (lane == 0) red_v[warp] = wv;
                        group_any(bar_id, false);
                        float m_new = m_run[ch], v_top = 0.f;
#pragma unroll
                        for (int w = 0; w < 4; w++) {
                            m_new = fmaxf(m_new, red[(4 * wg + w) * 32 + lane]);
                            v_top = fmaxf(v_top, red_v[4 * wg + w]);
                        }
                        const float lc = m_run[ch] == -INFINITY ? 0.f : fast_exp2(m_run[ch] - m_new);
                        float v_ratio = 1.f;
                        if (v_top > 0.f && (vs[ch] == 0.f || v_top * vs[ch] > kTreeGrowth)) {   // the largest |v| becomes 1 to 2
                            const float to = ldexpf(1.f, -ilogbf(v_top));
                            v_ratio = vs[ch] == 0.f ? 1.f : to / vs[ch];
                            vs[ch] = to;
                        }
                        m_run[ch] = m_new;
                        if (quarter == 0 && lane < CH) {
                            const_cast<float*>(s_nm)[ch * CH + lane] = -m_new;
                            s_lc[ch * CH + lane] = lc;
                            s_corr[ch * CH + lane] = lc * v_ratio;
                        }
                        group_any(bar_id, false);
#pragma unroll
                        for (int c = 0; c < CH; c++) l[ch][c] *= s_lc[ch * CH + c];
                        if (it > 0) {
                            wait(o_done + 8 * ((g - 1) % C::PST), (g - 1) / C::PST);
                            __syncwarp();
                            tc_fence_after();
#pragma unroll 1
                            for (int k = 0; k < C::MB * CH; k += 16) {
                                const int c = k % CH, mb = k / CH;
                                uint32_t o[16];
                                tc_ld16(tl + C::COL_O + mb * N + col + c, o);
                                tc_wait_ld(o);
#pragma unroll
                                for (int j = 0; j < 16; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * s_corr[ch * CH + c + j]);
                                tc_st16(tl + C::COL_O + mb * N + col + c, o);
                            }
                            tc_wait_st();
                        }
                        scores(boundary);
                    }
                    // (the scores of the last chunk are in registers: the next tile's may overwrite them)
                    if (ch == NCH - 1) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) {
                            mbar_arrive(s_free + 8 * sb);
                            mbar_arrive(norm_empty + 8 * (g % C::NORMS));
                        }
                    }
                    if (!p_free) {
                        if (g >= C::PST) wait(o_done + 8 * pb, g / C::PST - 1);
                        __syncwarp();
                        p_free = true;
                    }
                    const float vw = vn * vs[ch];
                    const u64 vw2 = pk2(vw, vw);
                    const uint32_t p_row = C::A_P + pb * C::P_BUF + (col / 64) * C::P_ATOM + my_tok * 128;
#pragma unroll
                    for (int c = 0; c < CH; c += 8) {
                        uint32_t h[4];
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const float e0 = fast_exp2(x[c + 2 * j]), e1 = fast_exp2(x[c + 2 * j + 1]);
                            upk2(add2(pk2(l[ch][c + 2 * j], l[ch][c + 2 * j + 1]), pk2(e0, e1)), l[ch][c + 2 * j], l[ch][c + 2 * j + 1]);
                            float w0, w1;
                            upk2(mul2(pk2(e0, e1), vw2), w0, w1);
                            if (boundary) {    // (what a row does not attend may have a norm that is not a number)
                                w0 = (bits >> (c + 2 * j)) & 1u ? w0 : 0.f;
                                w1 = (bits >> (c + 2 * j + 1)) & 1u ? w1 : 0.f;
                            }
                            h[j] = f2h2(w0, w1);
                        }
                        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};\n" ::"r"(p_row + (((((col & 63) + c) >> 3) ^ (my_tok & 7)) << 4)),
                                     "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + 8 * pb);
            }
            // ---- the piece's rows
            {
                const int g = g0 + n_tiles - 1;
                wait(o_done + 8 * (g % C::PST), g / C::PST);
                __syncwarp();
                tc_fence_after();
            }
#pragma unroll
            for (int ch = 0; ch < NCH; ch++) {
                const int col = wg * C::CW + ch * CH;
                // sums over the lanes, then over the warps: lane c gets row c's
                float sum;
                if constexpr (CH == 16) {
#pragma unroll
                    for (int c = 0; c < CH; c++) l[ch][c] += __shfl_xor_sync(0xffffffffu, l[ch][c], 16);
                }
#pragma unroll
                for (int d = CH / 2; d > 0; d >>= 1) {
#pragma unroll
                    for (int i = 0; i < d; i++) {
                        const bool hi = (lane & d) != 0;
                        const float send = hi ? l[ch][i] : l[ch][i + d], keep = hi ? l[ch][i + d] : l[ch][i];
                        l[ch][i] = keep + __shfl_xor_sync(0xffffffffu, send, d);
                    }
                }
                group_any(bar_id, false);        // (the buffer has been read)
                red[warp * 32 + lane] = l[ch][0];
                group_any(bar_id, false);
                sum = red[(4 * wg) * 32 + lane] + red[(4 * wg + 1) * 32 + lane] + red[(4 * wg + 2) * 32 + lane] + red[(4 * wg + 3) * 32 + lane];
                if (quarter == 0 && lane < CH && col + lane < rows) {
                    float* dst = pc.out + (col + lane) * ROW + D;
                    dst[0] = m_run[ch];
                    dst[1] = sum;
                }
                const float scale = p.inv_v_scale / (vs[ch] == 0.f ? 1.f : vs[ch]);
#pragma unroll 1
                for (int k = 0; k < C::MB * CH; k += 16) {
                    const int c = k % CH, mb = k / CH;
                    uint32_t o[16];
                    tc_ld16(tl + C::COL_O + mb * N + col + c, o);
                    tc_wait_ld(o);
                    // TMEM row m: atom m / 64, 16-byte chunk (m % 64) / 8 = 2 t + (jj & 1): coordinate 8 jj + m % 8 of run t
                    const int m = my_tok + 128 * mb, chunk = (m & 63) >> 3, jj = 2 * (m >> 6) + (chunk & 1);
                    const int coord = (chunk >> 1) * (D / 4) + 8 * jj + (m & 7);
                    if (D == 64 && m >= 64) continue;
#pragma unroll
                    for (int j = 0; j < 16; j++)
                        if (col + c + j < rows) pc.out[(col + c + j) * ROW + coord] = __uint_as_float(o[j]) * scale;
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(o_free);
                mbar_arrive(q_empty + 8 * qb);
            }
            g0 += n_tiles;
        }
    } else if (warp < W_MMA) {
        if constexpr (C::SPLIT) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(C::R_DQ));
        // ================= dequantisation: one stream of tiles, whatever pieces they belong to; the codes of AHEAD tiles are
        // under way in registers
        constexpr int KSB = C::PDK / 4, VSB = C::PDV / 4;                  // bytes of a lane's run of D / 4 codes
        constexpr int KW = (KSB + 3) / 4, VW = (VSB + 3) / 4, XW = KW > VW ? KW : VW;
        const int g8 = lane >> 2, t4 = lane & 3, dq = warp & 3;
        const bool is_k = warp < W_V;
        TreeCodes<XW> f[C::AHEAD];
        int n_tiles = INT_MAX;     // (known when the stream's end has been seen: places of -2)
        auto fetch = [&](int g, TreeCodes<XW>& f) {    // the codes of the stream's tile g
            if (g >= n_tiles) return;
            const int slot = g % C::PAGES;
            wait(page_full + 8 * slot, g / C::PAGES);
            __syncwarp();
            const int64_t* const where = reinterpret_cast<const int64_t*>(at(C::A_PAGE + slot * 64));
            const int64_t page[2] = {where[is_k ? 2 * dq : dq], where[is_k ? 2 * dq + 1 : 4 + dq]};
            __syncwarp();
            if (lane == 0) mbar_arrive(page_empty + 8 * slot);
            if (page[0] == -2 || __any_sync(0xffffffffu, *gave_up != 0)) {   // (then what stands there may be no place)
                n_tiles = g;
                return;
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint8_t* src = p.pool + page[i];
#pragma unroll
                for (int r = 0; r < 2; r++) {
#pragma unroll
                    for (int j = 0; j < XW; j++) f.w[i][r][j] = 0;
                    if (page[i] < 0) continue;
                    const int tok = g8 + 8 * r;
                    // (a V row has its halves exchanged where bit 1 of its token's place is set)
                    if (is_k) tree_fetch<KSB>(src + tok * C::PDK + t4 * KSB, f.w[i][r]);
                    else tree_fetch<VSB>(src + C::OFF_VC + tok * C::PDV + (t4 ^ (tok & 2)) * VSB, f.w[i][r]);
                }
            }
        };
#pragma unroll
        for (int i = 0; i < C::AHEAD; i++) fetch(i, f[i]);
        if (is_k) {
            // ================= keys: codes -> TMEM, rows of lanes = tokens
            const uint32_t base = C::WINDOW + (BK == 2 ? (lane & 15) * 8 : lane * 4);
            const uint32_t rows_at = tmem + (static_cast<uint32_t>(dq * 32) << 16) + C::COL_K;
            auto turn = [&](int g, TreeCodes<XW>& f) {
                const int st = g & 1;
                if (g >= 2) wait(k_empty + 8 * st, (g >> 1) - 1);
                __syncwarp();
                tc_fence_after();
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    typename Window<BK, false>::template Run<KW> r0, r1;
#pragma unroll
                    for (int j = 0; j < KW; j++) {
                        r0.w[j] = f.w[i][0][j];
                        r1.w[j] = f.w[i][1][j];
                    }
                    Window<BK, false>::shift(r0);
                    Window<BK, false>::shift(r1);
#pragma unroll
                    for (int q = 0; q < D / 64; q++) {
                        uint32_t x[16];
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            Window<BK, false>::pairs(r0, 4 * q + j, base, x[4 * j], x[4 * j + 1]);
                            Window<BK, false>::pairs(r1, 4 * q + j, base, x[4 * j + 2], x[4 * j + 3]);
                        }
                        tc_st_16x256b_x4(rows_at + (static_cast<uint32_t>(16 * i) << 16) + st * (D / 2) + 32 * q, x);
                    }
                }
                fetch(g + C::AHEAD, f);
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
#ifdef FTQ_TEST_WAIT_EXPIRY
                if (g == 1 && dq == 0 && cta == 0) return;
#endif
                if (lane == 0) mbar_arrive(k_full + 8 * st);
            };
#pragma unroll 1
            for (int g = 0; g < n_tiles; g += C::AHEAD) {
#pragma unroll
                for (int i = 0; i < C::AHEAD; i++)
                    if (g + i < n_tiles) turn(g + i, f[i]);
            }
        } else {
            // ================= values: codes -> fp16 tiles, MN-major with 128-byte swizzle
            const uint32_t base = C::WINDOW + 128 + (BV == 2 ? (lane & 15) * 8 : lane * 4);
            auto turn = [&](int g, TreeCodes<XW>& f) {
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int n = 2 * g + i, slot = n % C::VS, use = n / C::VS;
                    if (use > 0) wait(v_empty + 8 * slot, use - 1);
                    __syncwarp();
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        typename Window<BV, false>::template Run<VW> run;
#pragma unroll
                        for (int j = 0; j < VW; j++) run.w[j] = f.w[i][r][j];
                        Window<BV, false>::shift(run);
                        const int row = 16 * dq + g8 + 8 * r;
                        const uint32_t dst = C::A_V + slot * C::V_SLOT + row * 128;
#pragma unroll
                        for (int jj = 0; jj < D / 32; jj++) {
                            uint32_t x[4];
                            Window<BV, false>::pairs(run, 2 * jj, base, x[0], x[1]);
                            Window<BV, false>::pairs(run, 2 * jj + 1, base, x[2], x[3]);
                            // (eight lanes that store together have two rows and four chunks apart by two: no two on the same banks)
                            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};\n" ::"r"(dst + (jj >> 1) * 8192 + (((2 * t4 + (jj & 1)) ^ (row & 7)) << 4)),
                                         "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]) : "memory");
                        }
                    }
                    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(v_full + 8 * slot);
                }
                fetch(g + C::AHEAD, f);
            };
#pragma unroll 1
            for (int g = 0; g < n_tiles; g += C::AHEAD) {
#pragma unroll
                for (int i = 0; i < C::AHEAD; i++)
                    if (g + i < n_tiles) turn(g + i, f[i]);
            }
        }
    } else if (warp == W_MMA) {
        // ================= the products
        for (int np = 0, g0 = 0;; np++) {
            const int qb = np % C::QB, n_tiles = piece_at(np).n_tiles;
            if (n_tiles == 0) break;
            constexpr uint32_t kIdescS = (1u << 4) | (static_cast<uint32_t>(N / 8) << 17) | (8u << 24);
            constexpr uint32_t kIdescO = kIdescS | (1u << 15) | (1u << 16);
            constexpr uint32_t kHi = (1024u >> 4) | (1u << 14) | (2u << 29);
            constexpr uint32_t kQ = (static_cast<uint32_t>(C::A_Q) >> 4) | ((16u >> 4) << 16);
            constexpr uint32_t kV = (static_cast<uint32_t>(C::A_V) >> 4) | ((8192u >> 4) << 16);
            constexpr uint32_t kP = (static_cast<uint32_t>(C::A_P) >> 4) | ((static_cast<uint32_t>(C::P_ATOM) >> 4) << 16);
            auto pv = [&](int it) {
                const int g = g0 + it, pb = g % C::PST;
                wait(p_full + 8 * pb, g / C::PST);
                if (it == 0 && np > 0) wait(o_free, np - 1);
                __syncwarp();
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int n = 2 * g + h, slot = n % C::VS;
                    wait(v_full + 8 * slot, n / C::VS);
                    __syncwarp();
                    tc_fence_after();
                    const uint32_t v = kV + slot * (C::V_SLOT >> 4), q = kP + pb * (C::P_BUF >> 4) + h * (8192 >> 4);
                    if (elect_one()) {
#pragma unroll
                        for (int mb = 0; mb < C::MB; mb++)
#pragma unroll
                            for (int ks = 0; ks < 4; ks++)
                                one_mma_ss(tmem + C::COL_O + mb * N, v + mb * (16384 >> 4) + ks * (2048 >> 4), q + ks * (2048 >> 4), kHi, kIdescO,
                                           h > 0 || ks > 0 ? 1u : static_cast<uint32_t>(it));
                        tc_commit(v_empty + 8 * slot);
                        if (h == 1) tc_commit(o_done + 8 * pb);
                    }
                    __syncwarp();
                }
            };
            wait(q_full + 8 * qb, np / C::QB);
#pragma unroll 1
            for (int it = 0; it < n_tiles; it++) {
                const int g = g0 + it, st = g & 1;
                wait(k_full + 8 * st, g >> 1);
                if (g >= 2) wait(s_free + 8 * st, (g >> 1) - 1);
                __syncwarp();
                tc_fence_after();
                if (elect_one()) {
#pragma unroll
                    for (int kb = 0; kb < D / 16; kb++)
                        one_mma_ts(tmem + C::COL_S + st * N, tmem + C::COL_K + st * (D / 2) + 8 * kb,
                                   kQ + qb * (C::Q_BYTES >> 4) + ((kb >> 2) * (N * 128) + (kb & 3) * 32) / 16, kHi, kIdescS, kb > 0);
                    tc_commit(s_full + 8 * st);
                    tc_commit(k_empty + 8 * st);
                    if (it == n_tiles - 1) tc_commit(q_empty + 8 * qb);
                }
                __syncwarp();
                if (it > 0) pv(it - 1);
            }
            pv(n_tiles - 1);
            g0 += n_tiles;
        }
    } else if (warp == C::W_FEED) {
        // ================= the pieces; where the pages of their tiles lie; the norms of the tokens.  In step s the block ids of
        // tile s are requested, the norms of tile s - 2, and those of tile s - 4 are handed over.  Lane l has page l / 4 of a
        // tile and four of its tokens.  No token: norms of zero; a block id outside the pool: keys that are not numbers.
        int pos = begin;                                           // next place
        int n_pieces = 0, n_tiles = 0, head = 0;
        int tile = 0, tiles_left = 0, seq = 0;                     // of the piece that the ids are requested for
        const int32_t* btab = nullptr;
        bool more = true;
        const int page_of_lane = lane >> 2, part = lane & 3;
#pragma unroll 1
        for (int s = 0; more || s - 4 < n_tiles; s++) {
            if (more && tiles_left == 0) {
                const TreePiece pc = next_piece(pos);
                const int slot = n_pieces % C::PIECES;
                if (n_pieces >= C::PIECES) wait(piece_empty + 8 * slot, n_pieces / C::PIECES - 1);
                __syncwarp();
                if (lane == 0) *reinterpret_cast<TreePiece*>(at(C::A_PIECE + slot * 48)) = pc;
                __syncwarp();
                if (lane == 0) mbar_arrive(piece_full + 8 * slot);
                n_pieces++;
                more = pc.n_tiles > 0;
                tile = pc.tile0; tiles_left = pc.n_tiles; seq = pc.seq;
                btab = p.block_table + static_cast<int64_t>(pc.b) * p.max_blocks;
                head = pc.hkv;
            }
            if (more) {
                const int pg = tile * (kTreeTile / kPageTokens) + page_of_lane;
                const uint32_t dst = C::A_ID + s % C::PAGES * 32 + page_of_lane * 4;
                if (part == 0) {
                    if (pg * kPageTokens < seq) copy_async<4>(dst, btab + pg);
                    else *reinterpret_cast<int*>(at(dst)) = -2;
                }
                // (the KV head of the tile, for the step after next)
                if (lane == 0) misc[40 + s % C::PAGES] = head;
                n_tiles++;
                tile++;
                tiles_left--;
            }
            asm volatile("cp.async.commit_group;\n" ::: "memory");
            const int t = s - 2;
            if (t >= 0 && t <= n_tiles) {
                // (four younger groups: two of step s - 1, one each of steps s - 2 and s)
                asm volatile("cp.async.wait_group 4;\n" ::: "memory");
                __syncwarp();
                const int slot = t % C::PAGES, ns = t % C::NORMS;
                if (t >= C::PAGES) wait(page_empty + 8 * slot, t / C::PAGES - 1);
                __syncwarp();
                const bool last = t == n_tiles;        // (the end of the stream)
                const int id = *reinterpret_cast<const int*>(at(C::A_ID + slot * 32 + page_of_lane * 4));
                const bool ok = !last && static_cast<uint64_t>(static_cast<int64_t>(id)) < static_cast<uint64_t>(p.num_blocks), bad = !last && !ok && id != -2;
                const int64_t page = last ? -2 : ok ? (static_cast<int64_t>(id) * p.Hkv + static_cast<int>(misc[40 + slot])) * C::PAGE_BYTES : -1;
                if (bad) __stcg(p.errors + 1, p.epoch);
                if (part == 0) *reinterpret_cast<int64_t*>(at(C::A_PAGE + slot * 64 + page_of_lane * 8)) = page;
                __syncwarp();
                if (lane == 0) mbar_arrive(page_full + 8 * slot);
                if (!last) {
                    if (t >= C::NORMS) wait(norm_empty + 8 * ns, t / C::NORMS - 1);
                    __syncwarp();
                    const uint32_t dst = C::A_NORM + ns * 4 * kTreeTile + lane * 8;
                    if (ok) {
                        copy_async<8>(dst, p.pool + page + C::OFF_KN + 8 * part);
                        copy_async<8>(dst + 2 * kTreeTile, p.pool + page + C::OFF_VN + 8 * part);
                    } else {
                        *reinterpret_cast<uint2*>(at(dst)) = bad ? make_uint2(0x7e007e00u, 0x7e007e00u) : make_uint2(0u, 0u);
                        *reinterpret_cast<uint2*>(at(dst + 2 * kTreeTile)) = make_uint2(0u, 0u);
                    }
                }
            }
            asm volatile("cp.async.commit_group;\n" ::: "memory");
            if (s >= 4 && s - 4 < n_tiles) {
                // (younger than the norms' group of step s - 2: the two of step s - 1, the two of step s)
                asm volatile("cp.async.wait_group 4;\n" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(norm_full + 8 * ((s - 4) % C::NORMS));
            }
        }
    } else {
        // ================= queries and masks of the other pieces, one ahead where there is room
        if (lane == 0) mbar_arrive(q_full);     // (the first piece's)
        bool more = !group_any<32 * C::Q_WARPS>(3, piece_at(0).n_tiles == 0);
        for (int n = 1; more; n++) {
            const TreePiece pc = piece_at(n);
            more = !group_any<32 * C::Q_WARPS>(3, pc.n_tiles == 0);
            if (!more) break;
            const int qb = n % C::QB;
            if (n >= C::QB) wait(q_empty + 8 * qb, n / C::QB - 1);
            __syncwarp();
            prepare_piece(pc, qb, std::integral_constant<int, C::Q_WARPS>{}, tid - 32 * C::W_Q);
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full + 8 * qb);
        }
    }
    __syncwarp();
    __syncthreads();
    if (*gave_up) {   // all that this CTA has
        int pos = begin;
        for (TreePiece pc = next_piece(pos); pc.n_tiles > 0; pc = next_piece(pos))
            for (int r = tid; r < pc.rows; r += C::THREADS) pc.out[r * ROW + D] = __int_as_float(0x7fc00000);
        if (tid == 0) __stcg(p.errors, p.epoch);
    }
    if (warp == W_MMA) {   // nothing may be in flight when TMEM is given back
        if (lane == 0) tc_commit(drained);
        __syncwarp();
        for (int i = 0; i < kDrainSpinLimit && !mbar_try_wait(drained, 0); i++) {}
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem));
    }
}

// Joins the pieces of every (sequence, node, head) row by their maxima, rotates back (core/hadamard.py:93-100) and stores; nodes
// that do not exist and rows that attend nothing are zero.  OCTETS octets per row, as in attn_merge_kernel.
struct TreeMergeParams {
    const int* plan;
    const float *whole, *cut;
    const int32_t *tree_lens, *seq_lens;
    void* out;
    int B, T, Hq, Hkv, N, row_tiles, max_seq;
    FastDiv group;
    float rsqrt_d;
    SignBits signs;
    MergeStatus status;
    bool more;                  // the status of an earlier launch of the call stays
};
template <int D, typename OT, int OCTETS>
__global__ void __launch_bounds__(128) tree_merge_kernel(const __grid_constant__ TreeMergeParams p) {
    constexpr int E = D / kOctet, ROW = D + 4;
    const int lane = threadIdx.x & 31, t = lane & 7, o = (lane >> 3) & (OCTETS - 1);
    after_previous_kernel();
    if (p.status.status && blockIdx.x == 0 && threadIdx.x == 0) {
        *p.status.status = (p.more ? *p.status.status : 0) | (__ldcg(p.status.errors) == p.status.epoch ? kStatusWaitExpired : 0) |
                           (__ldcg(p.status.errors + 1) == p.status.epoch ? kStatusBadBlock : 0);
        p.status.errors[0] = p.status.errors[1] = 0ull;   // (a replayed launch has the same epoch)
    }
    const int64_t n_rows = static_cast<int64_t>(p.B) * p.T * p.Hq;
    const int64_t mine = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / (8 * OCTETS);
    const int64_t v = mine < n_rows ? mine : n_rows - 1;
    const int hq = static_cast<int>(v % p.Hq), i = static_cast<int>(v / p.Hq % p.T), b = static_cast<int>(v / p.Hq / p.T);
    const int group = static_cast<int>(p.group.d), hkv = fast_div(hq, p.group), r = i * group + hq - hkv * group;
    const int rt = r / p.N, n = r - rt * p.N, u = hkv * p.row_tiles + rt, U = p.Hkv * p.row_tiles;
    const int seq = max(0, min(p.seq_lens[b], p.max_seq));
    const int nodes = p.tree_lens ? min(max(p.tree_lens[b], 0), min(p.T, seq)) : min(p.T, seq);
    const int share = p.plan[p.B + 1], len = (p.plan[b + 1] - p.plan[b]) / U, pos = p.plan[b] + u * len;
    const int c0 = pos / share, c1 = (pos + len - 1) / share, parts = i < nodes ? c1 - c0 + 1 : 0;
    auto row_of = [&](int k) -> const float* {   // part k's row, NULL: it has no tiles
        const int c = c0 + k;
        const int from = max(pos, c * share), to = static_cast<int>(min(static_cast<int64_t>(pos) + len, static_cast<int64_t>(c + 1) * share));
        if (tree_tile_of(to - pos) <= tree_tile_of(from - pos)) return nullptr;
        return c0 == c1 ? p.whole + ((static_cast<int64_t>(b) * U + u) * p.N + n) * ROW
                        : p.cut + ((2 * static_cast<int64_t>(c) + (k == 0 ? 1 : 0)) * p.N + n) * ROW;
    };
    float M = -INFINITY;
    for (int k = 8 * o + t; k < parts; k += 8 * OCTETS) {
        const float* row = row_of(k);
        M = fmaxf(M, row ? row[D] : -INFINITY);
    }
#pragma unroll
    for (int d = 1; d < 8 * OCTETS; d <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
    float a[E];
#pragma unroll
    for (int k = 0; k < E; k++) a[k] = 0.f;
    float L = 0.f;
#pragma unroll 2
    for (int k = o; k < parts; k += OCTETS) {
        const float* row = row_of(k);
        const float m = row ? row[D] : -INFINITY, ls = row ? row[D + 1] : 0.f;
        const bool live = row && (m != -INFINITY || ls != 0.f);
        // (a row whose scores are not numbers knows no maximum: its sum says so)
        const float f = live ? (m == -INFINITY ? ls : exp2f(m - M)) : 0.f;
        L = live ? fmaf(ls, f, L) : L;
#pragma unroll
        for (int x = 0; x < E / 8; x++) {
            float tmp[8];
            if (row) load8<float>(row + 8 * (t + 8 * x), tmp);
#pragma unroll
            for (int c = 0; c < 8; c++) a[8 * x + c] = live ? fmaf(tmp[c], f, a[8 * x + c]) : a[8 * x + c];
        }
    }
#pragma unroll
    for (int d = 8; d < 8 * OCTETS; d <<= 1) {
        L += __shfl_xor_sync(0xffffffffu, L, d);
#pragma unroll
        for (int k = 0; k < E; k++) a[k] += __shfl_xor_sync(0xffffffffu, a[k], d);
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int k = 0; k < E; k++) a[k] *= inv;
    octet_fwht<E>(a, lane);
#pragma unroll
    for (int k = 0; k < E; k++) {
        if (mine >= n_rows || (k & (OCTETS - 1)) != o) continue;
        const float x = a[k] * p.rsqrt_d;
        reinterpret_cast<OT*>(p.out)[v * D + t + 8 * k] = from_float<OT>(__uint_as_float(__float_as_uint(x) ^ sign_mask(p.signs, t + 8 * k)));
    }
}

}  // namespace ftq
