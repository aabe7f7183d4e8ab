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
// Lazy maxima: a row's weights refer to the largest score of an earlier tile (m).  The one barrier of a tile, which its
// products need anyway, tells whether a score was above m + 13 (base 2); if so the warps find the new maxima, rescale O
// and the sums and write the tile's weights again.  (With a slack of 3, as in the decode kernels, half of the tiles
// did: of 32 rows there is always one that has found a larger score.)  Weights are fp16: |v| is scaled by a power of
// two, so that the largest so far is 1 to 2, and again when one of 4 or more comes; p * |v| is then at most 2^15, and a weight of
// 2^-14 of the largest still has all its bits (a row that attends none but values 2^14 times shorter than the longest that its column
// group has met loses some).  Queries have a common scale, and rows that are much smaller one of their own, so that
// no row costs another its precision.  Scores, sums and O are fp32.  Three operands are rounded to fp16, as in
// the decode kernels, for the tensor cores' sake: rotated queries, centroids and weights; against 64 bits an output is off by 4e-4 of its
// size, by 2e-4 if only the output were rounded to fp16, and by 1.7e-3 either way if to bf16.
//
// Work: units (sequence, KV head, row tile) in a line of places, a place per tile of 128 tokens and tree_piece more per
// unit, cut into equal shares, one per half of a CTA (one CTA per SM).  A half's eight warps do all that a tile takes of a
// thread, one thing after the other: keys to TMEM, softmax, values to shared memory, a barrier.  While one half waits for
// something the other has the SM.  Two helper warps a half (of the last four warps) do what would hold the others up: one issues the products (about
// 700 cycles a tile), one fetches codes and norms by bulk copies (400 cycles to issue one) as their places become free.
// Beyond 64 rows (products of 128), and for heads of 256, one half of sixteen warps has the
// CTA to itself: its rows share what was dequantised, and eight warps have the keys, eight the values.  Every piece leaves its rows
// (O, m, l) in the workspace; tree_merge_kernel joins the pieces of a unit, rotates back and stores.
//
// Bound: the latency of the chain of a tile, about 6000 cycles for a half: look-ups (a 16-bit pair of codes a 4-byte load), softmax,
// and the waits for shared memory and at barriers between them.  No unit is full: issue slots 38 (heads of 256) to 50 %, tensor cores
// 11 to 24 %, HBM 2 to 25 %; barriers and shared memory are the longest stalls.  Measured (K4V4, bf16): one sequence of 900 tokens,
// 8 nodes, 32 heads of 128 over 8: 17.5 us; 32 of 8192, 16 nodes: 175 us (floor by HBM 44), where dequantising and a CTA of 128 rows of one sequence after
// the other took 413, one CTA of specialised warps 261 to 350 (handing tiles over cost more than the work), two halves
// that fetched and issued for themselves 205; 2 of 131072, 64 nodes, 64 heads: 893 us (616 TFLOP/s, 38 % of the measured
// bf16 rate); 24 ragged of up to 16384, heads of 256: 99 us; 40 ragged of up to 4096, 25 nodes, 14 heads of 64 over 2: 41 us.
//
// Every wait is bounded.  After one has run out nothing waits any more, the half's rows become NaN and the status word says
// so.  Block ids outside the pool are not followed: the rows that attend a token of such a page are NaN.
#pragma once

#include "ftq_attn_chunk.cuh"
#include "ftq_serve_launch.h"

namespace ftq {

constexpr int kTreeTile = 128;         // tokens of a tile
// Places that a unit costs besides its tiles: its queries, its first maxima and its rows take as long as so many tiles.  (24 ragged
// sequences with heads of 256: 2, 3, 4, 6 places 124, 111, 99, 102 us; 40 with heads of 64: 42, 41, 43, 46 us.  Heads of 128, 2, 3, 4
// places: 40 ragged of up to 4096 51, 52, 53 us; 8 of 2048 28, 27, 28; 64 ragged of up to 500, 25 nodes, 59, 67, 69; 32 of 8192 all 175.)
__host__ __device__ constexpr int tree_piece(int head_dim) { return head_dim == 256 ? 4 : 3; }
constexpr int kTreeMaxSeqs = 1024;     // sequences of a launch
constexpr float kTreeSlack = 13.f, kTreeGrowth = 4.f;
constexpr float kTreeRounded = 1 << 20;    // (half a unit in its last place: 2^-4)
// Rows that differ by less have a common scale.  (Were every row given its own, a tile's scores would all be scaled back: 32 sequences of
// 8192 tokens, 16 nodes of ordinary queries 191 us instead of 175.)
constexpr int kTreeSpread = 12;

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
    float* whole;               // rows of units that one half has: [B][Hkv * row_tiles][N][D + 4]
    float* cut;                 // rows of the others: [halves][2][N][D + 4]
    unsigned long long* errors; // expired waits, bad block ids (see ChunkAttnParams)
    unsigned long long epoch;
    Codebook lk, lv;            // scaled for their fp16 rounding
    SignBits signs;
};

// The part of a unit that a half has: places [off, off_end) of its tiles + tree_piece.
__host__ __device__ __forceinline__ int tree_tile_of(int off, int piece) { return off > piece ? off - piece : 0; }

template <int D, int BK, int BV, int N>
struct TreeCfg {
    static constexpr int HALVES = D == 256 || N == 128 ? 1 : 2, WARPS = 16, THREADS = 640, PIECE = tree_piece(D);
    static constexpr int WH = WARPS / HALVES, HT = 32 * WH;        // warps and threads of a half, without its two helpers
    // softmax: column groups of four warps (a warp reaches the 32 tokens of its quarter), rows of a group
    static constexpr int CG = WH / 4 < N / 8 ? WH / 4 : N / 8, CW = N / CG;
    static constexpr int PDK = packed_dim(D, BK), PDV = packed_dim(D, BV);
    static constexpr int OFF_KN = kPageTokens * PDK;
    static constexpr int OFF_VC = OFF_KN + 2 * kPageTokens;
    static constexpr int OFF_VN = OFF_VC + kPageTokens * PDV;
    static constexpr int PAGE_BYTES = OFF_VN + 2 * kPageTokens;
    static constexpr int MB = D == 256 ? 2 : 1;                    // M blocks of O^T
    // Shared memory of a half: V (one buffer, two where there is room), P, queries, masks.  The look-up window takes 64 KB at 64 KB;
    // the dynamic part (the only one) starts in the first 4 KB.  (At head_dim 64 a product reads an atom beyond V, P's: unused rows.)
    static constexpr int VB = HALVES == 1 && D <= 128 ? 2 : 1, V_ATOM = kTreeTile * 128, V_BUF = V_ATOM * (D / 64);
    static constexpr bool LATE_V = HALVES == 2;     // a tile's values are looked up after its weights
    static constexpr int P_ATOM = kTreeTile * 128, P_BUF = P_ATOM * ((N + 63) / 64);
    static constexpr int Q_BYTES = N * D * 2, MW = (N + 31) / 32, MASK_BYTES = kTreeMaxNodes * MW * 4;
    static constexpr int WINDOW = 65536, LOW = 4096, A_V = 131072, A_P = A_V + HALVES * VB * V_BUF;
    static constexpr int A_Q = LOW, A_MASK = A_Q + HALVES * Q_BYTES;
    static constexpr int A_ROW = A_MASK + HALVES * MASK_BYTES, ROW_BYTES = 7 * N * 4 + 64;   // - maximum, factors of l and O, red[4][N], red_v
    // codes on their way: the page of a warp (at head_dim 256 the value warps' lie behind P)
    static constexpr int STAGE = 16 * (PDK > PDV ? PDK : PDV), LOW_STAGES = D == 256 ? 8 : 16;
    static constexpr int A_STAGE = (A_ROW + HALVES * ROW_BYTES + 127) / 128 * 128, A_STAGE_HI = A_P + HALVES * P_BUF;
    static constexpr int A_FIRST = A_STAGE + LOW_STAGES * STAGE, END_LOW = A_FIRST + (kTreeMaxSeqs + 1) * 4;     // [kTreeMaxSeqs + 1]
    static constexpr int A_NORM = A_STAGE_HI + (WARPS - LOW_STAGES) * STAGE;       // a half's norms: keys [128], values [128]
    static constexpr int A_MISC = A_NORM + HALVES * 512, A_BAR = A_MISC + 128, BARS = 9, A_PIECE = A_BAR + HALVES * BARS * 8;
    static constexpr int A_DOWN = A_PIECE + 128, DOWN_BYTES = N * 4 + 16;          // a half's scales of S, and whether it needs settle()
    static constexpr int SMEM_BYTES = A_DOWN + HALVES * DOWN_BYTES;
    static_assert(END_LOW <= WINDOW && SMEM_BYTES <= 227 * 1024 && Q_BYTES % 1024 == 0, "");
    // TMEM columns of a half: two key buffers, S, O
    static constexpr int COLS = 512 / HALVES, COL_S = D, COL_O = D + N;
    static_assert(COL_O + MB * N <= COLS, "");
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
    float* out;                 // [N][D + 4]
    int k_phase;                // of k_full and k_free at its first tile
};

// A load whose value is not looked at before its use: a select on it, or a conversion, would wait for memory here and now.
__device__ __forceinline__ int load_id_if(bool ok, const int32_t* p, int otherwise) {
    int v;
    asm volatile("{\n.reg .pred q;\nsetp.ne.u32 q, %1, 0;\nmov.b32 %0, %3;\n@q ld.global.b32 %0, [%2];\n}\n"
                 : "=&r"(v) : "r"(static_cast<uint32_t>(ok)), "l"(p), "r"(otherwise) : "memory");
    return v;
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
    } else if constexpr (NC == 16) {
        tc_ld16(addr, r);
        tc_wait_ld(r);
    } else {
        static_assert(NC == 8, "");
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\ntcgen05.wait::ld.sync.aligned;\n"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(addr) : "memory");
    }
}
__device__ __forceinline__ void tc_st8(uint32_t addr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}

// Run number `t` (SB bytes) of a row of codes in shared memory, codes from bit 0 on (rows start on 4 bytes).
template <int SB, class Run>
__device__ __forceinline__ void tree_run(uint32_t row, int t, Run& run) {
    const uint32_t a = row + t * SB;
    if constexpr (SB % 16 == 0) {
#pragma unroll
        for (int i = 0; i < SB / 16; i++)
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n" : "=r"(run.w[4 * i]), "=r"(run.w[4 * i + 1]), "=r"(run.w[4 * i + 2]), "=r"(run.w[4 * i + 3])
                         : "r"(a + 16 * i) : "memory");
    } else if constexpr (SB % 8 == 0) {
#pragma unroll
        for (int i = 0; i < SB / 8; i++)
            asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];\n" : "=r"(run.w[2 * i]), "=r"(run.w[2 * i + 1]) : "r"(a + 8 * i) : "memory");
    } else if constexpr (SB % 4 == 0) {
#pragma unroll
        for (int i = 0; i < SB / 4; i++) asm volatile("ld.shared.b32 %0, [%1];\n" : "=r"(run.w[i]) : "r"(a + 4 * i) : "memory");
    } else {        // (six bytes on a two-byte boundary, in two words)
        static_assert(SB == 6, "");
        uint32_t lo, hi;
        asm volatile("ld.shared.b32 %0, [%1];\n" : "=r"(lo) : "r"(a & ~3u) : "memory");
        asm volatile("ld.shared.b32 %0, [%1];\n" : "=r"(hi) : "r"((a & ~3u) + 4) : "memory");
        const int sh = (t & 1) * 16;
        run.w[0] = __funnelshift_r(lo, hi, sh);
        run.w[1] = hi >> sh;
    }
}
__device__ __forceinline__ void bulk_g2s(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

template <int D, int BK, int BV, int N>
__global__ void __launch_bounds__(TreeCfg<D, BK, BV, N>::THREADS, 1)
tree_attn_kernel(const __grid_constant__ TreeAttnParams p) {
    using C = TreeCfg<D, BK, BV, N>;
    constexpr int E = D / kOctet, ROW = D + 4, CW = C::CW;
    constexpr int KSB = C::PDK / 4, VSB = C::PDV / 4;                  // bytes of a lane's run of D / 4 codes
    constexpr int KW = (KSB + 3) / 4, VW = (VSB + 3) / 4;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    const uint32_t raw = static_cast<uint32_t>(__cvta_generic_to_shared(smem_raw));
    auto at = [&](uint32_t a) { return smem_raw + (a - raw); };
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    // half, warp and thread in it; of the last warps every half has two, one that issues its products and one that fetches its pages
    const bool helper = warp >= C::WARPS;
    const int half = helper ? (warp - C::WARPS) >> 1 : warp / C::WH, hw = warp % C::WH, me = helper ? C::HT + lane : tid - half * C::HT;
    uint32_t* const misc = reinterpret_cast<uint32_t*>(at(C::A_MISC));   // 0: TMEM, 1, 2: a half's wait ran out, 3, 4: its largest |q|, 8..: scan
    volatile uint32_t* const gave_up = misc + 1 + half;
    // a half's barriers: products; codes and norms that are there, and that were looked at (one phase each per tile)
    const uint32_t s_done = C::A_BAR + 8 * C::BARS * half, o_done = s_done + 8, drained = s_done + 16;
    const uint32_t k_full = s_done + 24, v_full = s_done + 32, n_full = s_done + 40, k_free = s_done + 48, v_free = s_done + 56, n_free = s_done + 64;

    // ---- look-up window (struct Window): 256 rows of 256 bytes, keys in the first half of a row, values in the second
    {
        auto build = [&](int off, auto bits, const Codebook& cb) {
            constexpr int NB = decltype(bits)::value;
            const float lev = cb.v[lane & 15];
#pragma unroll 4
            for (int e = warp; e < 256; e += C::THREADS / 32) {
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
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(static_cast<uint32_t>(C::A_MISC)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n");
        if (lane == 0) {
            for (int h = 0; h < C::HALVES; h++) {
                const uint32_t bars = C::A_BAR + 8 * C::BARS * h;
                for (int i = 0; i < C::BARS; i++) mbar_init(bars + 8 * i, i < 3 ? 1 : i == 5 ? 16 : i == 8 ? C::WH : 8);
            }
            mbar_fence_init();
        }
        tc_fence_before();
    }
    if (tid < 4) misc[1 + tid] = 0;
    after_previous_kernel();    // (nothing in global memory was touched so far)

    // ---- the line of places
    const int U = p.Hkv * p.row_tiles, workers = gridDim.x * C::HALVES, worker = blockIdx.x * C::HALVES + half;
    int* const first = reinterpret_cast<int*>(at(C::A_FIRST));
    {
        int base = 0;
        for (int b0 = 0; b0 < p.B; b0 += C::THREADS) {
            const int b = b0 + tid;
            const int len = b < p.B ? max(0, min(p.seq_lens[b], p.max_seq)) : 0;
            const int v = b < p.B ? U * ((len + kTreeTile - 1) / kTreeTile + C::PIECE) : 0;
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
            for (int w = 0; w < C::THREADS / 32; w++) {
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
    const uint32_t tmem_all = __shfl_sync(0xffffffffu, misc[0], 0), tmem = tmem_all + half * C::COLS;
    const int total = first[p.B], share = (total + workers - 1) / workers;
    const int end = static_cast<int>(min(static_cast<int64_t>(total), static_cast<int64_t>(worker + 1) * share));
    const int begin = static_cast<int>(min(static_cast<int64_t>(worker) * share, static_cast<int64_t>(end)));
    if (worker == 0 && !helper) {
        for (int b = me; b <= p.B; b += C::HT) p.plan[b] = first[b];
        if (me == 0) p.plan[p.B + 1] = share;
    }
    // bounded wait; once one has run out the half does not wait any more
    auto wait = [&](uint32_t bar, uint32_t parity) {
#pragma unroll 1
        for (int i = 0; i < kChunkSpinLimit; i++) {
            if (mbar_try_wait(bar, parity & 1u)) break;
            if ((i & 63) == 63 && *gave_up) break;
            if (i == kChunkSpinLimit - 1) *gave_up = 1;
        }
        __syncwarp();
        tc_fence_after();
    };
    // The same for copies, which are waited for whatever has happened to the products (none may be in flight when the CTA ends).
    bool stalled = false;
    auto copied = [&](uint32_t bar, uint32_t parity) {
        if (stalled) return;
        bool there = false;
#pragma unroll 1
        for (int i = 0; i < kDrainSpinLimit && !there; i++) there = mbar_try_wait(bar, parity & 1u);
        stalled = !__all_sync(0xffffffffu, there);
        if (stalled) *gave_up = 1;
    };
    // the warp has looked at what came
    auto taken = [&](uint32_t bar) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
    };
    // barriers of a half: its workers'; theirs and the issuer's (true if any thread says so); theirs and the feeder's
    auto meet = [&]() { group_any<C::HT>(3 + half, false); };
    auto meet_issuer = [&](bool mine) { return group_any<C::HT + 32>(1 + half, mine); };
    auto meet_feeder = [&]() { group_any<C::HT + 32>(5 + half, false); };
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
            const int off_end = min(len, off + end - pos), t0 = tree_tile_of(off, C::PIECE), t1 = tree_tile_of(off_end, C::PIECE);
            pos += off_end - off;
            if (t1 <= t0) continue;
            pc.b = lo;
            pc.hkv = u / p.row_tiles;
            pc.row0 = (u - pc.hkv * p.row_tiles) * N;
            pc.seq = max(0, min(p.seq_lens[lo], p.max_seq));
            pc.ctx = pc.seq - min(p.tree_lens ? max(p.tree_lens[lo], 0) : p.T, min(p.T, pc.seq));
            // (of the nodes that exist: what lies in the others' queries is not looked at, nor is a context that no node attends)
            pc.rows = min(N, (pc.seq - pc.ctx) * static_cast<int>(p.group.d) - pc.row0);
            if (pc.rows <= 0) continue;
            pc.tile0 = t0;
            pc.n_tiles = t1 - t0;
            pc.out = off == 0 && off_end == len ? p.whole + (static_cast<int64_t>(lo) * U + u) * N * ROW
                                                : p.cut + (2 * static_cast<int64_t>(worker) + (off == 0 ? 1 : 0)) * N * ROW;
        }
        return pc;
    };

    // ---- what a warp does in a tile
    const int quarter = warp & 3, cg = hw >> 2, my_tok = quarter * 32 + lane, col0 = cg * CW;
    const bool soft = cg < C::CG;                             // (small row tiles leave some warps without a column)
    const int g8 = lane >> 2, t4 = lane & 3;
    // its page of a tile: of the two of its quarter; with 16 warps eight have keys and eight values, with eight each has both
    const int odd = C::HALVES == 2 ? hw >> 2 : (hw >> 2) & 1, my_page = 2 * quarter + odd;
    const bool has_k = C::HALVES == 2 || hw < 8, has_v = C::HALVES == 2 || hw >= 8;
    const uint32_t tl = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t a_v = C::A_V + half * C::VB * C::V_BUF, a_p = C::A_P + half * C::P_BUF, a_q = C::A_Q + half * C::Q_BYTES;
    const uint32_t p_row = a_p + (col0 / 64) * C::P_ATOM + my_tok * 128;
    float* const s_nm = reinterpret_cast<float*>(at(C::A_ROW + half * C::ROW_BYTES));
    float *const s_lc = s_nm + N, *const s_corr = s_lc + N, *const red = s_corr + N, *const red_v = red + 4 * N;
    float* const s_down = reinterpret_cast<float*>(at(C::A_DOWN + half * C::DOWN_BYTES));
    volatile uint32_t* const special = reinterpret_cast<volatile uint32_t*>(s_down + N);
    uint32_t* const cm = reinterpret_cast<uint32_t*>(at(C::A_MASK + half * C::MASK_BYTES));
    const uint32_t k_base = C::WINDOW + (BK == 2 ? (lane & 15) * 8 : lane * 4), v_base = C::WINDOW + 128 + (BV == 2 ? (lane & 15) * 8 : lane * 4);
    const uint32_t a_norm = C::A_NORM + 512 * half;
    auto stage_of = [&](int w) { return w < C::LOW_STAGES ? C::A_STAGE + w * C::STAGE : C::A_STAGE_HI + (w - C::LOW_STAGES) * C::STAGE; };
    int done = 0;       // tiles of earlier pieces: barriers have a phase for each tile
    // ... those of the keys' codes (LATE_V) but for a piece's second tile, whose codes come with the first's, to a place of their own.
    // (With phases that the feeder alone completes a slow warp could find two of them over, and wait for the one after.)
    auto k_phases = [&](int n_tiles) { return C::LATE_V && n_tiles > 1 ? n_tiles - 1 : n_tiles; };
    auto k_phase_of = [&](int tile) { return C::LATE_V && tile > 1 ? tile - 1 : tile; };      // (not of tile 1)

    // (In shared memory: what is needed once a piece would take the registers that the tiles need.  One thread finds a piece and
    // keeps the place behind it; the barrier at the end of a piece is behind every look at it.)
    static_assert(sizeof(TreePiece) <= 56, "");
    volatile TreePiece& pc = *reinterpret_cast<volatile TreePiece*>(at(C::A_PIECE + 64 * half));
    volatile int& pos = *reinterpret_cast<volatile int*>(at(C::A_PIECE + 64 * half + 56));
    // Registers: the workers get some of what the last four warps do not need, 512 x 104 + 128 x 64 of the 640 x 96 of the launch.
    // (Products of 64 rows spilled in every tile: 180 -> 173 us for 32 sequences of 8192 tokens and 16 nodes, before scales of rows.)
    static_assert(C::THREADS == 640 && 512 * 104 + 128 * 64 <= 640 * 96, "");
    __syncwarp();
    if (helper) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;\n");
        if (half < C::HALVES && (warp & 1) == 0) {
            // ---- the products of a half: one lane of its first helper
            constexpr uint32_t kIdescS = (1u << 4) | (static_cast<uint32_t>(N / 8) << 17) | (8u << 24);
            constexpr uint32_t kIdescO = kIdescS | (1u << 15) | (1u << 16);
            constexpr uint32_t kHi = (1024u >> 4) | (1u << 14) | (2u << 29);
            auto scores = [&](int tile) {
                if (elect_one()) {
                    const uint32_t q = (a_q >> 4) | ((16u >> 4) << 16);
#pragma unroll
                    for (int kb = 0; kb < D / 16; kb++)
                        one_mma_ts(tmem + C::COL_S, tmem + (tile & 1) * (D / 2) + 8 * kb, q + ((kb >> 2) * (N * 128) + (kb & 3) * 32) / 16, kHi, kIdescS, kb > 0);
#ifdef FTQ_TEST_WAIT_EXPIRY
                    if (!(tile == 1 && worker == 0))
#endif
                    tc_commit(s_done);
                }
                __syncwarp();
            };
            auto sums = [&](int tile) {
                if (elect_one()) {
                    const uint32_t v = ((a_v + (tile % C::VB) * C::V_BUF) >> 4) | ((static_cast<uint32_t>(C::V_ATOM) >> 4) << 16);
                    const uint32_t w = (a_p >> 4) | ((static_cast<uint32_t>(C::P_ATOM) >> 4) << 16);
#pragma unroll
                    for (int mb = 0; mb < C::MB; mb++)
#pragma unroll
                        for (int ks = 0; ks < kTreeTile / 16; ks++)
                            one_mma_ss(tmem + C::COL_O + mb * N, v + mb * (2 * C::V_ATOM >> 4) + ks * (2048 >> 4), w + ks * (2048 >> 4), kHi, kIdescO,
                                       ks > 0 ? 1u : static_cast<uint32_t>(tile));
                    tc_commit(o_done);
                }
                __syncwarp();
            };
#pragma unroll 1
            while (true) {
                meet_issuer(false);
                tc_fence_after();
                const int n_tiles = pc.n_tiles;
                if (n_tiles == 0) break;
                scores(0);
#pragma unroll 1
                for (int it = 0; it < n_tiles; it++) {
                    if (meet_issuer(false)) meet_issuer(false);     // (new maxima: the tile's weights come again)
                    tc_fence_after();
                    if (it + 1 < n_tiles) scores(it + 1);
                    sums(it);
                }
            }
            // nothing may be in flight when TMEM is given back
            if (elect_one()) tc_commit(drained);
            __syncwarp();
#pragma unroll 1
            for (int i = 0; i < kDrainSpinLimit && !mbar_try_wait(drained, 0); i++) {}
        }
        // ---- the pages of a half: its second helper.  Codes and norms come by bulk copies, a page of codes a warp, as soon as what lay
        // in their place was looked at.  (Registers would be the wrong place for them: loads that share one of the few scoreboards
        // complete together, so that a look at anything waits for the newest; and a copy takes its issuer 400 cycles.)
        if (half < C::HALVES && (warp & 1) == 1) {
            int k_sent = 0, v_sent = 0, n_sent = 0;
#pragma unroll 1
            while (true) {
                meet_feeder();
                const int n_tiles = pc.n_tiles;
                if (n_tiles == 0) break;
                const int tile0 = pc.tile0, seq = pc.seq, k_phase = pc.k_phase;
                const int32_t* const btab = p.block_table + static_cast<int64_t>(pc.b) * p.max_blocks;
                const uint8_t* const pool = p.pool + static_cast<int64_t>(pc.hkv) * C::PAGE_BYTES;
                // block ids of four tiles' pages (idb: of the next four); -1: no tokens
                auto has_tokens = [&](int tile) { return ((tile0 + tile) * (kTreeTile / kPageTokens) + (lane & 7)) * kPageTokens < seq; };
                auto load_ids = [&](int tile) {
                    const int t = tile + (lane >> 3), pg = (tile0 + t) * (kTreeTile / kPageTokens) + (lane & 7);
                    return load_id_if(t < n_tiles && has_tokens(t), btab + pg, -1);
                };
                int ida = load_ids(0), idb = load_ids(4);
                // of lane's page of a tile, while `now` is the tile that ida begins with or one of the three behind it
                auto id_of = [&](int tile, int now) { return __shfl_sync(0xffffffffu, (tile ^ now) < 4 ? ida : idb, (tile & 3) * 8 + (lane & 7)); };
                auto in_pool = [&](int id) { return static_cast<uint64_t>(static_cast<int64_t>(id)) < static_cast<uint64_t>(p.num_blocks); };
                auto page_of = [&](int id) { return pool + static_cast<int64_t>(id) * p.Hkv * C::PAGE_BYTES; };
                // page g of a tile is warp 4 (g & 1) + g / 2's; values: of the warps behind, if there are any
                const int owner = half * C::WH + 4 * (lane & 1) + ((lane & 7) >> 1);
                const uint32_t k_stage = stage_of(owner), v_stage = C::LATE_V ? a_v + 2048 * (lane & 7) : stage_of(owner + 8);
                // (what lies in the place of a page that is not there is as good: its weights are zero, or no numbers)
                auto fetch = [&](uint32_t bar, uint32_t dst, int id, int off, uint32_t bytes, int& sent) {
                    if (stalled) return;
                    sent++;
                    if (lane < 8) {
                        if (in_pool(id)) {
                            mbar_expect_tx(bar, bytes);
                            bulk_g2s(dst, page_of(id) + off, bytes, bar);
                        } else {
                            mbar_arrive(bar);
                        }
                    }
                    __syncwarp();
                };
                constexpr uint32_t kKeys = kPageTokens * C::PDK, kValues = kPageTokens * C::PDV;
                auto fetch_k = [&](int tile, int now) { fetch(k_full, k_stage, id_of(tile, now), 0, kKeys, k_sent); };
                auto fetch_v = [&](int tile, int now) { fetch(v_full, v_stage, id_of(tile, now), C::OFF_VC, kValues, v_sent); };
                // norms of a tile; a key of a page that is not in the pool has one that is no number
                auto fetch_norms = [&](int tile, int now) {
                    const int id = id_of(tile, now);
                    if (stalled) return;
                    n_sent++;
                    if (lane < 16) {
                        const bool value = lane & 8;
                        const uint32_t to = a_norm + 32 * lane;
                        if (in_pool(id)) {
                            mbar_expect_tx(n_full, 32);
                            bulk_g2s(to, page_of(id) + (value ? C::OFF_VN : C::OFF_KN), 32, n_full);
                        } else {
                            if (has_tokens(tile)) {     // (by its place, not by its id: a table may hold any)
                                if (!value) {
                                    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};\n" ::"r"(to), "r"(0x7e007e00u) : "memory");
                                    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};\n" ::"r"(to + 16), "r"(0x7e007e00u) : "memory");
                                }
                                __stcg(p.errors + 1, p.epoch);
                            }
                            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                            mbar_arrive(n_full);
                        }
                    }
                    __syncwarp();
                };
                if (C::LATE_V) {
                    // The first two tiles' keys at once and in one phase; the second's to where the warp will write its first values, after it
                    // has looked at them.  (Values wait in the place that they are written to as fp16: a page's 2 KB there have room
                    // for two pages' codes.)
                    const int id0 = id_of(0, 0), id1 = id_of(1, 0);
                    if (!stalled) {
                        k_sent++;
                        if (lane < 8) {
                            const bool has0 = in_pool(id0), has1 = n_tiles > 1 && in_pool(id1);
                            mbar_expect_tx(k_full, (has0 ? kKeys : 0) + (has1 ? kKeys : 0));
                            if (has0) bulk_g2s(k_stage, page_of(id0), kKeys, k_full);
                            if (has1) bulk_g2s(v_stage + 1024, page_of(id1), kKeys, k_full);
                        }
                        __syncwarp();
                    }
                    fetch_norms(0, 0);
                    fetch_v(0, 0);
                    if (n_tiles > 2) {
                        copied(k_free, k_phase);
                        fetch_k(2, 0);
                    }
                } else {
                    fetch_k(0, 0);
                    fetch_v(0, 0);
                    fetch_norms(0, 0);
                    if (n_tiles > 1) {
                        copied(k_free, k_phase);
                        fetch_k(1, 0);
                        copied(v_free, done);
                        fetch_v(1, 0);
                    }
                    if (n_tiles > 2) {
                        copied(k_free, k_phase + 1);
                        fetch_k(2, 0);
                    }
                }
#pragma unroll 1
                for (int it = 0; it + 1 < n_tiles; it++) {
                    copied(n_free, done + it);
                    fetch_norms(it + 1, it + 1);
                    if (it + 3 < n_tiles) {
                        copied(k_free, k_phase + k_phase_of(it + 2));
                        fetch_k(it + 3, it + 1);
                    }
                    if (C::LATE_V) {
                        wait(o_done, done + it);
                        fetch_v(it + 1, it + 1);
                    } else if (it + 2 < n_tiles) {
                        copied(v_free, done + it + 1);
                        fetch_v(it + 2, it + 1);
                    }
                    if (((it + 2) & 3) == 0) {      // (ida has the ids of the next round's tile it + 1)
                        ida = idb;
                        idb = load_ids(it + 6);
                    }
                }
                done += n_tiles;
                meet_feeder();      // (after a wait that ran out the workers do not wait for what is fetched: the piece stays until it was read)
            }
            auto drain = [&](uint32_t bar, int sent) {
#pragma unroll 1
                for (int i = 0; i < kDrainSpinLimit && sent > 0 && !mbar_try_wait(bar, (sent - 1) & 1); i++) {}
            };
            drain(k_full, k_sent);
            drain(v_full, v_sent);
            drain(n_full, n_sent);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 104;\n");
        if (me == 0) {
            pos = begin;
            pc.n_tiles = pc.k_phase = 0;
        }
        const uint32_t stage = stage_of(warp);
#pragma unroll 1
        while (true) {
            if (me == 0) {
                int from = pos;
                const TreePiece x = next_piece(from);
                pc.k_phase = pc.k_phase + k_phases(pc.n_tiles);
                pc.b = x.b;
                pc.hkv = x.hkv;
                pc.row0 = x.row0;
                pc.rows = x.rows;
                pc.tile0 = x.tile0;
                pc.n_tiles = x.n_tiles;
                pc.seq = x.seq;
                pc.ctx = x.ctx;
                pc.out = x.out;
                pos = from;
            }
            meet_feeder();
            const int n_tiles = pc.n_tiles, group = static_cast<int>(p.group.d);
            if (n_tiles == 0) {
                meet_issuer(false);
                break;
            }
            const int first_masked = pc.ctx / kTreeTile - pc.tile0;       // (from here on tiles reach the tree or the sequence's end)
            // keys: codes -> TMEM, rows = tokens
            auto put_k = [&](int tile, uint32_t from) {
                const bool own_phase = !C::LATE_V || tile != 1;
                if (own_phase) copied(k_full, pc.k_phase + k_phase_of(tile));
                typename Window<BK, false>::template Run<KW> r0, r1;
                tree_run<KSB>(from + g8 * C::PDK, t4, r0);
                tree_run<KSB>(from + (g8 + 8) * C::PDK, t4, r1);
                if (own_phase) taken(k_free);
                Window<BK, false>::shift(r0);
                Window<BK, false>::shift(r1);
                const uint32_t dst = tmem + (static_cast<uint32_t>(16 * my_page) << 16) + (tile & 1) * (D / 2);
#pragma unroll
                for (int q = 0; q < D / 64; q++) {
                    uint32_t x[16];
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        Window<BK, false>::pairs(r0, 4 * q + j, k_base, x[4 * j], x[4 * j + 1]);
                        Window<BK, false>::pairs(r1, 4 * q + j, k_base, x[4 * j + 2], x[4 * j + 3]);
                    }
                    tc_st_16x256b_x4(dst + 32 * q, x);
                }
            };
            // values: codes -> fp16 tile, MN-major with 128-byte swizzle
            // (a V row has its halves exchanged where bit 1 of its token's place is set)
            auto put_v = [&](int tile) {
                copied(v_full, done + tile);
                const uint32_t from = (C::LATE_V ? a_v + 2048 * my_page : stage) + g8 * C::PDV;
                typename Window<BV, false>::template Run<VW> run[2];
#pragma unroll
                for (int r = 0; r < 2; r++) tree_run<VSB>(from + 8 * r * C::PDV, t4 ^ (g8 & 2), run[r]);
                if (C::LATE_V) __syncwarp();
                else taken(v_free);
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    Window<BV, false>::shift(run[r]);
                    const int row = 16 * my_page + g8 + 8 * r;
                    const uint32_t dst = a_v + (tile % C::VB) * C::V_BUF + row * 128;
#pragma unroll
                    for (int jj = 0; jj < D / 32; jj++) {
                        uint32_t x[4];
                        Window<BV, false>::pairs(run[r], 2 * jj, v_base, x[0], x[1]);
                        Window<BV, false>::pairs(run[r], 2 * jj + 1, v_base, x[2], x[3]);
                        // (eight lanes that store together have two rows and four chunks apart by two: no two on the same banks)
                        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};\n" ::"r"(dst + (jj >> 1) * C::V_ATOM + (((2 * t4 + (jj & 1)) ^ (row & 7)) << 4)),
                                     "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]) : "memory");
                    }
                }
            };
            // ---- the queries: rotated, scaled, fp16, K-major with 128-byte swizzle
            float q_down;           // of the common scale
            {
                const int b = pc.b, hkv = pc.hkv, row0 = pc.row0, rows = pc.rows, ctx = pc.ctx;
                constexpr int OCTETS = C::HT / 8;
                const int t8 = lane & 7, octet = me >> 3;
                auto query = [&](int r) {   // row r's 16-byte pieces: eight coordinates each
                    const int i = fast_div(row0 + r, p.group), h = row0 + r - i * group;
                    return static_cast<const uint4*>(p.q) + (((static_cast<int64_t>(b) * p.T + i) * p.Hq + hkv * group + h) * D) / 8;
                };
                auto widen = [&](const uint4& x, float (&o)[8]) {
                    if (p.q_dtype == kBF16) load8<__nv_bfloat16>(reinterpret_cast<const __nv_bfloat16*>(&x), o);
                    else load8<__half>(reinterpret_cast<const __half*>(&x), o);
                };
                // (read once: two rows an octet at most)
                constexpr int NR = (N + OCTETS - 1) / OCTETS;
                uint4 raw[NR][D / 64];
#pragma unroll
                for (int k = 0; k < NR; k++)
#pragma unroll
                    for (int j = 0; j < D / 64; j++) {
                        const int r = octet + k * OCTETS;
                        raw[k][j] = r < rows ? query(r)[t8 + 8 * j] : make_uint4(0, 0, 0, 0);
                    }
                // the mask words of the rows' nodes (to where weights will be)
                const bool trees = (pc.tile0 + n_tiles) * kTreeTile > ctx;
                const int i0 = fast_div(row0, p.group), words = (p.T + 31) / 32;
                uint32_t* const mask_words = reinterpret_cast<uint32_t*>(at(a_p));
                static_assert(N * (kTreeMaxNodes / 32) * 4 <= C::P_BUF, "");
                if (trees)
                    for (int k = me; k < (fast_div(row0 + rows - 1, p.group) - i0 + 1) * words; k += C::HT)
                        mask_words[k] = p.masks[(static_cast<int64_t>(b) * p.T + i0 + k / words) * p.W + k % words];
                // the largest of each row and of all, for their scale: |rotated| <= D * largest |q|, and that shall be below 2^15
                float row_top[NR], top = 0.f;
#pragma unroll
                for (int k = 0; k < NR; k++) {
                    row_top[k] = 0.f;
#pragma unroll
                    for (int j = 0; j < D / 64; j++) {
                        float v[8];
                        widen(raw[k][j], v);
#pragma unroll
                        for (int c = 0; c < 8; c++) row_top[k] = fabsf(v[c]) <= FLT_MAX ? fmaxf(row_top[k], fabsf(v[c])) : row_top[k];
                    }
#pragma unroll
                    for (int x = 1; x < 8; x <<= 1) row_top[k] = fmaxf(row_top[k], __shfl_xor_sync(0xffffffffu, row_top[k], x));
                    top = fmaxf(top, row_top[k]);
                }
                top = warp_max(top);
                if (lane == 0) red[hw] = top;
                if (me < N) s_nm[me] = INFINITY;
                if (me == 0) *special = 0;
                meet();
#pragma unroll
                for (int w = 0; w < C::WH; w++) top = fmaxf(top, red[w]);
                // powers of two: the exponent of a scale, and the scale
                auto exponent = [&](float t) {
                    const int x = (__float_as_int(t * (fabsf(p.q_scale) * D)) >> 23) - 127;      // (128: infinite, that is below 2^134)
                    return max(-120, min(120, 14 - (x == 128 ? 134 : x)));
                };
                auto two_to = [](int e) { return __int_as_float((127 + e) << 23); };
                // A common scale where it costs nothing: rows of up to 2^kTreeSpread times less than the largest keep all their bits, or
                // lose some of 2^-15 of their size.  Smaller ones are scaled up, and their scores down again.
                const int e = top > 0.f ? exponent(top) : 0;
                q_down = two_to(-e);
#pragma unroll
                for (int k2 = 0; k2 < NR; k2++) {
                    const int r = octet + k2 * OCTETS;
                    const int more = row_top[k2] > 0.f ? min(120, exponent(row_top[k2]) - e) : 0, own = more > kTreeSpread ? more : 0;
                    const float up = p.q_scale * two_to(e + own);
                    if (t8 == 0 && r < N) s_down[r] = two_to(-own);
                    if (own > 0) *special = 1;
                    float a[E];
#pragma unroll
                    for (int k = 0; k < D / 64; k++) {
                        float v[8];
                        widen(raw[k2][k], v);
#pragma unroll
                        for (int c = 0; c < 8; c++)
                            a[8 * k + c] = __uint_as_float(__float_as_uint(v[c] * up) ^ sign_mask(p.signs, load_coord(t8, 8 * k + c)));
                    }
                    octet_fwht<E>(a, lane);
                    // Coordinate c = t8 + 8 k is code 4 jj + (c & 3) of lane t's run: place 16 jj + 4 t + (c & 3).  Two lanes have two
                    // neighbours: of two k's the even lane stores the first, the odd lane the second.
                    uint8_t* dst = at(a_q) + r * 128;
#pragma unroll
                    for (int k = 0; k < E; k += 2) {
                        const float other = __shfl_xor_sync(0xffffffffu, (t8 & 1) ? a[k] : a[k + 1], 1);
                        const int c = (t8 & 6) + 8 * (k + (t8 & 1)), t = c / (D / 4), jj = (c % (D / 4)) / 4, place = 16 * jj + 4 * t + (c & 3);
                        const uint32_t h = (t8 & 1) ? f2h2(other, a[k + 1]) : f2h2(a[k], other);
                        if (r < N) *reinterpret_cast<uint32_t*>(dst + (place >> 6) * (N * 128) + ((((place & 63) >> 3) ^ (r & 7)) << 4) + (place & 7) * 2) = h;
                    }
                }
                // which rows attend a node: bit r of its words
                if (trees) {
                    const int nodes = pc.seq - ctx;
                    for (int k = me; k < nodes * C::MW; k += C::HT) {
                        const int node = k / C::MW, w = k % C::MW;
                        uint32_t bits = 0;
                        // (a node's heads are neighbours: a run of bits)
                        const int r1 = min(rows, 32 * w + 32);
#pragma unroll 1
                        for (int r = 32 * w; r < r1;) {
                            const int i = fast_div(row0 + r, p.group), stop = min(r1, (i + 1) * group - row0);
                            if ((mask_words[(i - i0) * words + (node >> 5)] >> (node & 31)) & 1u)
                                bits |= (0xffffffffu >> (32 - (stop - r))) << (r & 31);
                            r = stop;
                        }
                        cm[k] = bits;
                    }
                }
            }
            if (has_k) put_k(0, stage);
            if (has_v && !C::LATE_V) put_v(0);
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            tc_wait_st();
            tc_fence_before();
            meet_issuer(false);
            if (has_k && n_tiles > 1) put_k(1, C::LATE_V ? a_v + 2048 * my_page + 1024 : stage);
            float l[CW], vs = 0.f;      // sums of the thread's tokens; scale of |v|
#pragma unroll
            for (int c = 0; c < CW; c++) l[c] = 0.f;

#pragma unroll 1
            for (int it = 0; it < n_tiles; it++) {
                const bool masked = it >= first_masked;
                uint32_t nk, nv;
                copied(n_full, done + it);
                asm volatile("ld.shared.u16 %0, [%1];\n" : "=r"(nk) : "r"(a_norm + 2 * my_tok) : "memory");
                asm volatile("ld.shared.u16 %0, [%1];\n" : "=r"(nv) : "r"(a_norm + 256 + 2 * my_tok) : "memory");
                taken(n_free);
                const bool settled = *special != 0;
                float kn = half_bits_to_float(nk) * q_down;
                const float vn = half_bits_to_float(nv);
                // which of the group's rows attend the token; |v| where one does and it is finite
                uint32_t bits = 0xffffffffu;
                if (masked) {
                    const int node = (pc.tile0 + it) * kTreeTile + my_tok - pc.ctx;
                    if (node >= 0) bits = node >= pc.seq - pc.ctx ? 0u : cm[node * C::MW + col0 / 32] >> (col0 & 31);
                }
                if (CW < 32) bits &= (1u << (CW & 31)) - 1u;
                const float av = bits != 0 && fabsf(vn) <= FLT_MAX ? fabsf(vn) : 0.f;
                const uint32_t s_at = tl + C::COL_S + col0;
                // Where rows have scales of their own, or a maximum is so large that what an fma does not round is far from zero as an
                // exponent: S becomes the scores, rounded as they were when a maximum was taken.
                auto settle = [&]() {
#pragma unroll 1
                    for (int c0 = 0; c0 < CW; c0 += 8) {
                        uint32_t s[8];
                        tc_load(s_at + c0, s);
#pragma unroll
                        for (int c = 0; c < 8; c++) s[c] = __float_as_uint(__uint_as_float(s[c]) * s_down[col0 + c0 + c] * kn);
                        tc_st8(s_at + c0, s);
                    }
                    tc_wait_st();
                    kn = 1.f;
                };
                // scores - maxima (base 2)
                auto exponents = [&](float* x) {
                    uint32_t s[CW];
                    tc_load(s_at, s);
                    const u64 kn2 = pk2(kn, kn);
#pragma unroll
                    for (int c = 0; c < CW; c += 4) {
                        const float4 nm = *reinterpret_cast<const float4*>(s_nm + col0 + c);
                        upk2(fma2(pk2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), kn2, pk2(nm.x, nm.y)), x[c], x[c + 1]);
                        upk2(fma2(pk2(__uint_as_float(s[c + 2]), __uint_as_float(s[c + 3])), kn2, pk2(nm.z, nm.w)), x[c + 2], x[c + 3]);
                    }
                };
                // weights to shared memory and into the sums
                auto weights = [&](const float* x, auto with_masks, bool add) {
                    const float vw = vn * vs;
                    const u64 vw2 = pk2(vw, vw);
#pragma unroll
                    for (int c = 0; c < CW; c += 8) {
                        uint32_t h[4];
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const int k = c + 2 * j;
                            const float e0 = fast_exp2(x[k]), e1 = fast_exp2(x[k + 1]);
                            if (!decltype(with_masks)::value || add) upk2(add2(pk2(l[k], l[k + 1]), pk2(e0, e1)), l[k], l[k + 1]);
                            float w0, w1;
                            upk2(mul2(pk2(e0, e1), vw2), w0, w1);
                            if constexpr (decltype(with_masks)::value) {    // (what a row does not attend may have a norm that is not a number)
                                w0 = (bits >> k) & 1u ? w0 : 0.f;
                                w1 = (bits >> (k + 1)) & 1u ? w1 : 0.f;
                            }
                            h[j] = f2h2(w0, w1);
                        }
                        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};\n" ::"r"(p_row + (((((col0 & 63) + c) >> 3) ^ (my_tok & 7)) << 4)),
                                     "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
                    }
                };
                auto apply_masks = [&](float* x) {
#pragma unroll
                    for (int c = 0; c < CW; c++) x[c] = (bits >> c) & 1u ? x[c] : -INFINITY;
                };
                wait(s_done, done + it);
                if (soft && settled) settle();
                if (!C::LATE_V && C::VB == 2 && it > 0) wait(o_done, done + it - 1);       // (P.V of the tile before has read the weights)
                bool above = false;
                float x[CW];
                auto too_high = [&](const float* y) {
                    float top = fmaxf(y[0], y[1]);
#pragma unroll
                    for (int c = 2; c < CW; c += 2) top = fmaxf(fmaxf(top, y[c]), y[c + 1]);
                    return __any_sync(0xffffffffu, top > kTreeSlack || (vs == 0.f ? av > 0.f : av * vs > kTreeGrowth)) != 0;
                };
                // (two paths down to the vote: a branch around the selects alone becomes selects in every tile)
                if (soft && !masked) {
                    exponents(x);
                    above = too_high(x);
                } else if (soft) {
                    exponents(x);
                    apply_masks(x);
                    above = too_high(x);
                }
                if (C::LATE_V && it > 0) wait(o_done, done + it - 1);
                if (soft && !above) {
                    if (masked) weights(x, std::true_type{}, true);
                    else weights(x, std::false_type{}, true);
                }
                if (C::LATE_V) {
                    put_v(it);
                }
                asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                tc_wait_st();
                tc_fence_before();
                if (meet_issuer(above)) {
                    // ---- new maxima; O, the sums and the tile's weights refer to them
                    const float m_run = soft && lane < CW ? -s_nm[col0 + lane] : 0.f;
                    if (soft) {
                        float mine = -INFINITY;
#pragma unroll 1
                        for (int c0 = 0; c0 < CW; c0 += 8) {
                            uint32_t s[8];
                            tc_load(s_at + c0, s);
#pragma unroll
                            for (int c = 0; c < 8; c++) {
                                const float r = warp_max((bits >> (c0 + c)) & 1u ? __uint_as_float(s[c]) * kn : -INFINITY);
                                if (lane == c0 + c) mine = r;
                            }
                        }
                        const float wv = warp_max(av);
                        if (lane < CW) red[quarter * N + col0 + lane] = mine;
                        if (lane == 0) red_v[hw] = wv;
                    }
                    meet();
                    float v_ratio = 1.f;
                    if (soft) {
                        float v_top = 0.f;
#pragma unroll
                        for (int w = 0; w < 4; w++) v_top = fmaxf(v_top, red_v[4 * cg + w]);
                        if (v_top > 0.f && (vs == 0.f || v_top * vs > kTreeGrowth)) {   // the largest |v| becomes 1 to 2
                            const float to = ldexpf(1.f, -ilogbf(v_top));
                            v_ratio = vs == 0.f ? 1.f : to / vs;
                            vs = to;
                        }
                        if (lane < CW) {
                            float m_new = m_run;
#pragma unroll
                            for (int w = 0; w < 4; w++) m_new = fmaxf(m_new, red[w * N + col0 + lane]);
                            const float lc = m_run == -INFINITY ? 0.f : fast_exp2(m_run - m_new);
                            if (quarter == 0) {
                                s_nm[col0 + lane] = -m_new;
                                s_lc[col0 + lane] = lc;
                                s_corr[col0 + lane] = lc * v_ratio;
                                if (fabsf(m_new) > kTreeRounded && m_new != -INFINITY) *special = 1;
                            }
                        }
                    }
                    meet();
                    if (soft && !settled && *special) settle();
                    if (soft) {
#pragma unroll
                        for (int c = 0; c < CW; c += 4) {
                            const float4 f = *reinterpret_cast<const float4*>(s_lc + col0 + c);
                            l[c] *= f.x;
                            l[c + 1] *= f.y;
                            l[c + 2] *= f.z;
                            l[c + 3] *= f.w;
                        }
                        if (it > 0) {       // (P.V of the tile before is complete)
#pragma unroll
                            for (int mb = 0; mb < C::MB; mb++) {
#pragma unroll 1
                                for (int c = 0; c < CW; c += 8) {       // (few registers: what this path spills the others pay for)
                                    uint32_t o[8];
                                    const uint32_t o_at = tl + C::COL_O + mb * N + col0 + c;
                                    const float4 f = *reinterpret_cast<const float4*>(s_corr + col0 + c), g = *reinterpret_cast<const float4*>(s_corr + col0 + c + 4);
                                    const float by[8] = {f.x, f.y, f.z, f.w, g.x, g.y, g.z, g.w};
                                    tc_load(o_at, o);
#pragma unroll
                                    for (int k = 0; k < 8; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) * by[k]);
                                    tc_st8(o_at, o);
                                }
                            }
                        }
                        exponents(x);
                        apply_masks(x);
                        weights(x, std::true_type{}, above);
                    }
                    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                    tc_wait_st();
                    tc_fence_before();
                    meet_issuer(false);
                }
                tc_fence_after();
                if (it + 1 == n_tiles) break;
                // ---- the tiles to come
                if (has_k && it + 2 < n_tiles) put_k(it + 2, stage);
                if (!C::LATE_V) {
                    if (C::VB == 1) wait(o_done, done + it);
                    if (has_v) put_v(it + 1);
                }
            }
            // ---- the piece's rows
            wait(o_done, done + n_tiles - 1);
            done += n_tiles;
            const int rows = pc.rows;
            float* const to = pc.out;
            if (soft) {
                // sums over the lanes, then over the warps: lane c gets row c's
                float sum[CW];
#pragma unroll
                for (int c = 0; c < CW; c++) {
                    sum[c] = l[c];
#pragma unroll
                    for (int d = CW; d < 32; d <<= 1) sum[c] += __shfl_xor_sync(0xffffffffu, sum[c], d);
                }
#pragma unroll
                for (int d = CW / 2; d > 0; d >>= 1) {
#pragma unroll
                    for (int i = 0; i < d; i++) {
                        const bool hi = (lane & d) != 0;
                        const float send = hi ? sum[i] : sum[i + d], keep = hi ? sum[i + d] : sum[i];
                        sum[i] = keep + __shfl_xor_sync(0xffffffffu, send, d);
                    }
                }
                if (lane < CW) red[quarter * N + col0 + lane] = sum[0];
            }
            meet();
            if (soft) {
                if (quarter == 0 && lane < CW && col0 + lane < rows) {
                    float* dst = to + (col0 + lane) * ROW + D;
                    const float* r = red + col0 + lane;
                    dst[0] = -s_nm[col0 + lane];
                    dst[1] = r[0] + r[N] + r[2 * N] + r[3 * N];
                }
                const float scale = p.inv_v_scale / (vs == 0.f ? 1.f : vs);
#pragma unroll
                for (int mb = 0; mb < C::MB; mb++) {
                    uint32_t o[CW];
                    tc_load(tl + C::COL_O + mb * N + col0, o);
                    // TMEM row m: atom m / 64, 16-byte chunk (m % 64) / 8 = 2 t + (jj & 1): coordinate 8 jj + m % 8 of run t
                    const int m = my_tok + 128 * mb, chunk = (m & 63) >> 3, jj = 2 * (m >> 6) + (chunk & 1);
                    const int coord = (chunk >> 1) * (D / 4) + 8 * jj + (m & 7);
                    if (D == 64 && m >= 64) continue;
#pragma unroll
                    for (int c = 0; c < CW; c++)
                        if (col0 + c < rows) to[(col0 + c) * ROW + coord] = __uint_as_float(o[c]) * scale;
                }
            }
            tc_fence_before();
            meet_feeder();      // (the next piece writes to what these reads came from)
            tc_fence_after();
        }
    }
    __syncwarp();
    __syncthreads();
    if (*gave_up && !helper) {   // all that this half has
        int at_pos = begin;
        for (TreePiece pc = next_piece(at_pos); pc.n_tiles > 0; pc = next_piece(at_pos))
            for (int r = me; r < N; r += C::HT) pc.out[r * ROW + D] = __int_as_float(0x7fc00000);
        if (me == 0) __stcg(p.errors, p.epoch);
    }
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem_all));
    }
}

// Joins the pieces of every (sequence, node, head) row by their maxima, rotates back (core/hadamard.py:93-100) and stores; nodes
// that do not exist and rows that attend nothing are zero.  OCTETS octets per row, as in attn_merge_kernel.
struct TreeMergeParams {
    const int* plan;
    const float *whole, *cut;
    const int32_t *tree_lens, *seq_lens;
    void* out;
    int B, T, Hq, Hkv, N, row_tiles, max_seq, piece;
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
        if (tree_tile_of(to - pos, p.piece) <= tree_tile_of(from - pos, p.piece)) return nullptr;
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
