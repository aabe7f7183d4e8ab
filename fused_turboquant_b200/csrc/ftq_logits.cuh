// Logits of a serving step: penalties for repeated tokens, biases, grammar masks, best token.
//
//   y = x > 0 ? x / repetition : x * repetition     where the token is in the prompt or the answer so far
//   y = y - frequency * count - presence * [count > 0]   count: how often it is in the answer so far
//   y = y + bias;   y = -inf where it is not allowed;   best = the lowest index of the largest y
//
// With a drafted tree a request has a row of logits for each node, and the tokens on a node's path count as its answer.
// Each operation is rounded once in fp32, in this order.
//
// A CTA has a segment of the vocabulary of one request and some of its rows.  It counts the history's tokens of its
// segment in shared memory (a word a token: the count, a bit each for the prompt, a bias and a node of the tree) once for all its
// rows, lists each warp's tokens that have a word, and then streams the rows: a warp works on its listed tokens side by side, the
// others are converted and stored.  Between rows the counts change by the nodes on whose paths the rows differ.  No dense
// [requests, vocabulary] count exists in memory.
//
// A row's 2 bytes in, 4 out and a bit of mask per token are 63 us of HBM for 32 requests of 16 nodes, 131072 tokens, 8192 of
// history and 100 biases; it takes 127 us (3.25 TB/s).  68 % of the issue slots are in use (240 instructions for a warp's 256 tokens of a
// row: masks, maxima, listed tokens); the longest stalls are loads from global memory (one row is on its way), then the barriers between
// rows, whose counts change, and 2.8 rounds of CTAs begin with the history.  152 us had the eight tokens of a thread adjusted where
// they lie (a division for one or two lanes at a time), the index of the largest carried from token to token and two barriers a
// row.  Segments of 4096 tokens, CTAs of 512: 130 us.  The row on its way and 48 registers (five CTAs an SM; fp32 logits spill eight
// words) go together: without the one 154 us, with 40 or 32 registers, which spill more, 175 and 193; four tokens and four more a
// lane, for whole sectors in a store, 147.
#pragma once

#include "ftq_serve_launch.h"

namespace ftq {

constexpr int kLogitThreads = 256;
constexpr uint32_t kInPrompt = 1u << 31, kHasBias = 1u << 30, kHasNode = 1u << 29, kCountMask = kHasNode - 1;
static_assert(kLogitSegment == 8 * kLogitThreads, "a thread has eight tokens of a segment");

// Orders as the value does; NaN above all.  Lower indexes are larger.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t u = __float_as_uint(x);
    return x != x ? 0xffffffffu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float max_or_nan(float a, float b) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(m) : "f"(a), "f"(b));
    return m;
}

__device__ __forceinline__ float warp_max_or_nan(float x) {
    float m;
    asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;\n" : "=f"(m) : "f"(x));
    return m;
}

// (A call: few tokens come here, and inlined for each of a thread's tokens it took half of the registers.)
__device__ __noinline__ float adjusted(float x, uint32_t word, float repetition, float frequency, float presence, float bias) {
    const uint32_t count = word & kCountMask;
    if (word & (kInPrompt | kCountMask)) x = x > 0.f ? __fdiv_rn(x, repetition) : __fmul_rn(x, repetition);
    if (count) x = __fsub_rn(__fsub_rn(x, __fmul_rn(frequency, static_cast<float>(count))), presence);
    if (word & kHasBias) x = __fadd_rn(x, bias);
    return x;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kLogitThreads, 5) logits_kernel(const LogitParams p) {
    extern __shared__ uint32_t s_words[];
    uint32_t* const s_word = s_words;                                           // [segment]
    float* const s_y = reinterpret_cast<float*>(s_words + kLogitSegment);        // [segment]: a row's values of the tokens that have a word
    uint8_t* const s_list = reinterpret_cast<uint8_t*>(s_words + 2 * kLogitSegment);   // [segment]: each warp's such tokens
    int* const s_bias = reinterpret_cast<int*>(s_list + kLogitSegment);        // [segment]: place in the list (K > 0 only)
    __shared__ int s_node[kTreeMaxNodes], s_place[kTreeMaxNodes];          // nodes whose token lies in the segment
    __shared__ int s_nodes;
    __shared__ unsigned long long s_best[kTreeMaxNodes];                  // of each row
    const int tid = threadIdx.x, lane = tid & 31, r = blockIdx.y;
    const int seg0 = blockIdx.x * kLogitSegment, n = min(kLogitSegment, p.V - seg0);
    const int row0 = blockIdx.z * p.rows_per_cta, row1 = min(p.T, row0 + p.rows_per_cta);
    const int W = (p.T + 31) / 32;
    for (int i = tid; i < kLogitSegment / 4; i += kLogitThreads) {
        reinterpret_cast<uint4*>(s_word)[i] = make_uint4(0, 0, 0, 0);
        if (p.K > 0) reinterpret_cast<int4*>(s_bias)[i] = make_int4(-1, -1, -1, -1);
    }
    if (tid == 0) s_nodes = 0;
    for (int i = tid; i < row1 - row0; i += kLogitThreads) s_best[i] = 0;
    after_previous_kernel();
    let_next_kernel_start();
    __syncthreads();
    auto in_segment = [&](int token) { return static_cast<uint32_t>(token) - static_cast<uint32_t>(seg0) < static_cast<uint32_t>(n); };
    if (p.history) {
        const int len = min(max(p.history_lens[r], 0), p.H), prompt = p.prompt_lens ? p.prompt_lens[r] : 0;
        const int32_t* h = p.history + static_cast<int64_t>(r) * p.H;
        auto count = [&](int t, int i) {
            if (!in_segment(t)) return;
            if (i < prompt) atomicOr(&s_word[t - seg0], kInPrompt);
            else atomicAdd(&s_word[t - seg0], 1u);
        };
        const int fours = (reinterpret_cast<uintptr_t>(h) & 15) == 0 ? len / 4 : 0;
#pragma unroll 4
        for (int i = tid; i < fours; i += kLogitThreads) {
            const int4 t = reinterpret_cast<const int4*>(h)[i];
            count(t.x, 4 * i);
            count(t.y, 4 * i + 1);
            count(t.z, 4 * i + 2);
            count(t.w, 4 * i + 3);
        }
#pragma unroll 4
        for (int i = 4 * fours + tid; i < len; i += kLogitThreads) count(h[i], i);
    }
    for (int k = tid; k < p.K; k += kLogitThreads) {
        const int t = p.bias_ids[static_cast<int64_t>(r) * p.K + k];
        if (in_segment(t)) {
            atomicOr(&s_word[t - seg0], kHasBias);
            atomicMax(&s_bias[t - seg0], k);   // (of a token's entries the last counts)
        }
    }
    if (p.tree_masks) {
        for (int j = tid; j < p.T; j += kLogitThreads) {
            const int t = p.tree_tokens[static_cast<int64_t>(r) * p.T + j];
            if (in_segment(t)) {
                const int k = atomicAdd(&s_nodes, 1);
                s_node[k] = j;
                s_place[k] = t - seg0;
                atomicOr(&s_word[t - seg0], kHasNode);
            }
        }
    }
    __syncthreads();
    const int nodes = s_nodes;
    const float rep = p.repetition ? p.repetition[r] : 1.f, freq = p.frequency ? p.frequency[r] : 0.f,
                pres = p.presence ? p.presence[r] : 0.f;
    auto adjust = [&](float x, uint32_t word, int place) {
        return adjusted(x, word, rep, freq, pres, (word & kHasBias) ? p.bias[static_cast<int64_t>(r) * p.K + s_bias[place]] : 0.f);
    };
    // A thread has eight tokens; its warp's that have a word are listed once for all rows, so that a row's few are worked on side by
    // side.  (Where they lie, each of the eight in turn, nearly every warp took the branch, for one lane or two.)
    const int e = 8 * tid, warp0 = 256 * (tid >> 5);
    uint32_t touched = 0, listed = 0;
    if constexpr (VEC) {
        if (e < n) {
            const uint4 a = *reinterpret_cast<const uint4*>(s_word + e), b = *reinterpret_cast<const uint4*>(s_word + e + 4);
            const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
            for (int c = 0; c < 8; c++) touched |= w[c] ? 1u << c : 0u;
        }
        const uint32_t mine = __popc(touched);
        uint32_t sum = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= d) sum += y;
        }
        listed = __shfl_sync(0xffffffffu, sum, 31);
        uint8_t* to = s_list + warp0 + sum - mine;
        for (uint32_t t = touched; t; t &= t - 1) *to++ = static_cast<uint8_t>(8 * lane + __ffs(t) - 1);
        __syncwarp();
    }
    // a row's tokens as they come: the next row's are on their way while one is worked on
    constexpr int PARTS = sizeof(T) / 2;
    uint4 raw[PARTS];
    uint32_t raw_bits = 0xff;
    T raw_listed;       // of the lane's entry of the list
    const int listed_at = VEC && lane < listed ? warp0 + s_list[warp0 + lane] : -1;
    // (of the row to fetch next: pointers that move on, a row's 64-bit products would be a sixth of its instructions)
    const int64_t at0 = static_cast<int64_t>(r) * p.T + row0;
    const T* next_src = static_cast<const T*>(p.logits) + at0 * p.row_stride + seg0;
    const uint8_t* next_ok = p.allowed ? p.allowed + at0 * p.allowed_stride + seg0 / 8 + tid : nullptr;
    float* dst = p.out ? p.out + at0 * p.V + seg0 : nullptr;
    auto fetch = [&]() {
        if (e < n) {
#pragma unroll
            for (int i = 0; i < PARTS; i++) raw[i] = reinterpret_cast<const uint4*>(next_src + e)[i];
            if (next_ok) raw_bits = *next_ok;
        }
        if (listed_at >= 0) raw_listed = next_src[listed_at];
        next_src += p.row_stride;
        if (next_ok) next_ok += p.allowed_stride;
    };
    // the warp's best of the 32 rows so far, a row a lane
    float kept = 0.f;
    uint32_t kept_at = 0xffffffffu;
    auto keep = [&](int from) {     // rows from .. from + 31
        if (kept_at != 0xffffffffu)
            atomicMax(&s_best[from - row0 + lane], static_cast<unsigned long long>(order_of(__fadd_rn(kept, 0.f))) << 32 | (0xffffffffu - (seg0 + kept_at)));
        kept_at = 0xffffffffu;
    };
    if (VEC) fetch();
    for (int row = row0; row < row1; row++) {
        const int64_t at = static_cast<int64_t>(r) * p.T + row;
        if (nodes > 0) {
            // the counts are those of the row before: add what this path has more, take what it has less
            if (row > row0) __syncthreads();
            const int32_t *now = p.tree_masks + at * W, *was = now - W;
            for (int k = tid; k < nodes; k += kLogitThreads) {
                const int j = s_node[k], on = (now[j >> 5] >> (j & 31)) & 1, before = row > row0 ? (was[j >> 5] >> (j & 31)) & 1 : 0;
                if (on != before) atomicAdd(&s_word[s_place[k]], static_cast<uint32_t>(on - before));
            }
            __syncthreads();
        }
        if constexpr (VEC) {
            float x[8];
            load8<T>(reinterpret_cast<const T*>(raw), x);
            const uint32_t bits = raw_bits;
            if (listed_at >= 0) s_y[listed_at] = adjust(to_float<T>(raw_listed), s_word[listed_at], listed_at);
            const T* const src = next_src - p.row_stride;
            if (row + 1 < row1) fetch();
            if (listed > 0) {
                for (int j = lane + 32; j < listed; j += 32) {
                    const int place = warp0 + s_list[warp0 + j];
                    s_y[place] = adjust(to_float<T>(src[place]), s_word[place], place);
                }
                __syncwarp();
                if (touched) {
                    const float4 a = *reinterpret_cast<const float4*>(s_y + e), b = *reinterpret_cast<const float4*>(s_y + e + 4);
                    const float y[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
                    for (int c = 0; c < 8; c++) x[c] = (touched >> c) & 1 ? y[c] : x[c];
                }
                __syncwarp();
            }
            if (bits != 0xff) {
#pragma unroll
                for (int c = 0; c < 8; c++) x[c] = (bits >> c) & 1 ? x[c] : -INFINITY;
            }
            float top = x[0];
#pragma unroll
            for (int c = 1; c < 8; c++) top = max_or_nan(top, x[c]);
            if (dst && e < n) {
                __stcs(reinterpret_cast<float4*>(dst + e), make_float4(x[0], x[1], x[2], x[3]));
                __stcs(reinterpret_cast<float4*>(dst + e + 4), make_float4(x[4], x[5], x[6], x[7]));
            }
            if (p.keys) {
                // the largest of the warp, then the first place that has it
                const float most = warp_max_or_nan(e < n ? top : -INFINITY);
                uint32_t first = 0xffffffffu;
                if (most == most) {
#pragma unroll
                    for (int c = 7; c >= 0; c--) first = x[c] == most ? e + c : first;
                } else {
#pragma unroll
                    for (int c = 7; c >= 0; c--) first = x[c] != x[c] ? e + c : first;
                }
                first = __reduce_min_sync(0xffffffffu, e < n ? first : 0xffffffffu);
                const int k = (row - row0) & 31;
                if (lane == k) {
                    kept = most;
                    kept_at = first;
                }
                if (k == 31 || row + 1 == row1) keep(row - k);
            }
        } else {
            const T* src = static_cast<const T*>(p.logits) + at * p.row_stride + seg0;
            const uint8_t* ok = p.allowed ? p.allowed + at * p.allowed_stride + seg0 / 8 : nullptr;
            uint32_t best = 0, best_at = 0;
            auto consider = [&](float y, int place) {   // (places ascend)
                const uint32_t o = order_of(__fadd_rn(y, 0.f));
                if (o > best) {
                    best = o;
                    best_at = place;
                }
            };
            constexpr int ONES = kLogitSegment / kLogitThreads;
            float x[ONES];
#pragma unroll
            for (int k = 0; k < ONES; k++) {
                const int at1 = k * kLogitThreads + tid;
                x[k] = at1 < n ? to_float<T>(src[at1]) : 0.f;
            }
#pragma unroll
            for (int k = 0; k < ONES; k++) {
                const int at1 = k * kLogitThreads + tid;
                if (at1 >= n) break;
                const uint32_t w = s_word[at1];
                if (w) x[k] = adjust(x[k], w, at1);
                if (ok && !((ok[at1 / 8] >> (at1 % 8)) & 1)) x[k] = -INFINITY;
                if (p.keys) consider(x[k], at1);
                if (dst) dst[at1] = x[k];
            }
            if (p.keys) {
                const uint32_t most = __reduce_max_sync(0xffffffffu, best);
                const uint32_t first = __reduce_min_sync(0xffffffffu, best == most ? best_at : 0xffffffffu);
                if (lane == 0 && most) atomicMax(&s_best[row - row0], static_cast<unsigned long long>(most) << 32 | (0xffffffffu - (seg0 + first)));
            }
        }
        if (dst) dst += p.V;
    }
    if (p.keys) {
        __syncthreads();
        for (int i = tid; i < row1 - row0; i += kLogitThreads) p.keys[(static_cast<int64_t>(r) * p.T + row0 + i) * p.segments + blockIdx.x] = s_best[i];
    }
}

// The best of a row's segments: a warp per row.
__global__ void __launch_bounds__(128) logits_best_kernel(const unsigned long long* keys, int32_t* best, int64_t rows, int segments) {
    const int lane = threadIdx.x & 31;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
    after_previous_kernel();
    let_next_kernel_start();
    if (row >= rows) return;
    unsigned long long k = 0;
    for (int s = lane; s < segments; s += 32) k = max(k, keys[row * segments + s]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) k = max(k, __shfl_xor_sync(0xffffffffu, k, d));
    if (lane == 0) best[row] = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(k));
}

}  // namespace ftq
