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
// segment in shared memory (a word a token: the count, a bit for the prompt, a bit for a bias) once for all its rows,
// and then streams the rows: nearly all tokens have a zero word and are converted and stored.  Between rows the counts change
// by the nodes on whose paths the rows differ.  No dense [requests, vocabulary] count exists in memory.
//
// Bound by HBM: a row's 2 bytes in, 4 out and a bit of mask per token.
#pragma once

#include "ftq_serve_launch.h"

namespace ftq {

constexpr int kLogitThreads = 256;
constexpr uint32_t kInPrompt = 1u << 31, kHasBias = 1u << 30, kCountMask = kHasBias - 1;


// Orders as the value does; NaN above all.  Lower indexes are larger.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t u = __float_as_uint(x);
    return x != x ? 0xffffffffu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kLogitThreads) logits_kernel(const LogitParams p) {
    extern __shared__ uint32_t s_words[];
    uint32_t* const s_word = s_words;                                           // [segment]
    int* const s_bias = reinterpret_cast<int*>(s_words + kLogitSegment);        // [segment]: place in the list (K > 0 only)
    __shared__ int s_node[kTreeMaxNodes], s_place[kTreeMaxNodes];          // nodes whose token lies in the segment
    __shared__ int s_nodes;
    __shared__ unsigned long long s_best;
    const int tid = threadIdx.x, lane = tid & 31, r = blockIdx.y;
    const int seg0 = blockIdx.x * kLogitSegment, n = min(kLogitSegment, p.V - seg0);
    const int row0 = blockIdx.z * p.rows_per_cta, row1 = min(p.T, row0 + p.rows_per_cta);
    const int W = (p.T + 31) / 32;
    for (int i = tid; i < kLogitSegment / 4; i += kLogitThreads) {
        reinterpret_cast<uint4*>(s_word)[i] = make_uint4(0, 0, 0, 0);
        if (p.K > 0) reinterpret_cast<int4*>(s_bias)[i] = make_int4(-1, -1, -1, -1);
    }
    if (tid == 0) {
        s_nodes = 0;
        s_best = 0;
    }
    after_previous_kernel();
    let_next_kernel_start();
    __syncthreads();
    auto in_segment = [&](int token) { return static_cast<uint32_t>(token) < static_cast<uint32_t>(p.V) && token >= seg0 && token - seg0 < n; };
    if (p.history) {
        const int len = min(max(p.history_lens[r], 0), p.H), prompt = p.prompt_lens ? p.prompt_lens[r] : 0;
        const int32_t* h = p.history + static_cast<int64_t>(r) * p.H;
#pragma unroll 8
        for (int i = tid; i < len; i += kLogitThreads) {
            const int t = h[i];
            if (in_segment(t)) {
                if (i < prompt) atomicOr(&s_word[t - seg0], kInPrompt);
                else atomicAdd(&s_word[t - seg0], 1u);
            }
        }
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
            }
        }
    }
    __syncthreads();
    const int nodes = s_nodes;
    const float rep = p.repetition ? p.repetition[r] : 1.f, freq = p.frequency ? p.frequency[r] : 0.f,
                pres = p.presence ? p.presence[r] : 0.f;
    auto adjust = [&](float x, uint32_t word, int place) {
        const uint32_t count = word & kCountMask;
        if (word & ~kHasBias) x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
        if (count) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, static_cast<float>(count))), pres);
        if (word & kHasBias) x = __fadd_rn(x, p.bias[static_cast<int64_t>(r) * p.K + s_bias[place]]);
        return x;
    };
    for (int row = row0; row < row1; row++) {
        const int64_t at = static_cast<int64_t>(r) * p.T + row;
        if (nodes > 0) {
            // the counts are those of the row before: add what this path has more, take what it has less
            const int32_t *now = p.tree_masks + at * W, *was = now - W;
            for (int k = tid; k < nodes; k += kLogitThreads) {
                const int j = s_node[k], on = (now[j >> 5] >> (j & 31)) & 1, before = row > row0 ? (was[j >> 5] >> (j & 31)) & 1 : 0;
                if (on != before) atomicAdd(&s_word[s_place[k]], static_cast<uint32_t>(on - before));
            }
            __syncthreads();
        }
        const T* src = static_cast<const T*>(p.logits) + at * p.row_stride + seg0;
        float* dst = p.out ? p.out + at * p.V + seg0 : nullptr;
        const uint8_t* ok = p.allowed ? p.allowed + at * p.allowed_stride + seg0 / 8 : nullptr;
        uint32_t best = 0, best_at = 0;
        auto consider = [&](float y, int place) {   // (places ascend)
            const uint32_t o = order_of(__fadd_rn(y, 0.f));   // (-0 is 0)
            if (o > best) {
                best = o;
                best_at = place;
            }
        };
        if constexpr (VEC) {
            constexpr int ROUNDS = kLogitSegment / 8 / kLogitThreads;
            float x[ROUNDS][8];
            uint32_t bits[ROUNDS];
#pragma unroll
            for (int k = 0; k < ROUNDS; k++) {
                const int e = 8 * (k * kLogitThreads + tid);
                bits[k] = 0xff;
                if (e < n) {
                    load8<T>(src + e, x[k]);
                    if (ok) bits[k] = ok[e / 8];
                }
            }
#pragma unroll
            for (int k = 0; k < ROUNDS; k++) {
                const int e = 8 * (k * kLogitThreads + tid);
                if (e >= n) break;
                const uint4 a = *reinterpret_cast<const uint4*>(s_word + e), b = *reinterpret_cast<const uint4*>(s_word + e + 4);
                const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
                if (a.x | a.y | a.z | a.w | b.x | b.y | b.z | b.w) {
#pragma unroll
                    for (int c = 0; c < 8; c++)
                        if (w[c]) x[k][c] = adjust(x[k][c], w[c], e + c);
                }
#pragma unroll
                for (int c = 0; c < 8; c++) {
                    if (!((bits[k] >> c) & 1)) x[k][c] = -INFINITY;
                    if (p.keys) consider(x[k][c], e + c);
                }
                if (dst) {
                    *reinterpret_cast<float4*>(dst + e) = make_float4(x[k][0], x[k][1], x[k][2], x[k][3]);
                    *reinterpret_cast<float4*>(dst + e + 4) = make_float4(x[k][4], x[k][5], x[k][6], x[k][7]);
                }
            }
        } else {
            constexpr int ROUNDS = kLogitSegment / kLogitThreads;
            float x[ROUNDS];
#pragma unroll
            for (int k = 0; k < ROUNDS; k++) {
                const int e = k * kLogitThreads + tid;
                x[k] = e < n ? to_float<T>(src[e]) : 0.f;
            }
#pragma unroll
            for (int k = 0; k < ROUNDS; k++) {
                const int e = k * kLogitThreads + tid;
                if (e >= n) break;
                const uint32_t w = s_word[e];
                if (w) x[k] = adjust(x[k], w, e);
                if (ok && !((ok[e / 8] >> (e % 8)) & 1)) x[k] = -INFINITY;
                if (p.keys) consider(x[k], e);
                if (dst) dst[e] = x[k];
            }
        }
        if (p.keys) {
            const uint32_t top = __reduce_max_sync(0xffffffffu, best);
            const uint32_t first = __reduce_min_sync(0xffffffffu, best == top ? best_at : 0xffffffffu);
            if (lane == 0 && top) atomicMax(&s_best, static_cast<unsigned long long>(top) << 32 | (0xffffffffu - (seg0 + first)));
            __syncthreads();
            if (tid == 0) {
                p.keys[at * p.segments + blockIdx.x] = s_best;
                s_best = 0;
            }
        }
        if (p.keys || nodes > 0) __syncthreads();
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
