// Beam search's selection: the best continuations of every request's beams, over beams and vocabulary.
//
//   total(b, v) = scores[b] + x[b][v] - log sum_u exp x[b][u]
//
// the n largest of a request, of equal ones the lowest beam's lowest token; tokens that end an answer are left out and
// their totals returned by themselves.
//
// The logits are read once.  A CTA has a chunk of a row: every thread keeps the maximum and the sum of exponentials of its 16-byte
// vectors, and which vector the maximum came from.  Any of the chunk's `keep` largest tokens lies in one of the `keep` threads,
// and there in one of the `keep` vectors, that are first when ordered by their largest token (of equal ones the
// first): otherwise as many threads or vectors would each hold a token that goes before it.  So a sort of the threads, one of
// their vectors' maxima, and one of those vectors' tokens leave the exact order, whatever the logits are, and what is read again
// is a few hundred vectors.  keep = n + the tokens that end an answer.  beam_join_kernel adds up a request's rows and sorts their
// tokens by their totals, in 64 bits (totals of different beams may lie closer than fp32 tells apart).
#pragma once

#include "ftq_beam_launch.h"

namespace ftq {

constexpr int kSelectThreads = 512, kSelectMaxKeep = kBeamMax + kBeamMaxEnds;
constexpr int kSelectVectors = 32;      // vectors of a thread at most, so that those of `keep` threads can be sorted

__host__ __device__ constexpr int select_pow2(int n) {
    int x = 1;
    while (x < n) x *= 2;
    return x;
}
// tokens that beam_join_kernel sorts at a time
constexpr int kSelectJoin = 4096;
__host__ __device__ constexpr int select_join_size(int beams, int chunks, int keep, int n) {
    const int64_t all = static_cast<int64_t>(beams) * chunks * keep + n;
    return all > kSelectJoin ? kSelectJoin : select_pow2(static_cast<int>(all));
}

// Orders as the value does (no NaN comes here).
__device__ __forceinline__ uint32_t select_order(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);        // (-0 and 0 are equal)
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float select_value(uint32_t o) { return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ unsigned long long select_key(float x, uint32_t place) {     // (lower places are larger)
    return static_cast<unsigned long long>(select_order(x)) << 32 | static_cast<uint32_t>(~place);
}

// Sorts n = 2^k keys in shared memory, the largest first; by the whole CTA.
__device__ __forceinline__ void select_sort(unsigned long long* s, int n) {
    for (int k = 2; k <= n; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            __syncthreads();
            for (int i = threadIdx.x; i < n / 2; i += blockDim.x) {
                const int a = 2 * i - (i & (j - 1)), b = a + j;
                const unsigned long long x = s[a], y = s[b];
                if ((x < y) == ((a & k) == 0)) {
                    s[a] = y;
                    s[b] = x;
                }
            }
        }
    __syncthreads();
}

// a vector's 16 bytes as values
template <typename T>
struct SelectVec {
    static constexpr int N = 16 / sizeof(T);
    float v[N];
    // vector i of the row part [begin, end) of x, where vectors lie on 16-byte boundaries and the first one `head` tokens before
    // begin: what does not belong to it is -inf
    __device__ __forceinline__ void load(const T* x, int head, int len, int i) {
        const int at = i * N - head;
        if (at >= 0 && at + N <= len) {
            unpack(*reinterpret_cast<const uint4*>(x + at));
        } else {
#pragma unroll
            for (int k = 0; k < N; k++) v[k] = at + k >= 0 && at + k < len ? to_float<T>(x[at + k]) : -INFINITY;
        }
    }
    __device__ __forceinline__ void unpack(uint4 u) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if constexpr (sizeof(T) == 4) {
                v[k] = __uint_as_float(w[k]);
            } else if constexpr (std::is_same<T, __half>::value) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
                v[2 * k] = f.x;
                v[2 * k + 1] = f.y;
            } else {
                v[2 * k] = bf16_lo(w[k]);
                v[2 * k + 1] = bf16_hi(w[k]);
            }
        }
    }
    __device__ __forceinline__ float largest() const {
        float m = v[0];
#pragma unroll
        for (int k = 1; k < N; k++) m = fmaxf(m, v[k]);
        return m;
    }
};

template <typename T>
__global__ void __launch_bounds__(kSelectThreads) beam_rows_kernel(const SelectParams p) {
    constexpr int N = SelectVec<T>::N;
    extern __shared__ unsigned long long s_keys[];
    __shared__ float s_max[kSelectThreads / 32], s_sum[kSelectThreads / 32];
    const int tid = threadIdx.x, lane = tid & 31, row = blockIdx.x / p.chunks, chunk = blockIdx.x - row * p.chunks;
    after_previous_kernel();
    let_next_kernel_start();
    if (!(p.scores[row] > -INFINITY)) return;     // (a beam that is not alive; beam_join_kernel asks the same)
    const int begin = chunk * p.chunk, len = min(p.chunk, p.V - begin);
    const T* const x = static_cast<const T*>(p.logits) + row * p.row_stride + begin;
    const int head = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T)), n_vec = (head + len + N - 1) / N;
    float m = -INFINITY, sum = 0.f;
    int where = tid;        // the vector that the maximum came from
    constexpr float kLog2 = 1.4426950408889634f;
    for (int i0 = tid; i0 < n_vec; i0 += 4 * kSelectThreads) {
        SelectVec<T> v[4];
        float top[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int i = i0 + k * kSelectThreads;
            if (i < n_vec) {
                v[k].load(x, head, len, i);
            } else {
#pragma unroll
                for (int c = 0; c < N; c++) v[k].v[c] = -INFINITY;
            }
        }
        const float before = m;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            top[k] = v[k].largest();
            where = top[k] > m ? i0 + k * kSelectThreads : where;
            m = fmaxf(m, top[k]);
        }
        const float ref = m == -INFINITY ? 0.f : m;
        if (m > before) sum *= fast_exp2((before - ref) * kLog2);
        // (x - m first: logits far from zero lose nothing that way.  Packed: half the instructions)
        const u64 ref2 = pk2(ref, ref), log2 = pk2(kLog2, kLog2);
        u64 part[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            part[k] = 0;
#pragma unroll
            for (int c = 0; c < N; c += 2) {
                float a, b;
                upk2(mul2(sub2(pk2(v[k].v[c], v[k].v[c + 1]), ref2), log2), a, b);
                part[k] = add2(part[k], pk2(fast_exp2(a), fast_exp2(b)));
            }
        }
        float a, b;
        upk2(add2(add2(part[0], part[1]), add2(part[2], part[3])), a, b);
        sum += a + b;
    }
    // ---- the chunk's maximum and sum, in an order of their own
    {
        float mw = m;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) mw = fmaxf(mw, __shfl_xor_sync(0xffffffffu, mw, d));
        float s = m == -INFINITY ? sum : sum * fast_exp2((m - mw) * kLog2);     // (not a number stays so)
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        if (lane == 0) {
            s_max[tid / 32] = mw;
            s_sum[tid / 32] = s;
        }
    }
    s_keys[tid] = tid < n_vec ? select_key(m, where) : 0;
    __syncthreads();
    if (tid == 0) {
        float mc = s_max[0];
        for (int w = 1; w < kSelectThreads / 32; w++) mc = fmaxf(mc, s_max[w]);
        float s = 0.f;
        for (int w = 0; w < kSelectThreads / 32; w++) s += s_max[w] == -INFINITY ? s_sum[w] : s_sum[w] * fast_exp2((s_max[w] - mc) * kLog2);
        p.sums[blockIdx.x] = make_float2(mc, s);
    }
    // ---- the first `keep` threads by their largest token
    select_sort(s_keys, kSelectThreads);
    const int threads = min(p.keep, min(n_vec, kSelectThreads)), rounds = (n_vec + kSelectThreads - 1) / kSelectThreads;
    __shared__ int s_first[kSelectMaxKeep];
    if (tid < threads) s_first[tid] = static_cast<int>(~static_cast<uint32_t>(s_keys[tid])) % kSelectThreads;
    __syncthreads();
    // ---- of their vectors the first `keep`
    int n = select_pow2(threads * rounds);
    for (int e = tid; e < n; e += kSelectThreads) {
        const int i = e < threads * rounds ? s_first[e / rounds] + e % rounds * kSelectThreads : n_vec;
        unsigned long long key = 0;
        if (i < n_vec) {
            SelectVec<T> v;
            v.load(x, head, len, i);
            key = select_key(v.largest(), i);
        }
        s_keys[e] = key;
    }
    select_sort(s_keys, n);
    const int vectors = min(p.keep, min(n, n_vec));
    if (tid < vectors) s_first[tid] = static_cast<int>(~static_cast<uint32_t>(s_keys[tid]));
    __syncthreads();
    // ---- of their tokens the first `keep`
    n = select_pow2(max(vectors * N, p.keep));
    for (int e = tid; e < n; e += kSelectThreads) {
        unsigned long long key = 0;
        if (e < vectors * N && s_first[e / N] < n_vec) {
            const int t = s_first[e / N] * N - head + e % N;
            if (t >= 0 && t < len) key = select_key(to_float<T>(x[t]), begin + t);
        }
        s_keys[e] = key;
    }
    select_sort(s_keys, n);
    for (int e = tid; e < p.keep; e += kSelectThreads) p.keys[static_cast<int64_t>(blockIdx.x) * p.keep + e] = s_keys[e];
}

// Orders as the value does.
__device__ __forceinline__ unsigned long long select_order64(double x) {
    const long long u = __double_as_longlong(x + 0.0);
    return u < 0 ? ~static_cast<unsigned long long>(u) : static_cast<unsigned long long>(u) | 1ull << 63;
}
__device__ __forceinline__ double select_value64(unsigned long long o) {
    return __longlong_as_double(static_cast<long long>(o >> 63 ? o & ~(1ull << 63) : ~o));
}

// A CTA has a request: its rows' sums, the ends' totals, and the order of the tokens that the rows kept.
template <typename T>
__global__ void __launch_bounds__(kSelectThreads) beam_join_kernel(const SelectParams p) {
    extern __shared__ unsigned long long s_keys[];
    // a beam's score (-inf: it has no continuation), its row's maximum, and the logarithm of the sum of exponentials less that
    __shared__ double s_score[kBeamMax], s_max[kBeamMax], s_log[kBeamMax];
    const int tid = threadIdx.x, r = blockIdx.x;
    after_previous_kernel();
    let_next_kernel_start();
    for (int b = tid / 32; b < p.K; b += kSelectThreads / 32) {
        const int64_t row = static_cast<int64_t>(r) * p.K + b;
        const float score = p.scores[row];
        double s = 0.0;
        float m = -INFINITY;
        if (score > -INFINITY) {
            const float2* at = p.sums + row * p.chunks;
            for (int c = tid & 31; c < p.chunks; c += 32) m = fmaxf(m, __ldcg(at + c).x);
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
            for (int c = tid & 31; c < p.chunks; c += 32) {
                const float2 x = __ldcg(at + c);
                // (a sum that is not a number says so whatever its maximum is)
                s += x.x == -INFINITY ? static_cast<double>(x.y) : x.y * exp(static_cast<double>(x.x) - m);
            }
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        }
        if ((tid & 31) == 0) {
            s_score[b] = s > 0.0 && m > -INFINITY && m < INFINITY ? score : -INFINITY;
            s_max[b] = m;
            s_log[b] = log(s);
        }
    }
    auto total_of = [&](int b, float x) { return (x - s_max[b]) - s_log[b] + s_score[b]; };
    __syncthreads();
    for (int e = tid; e < p.K * p.n_ends; e += kSelectThreads) {
        const int b = e / p.n_ends, id = p.ends[e - b * p.n_ends];
        double total = -INFINITY;
        if (s_score[b] > -INFINITY && id >= 0 && id < p.V)
            total = total_of(b, to_float<T>(static_cast<const T*>(p.logits)[(static_cast<int64_t>(r) * p.K + b) * p.row_stride + id]));
        p.end_scores[static_cast<int64_t>(r) * p.K * p.n_ends + e] = static_cast<float>(total);
    }
    // ---- the n best so far and as many others as there is room for, until there are no others
    const int per_row = p.chunks * p.keep, all = p.K * per_row, n = select_join_size(p.K, p.chunks, p.keep, p.n);
    unsigned long long* const s_place = s_keys + n;
    for (int e = tid; e < p.n; e += kSelectThreads) {
        s_keys[e] = 0;
        s_place[e] = ~0ull;
    }
    for (int done = 0; done < all; done += n - p.n) {
        for (int e = p.n + tid; e < n; e += kSelectThreads) {
            unsigned long long key = 0, place = ~0ull;
            const int i = done + e - p.n, b = i / per_row;
            if (i < all && s_score[b] > -INFINITY) {
                const unsigned long long k = __ldcg(p.keys + static_cast<int64_t>(r) * all + i);
                const uint32_t token = ~static_cast<uint32_t>(k);
                const double total = total_of(b, select_value(static_cast<uint32_t>(k >> 32)));
                bool end = k == 0;
                for (int c = 0; c < p.n_ends; c++) end |= static_cast<uint32_t>(p.ends[c]) == token;
                if (!end && total > -INFINITY) {
                    key = select_order64(total);
                    place = static_cast<unsigned long long>(b) << 32 | token;
                }
            }
            s_keys[e] = key;
            s_place[e] = place;
        }
        for (int k = 2; k <= n; k <<= 1)
            for (int j = k >> 1; j > 0; j >>= 1) {
                __syncthreads();
                for (int i = tid; i < n / 2; i += kSelectThreads) {
                    const int a = 2 * i - (i & (j - 1)), b = a + j;
                    const unsigned long long x = s_keys[a], y = s_keys[b], px = s_place[a], py = s_place[b];
                    const bool less = x < y || (x == y && px > py);
                    if (less == ((a & k) == 0)) {
                        s_keys[a] = y; s_keys[b] = x;
                        s_place[a] = py; s_place[b] = px;
                    }
                }
            }
        __syncthreads();
    }
    for (int e = tid; e < p.n; e += kSelectThreads) {
        const unsigned long long key = s_keys[e], place = s_place[e];
        const int64_t at = static_cast<int64_t>(r) * p.n + e;
        p.out_scores[at] = key ? static_cast<float>(select_value64(key)) : -INFINITY;
        p.parents[at] = key ? static_cast<int>(place >> 32) : -1;
        p.tokens[at] = key ? static_cast<int>(place & 0xffffffffu) : -1;
    }
}

}  // namespace ftq
