// Beam search's selection: the best continuations of every request's beams, over beams and vocabulary.
//
//   total(b, v) = scores[b] + x[b][v] - log sum_u exp x[b][u]
//
// the n largest of a request, of equal ones the lowest beam's lowest token; tokens that end an answer are left out and
// their totals returned by themselves.
//
// The logits are read once.  A CTA has a chunk of a row: every thread keeps the maximum and the sum of exponentials of its 16-byte
// vectors.  Any `keep` of the threads' maxima bound the chunk's keep-th largest token from below (keep = n + the tokens that end
// an answer), so the keep-th of the warps' few largest is a threshold: threads whose maximum reaches it are few, their vectors are
// looked at again, and the few tokens that reach it are ranked by counting (threshold, push and rank below).  Masked tokens (-inf) never do: a chunk
// whose mask leaves fewer than `keep` threads a token has all of its others looked at.  Where more tokens reach it than there is
// room for (equal logits, or large ones in a few threads' vectors only) sorts leave the exact order whatever the logits are: any of the `keep` largest tokens lies in
// one of the `keep` threads, and there in one of the `keep` vectors, that are first by their largest token (of equal ones
// the first), since otherwise as many threads or vectors would each hold a token that goes before it.
// beam_join_kernel adds up a request's rows and does the same with their tokens' totals, in 64 bits (totals of different beams
// may lie closer than fp32 tells apart).  A chunk's sum is fp32's: the logarithm of a row's is good to some 1e-7, and beams whose totals
// lie closer come in either order.  Those with the same logits and scores have the same totals.
//
// 64 requests of 8 beams, 131072 bf16 logits: 41 us, 35 of them the rows (134 MB: 20.5 us of HBM).  A logit takes 7 instructions (its
// exponential one of 16 a cycle and SM: 15 us), threshold and ranks a quarter of all; issue is busy half of the time, and what
// keeps the rest is loads and the few barriers of CTAs of 32768 tokens.  With three bitonic sorts a CTA 133 us; thresholds 54; the
// chunk prefetched and the join's loads side by side 47; vectors looked at again one a thread 44; no batch of vectors on its way while the
// one before is added up, which only took registers, 42 -> 41.  With a
// mask that leaves 50 tokens a row 38 us (120 with masked tokens as candidates, which went to the sorts).
#pragma once

#include <type_traits>

#include "ftq_beam_launch.h"

namespace ftq {

constexpr int kSelectThreads = 256, kSelectWarps = kSelectThreads / 32;     // of beam_rows_kernel
constexpr int kJoinFew = 1024;          // tokens of a request that 256 threads of beam_join_kernel take as they come; more take 512
constexpr int kSelectMaxKeep = kBeamMax + kBeamMaxEnds;
constexpr int kSelectVectors = 32;      // vectors of a thread at most, so that those of `keep` threads can be sorted
constexpr int kSelectBatch = 2;         // of which a thread loads so many at a time
constexpr int kSelectRoom = 1024;       // tokens that are ranked by counting
constexpr int kSelectTop = 16;          // a warp's largest keys that a threshold is made of, at most
constexpr uint32_t kSelectLeast = 0x00800000u;      // select_order of the least finite value: what is masked (-inf) is no candidate

__host__ __device__ constexpr int select_pow2(int n) {
    int x = 1;
    while (x < n) x *= 2;
    return x;
}
// tokens that beam_join_kernel sorts at a time, where it has to
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

// A key that at least `keep` of the CTA's threads' keys reach, 0 where fewer are above 0; by the whole CTA.  `s` has room for
// kSelectTop keys of each warp and one more.
template <int WARPS>
__device__ __forceinline__ uint32_t select_threshold(uint32_t key, int keep, uint32_t* s) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // (two more of each warp than an even spread needs)
    const int top = min(kSelectTop, (keep + WARPS - 1) / WARPS + 2), all = top * WARPS;
    for (int i = 0; i < top; i++) {
        const uint32_t m = __reduce_max_sync(0xffffffffu, key);
        if (lane == 0) s[warp * top + i] = m;
        if (lane == __ffs(__ballot_sync(0xffffffffu, key == m)) - 1) key = 0;
    }
    __syncthreads();
    if (static_cast<int>(threadIdx.x) < all) {
        const uint32_t mine = s[threadIdx.x];
        int rank = 0;
#pragma unroll 8
        for (int i = 0; i < all; i++) rank += s[i] > mine || (s[i] == mine && i < static_cast<int>(threadIdx.x));
        if (rank == keep - 1) s[kSelectTop * WARPS] = mine;
    }
    __syncthreads();
    return s[kSelectTop * WARPS];
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
    static __device__ __forceinline__ void unpack(uint4 u, float (&v)[N]) {
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
    // the N values that begin `head` values into two neighbouring vectors; HEAD: known to the compiler, or -1
    template <int HEAD>
    static __device__ __forceinline__ uint4 shifted(uint4 a, uint4 b, int head) {
        const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        const int bytes = (HEAD < 0 ? head : HEAD) * static_cast<int>(sizeof(T));
        uint32_t t[6], u[5], out[4];
#pragma unroll
        for (int k = 0; k < 6; k++) t[k] = (bytes & 8) ? w[k + 2] : w[k];
#pragma unroll
        for (int k = 0; k < 5; k++) u[k] = (bytes & 4) ? t[k + 1] : t[k];
#pragma unroll
        for (int k = 0; k < 4; k++) out[k] = sizeof(T) == 4 ? u[k] : __funnelshift_r(u[k], u[k + 1], 8 * (bytes & 3));
        return make_uint4(out[0], out[1], out[2], out[3]);
    }
    // whether the two are nothing but tokens of the row part [x, x + len), which begins `head` tokens behind a 16-byte boundary
    static __device__ __forceinline__ bool inside(int head, int len, int i) { return i * N >= head && i * N - head + 2 * N <= len; }
    // vector i of it, tokens i N .. i N + N - 1: what does not belong to it is -inf
    static __device__ __forceinline__ void load(const T* x, int head, int len, int i, float (&v)[N]) {
        const uint4* const from = reinterpret_cast<const uint4*>(x - head) + i;
        if (head == 0 && i * N + N <= len) {
            unpack(*from, v);
        } else if (head > 0 && inside(head, len, i)) {
            unpack(shifted<-1>(from[0], from[1], head), v);
        } else {
#pragma unroll
            for (int k = 0; k < N; k++) v[k] = i * N + k < len ? to_float<T>(x[i * N + k]) : -INFINITY;
        }
    }
    // f(std::integral_constant<int, head>), 0 <= head < N
    template <int HEAD = 0, typename F>
    static __device__ __forceinline__ void with_head(int head, F&& f) {
        if constexpr (HEAD + 1 < N) {
            if (head != HEAD) return with_head<HEAD + 1>(head, f);
        }
        f(std::integral_constant<int, HEAD>{});
    }
    static __device__ __forceinline__ float largest(const float (&v)[N]) {
        float m = v[0];
#pragma unroll
        for (int k = 1; k < N; k++) m = fmaxf(m, v[k]);
        return m;
    }
};

// Asks for bytes that will be read (16-byte aligned, a multiple of 16): a CTA's whole chunk is on its way to L2 while its first
// vectors are waited for, and while other CTAs look for their largest tokens.
__device__ __forceinline__ void prefetch_l2(const void* p, uint32_t bytes) {
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;\n" ::"l"(p), "r"(bytes) : "memory");
}

// a thread's maximum, and the sum of exp(x - maximum)
struct SelectSum {
    float m = -INFINITY, sum = 0.f;
    // (x - m first: logits far from zero lose nothing that way.  Packed: half the instructions)
    template <int N, int B>
    __device__ __forceinline__ void add(const float (&v)[B][N]) {
        constexpr float kLog2 = 1.4426950408889634f;
        float top[B];
#pragma unroll
        for (int k = 0; k < B; k++) {
            top[k] = v[k][0];
#pragma unroll
            for (int c = 1; c < N; c++) top[k] = fmaxf(top[k], v[k][c]);
        }
        const float before = m;
#pragma unroll
        for (int k = 0; k < B; k++) m = fmaxf(m, top[k]);
        const float ref = m == -INFINITY ? 0.f : m;
        if (m > before) sum *= fast_exp2((before - ref) * kLog2);
        const u64 ref2 = pk2(ref, ref), log2 = pk2(kLog2, kLog2);
        u64 part[B];
#pragma unroll
        for (int k = 0; k < B; k++) {
            part[k] = 0;
#pragma unroll
            for (int c = 0; c < N; c += 2) {
                float a, b;
                upk2(mul2(sub2(pk2(v[k][c], v[k][c + 1]), ref2), log2), a, b);
                part[k] = add2(part[k], pk2(fast_exp2(a), fast_exp2(b)));
            }
        }
#pragma unroll
        for (int k = 1; k < B; k++) part[0] = add2(part[0], part[k]);
        float a, b;
        upk2(part[0], a, b);
        sum += a + b;
    }
};

// Which tokens a thread adds up, and in which order, is the same for all rows, wherever they begin in memory: beams that say the same
// have the same sums.  A vector of a row that begins between 16-byte boundaries is made of two that lie on them, by shifts that
// the compiler knows (64 requests of 8 beams, 131071 bf16 logits 49 us, 50257 fp32 ones 33, where vectors that lie on boundaries, so that
// sums differed by row, took 45 and 32; shifts that it does not know 52 and 35, tokens loaded one by one, 32 apart, 56 and 33).
template <typename T>
__global__ void __launch_bounds__(kSelectThreads, 5) beam_rows_kernel(const SelectParams p) {
    using V = SelectVec<T>;
    constexpr int N = V::N, B = kSelectBatch;
    extern __shared__ __align__(16) unsigned long long s_keys[];
    __shared__ float s_max[kSelectWarps], s_sum[kSelectWarps];
    __shared__ uint32_t s_top[kSelectTop * kSelectWarps + 1];
    __shared__ int s_first[kSelectThreads], s_n[2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = blockIdx.x / p.chunks, chunk = blockIdx.x - row * p.chunks;
    after_previous_kernel();
    let_next_kernel_start();
    if (!(p.scores[row] > -INFINITY)) return;     // (a beam that is not alive; beam_join_kernel asks the same)
    const int begin = chunk * p.chunk, len = min(p.chunk, p.V - begin);
    const T* const x = static_cast<const T*>(p.logits) + row * p.row_stride + begin;
    const int head = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T)), n_vec = (len + N - 1) / N;
    if (tid < 2) s_n[tid] = 0;
    constexpr float kLog2 = 1.4426950408889634f;
    SelectSum own;
    {
        const uint4* const from = reinterpret_cast<const uint4*>(x - head);
        const int lo = head > 0 ? 1 : 0, hi = (head + len) / N, whole = len / N;     // vectors between boundaries; tokens' whole ones
        if (tid == 0 && hi > lo) prefetch_l2(from + lo, 16 * (hi - lo));
        V::with_head(head, [&](auto head_tag) {
            constexpr int HEAD = decltype(head_tag)::value, S = HEAD > 0 ? 2 : 1;
            int i = tid;
            for (; i + (B - 1) * kSelectThreads < whole; i += B * kSelectThreads) {
                uint4 u[B][S];
                float v[B][N];
#pragma unroll
                for (int k = 0; k < B; k++) {
                    const int j = i + k * kSelectThreads;
                    if (HEAD > 0 && !V::inside(HEAD, len, j)) continue;
#pragma unroll
                    for (int c = 0; c < S; c++) u[k][c] = from[j + c];
                }
#pragma unroll
                for (int k = 0; k < B; k++) {
                    const int j = i + k * kSelectThreads;
                    if (HEAD == 0) V::unpack(u[k][0], v[k]);
                    else if (V::inside(HEAD, len, j)) V::unpack(V::template shifted<HEAD>(u[k][0], u[k][S - 1], HEAD), v[k]);
                    else V::load(x, HEAD, len, j, v[k]);
                }
                own.add(v);
            }
            for (; i < n_vec; i += kSelectThreads) {
                float v[1][N];
                V::load(x, HEAD, len, i, v[0]);
                own.add(v);
            }
        });
    }
    // ---- the chunk's maximum and sum, in an order of their own
    {
        float mw = own.m;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) mw = fmaxf(mw, __shfl_xor_sync(0xffffffffu, mw, d));
        float s = own.m == -INFINITY ? own.sum : own.sum * fast_exp2((own.m - mw) * kLog2);     // (not a number stays so)
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        if (lane == 0) {
            s_max[warp] = mw;
            s_sum[warp] = s;
        }
    }
    const uint32_t mine = own.m > -INFINITY ? select_order(own.m) : 0;
    const uint32_t least = max(select_threshold<kSelectWarps>(mine, p.keep, s_top), kSelectLeast);
    if (tid == 0) {
        float mc = s_max[0];
        for (int w = 1; w < kSelectWarps; w++) mc = fmaxf(mc, s_max[w]);
        float s = 0.f;
        for (int w = 0; w < kSelectWarps; w++) s += s_max[w] == -INFINITY ? s_sum[w] : s_sum[w] * fast_exp2((s_max[w] - mc) * kLog2);
        p.sums[blockIdx.x] = make_float2(mc, s);
    }
    // ---- the vectors of the threads whose maximum reaches it: their tokens that do
    if (mine >= least) s_first[atomicAdd(&s_n[0], 1)] = tid;
    __syncthreads();
    const int rounds = (n_vec + kSelectThreads - 1) / kSelectThreads;
    for (int e = tid; e < s_n[0] * rounds; e += kSelectThreads) {
        const int c = e / rounds, i = s_first[c] + (e - c * rounds) * kSelectThreads;
        if (i >= n_vec || s_n[1] > kSelectRoom) continue;
        float v[N];
        V::load(x, head, len, i, v);
#pragma unroll
        for (int k = 0; k < N; k++) {
            const int t = i * N + k;
            if (select_order(v[k]) >= least && t < len) {
                const int at = atomicAdd(&s_n[1], 1);
                if (at < kSelectRoom) s_keys[at] = select_key(v[k], begin + t);
            }
        }
    }
    __syncthreads();
    unsigned long long* const to = p.keys + static_cast<int64_t>(blockIdx.x) * p.keep;
    if (s_n[1] <= kSelectRoom) {
        const int n = s_n[1];
        for (int e = tid; e < n; e += kSelectThreads) {
            const unsigned long long key = s_keys[e];
            int rank = 0;
#pragma unroll 8
            for (int i = 0; i < n; i++) rank += s_keys[i] > key;
            if (rank < p.keep) to[rank] = key;
        }
        for (int e = n + tid; e < p.keep; e += kSelectThreads) to[e] = 0;
        return;
    }
    // ---- too many of them.  The first `keep` threads by their largest token (and the vector that it lies in)
    {
        float best = -INFINITY;
        int where = tid;
        for (int i = tid; i < n_vec; i += kSelectThreads) {
            float v[N];
            V::load(x, head, len, i, v);
            const float t = V::largest(v);
            where = t > best ? i : where;
            best = fmaxf(best, t);
        }
        __syncthreads();
        s_keys[tid] = tid < n_vec ? select_key(best, where) : 0;
    }
    select_sort(s_keys, kSelectThreads);
    const int threads = min(p.keep, min(n_vec, kSelectThreads));
    if (tid < threads) s_first[tid] = static_cast<int>(~static_cast<uint32_t>(s_keys[tid])) % kSelectThreads;
    __syncthreads();
    // of their vectors the first `keep`
    int n = select_pow2(threads * rounds);
    for (int e = tid; e < n; e += kSelectThreads) {
        const int i = e < threads * rounds ? s_first[e / rounds] + e % rounds * kSelectThreads : n_vec;
        unsigned long long key = 0;
        if (i < n_vec) {
            float v[N];
            V::load(x, head, len, i, v);
            key = select_key(V::largest(v), i);
        }
        s_keys[e] = key;
    }
    select_sort(s_keys, n);
    const int vectors = min(p.keep, min(n, n_vec));
    if (tid < vectors) s_first[tid] = static_cast<int>(~static_cast<uint32_t>(s_keys[tid]));
    __syncthreads();
    // of their tokens the first `keep`
    n = select_pow2(max(vectors * N, p.keep));
    for (int e = tid; e < n; e += kSelectThreads) {
        unsigned long long key = 0;
        if (e < vectors * N && s_first[e / N] < n_vec) {
            const int t = s_first[e / N] * N + e % N;
            if (t < len) key = select_key(to_float<T>(x[t]), begin + t);
        }
        s_keys[e] = key;
    }
    select_sort(s_keys, n);
    for (int e = tid; e < p.keep; e += kSelectThreads) to[e] = s_keys[e];
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
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS) beam_join_kernel(const SelectParams p) {
    extern __shared__ __align__(16) unsigned long long s_keys[];
    // a beam's score (-inf: it has no continuation), its row's maximum, and the logarithm of the sum of exponentials less that
    __shared__ double s_score[kBeamMax], s_max[kBeamMax], s_log[kBeamMax];
    __shared__ uint32_t s_top[kSelectTop * THREADS / 32 + 1];
    __shared__ int s_end[kBeamMaxEnds], s_n;
    const int tid = threadIdx.x, r = blockIdx.x;
    after_previous_kernel();
    let_next_kernel_start();
    if (tid == 0) s_n = 0;
    if (tid < p.n_ends) s_end[tid] = p.ends[tid];
    const int per_row = p.chunks * p.keep, all = p.K * per_row;
    // (the thread's first tokens are on their way while the sums are made)
    constexpr int FEW = kJoinFew / THREADS;
    unsigned long long kept[FEW];
#pragma unroll
    for (int j = 0; j < FEW; j++) {
        const int i = tid + j * THREADS;
        kept[j] = i < all ? __ldcg(p.keys + static_cast<int64_t>(r) * all + i) : 0;     // (of a row that is not alive: anything)
    }
    for (int b = tid / 32; b < p.K; b += THREADS / 32) {
        const int64_t row = static_cast<int64_t>(r) * p.K + b;
        const float2* const at = p.sums + row * p.chunks;
        const float score = p.scores[row];
        const float2 first = (tid & 31) < p.chunks ? __ldcg(at + (tid & 31)) : make_float2(-INFINITY, 0.f);
        float m = first.x;
        for (int c = 32 + (tid & 31); c < p.chunks; c += 32) m = fmaxf(m, __ldcg(at + c).x);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
        // (a sum that is not a number says so whatever its maximum is)
        auto part = [&](float2 x) { return x.x == -INFINITY ? static_cast<double>(x.y) : x.y * exp(static_cast<double>(x.x) - m); };
        double s = part(first);
        for (int c = 32 + (tid & 31); c < p.chunks; c += 32) s += part(__ldcg(at + c));
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        if ((tid & 31) == 0) {
            s_score[b] = score > -INFINITY && s > 0.0 && m > -INFINITY && m < INFINITY ? score : -INFINITY;
            s_max[b] = m;
            s_log[b] = log(s);
        }
    }
    auto total_of = [&](int b, float x) { return (x - s_max[b]) - s_log[b] + s_score[b]; };
    __syncthreads();
    for (int e = tid; e < p.K * p.n_ends; e += THREADS) {
        const int b = e / p.n_ends, id = s_end[e - b * p.n_ends];
        double total = -INFINITY;
        if (s_score[b] > -INFINITY && id >= 0 && id < p.V)
            total = total_of(b, to_float<T>(static_cast<const T*>(p.logits)[(static_cast<int64_t>(r) * p.K + b) * p.row_stride + id]));
        p.end_scores[static_cast<int64_t>(r) * p.K * p.n_ends + e] = static_cast<float>(total);
    }
    // token i of those that the request's rows kept, of the key k: (order of its total, place); 0: none
    auto total_key = [&](int i, unsigned long long k, unsigned long long& place) -> unsigned long long {
        const int b = i / per_row;
        if (!(s_score[b] > -INFINITY)) return 0;
        const uint32_t token = ~static_cast<uint32_t>(k);
        bool end = k == 0;
        for (int c = 0; c < p.n_ends; c++) end |= static_cast<uint32_t>(s_end[c]) == token;
        const double total = total_of(b, select_value(static_cast<uint32_t>(k >> 32)));
        place = static_cast<unsigned long long>(b) << 32 | token;
        return !end && total > -INFINITY ? select_order64(total) : 0;
    };
    auto token_of = [&](int i, unsigned long long& place) { return total_key(i, __ldcg(p.keys + static_cast<int64_t>(r) * all + i), place); };
    auto store = [&](int e, unsigned long long key, unsigned long long place) {
        const int64_t at = static_cast<int64_t>(r) * p.n + e;
        p.out_scores[at] = key ? static_cast<float>(select_value64(key)) : -INFINITY;
        p.parents[at] = key ? static_cast<int>(place >> 32) : -1;
        p.tokens[at] = key ? static_cast<int>(place & 0xffffffffu) : -1;
    };
    // ---- those that reach a threshold, by counting
    {
        uint32_t most = 0;
        unsigned long long place[FEW], other;
#pragma unroll
        for (int j = 0; j < FEW; j++) {
            const int i = tid + j * THREADS;
            kept[j] = i < all ? total_key(i, kept[j], place[j]) : 0;
            most = max(most, static_cast<uint32_t>(kept[j] >> 32));
        }
        for (int i = tid + FEW * THREADS; i < all; i += THREADS) most = max(most, static_cast<uint32_t>(token_of(i, other) >> 32));
        const uint32_t least = select_threshold<THREADS / 32>(most, p.n, s_top);
        auto push = [&](unsigned long long key, unsigned long long at) {
            if (key == 0 || static_cast<uint32_t>(key >> 32) < least) return;
            const int n = atomicAdd(&s_n, 1);
            if (n < kSelectRoom) {
                s_keys[2 * n] = key;
                s_keys[2 * n + 1] = at;
            }
        };
        if (most >= least) {
#pragma unroll
            for (int j = 0; j < FEW; j++) push(kept[j], place[j]);
            for (int i = tid + FEW * THREADS; i < all; i += THREADS) {
                const unsigned long long key = token_of(i, other);
                push(key, other);
            }
        }
        __syncthreads();
    }
    if (s_n <= kSelectRoom) {
        const int n = s_n;
        const ulonglong2* const s = reinterpret_cast<const ulonglong2*>(s_keys);
        for (int e = tid; e < n; e += THREADS) {
            const ulonglong2 mine = s[e];
            int rank = 0;
#pragma unroll 4
            for (int i = 0; i < n; i++) {
                const ulonglong2 x = s[i];
                rank += x.x > mine.x || (x.x == mine.x && x.y < mine.y);
            }
            if (rank < p.n) store(rank, mine.x, mine.y);
        }
        for (int e = n + tid; e < p.n; e += THREADS) store(e, 0, 0);
        return;
    }
    // ---- too many of them: the n best so far and as many others as there is room for, until there are no others
    const int n = select_join_size(p.K, p.chunks, p.keep, p.n);
    unsigned long long* const s_place = s_keys + n;
    __syncthreads();
    for (int e = tid; e < p.n; e += THREADS) {
        s_keys[e] = 0;
        s_place[e] = ~0ull;
    }
    for (int done = 0; done < all; done += n - p.n) {
        for (int e = p.n + tid; e < n; e += THREADS) {
            unsigned long long place = ~0ull;
            const int i = done + e - p.n;
            s_keys[e] = i < all ? token_of(i, place) : 0;
            s_place[e] = place;
        }
        for (int k = 2; k <= n; k <<= 1)
            for (int j = k >> 1; j > 0; j >>= 1) {
                __syncthreads();
                for (int i = tid; i < n / 2; i += THREADS) {
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
    for (int e = tid; e < p.n; e += THREADS) store(e, s_keys[e], s_place[e]);
}

}  // namespace ftq
