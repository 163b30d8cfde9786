// Log probabilities of given tokens, the entropy of the distribution and the likeliest tokens, from a row of logits:
//   m = max x, s = sum exp(x - m), lse = m + log s;   log p = x - lse;   H = log s - sum exp(x - m) (x - m) / s.
//
// One CTA per row and one pass over it: every thread keeps the maximum of what it has seen, the sum and the weighted sum relative to
// it, and rescales them when the maximum grows; the maximum of every run of pieces (an eighth of the thread's) is kept besides.  The maxima of
// 32 groups of threads bound the k-th largest logit from below (k of them are reached by k logits), so only the runs whose maximum
// reaches that bound are looked at again, about k of 2048, by all threads together, and the handful of logits that do is ranked by
// counting.  A row whose list would not fit (hundreds of equal logits at the bound; fewer logits above -inf, or above the
// lowest value that masks the others, than alternatives) or that holds a NaN is walked once for every alternative instead: 8 rows of 32000 with four finite
// logits and five alternatives take 38 us instead of 5.6, with sixty finite ones 5.6.  256 threads whatever the row: 1024 of them took 6.6 us instead of 5.3 for 8 rows of 32000, 12.7 instead of 12.6 for 8 of
// 152064, and 512 took 49 instead of 37 for 2048 rows of 32000.
// 2048 rows of 50257 float32 logits with twenty alternatives take 82 us (0.41 GB, 5.0 TB/s; 69 without alternatives, whose small dependent steps end each
// row); in bfloat16, 2048 rows of 32000, 37 us (3.5 TB/s): there exponentials and sums bound it, two bytes a logit.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace ade {

constexpr int LP_MAX_TOP = 32;
constexpr int LP_LIST = 512;       // logits that may reach the bound
constexpr int LP_THREADS = 256;
constexpr int LP_RUNS = 8;         // runs of a thread's pieces

struct LogprobParams {
    const void* x;                 // [rows][vocab], rows `stride` elements apart
    const long long* tokens;       // [rows] or nullptr; negative: no token, the log probability is 0; >= vocab: NaN
    float *logprob, *entropy;      // [rows]; logprob is nullptr without tokens
    float* top_logprob;            // [rows][top]
    long long* top_token;          // [rows][top]
    long long stride;
    int rows, vocab, top;
};

__device__ __forceinline__ float lp_float(float v) { return v; }
__device__ __forceinline__ float lp_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float lp_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// the logits of a 16-byte piece
template <typename T>
struct LpPiece {
    static constexpr int N = 16 / sizeof(T);
    // a piece of nothing but -inf
    static __device__ __forceinline__ uint4 none() {
        constexpr uint32_t w = sizeof(T) == 4 ? 0xFF800000u : std::is_same<T, __half>::value ? 0xFC00FC00u : 0xFF80FF80u;
        return make_uint4(w, w, w, w);
    }
    static __device__ __forceinline__ void get(const uint4& w, float (&v)[N]) {
        const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = lp_float(e[i]);
    }
};

// Order of the alternatives: larger logits first, NaN before all, equal ones by the lower index.  The larger key comes first.
__device__ __forceinline__ unsigned long long lp_key(float v, int i) {
    uint32_t u = __float_as_uint(v + 0.0f);                  // -0 counts as +0
    u = v != v ? 0xFFFFFFFFu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
    return static_cast<unsigned long long>(u) << 32 | ~static_cast<uint32_t>(i);
}

__device__ __forceinline__ float lp_exp2(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// the logit of a key
__device__ __forceinline__ float lp_value(unsigned long long key) {
    const uint32_t u = static_cast<uint32_t>(key >> 32);
    return __uint_as_float(u == 0xFFFFFFFFu ? u : u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}

// maximum m of some logits, sum of w = 2^z and of w z, where z = (x - m) log2(e)
struct LpSums {
    float m, s, e;
    // the same relative to another maximum, which is at least as large; the difference is kept where its product with a sum is finite (a logit may
    // be the lowest float32), exp is 0 long before that
    __device__ __forceinline__ void move(float to) {
        const float d = fmaxf((m - to) * 1.44269504088896340736f, -1e30f), f = lp_exp2(d);
        if (m != -INFINITY) {                                // without a maximum the sums are 0, or NaN
            e = f * (e + s * d);
            s *= f;
        }
        m = to;
    }
    // what the logits are taken relative to: without a maximum (nothing but -inf so far, which adds nothing, and NaN, which shows) the logits themselves
    __device__ __forceinline__ float base() const { return m == -INFINITY ? 0.f : m; }
    __device__ __forceinline__ void add(float x, float base) {
        const float z = (x - base) * 1.44269504088896340736f, w = lp_exp2(z);
        s += w;
        e += w * fmaxf(z, -1e30f);                           // a token of no probability adds nothing, -inf among them
    }
};

// Pieces of 16 bytes from the first 16-byte boundary of the row; what stands before it and behind the last whole piece goes to the first threads
// one by one.  A batch of pieces is requested while the one before it is added.
template <typename T>
__global__ void __launch_bounds__(LP_THREADS, 4) logprob_kernel(const LogprobParams p) {
    using P = LpPiece<T>;
    constexpr int THREADS = LP_THREADS, NW = THREADS / 32, U = 4;      // pieces of a batch
    __shared__ LpSums ws[NW];
    __shared__ float tmax[THREADS], rmax[LP_RUNS][THREADS];
    __shared__ unsigned short runs[LP_RUNS * THREADS];
    __shared__ unsigned long long list[LP_LIST], wk[NW];
    __shared__ int listed, found;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const T* x = static_cast<const T*>(p.x) + blockIdx.x * p.stride;
    const int V = p.vocab;
    const int head = min(V, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / static_cast<int>(sizeof(T)));
    const int pieces = (V - head) / P::N, tail = head + pieces * P::N;
    const uint4* body = reinterpret_cast<const uint4*>(x + head);
    // this thread's logit outside the pieces, if below V; behind the last of them it may pass 31 bits
    const uint32_t edge = tid < head ? tid : static_cast<uint32_t>(tail) + tid - head, end = V;
    if (tid == 0) listed = found = 0;
    float given = 0.f;                                                       // the given token's logit, under way from the start
    if (tid == 0 && p.tokens) {
        const long long k = p.tokens[blockIdx.x];
        given = k >= 0 && k < V ? lp_float(x[k]) : __uint_as_float(0x7FC00000u);
    }

    LpSums a = {-INFINITY, 0.f, 0.f};
    if (edge < end) {
        const float v = lp_float(x[edge]);
        a.m = fmaxf(a.m, v);
        a.add(v, a.base());
    }
    uint4 cur[U], next[U];
    auto load = [&](uint4 (&w)[U], int i) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            w[u] = P::none();
            if (i + u * THREADS < pieces) w[u] = __ldg(body + i + u * THREADS);
        }
    };
    load(cur, tid);
    const int batches = (pieces + U * THREADS - 1) / (U * THREADS), length = (batches + LP_RUNS - 1) / LP_RUNS;      // of a run, in batches
    float top = -INFINITY;                                                   // maximum of the run
    for (int i = tid, n = 0; n < batches; i += U * THREADS, ++n) {
        load(next, i + U * THREADS);
        float v[U][P::N], mx = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            P::get(cur[u], v[u]);
#pragma unroll
            for (int j = 0; j < P::N; ++j) mx = fmaxf(mx, v[u][j]);
        }
        if (mx > a.m) a.move(mx);
        const float base = a.base();
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int j = 0; j < P::N; ++j) a.add(v[u][j], base);
            cur[u] = next[u];
        }
        top = fmaxf(top, mx);
        if ((n + 1) % length == 0 || n + 1 == batches) {
            rmax[n / length][tid] = top;
            top = -INFINITY;
        }
    }
    const float mine = a.m;
    // maxima of the groups, then everything relative to the row's maximum.  A group is the threads of one lane, so that few pieces fall to 32 groups
    // too and the bound holds for short rows (10 rows of 532 bfloat16, twenty alternatives: 4.5 us; 16 with groups of neighbours, most of them
    // empty, and every logit on the list).
    tmax[tid] = mine;
    __syncthreads();
    float g = mine;
#pragma unroll
    for (int w = 0; w < NW; ++w) g = fmaxf(g, tmax[w * 32 + lane]);
    float m = g;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    a.move(m);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a.s += __shfl_xor_sync(0xFFFFFFFFu, a.s, o);
        a.e += __shfl_xor_sync(0xFFFFFFFFu, a.e, o);
    }
    if (lane == 0) ws[warp] = a;
    __syncthreads();
    float s = 0.f, e = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        s += ws[w].s;
        e += ws[w].e;
    }
    const float ls = logf(s);
    auto logp = [&](float v) { return (v - m) - ls; };
    if (tid == 0) {
        p.entropy[blockIdx.x] = ls - 0.69314718055994530942f * (e / s);
        if (p.tokens) {
            p.logprob[blockIdx.x] = p.tokens[blockIdx.x] < 0 ? 0.f : logp(given);
        }
    }
    if (p.top == 0) return;
    auto put = [&](int j, unsigned long long key) {
        const uint32_t at = ~static_cast<uint32_t>(key);
        p.top_token[static_cast<long long>(blockIdx.x) * p.top + j] = at;
        p.top_logprob[static_cast<long long>(blockIdx.x) * p.top + j] = logp(lp_value(key));
    };
    bool walk = !(s > 0.f);                                                  // NaN, an infinity, or nothing but -inf
    if (!walk) {
        // the top-th largest of the 32 maxima (equal ones by their place)
        int rank = 0;
#pragma unroll
        for (int o = 0; o < 32; ++o) {
            const float u = __shfl_sync(0xFFFFFFFFu, g, o);
            rank += u > g || (u == g && o < lane);
        }
        const float bound = __shfl_sync(0xFFFFFFFFu, g, __ffs(__ballot_sync(0xFFFFFFFFu, rank == p.top - 1)) - 1);
        auto list_it = [&](float v, int at) {
            if (!(v >= bound)) return;
            const int n = atomicAdd(&listed, 1);
            if (n < LP_LIST) list[n] = lp_key(v, at);
        };
        if (edge < end) list_it(lp_float(x[edge]), edge);
        if (mine >= bound)
            for (int r = 0; r * length < batches; ++r)
                if (rmax[r][tid] >= bound) runs[atomicAdd(&found, 1)] = static_cast<unsigned short>(r * THREADS + tid);
        __syncthreads();
        const int size = length * U, all = found * size;
        for (int w = tid; w < all; w += THREADS) {
            const int id = runs[w / size], k = (id / THREADS * size + w % size) * THREADS + id % THREADS;
            if (k >= pieces) continue;
            float v[P::N];
            P::get(__ldg(body + k), v);
#pragma unroll
            for (int j = 0; j < P::N; ++j) list_it(v[j], head + k * P::N + j);
        }
        __syncthreads();
        const int n = listed;
        walk = n > LP_LIST;
        if (!walk)
            for (int k = tid; k < n; k += THREADS) {
                const unsigned long long key = list[k];
                int before = 0;
                for (int j = 0; j < n; ++j) before += list[j] > key;
                if (before < p.top) put(before, key);
            }
    }
    if (!walk) return;
    unsigned long long below = ~0ull;
    for (int j = 0; j < p.top; ++j) {
        unsigned long long best = 0;
        auto look = [&](float v, int at) {
            const unsigned long long key = lp_key(v, at);
            if ((j == 0 || key < below) && key > best) best = key;
        };
        if (edge < end) look(lp_float(x[edge]), edge);
        for (int k = tid; k < pieces; k += THREADS) {
            float v[P::N];
            P::get(__ldg(body + k), v);
#pragma unroll
            for (int q = 0; q < P::N; ++q) look(v[q], head + k * P::N + q);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const unsigned long long u = __shfl_xor_sync(0xFFFFFFFFu, best, o);
            best = u > best ? u : best;
        }
        __syncthreads();
        if (lane == 0) wk[warp] = best;
        __syncthreads();
        below = wk[0];
        for (int w = 1; w < NW; ++w) below = wk[w] > below ? wk[w] : below;
        if (tid == 0) put(j, below);
    }
}

}  // namespace ade
