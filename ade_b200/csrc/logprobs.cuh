// Log probabilities of given tokens, the entropy of the distribution and the likeliest tokens, from a row of logits:
//   m = max x, s = sum exp(x - m), lse = m + log s;   log p = x - lse;   H = log s - sum exp(x - m) (x - m) / s.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace ade {

constexpr int LP_THREADS = 256;
constexpr int LP_MAX_TOP = 32;

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

// Order of the alternatives: larger logits first, NaN before all, equal ones by the lower index.  The larger key comes first.
__device__ __forceinline__ unsigned long long lp_key(float v, int i) {
    uint32_t u = __float_as_uint(v + 0.0f);                  // -0 counts as +0
    u = v != v ? 0xFFFFFFFFu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
    return static_cast<unsigned long long>(u) << 32 | ~static_cast<uint32_t>(i);
}

template <typename Op, typename T>
__device__ __forceinline__ T lp_reduce(T v, T* ws, Op op) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) ws[threadIdx.x >> 5] = v;
    __syncthreads();
    v = ws[0];
    for (int w = 1; w < LP_THREADS / 32; ++w) v = op(v, ws[w]);
    return v;
}

// One CTA per row: a pass for the maximum, one for the sums, one for each alternative.
template <typename T>
__global__ void __launch_bounds__(LP_THREADS) logprob_kernel(const LogprobParams p) {
    __shared__ float wf[LP_THREADS / 32];
    __shared__ unsigned long long wk[LP_THREADS / 32];
    const int tid = threadIdx.x;
    const T* x = static_cast<const T*>(p.x) + blockIdx.x * p.stride;
    auto add = [](float a, float b) { return a + b; };
    float m = -INFINITY;
    for (int i = tid; i < p.vocab; i += LP_THREADS) m = fmaxf(m, lp_float(x[i]));
    m = lp_reduce(m, wf, [](float a, float b) { return fmaxf(a, b); });
    float s = 0.f, e = 0.f;
    for (int i = tid; i < p.vocab; i += LP_THREADS) {
        const float z = lp_float(x[i]) - m, w = expf(z);
        s += w;
        e += w == 0.f ? 0.f : w * z;                           // a token of no probability adds nothing, -inf among them
    }
    s = lp_reduce(s, wf, add);
    e = lp_reduce(e, wf, add);
    const float ls = logf(s);
    if (tid == 0) {
        p.entropy[blockIdx.x] = ls - e / s;
        if (p.tokens) {
            const long long k = p.tokens[blockIdx.x];
            p.logprob[blockIdx.x] = k < 0 ? 0.f : k >= p.vocab ? __uint_as_float(0x7FC00000u) : (lp_float(x[k]) - m) - ls;
        }
    }
    unsigned long long below = ~0ull;
    for (int j = 0; j < p.top; ++j) {
        unsigned long long best = 0;
        for (int i = tid; i < p.vocab; i += LP_THREADS) {
            const unsigned long long k = lp_key(lp_float(x[i]), i);
            if ((j == 0 || k < below) && k > best) best = k;
        }
        below = lp_reduce(best, wk, [](unsigned long long a, unsigned long long b) { return a > b ? a : b; });
        if (tid == 0) {
            const uint32_t i = ~static_cast<uint32_t>(below);
            p.top_token[static_cast<long long>(blockIdx.x) * p.top + j] = i;
            p.top_logprob[static_cast<long long>(blockIdx.x) * p.top + j] = (lp_float(x[i]) - m) - ls;
        }
    }
}

}  // namespace ade
