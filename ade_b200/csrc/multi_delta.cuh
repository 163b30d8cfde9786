// Deltas of many fine-tuned models beside one shared projection:  out[t] = y[t] + U_d^ (V_d^^T x[t]),  d = ids[t].
//
// The deltas lie in a bank, rank group by rank group (128 ranks): delta d owns groups start[d] .. start[d + 1] - 1.
//   vt uint8 [G][128][N/2], vs bf16 [G][N], vz uint8 [G][N]     V^^T = vs (code - vz), packed along d_i
//   uq uint8 [G][M][64],    us bf16 [G][M], uz uint8 [G][M]     U^  = us (code - uz), packed along the rank axis
// Rows whose id is outside 0 .. deltas - 1 get y alone.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace ade {

constexpr int MD_MAX_GROUPS = 16;         // rank groups of one delta (ADE_B200_MAX_RANK / 128)

struct MultiDeltaParams {
    const __nv_bfloat16 *x, *y;           // [T][N], [T][M]
    __nv_bfloat16* out;                   // [T][M]
    const uint8_t *uq, *uz, *vt, *vz;
    const __nv_bfloat16 *us, *vs;
    const int *start, *ids;               // [deltas + 1], [T]
    float* h;                             // [T][MD_MAX_GROUPS * 128]
    int M, N, G, deltas, T;
};

// groups of row t's delta: first one and how many (0: the row has no delta)
__device__ __forceinline__ int md_groups(const MultiDeltaParams& p, int t, int& first) {
    const int d = p.ids[t];
    first = 0;
    if (d < 0 || d >= p.deltas) return 0;
    first = max(p.start[d], 0);
    return max(0, min(min(p.start[d + 1], p.G) - first, MD_MAX_GROUPS));
}

// h[t][128 j + k] = sum_n vs (code - vz) x[t][n] for rank k of the j-th group: one CTA per (row, group), 16 ranks per warp
__global__ void __launch_bounds__(256) multi_delta_v_kernel(const MultiDeltaParams p) {
    int first;
    const int t = blockIdx.x, j = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (j >= md_groups(p, t, first)) return;
    const size_t g = first + j;
    for (int k = warp * 16; k < warp * 16 + 16; ++k) {
        float s = 0.f;
        const uint32_t* row = reinterpret_cast<const uint32_t*>(p.vt + (g * 128 + k) * (p.N / 2));
        for (int w = lane; w < p.N / 8; w += 32) {
            const uint32_t code = row[w];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int n = w * 8 + i;
                const int c = code >> (4 * (i >> 1) + 16 * (i & 1)) & 15;
                s += static_cast<float>(c - p.vz[g * p.N + n]) * __bfloat162float(p.vs[g * p.N + n]) * __bfloat162float(p.x[static_cast<size_t>(t) * p.N + n]);
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
        if (lane == 0) p.h[static_cast<size_t>(t) * (MD_MAX_GROUPS * 128) + j * 128 + k] = s;
    }
}

// out[t][m] = y[t][m] + sum_g us sum_k (code - uz) h: one thread per (row, output)
__global__ void __launch_bounds__(256) multi_delta_u_kernel(const MultiDeltaParams p) {
    __shared__ float h[MD_MAX_GROUPS * 128];
    int first;
    const int t = blockIdx.x, m = blockIdx.y * 256 + threadIdx.x;
    const int ng = md_groups(p, t, first);
    for (int k = threadIdx.x; k < ng * 128; k += 256) h[k] = p.h[static_cast<size_t>(t) * (MD_MAX_GROUPS * 128) + k];
    __syncthreads();
    if (m >= p.M) return;
    float acc = __bfloat162float(p.y[static_cast<size_t>(t) * p.M + m]);
    for (int j = 0; j < ng; ++j) {
        const size_t gm = static_cast<size_t>(first + j) * p.M + m;
        const uint32_t* row = reinterpret_cast<const uint32_t*>(p.uq + gm * 64);
        const int z = p.uz[gm];
        float s = 0.f;
        for (int w = 0; w < 16; ++w) {
            const uint32_t code = row[w];
#pragma unroll
            for (int i = 0; i < 8; ++i) s += static_cast<float>(static_cast<int>(code >> (4 * (i >> 1) + 16 * (i & 1)) & 15) - z) * h[j * 128 + w * 8 + i];
        }
        acc += __bfloat162float(p.us[gm]) * s;
    }
    p.out[static_cast<size_t>(t) * p.M + m] = __float2bfloat16_rn(acc);
}

}  // namespace ade
