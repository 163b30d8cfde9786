// Deltas of many fine-tuned models beside one shared projection:  out[t] = y[t] + U_d^ (V_d^^T x[t]),  d = ids[t].
//
// The deltas lie in a bank, rank group by rank group (128 ranks): delta d owns groups start[d] .. start[d + 1] - 1.
//   vt uint8 [G][128][N/2], vs bf16 [G][N], vz uint8 [G][N]     V^^T = vs (code - vz), packed along d_i
//   uq uint8 [G][M][64],    us bf16 [G][M], uz uint8 [G][M]     U^  = us (code - uz), packed along the rank axis
// Rows whose id is outside 0 .. deltas - 1 get y alone.
//
// Two launches, h = V^^T x and out = y + U^ h; the second is set up under the first.  Both find out on the device which rows share a
// delta (ids may change from replay to replay of a graph) and cut them into entries of up to eight rows, so that a delta's codes
// are read once for each entry, and from DRAM once.  Both are streams of 4-bit codes against a handful of token columns, on the warp matrix
// instruction m16n8k16: the codes, as bfloat16 128 + c (one or two integer instructions for a pair), are its 16 rows, four token rows its
// eight columns: columns 0-3 hold the bfloat16 rounding of a float32 operand (x vs, or h), columns 4-7 what that rounding left over, which
// is free as long as an entry has at most four rows.  The zero-points come off afterwards: sum a (c - z) = sum a (128 + c) - sum a (128 + z),
// whose second term is one more row of the product for V and a multiple of sum a for U; both sums are float32.
// Every thread copies the 16-byte pieces of codes that it will use itself with cp.async into a queue of its own, so the
// stream runs through the barriers of an item and into the next one.  Sums have a fixed order; there are no atomics.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "ptx.cuh"

namespace ade {

constexpr int MD_MAX_GROUPS = 16;                 // rank groups of one delta (ADE_B200_MAX_RANK / 128)
constexpr int MD_MAX_ROWS = 128;                  // ADE_B200_MAX_TOKENS
constexpr int MD_THREADS = 256;
constexpr int MD_ENTRY = 8;                       // rows of an entry
constexpr int MD_COLS = 1024;                     // columns of V^T that one item covers, 128 per warp
constexpr int MD_H = MD_MAX_GROUPS * 128;         // floats of h kept per row and slice of columns
constexpr int MD_CHUNK = 8;                       // rank groups of h in shared memory at a time
constexpr int MD_UROWS = 256;                     // rows of U that one item covers, 32 per warp
constexpr int MD_PART = 132;                      // row pitch of the warps' partial h, in floats
constexpr int MD_HCOL = MD_CHUNK * 256 + 64;      // bytes of a column of h in shared memory; 64 over a multiple of 128: no bank conflicts
constexpr int MD_UDEPTH = 4;                      // steps in the queue of the second launch
constexpr uint32_t kMd128 = 0x43004300u;          // bf16x2 (128, 128)

struct MultiDeltaParams {
    const __nv_bfloat16 *x, *y;           // [T][N], [T][M]
    __nv_bfloat16* out;                   // [T][M]
    const uint8_t *uq, *uz, *vt, *vz;
    const __nv_bfloat16 *us, *vs;
    const int *start, *ids;               // [deltas + 1], [T]
    float* h;                             // [slices][T][MD_H] sums over the columns of a slice
    int M, N, G, deltas, T;
};

// Rows that share a delta, in entries of up to MD_ENTRY rows.
struct MdEntries {
    int n;
    int first[MD_MAX_ROWS], ng[MD_MAX_ROWS], rows[MD_MAX_ROWS];   // first rank group, their number, rows of the entry
    int groups_end[MD_MAX_ROWS];                                  // rank groups of this entry and those before it
    uint8_t row[MD_MAX_ROWS][MD_ENTRY];
    int key[MD_MAX_ROWS], base[MD_MAX_ROWS], wsum[8];
};

constexpr size_t md_v_smem() { return 8 * 2 * MD_THREADS * 16 + 8 * MD_ENTRY * MD_PART * sizeof(float); }
constexpr size_t md_u_smem() { return MD_UDEPTH * 4 * MD_THREADS * 16 + 16 * MD_HCOL + MD_CHUNK * 16 * sizeof(float); }
inline int md_slices(int N) { return (N + MD_COLS - 1) / MD_COLS; }

__device__ __forceinline__ void md_cp16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void md_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void md_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ float md_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float md_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
__device__ __forceinline__ uint32_t md_pack(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// codes 2 j, 2 j + 1 of a packed word as bfloat16 128 + c
__device__ __forceinline__ uint32_t md_pair(uint32_t w, int j) { return (w >> (4 * j) & 0x000F000Fu) | kMd128; }

__device__ __forceinline__ void md_entries(const MultiDeltaParams& p, MdEntries& e) {
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    int first = 0, ng = 0;
    if (t < p.T) {
        const int d = p.ids[t];
        if (d >= 0 && d < p.deltas) {
            first = max(p.start[d], 0);
            ng = max(0, min(min(p.start[d + 1], p.G) - first, MD_MAX_GROUPS));
        }
        e.key[t] = ng ? d : -1;                             // rows without a delta share an entry of no groups
    }
    __syncthreads();
    int before = 0, same = 0, leader = t;
    if (t < p.T) {
        const int mine = e.key[t];
        for (int u = p.T - 1; u >= 0; --u)
            if (e.key[u] == mine) {
                ++same;
                before += u < t;
                leader = u;
            }
    }
    // entries and rank groups of each group of rows, at its first row, summed over the rows
    const int mine = t < p.T && leader == t ? (same + MD_ENTRY - 1) / MD_ENTRY : 0;
    int run = mine << 16 | mine * ng;                       // at most 128 entries, 128 * 16 rank groups
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xFFFFFFFFu, run, o);
        if (lane >= o) run += u;
    }
    if (lane == 31) e.wsum[warp] = run;
    __syncthreads();
    run -= mine << 16 | mine * ng;
    for (int w = 0; w < warp; ++w) run += e.wsum[w];
    if (t < p.T) e.base[t] = run;
    if (t == 0) {
        int all = 0;
        for (int w = 0; w < MD_MAX_ROWS / 32; ++w) all += e.wsum[w];
        e.n = all >> 16;
    }
    for (int k = 0; k < mine; ++k) {
        const int i = (run >> 16) + k;
        e.first[i] = first;
        e.ng[i] = ng;
        e.rows[i] = min(MD_ENTRY, same - k * MD_ENTRY);
        e.groups_end[i] = (run & 0xFFFF) + (k + 1) * ng;
    }
    __syncthreads();
    if (t < p.T) e.row[(e.base[leader] >> 16) + before / MD_ENTRY][before % MD_ENTRY] = static_cast<uint8_t>(t);
    __syncthreads();
}

// ------------------------------------------------------------------ h = V^T x
// An item is one rank group of one entry over MD_COLS columns: a warp multiplies the group's 128 ranks with 128 columns, eight tiles of 16
// ranks one behind the other, and the warps' sums are added through shared memory.
template <int N>
struct MdTiles {
    static constexpr int value = N;
};

struct MdVItem {
    int e, j, slice;                       // entry, its rank group, slice of columns
};

__device__ __forceinline__ MdVItem md_v_item(const MdEntries& e, int item, int slices) {
    const int g = item / slices;
    int lo = 0, hi = e.n - 1;              // first entry with groups_end > g
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (e.groups_end[mid] > g) hi = mid;
        else lo = mid + 1;
    }
    return {lo, g - (e.groups_end[lo] - e.ng[lo]), item - g * slices};
}

template <int NT>
__device__ __forceinline__ void md_v_compute(const MultiDeltaParams& p, const MdEntries& e, const MdVItem& it, int cb, uint32_t fifo, float* part, bool more,
                                             const uint8_t* next) {
    const int lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
    const size_t g = e.first[it.e] + it.j, col = static_cast<size_t>(cb) * 128 + tig * 32;
    uint32_t xs[NT][16], z[16];
    {
        uint4 zv[2], sv[4];
        const uint4* zp = reinterpret_cast<const uint4*>(p.vz + g * p.N + col);
        const uint4* sp = reinterpret_cast<const uint4*>(p.vs + g * p.N + col);
        zv[0] = ldg16(zp);
        zv[1] = ldg16(zp + 1);
#pragma unroll
        for (int i = 0; i < 4; ++i) sv[i] = ldg16(sp + i);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int r = n * 4 + (gid & 3);
            uint4 xv[4] = {};
            if (r < e.rows[it.e]) {
                const uint4* xp = reinterpret_cast<const uint4*>(p.x + static_cast<size_t>(e.row[it.e][r]) * p.N + col);
#pragma unroll
                for (int i = 0; i < 4; ++i) xv[i] = ldg16(xp + i);
            }
            const uint32_t *xw = reinterpret_cast<const uint32_t*>(xv), *sw = reinterpret_cast<const uint32_t*>(sv);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float a = md_lo(xw[i]) * md_lo(sw[i]), b = md_hi(xw[i]) * md_hi(sw[i]);
                const uint32_t hi = md_pack(a, b);
                xs[n][i] = gid < 4 ? hi : md_pack(a - md_lo(hi), b - md_hi(hi));
            }
        }
        const uint32_t* zw = reinterpret_cast<const uint32_t*>(zv);
#pragma unroll
        for (int i = 0; i < 8; ++i) {                                 // zero-points 4 i .. 4 i + 3 as bfloat16 128 + z
            z[2 * i] = __byte_perm(zw[i], 0, 0x4140) | kMd128;
            z[2 * i + 1] = __byte_perm(zw[i], 0, 0x4342) | kMd128;
        }
    }
    float zero[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        zero[n][0] = zero[n][1] = zero[n][2] = zero[n][3] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) mma_bf16(zero[n], z[2 * i], z[2 * i], z[2 * i + 1], z[2 * i + 1], xs[n][2 * i], xs[n][2 * i + 1]);
    }
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) {
        md_wait<7>();
        const uint4 r0 = lds16(fifo + (mt * 2) * MD_THREADS * 16), r1 = lds16(fifo + (mt * 2 + 1) * MD_THREADS * 16);
        const uint32_t w0[4] = {r0.x, r0.y, r0.z, r0.w}, w1[4] = {r1.x, r1.y, r1.z, r1.w};
        float d[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) d[n][0] = d[n][1] = d[n][2] = d[n][3] = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const uint32_t a0 = md_pair(w0[w], 2 * q), a1 = md_pair(w1[w], 2 * q), a2 = md_pair(w0[w], 2 * q + 1), a3 = md_pair(w1[w], 2 * q + 1);
#pragma unroll
                for (int n = 0; n < NT; ++n) mma_bf16(d[n], a0, a1, a2, a3, xs[n][w * 4 + 2 * q], xs[n][w * 4 + 2 * q + 1]);
            }
        if (more) {                                                   // the same tile of the next item into the pieces just used
            md_cp16(fifo + (mt * 2) * MD_THREADS * 16, next + static_cast<size_t>(mt * 16) * (p.N / 2));
            md_cp16(fifo + (mt * 2 + 1) * MD_THREADS * 16, next + static_cast<size_t>(mt * 16 + 8) * (p.N / 2));
        }
        md_commit();
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v = d[n][i] - zero[n][i];                        // rank gid + 8 (i / 2), column 2 tig + i % 2
                v += __shfl_xor_sync(0xFFFFFFFFu, v, 2);
                if (tig < 2) part[(n * 4 + tig * 2 + (i & 1)) * MD_PART + mt * 16 + gid + (i >> 1) * 8] = v;
            }
    }
}

__global__ void __launch_bounds__(MD_THREADS, 2) multi_delta_v_kernel(const MultiDeltaParams p, int slices) {
    extern __shared__ __align__(16) uint8_t md_smem[];
    __shared__ MdEntries e;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gid = lane >> 2, tig = lane & 3;
    float* part = reinterpret_cast<float*>(md_smem + 8 * 2 * MD_THREADS * 16);
    const uint32_t fifo = smem_u32(md_smem) + tid * 16;
    md_entries(p, e);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int blocks = p.N / 128, items = (e.n ? e.groups_end[e.n - 1] : 0) * slices;
    // this thread's first piece of an item's codes, or nullptr where the warp has no columns
    auto codes = [&](const MdVItem& it) -> const uint8_t* {
        const int cb = it.slice * (MD_COLS / 128) + warp;
        if (cb >= blocks) return nullptr;
        return p.vt + (static_cast<size_t>(e.first[it.e] + it.j) * 128 + gid) * (p.N / 2) + cb * 64 + tig * 16;
    };
    int item = blockIdx.x;
    if (item >= items) return;
    MdVItem it = md_v_item(e, item, slices);
    const uint8_t* src = codes(it);
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) {
        if (src) {
            md_cp16(fifo + (mt * 2) * MD_THREADS * 16, src + static_cast<size_t>(mt * 16) * (p.N / 2));
            md_cp16(fifo + (mt * 2 + 1) * MD_THREADS * 16, src + static_cast<size_t>(mt * 16 + 8) * (p.N / 2));
        }
        md_commit();
    }
    while (true) {
        const int next_item = item + gridDim.x;
        const bool go_on = next_item < items;
        const MdVItem nx = go_on ? md_v_item(e, next_item, slices) : it;
        const uint8_t* nsrc = go_on ? codes(nx) : nullptr;
        const int cb = it.slice * (MD_COLS / 128) + warp, rows = e.rows[it.e];
        if (src) {
            float* mine = part + warp * (MD_ENTRY * MD_PART);
            if (rows <= 4) md_v_compute<1>(p, e, it, cb, fifo, mine, nsrc != nullptr, nsrc);
            else md_v_compute<2>(p, e, it, cb, fifo, mine, nsrc != nullptr, nsrc);
        } else {
#pragma unroll
            for (int mt = 0; mt < 8; ++mt) {
                if (nsrc) {
                    md_cp16(fifo + (mt * 2) * MD_THREADS * 16, nsrc + static_cast<size_t>(mt * 16) * (p.N / 2));
                    md_cp16(fifo + (mt * 2 + 1) * MD_THREADS * 16, nsrc + static_cast<size_t>(mt * 16 + 8) * (p.N / 2));
                }
                md_commit();
            }
        }
        __syncthreads();
        const int warps = min(8, blocks - it.slice * (MD_COLS / 128));
        for (int i = tid; i < rows * 128; i += MD_THREADS) {
            const int r = i >> 7, k = i & 127;
            float s = 0.f;
            for (int w = 0; w < warps; ++w) s += part[(w * MD_ENTRY + r) * MD_PART + k];
            p.h[(static_cast<size_t>(it.slice) * p.T + e.row[it.e][r]) * MD_H + it.j * 128 + k] = s;
        }
        if (!go_on) return;
        __syncthreads();
        item = next_item;
        it = nx;
        src = nsrc;
    }
}

// ------------------------------------------------------------------ out = y + U h
// An item is MD_UROWS rows of one entry's U: a warp multiplies 32 of them, in two tiles of 16, with the entry's columns of h, a rank group at a
// step, and adds us (sum - (128 + uz) sum h) to its float32 results.
template <int NT>
__device__ __forceinline__ void md_u_step(const uint4 (&c)[4], const uint8_t* hcol, const float* hsum, int j, const float (&us)[4], const float (&uz)[4],
                                          float (&acc)[2][NT][4]) {
    const int lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
    float d[2][NT][4];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) d[m][n][0] = d[m][n][1] = d[m][n][2] = d[m][n][3] = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        uint4 b[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) b[n] = *reinterpret_cast<const uint4*>(hcol + (n * 8 + gid) * MD_HCOL + j * 256 + (w * 4 + tig) * 16);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const uint32_t w0 = reinterpret_cast<const uint32_t*>(&c[m * 2])[w], w1 = reinterpret_cast<const uint32_t*>(&c[m * 2 + 1])[w];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                mma_bf16(d[m][n], md_pair(w0, 0), md_pair(w1, 0), md_pair(w0, 1), md_pair(w1, 1), b[n].x, b[n].y);
                mma_bf16(d[m][n], md_pair(w0, 2), md_pair(w1, 2), md_pair(w0, 3), md_pair(w1, 3), b[n].z, b[n].w);
            }
        }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const float2 s = *reinterpret_cast<const float2*>(hsum + j * 16 + n * 8 + tig * 2);
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[m][n][i] += us[m * 2 + (i >> 1)] * (d[m][n][i] - uz[m * 2 + (i >> 1)] * (i & 1 ? s.y : s.x));
    }
}

__global__ void __launch_bounds__(MD_THREADS, 2) multi_delta_u_kernel(const MultiDeltaParams p, int slices) {
    extern __shared__ __align__(16) uint8_t md_smem[];
    __shared__ MdEntries e;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gid = lane >> 2, tig = lane & 3;
    const uint32_t fifo = smem_u32(md_smem) + tid * 16;
    uint8_t* hcol = md_smem + MD_UDEPTH * 4 * MD_THREADS * 16;                   // [16 columns][MD_HCOL]
    float* hsum = reinterpret_cast<float*>(hcol + 16 * MD_HCOL);                 // [MD_CHUNK][16 columns]
    md_entries(p, e);
    const int chunks = (p.M + MD_UROWS - 1) / MD_UROWS, items = e.n * chunks;
    // the stream of (item, rank group) steps, MD_UDEPTH - 1 ahead of the arithmetic
    int a_item = blockIdx.x, a_j = 0;
    auto settle = [&] {                                                          // items of entries without rank groups have no steps
        while (a_item < items && a_j >= e.ng[a_item / chunks]) {
            a_item += gridDim.x;
            a_j = 0;
        }
    };
    auto issue = [&](int slot) {
        settle();
        if (a_item < items) {
            const int en = a_item / chunks, m = (a_item - en * chunks) * MD_UROWS + warp * 32 + gid;
            const uint8_t* src = p.uq + (static_cast<size_t>(e.first[en] + a_j) * p.M + m) * 64 + tig * 16;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (m + 8 * i < p.M) md_cp16(fifo + (slot * 4 + i) * MD_THREADS * 16, src + i * 8 * 64);
            ++a_j;
        }
        md_commit();
    };
#pragma unroll
    for (int s = 0; s < MD_UDEPTH - 1; ++s) issue(s);
    int slot = 0;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    auto work = [&](int item, auto tiles) {
        constexpr int NT = decltype(tiles)::value;                               // tiles of eight columns: two parts of four rows each
        const int en = item / chunks, ng = e.ng[en], rows = e.rows[en], first = e.first[en];
        const int m0 = (item - en * chunks) * MD_UROWS + warp * 32 + gid;          // rows m0 + 8 i of U, i = 0 .. 3
        float acc[2][NT][4] = {};
        for (int j0 = 0; j0 < ng; j0 += MD_CHUNK) {
            const int jn = min(MD_CHUNK, ng - j0);
            __syncthreads();                                                       // nobody reads the columns of h in place any more
            // h of (row, rank group), one of them per warp and round, four ranks per lane: the slices' sums, as two bfloat16 parts in the
            // order in which the products take them
            for (int i = warp; i < rows * jn; i += MD_THREADS / 32) {
                const int r = i / jn, j = i - r * jn;
                const float* src = p.h + static_cast<size_t>(e.row[en][r]) * MD_H + (j0 + j) * 128 + lane * 4;
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
                for (int s = 0; s < slices; ++s) {
                    const float4 a = *reinterpret_cast<const float4*>(src + static_cast<size_t>(s) * p.T * MD_H);
                    v.x += a.x;
                    v.y += a.y;
                    v.z += a.z;
                    v.w += a.w;
                }
                const uint32_t h0 = md_pack(v.x, v.y), h1 = md_pack(v.z, v.w);
                const uint32_t l0 = md_pack(v.x - md_lo(h0), v.y - md_hi(h0)), l1 = md_pack(v.z - md_lo(h1), v.w - md_hi(h1));
                float sh = md_lo(h0) + md_hi(h0) + md_lo(h1) + md_hi(h1), sl = md_lo(l0) + md_hi(l0) + md_lo(l1) + md_hi(l1);
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    sh += __shfl_xor_sync(0xFFFFFFFFu, sh, o);
                    sl += __shfl_xor_sync(0xFFFFFFFFu, sl, o);
                }
                const int c = (r >> 2) * 8 + (r & 3);                              // column of the rounded part; the rest stands four behind it
                uint8_t* to = hcol + c * MD_HCOL + j * 256 + ((lane >> 1 & 3) * 4 + (lane >> 3)) * 16 + (lane & 1) * 8;
                *reinterpret_cast<uint2*>(to) = make_uint2(h0, h1);
                *reinterpret_cast<uint2*>(to + 4 * MD_HCOL) = make_uint2(l0, l1);
                if (lane == 0) {
                    hsum[j * 16 + c] = sh;
                    hsum[j * 16 + c + 4] = sl;
                }
            }
            __syncthreads();
            for (int j = 0; j < jn; ++j) {
                float us[4], uz[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const size_t at = static_cast<size_t>(first + j0 + j) * p.M + min(m0 + 8 * i, p.M - 1);
                    us[i] = __bfloat162float(p.us[at]);
                    uz[i] = 128.f + p.uz[at];
                }
                md_wait<MD_UDEPTH - 2>();
                uint4 c[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) c[i] = lds16(fifo + (slot * 4 + i) * MD_THREADS * 16);
                issue(slot == 0 ? MD_UDEPTH - 1 : slot - 1);
                slot = slot + 1 == MD_UDEPTH ? 0 : slot + 1;
                md_u_step<NT>(c, hcol, hsum, j, us, uz, acc);
            }
        }
        // the two parts of a column are added; lane (gid, tig < 2) then has rows 2 tig, 2 tig + 1 of the entry at outputs m0 + 8 i
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 8; ++i) {                                           // tile i / 4, upper or lower rows, column
                float v = acc[i >> 2][n][i & 3];
                v += __shfl_xor_sync(0xFFFFFFFFu, v, 2);
                const int r = n * 4 + tig * 2 + (i & 1), m = m0 + 8 * (i >> 1);
                if (tig < 2 && r < rows && m < p.M) {
                    const size_t at = static_cast<size_t>(e.row[en][r]) * p.M + m;
                    p.out[at] = __float2bfloat16_rn(__bfloat162float(p.y[at]) + v);
                }
            }
    };
    for (int item = blockIdx.x; item < items; item += gridDim.x) {
        if (e.rows[item / chunks] <= 4) work(item, MdTiles<1>{});
        else work(item, MdTiles<2>{});
    }
}

}  // namespace ade
