// Deltas of many fine-tuned models beside one shared projection:  out[t] = y[t] + U_d^ (V_d^^T x[t]),  d = ids[t].
//
// The deltas lie in a bank, rank group by rank group (128 ranks): delta d owns groups start[d] .. start[d + 1] - 1.
//   vt uint8 [G][128][N/2], vs bf16 [G][N], vz uint8 [G][N]     V^^T = vs (code - vz), packed along d_i
//   uq uint8 [G][M][64],    us bf16 [G][M], uz uint8 [G][M]     U^  = us (code - uz), packed along the rank axis
// Rows whose id is outside 0 .. deltas - 1 get y alone.
//
// Two launches, h = V^^T x and out = y + U^ h; the second is set up under the first.  Both find out on the device which rows share a
// delta (ids may change from replay to replay of a graph) and cut them into entries of up to eight rows, so that a delta's codes
// are read once for each entry, and from DRAM once.
//
// Both are streams of 4-bit codes against a handful of token columns, and what costs is the unpacking: integer instructions issue every other
// cycle.  As bytes, eight codes take three of them (two ANDs and a shift) for the warp matrix instruction m16n8k32 of 8-bit
// integers, which has twice the rate of m16n8k16; as bfloat16 pairs they take eleven (128 rows of 48 deltas, 11008 x 4096: 96.5 us
// then, 70 as bytes in the same layout).
// So the codes are the instruction's 16 rows, and the token rows enter in fixed point: x vs over 128 columns, or h over the 128 ranks of a
// group, scaled by a power of two to 16 bits, the upper eight in an even column, the lower eight in the odd one beside it (so one thread has both
// results of a token row, and four rows fill the eight columns).  An operand
// is thus held to 2^-16 to 2^-15 of the largest of its 128.  Products with the codes and their sums are exact integers; zero-points come off as integers
// in the first launch and in float32 in the second (scale times zero-point times the sum of h), and what is added across groups, columns and
// warps is float32.  Sixteen bits are the choice between the bytes of one column and of three: off by 4e-5 to 1.3e-4 of the delta's root mean square (4096 x
// 4096, 512 ranks, eight rows of normal x), by 5e-5 to 1.9e-4 with columns of x that are a hundred to a thousand times larger; the
// single-delta launch, with bfloat16 operands, is off by 3e-4 to 1.2e-3 there, the output's rounding by 1.7e-3.
// Every thread copies the 16-byte pieces of codes that it will use itself with cp.async into a queue of its own, so the
// stream runs through the barriers of an item and into the next one.  Sums have a fixed order; there are no floating-point atomics.
//
// Measured: 50.4 us for 128 rows of 48 deltas, 11008 x 4096 (178 MB, 3.5 TB/s): alone, 19 us for the first launch, which has a quarter of the bytes and is
// bound by bringing the activations to fixed point and by the latency of its short items, and 39 for the second; no pipe of either is above 40 %.
// 13.0 us for 16 rows of 12 deltas, 4096 x 4096, and 9.1 for 3 rows, 1000 x 2048: launches, and what depends on what in them.
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
constexpr int MD_PART = 132;                      // row pitch of the warps' partial h, in floats
constexpr int MD_HCOL = MD_MAX_GROUPS * 128 + 64; // bytes of a column of h in shared memory; 64 over a multiple of 128: no bank conflicts
constexpr int MD_TILE = 64;                       // rows of U that a warp takes at a time
constexpr int MD_UDEPTH = 2;                      // steps in the queue of the second launch
constexpr int MD_STAGE = 36;                      // row pitch of half a tile's results, in floats
constexpr int MD_SIDE = 224;                      // bytes of a step's scales (nine pieces) and zero-points (five)
constexpr float kMdMagic = 12582912.f;            // 1.5 * 2^23: what is added to it is rounded to an integer, in the lower bits of the sum

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
    alignas(16) int key[MD_MAX_ROWS];
    int first[MD_MAX_ROWS];                                       // first rank group
    int groups_end[MD_MAX_ROWS];                                  // rank groups of this entry and those before it
    int cost_end[MD_MAX_ROWS];                                    // md_u_cost, summed the same way
    uint8_t ng[MD_MAX_ROWS], rows[MD_MAX_ROWS];                   // rank groups and rows of the entry
    uint8_t row[MD_MAX_ROWS][MD_ENTRY], base[MD_MAX_ROWS];
    int wsum[8], wcost[8];
};

// What a tile of the second launch costs with an entry of so many rank groups and rows, in about 25 cycles of a warp.  128 rows of 48 deltas of 256 to 768
// ranks, 11008 x 4096, calls back to back in a graph: 47.7 us; 50.3 if entries of more than four rows cost the same as the others, 56.4 with one cost for all; 47.8 with 14 instead of 11.
// 128 rows of 24 deltas, 4096 x 4096: 25.1, 25.4, 26.5, 25.3; 40 rows of 30, 4096 x 11008: 30.2, 30.8, 30.8, 30.1; 64 rows of 8, or all of one delta: the same.
__device__ __forceinline__ int md_u_cost(int ng, int rows) { return ng == 0 ? 10 : rows <= 4 ? ng * 8 + 7 : ng * 11 + 6; }

constexpr size_t md_v_smem() { return 8 * 2 * MD_THREADS * 16 + 8 * MD_ENTRY * MD_PART * sizeof(float) + 8 * 384; }
constexpr size_t md_u_smem() { return MD_UDEPTH * 8 * MD_THREADS * 16 + 16 * MD_HCOL + MD_MAX_GROUPS * MD_ENTRY * sizeof(float2) + 8 * (4 * MD_STAGE * sizeof(float) + MD_UDEPTH * MD_SIDE); }
inline int md_slices(int N) { return (N + MD_COLS - 1) / MD_COLS; }

__device__ __forceinline__ void md_cp16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// the first `bytes` of 16, zeros behind them
__device__ __forceinline__ void md_cp16_part(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
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
// D(16x8, s32) = A(16x32, u8, row) * B(32x8, s8, col) + C
__device__ __forceinline__ void md_mma(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, const int (&c)[4]) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]));
}
// The product of a packed word of two rows (eight codes each, as bytes 0 4 1 5 and 2 6 3 7) with those of a column, added to d.
__device__ __forceinline__ void md_mma_word(int (&d)[4], uint32_t w0, uint32_t w1, uint32_t b0, uint32_t b1, const int (&c)[4]) {
    md_mma(d, w0 & 0x0F0F0F0Fu, w1 & 0x0F0F0F0Fu, w0 >> 4 & 0x0F0F0F0Fu, w1 >> 4 & 0x0F0F0F0Fu, b0, b1, c);
}
__device__ __forceinline__ float md_max(float a, float b) {              // NaN if either is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// What the sums of upper and lower bytes come to: their integer is exact, below 2^26, and rounded once.
__device__ __forceinline__ float md_join(int up, int lo, float unit) { return static_cast<float>(up * 256 + lo) * unit; }
// Fixed point for values of magnitude up to m: v * scale is at most 32637, so its upper and lower eight bits are signed bytes; `unit` = 1 / scale, a
// power of two (infinite or NaN where m is, so that results show it).
struct MdFixed {
    float scale, unit;
};
__device__ __forceinline__ MdFixed md_fixed(float m) {
    const int e = max(static_cast<int>(__float_as_uint(m * 1.004f) >> 23 & 255u), 27);
    return {__uint_as_float(static_cast<uint32_t>(268 - e) << 23), e == 255 ? m : __uint_as_float(static_cast<uint32_t>(e - 14) << 23)};
}

__device__ __forceinline__ void md_entries(const MultiDeltaParams& p, MdEntries& e) {
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    // the table of first rank groups is fetched beside the ids where it is short enough to keep (cost_end is free until the end)
    const bool kept = p.deltas < MD_MAX_ROWS;
    if (kept && t <= p.deltas) e.cost_end[t] = p.start[t];
    const int d = t < p.T ? p.ids[t] : -1;
    if (kept) __syncthreads();
    int first = 0, ng = 0;
    if (d >= 0 && d < p.deltas) {
        first = max(kept ? e.cost_end[d] : p.start[d], 0);
        ng = max(0, min(min(kept ? e.cost_end[d + 1] : p.start[d + 1], p.G) - first, MD_MAX_GROUPS));
    }
    if (t < MD_MAX_ROWS) e.key[t] = t >= p.T ? -2 : ng ? d : -1;     // rows without a delta share an entry of no groups
    __syncthreads();
    int before = 0, same = 0, leader = t;
    if (t < p.T) {
        const int mine = e.key[t];
#pragma unroll 4
        for (int u = (p.T - 1) & ~3; u >= 0; u -= 4) {
            const int4 k = *reinterpret_cast<const int4*>(&e.key[u]);
            const int is[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
            for (int i = 3; i >= 0; --i)
                if (is[i] == mine) {
                    ++same;
                    before += u + i < t;
                    leader = u + i;
                }
        }
    }
    // entries, rank groups and cost of each group of rows, at its first row, summed over the rows
    const int mine = t < p.T && leader == t ? (same + MD_ENTRY - 1) / MD_ENTRY : 0;
    const int full = md_u_cost(ng, MD_ENTRY), my_cost = mine ? (mine - 1) * full + md_u_cost(ng, same - (mine - 1) * MD_ENTRY) : 0;
    int run = mine << 16 | mine * ng, cost = my_cost;       // at most 128 entries, 128 * 16 rank groups
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xFFFFFFFFu, run, o), v = __shfl_up_sync(0xFFFFFFFFu, cost, o);
        if (lane >= o) {
            run += u;
            cost += v;
        }
    }
    if (lane == 31) {
        e.wsum[warp] = run;
        e.wcost[warp] = cost;
    }
    __syncthreads();
    run -= mine << 16 | mine * ng;
    cost -= my_cost;
#pragma unroll
    for (int w = 0; w < MD_MAX_ROWS / 32; ++w)
        if (w < warp) {
            run += e.wsum[w];
            cost += e.wcost[w];
        }
    if (t < p.T) e.base[t] = static_cast<uint8_t>(run >> 16);
    if (t == MD_MAX_ROWS) e.n = run >> 16;
    for (int k = 0; k < mine; ++k) {
        const int i = (run >> 16) + k, rows = min(MD_ENTRY, same - k * MD_ENTRY);
        cost += md_u_cost(ng, rows);
        e.first[i] = first;
        e.ng[i] = static_cast<uint8_t>(ng);
        e.rows[i] = static_cast<uint8_t>(rows);
        e.groups_end[i] = (run & 0xFFFF) + (k + 1) * ng;
        e.cost_end[i] = cost;
    }
    __syncthreads();
    if (t < p.T) e.row[e.base[leader] + before / MD_ENTRY][before % MD_ENTRY] = static_cast<uint8_t>(t);
    __syncthreads();
}

// where the share of block b of n things begins
__device__ __forceinline__ int md_share(int n, int b) {
    const int each = n / static_cast<int>(gridDim.x), more = n - each * static_cast<int>(gridDim.x);
    return each * b + min(b, more);
}

// How many of the ascending sums, times `by`, do not exceed `value`; by the whole warp.
__device__ __forceinline__ int md_count(const int* sums, int n, int by, int value) {
    int c = 0;
#pragma unroll
    for (int i = 0; i < MD_MAX_ROWS; i += 32) {
        const int k = i + static_cast<int>(threadIdx.x & 31);
        c += k < n && sums[k] * by <= value;
    }
    return __reduce_add_sync(0xFFFFFFFFu, c);
}

// ------------------------------------------------------------------ h = V^T x
// An item is one rank group of one entry over MD_COLS columns: a warp multiplies the group's 128 ranks with 128 columns, eight tiles of 16
// ranks one behind the other, and the warps' sums are added through shared memory.  Items go entry by entry, slice by slice, group by group, and a
// CTA has a run of them.  The codes, scales and zero-points of an item are under way while the item before it is computed.
struct MdVItem {
    int e, slice, j;                       // entry, slice of columns, rank group of the entry
};

__device__ __forceinline__ MdVItem md_v_item(const MdEntries& e, int item, int slices) {
    const int lo = md_count(e.groups_end, e.n, slices, item);             // the entry with groups_end * slices > item
    const int rest = item - (e.groups_end[lo] - e.ng[lo]) * slices;
    return {lo, rest / e.ng[lo], rest % e.ng[lo]};
}

// The copies of one item: a warp's scales and zero-points, then the tiles of codes, each thread its own pieces.
struct MdVCopy {
    const uint8_t *codes, *scale;          // nullptr where there is nothing to copy
    uint32_t fifo, side;                   // this thread's place in the queue; the warp's scales (256 bytes) and zero-points (128)
    size_t pitch;                          // bytes of a row of codes
    const uint8_t* zero;

    __device__ __forceinline__ void sides(int lane) const {
        if (codes) {
            if (lane < 16) md_cp16(side + lane * 16, scale + lane * 16);
            else if (lane < 24) md_cp16(side + lane * 16, zero + (lane - 16) * 16);
        }
        md_commit();
    }
    __device__ __forceinline__ void tile(int mt) const {
        if (codes) {
            md_cp16(fifo + (mt * 2) * MD_THREADS * 16, codes + static_cast<size_t>(mt * 16) * pitch);
            md_cp16(fifo + (mt * 2 + 1) * MD_THREADS * 16, codes + static_cast<size_t>(mt * 16 + 8) * pitch);
        }
        md_commit();
    }
};

// x of the entry's rows gid / 2 and gid / 2 + 4 at this lane's 32 columns, asked for an item ahead
__device__ __forceinline__ void md_v_x(const MultiDeltaParams& p, const MdEntries& e, const MdVItem& it, int cb, uint4 (&xv)[2][4]) {
    const int lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        const int r = n * 4 + (gid >> 1);
        const bool on = r < e.rows[it.e];
        const uint4* xp = reinterpret_cast<const uint4*>(p.x + static_cast<size_t>(e.row[it.e][on ? r : 0]) * p.N + cb * 128 + tig * 32);
#pragma unroll
        for (int i = 0; i < 4; ++i) xv[n][i] = on ? ldg16(xp + i) : make_uint4(0u, 0u, 0u, 0u);
    }
}

template <int NT>
__device__ __forceinline__ void md_v_compute(const uint4 (&xv)[2][4], float* part, const MdVCopy& next) {
    const int lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
    md_wait<8>();                                                     // the scales and zero-points are there; the tiles may be under way
    __syncwarp();
    uint32_t z[8];                                                    // zero-points in the order of the codes' bytes
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint4 v = lds16(next.side + 256 + (tig * 2 + i) * 16);
        z[i * 4] = __byte_perm(v.x, v.y, 0x5140);
        z[i * 4 + 1] = __byte_perm(v.x, v.y, 0x7362);
        z[i * 4 + 2] = __byte_perm(v.z, v.w, 0x5140);
        z[i * 4 + 3] = __byte_perm(v.z, v.w, 0x7362);
    }
    // x vs of row gid / 2 at this lane's 32 columns: the largest of the row's 128, then the upper (gid even) or lower bytes of the fixed-point values
    uint32_t xs[NT][8];
    float weight[NT];                                                 // what an integer of lower bytes counts for row tig
    int base[NT][4];                                                  // what the sums begin with: the zero-points' part off
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint4 sv = lds16(next.side + (tig * 4 + i) * 16);
            const uint32_t sw[4] = {sv.x, sv.y, sv.z, sv.w}, xw[4] = {xv[n][i].x, xv[n][i].y, xv[n][i].z, xv[n][i].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) m = md_max(m, md_max(fabsf(md_lo(xw[k]) * md_lo(sw[k])), fabsf(md_hi(xw[k]) * md_hi(sw[k]))));
        }
        m = md_max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
        m = md_max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
        const MdFixed fx = md_fixed(m);
        const float add = gid & 1 ? kMdMagic : kMdMagic + 128.f;        // the upper byte is the one of v + 128
        const uint32_t pick = gid & 1 ? 0x40u : 0x51u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint4 sv = lds16(next.side + (tig * 4 + i) * 16);
            const uint32_t sw[4] = {sv.x, sv.y, sv.z, sv.w}, xw[4] = {xv[n][i].x, xv[n][i].y, xv[n][i].z, xv[n][i].w};
            uint32_t q[8];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                q[2 * k] = __float_as_uint(fmaf(md_lo(xw[k]) * md_lo(sw[k]), fx.scale, add));
                q[2 * k + 1] = __float_as_uint(fmaf(md_hi(xw[k]) * md_hi(sw[k]), fx.scale, add));
            }
#pragma unroll
            for (int k = 0; k < 2; ++k)
                xs[n][i * 2 + k] = __byte_perm(__byte_perm(q[2 * k], q[2 * k + 4], pick), __byte_perm(q[2 * k + 1], q[2 * k + 5], pick), 0x5410);
        }
        weight[n] = __shfl_sync(0xFFFFFFFFu, fx.unit, tig * 8);
        int zero[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) md_mma(zero, z[2 * i], z[2 * i], z[2 * i + 1], z[2 * i + 1], xs[n][2 * i], xs[n][2 * i + 1], zero);
#pragma unroll
        for (int i = 0; i < 4; ++i) base[n][i] = -zero[i];
    }
    __syncwarp();                                                     // every lane has read the scales and zero-points
    next.sides(lane);
    constexpr int PAIR = 2 / NT;                                      // tiles of 16 ranks at a time: two chains of products in flight
#pragma unroll
    for (int m0 = 0; m0 < 8; m0 += PAIR) {
        md_wait<8 - (PAIR - 1)>();
        uint4 r0[PAIR], r1[PAIR];
#pragma unroll
        for (int k = 0; k < PAIR; ++k) {
            r0[k] = lds16(next.fifo + ((m0 + k) * 2) * MD_THREADS * 16);
            r1[k] = lds16(next.fifo + ((m0 + k) * 2 + 1) * MD_THREADS * 16);
        }
        int d[PAIR][NT][4];
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int k = 0; k < PAIR; ++k) {
                const uint32_t w0 = w == 0 ? r0[k].x : w == 1 ? r0[k].y : w == 2 ? r0[k].z : r0[k].w;
                const uint32_t w1 = w == 0 ? r1[k].x : w == 1 ? r1[k].y : w == 2 ? r1[k].z : r1[k].w;
#pragma unroll
                for (int n = 0; n < NT; ++n) md_mma_word(d[k][n], w0, w1, xs[n][2 * w], xs[n][2 * w + 1], w == 0 ? base[n] : d[k][n]);
            }
#pragma unroll
        for (int k = 0; k < PAIR; ++k) next.tile(m0 + k);             // into the pieces just used
#pragma unroll
        for (int k = 0; k < PAIR; ++k)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    part[(n * 4 + tig) * MD_PART + (m0 + k) * 16 + gid + i * 8] = md_join(d[k][n][2 * i], d[k][n][2 * i + 1], weight[n]);
    }
}

__global__ void __launch_bounds__(MD_THREADS, 2) multi_delta_v_kernel(const MultiDeltaParams p, int slices) {
    extern __shared__ __align__(16) uint8_t md_smem[];
    __shared__ MdEntries e;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gid = lane >> 2, tig = lane & 3;
    float* part = reinterpret_cast<float*>(md_smem + 8 * 2 * MD_THREADS * 16);
    const uint32_t side = smem_u32(md_smem) + 8 * 2 * MD_THREADS * 16 + 8 * MD_ENTRY * MD_PART * 4 + warp * 384;
    md_entries(p, e);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int blocks = p.N / 128, items = (e.n ? e.groups_end[e.n - 1] : 0) * slices;
    int item = md_share(items, blockIdx.x);
    const int end = md_share(items, blockIdx.x + 1);
    if (item >= end) return;
    auto copy = [&](const MdVItem& it, bool on) {
        MdVCopy c = {nullptr, nullptr, smem_u32(md_smem) + tid * 16, side, static_cast<size_t>(p.N / 2), nullptr};
        const int cb = it.slice * (MD_COLS / 128) + warp;
        if (on && cb < blocks) {
            const size_t g = e.first[it.e] + it.j;
            c.codes = p.vt + (g * 128 + gid) * c.pitch + cb * 64 + tig * 16;
            c.scale = reinterpret_cast<const uint8_t*>(p.vs + g * p.N + cb * 128);
            c.zero = p.vz + g * p.N + cb * 128;
        }
        return c;
    };
    MdVItem it = md_v_item(e, item, slices);
    uint4 xv[2][4];
    {
        const MdVCopy c = copy(it, true);
        c.sides(lane);
#pragma unroll
        for (int mt = 0; mt < 8; ++mt) c.tile(mt);
        if (c.codes) md_v_x(p, e, it, it.slice * (MD_COLS / 128) + warp, xv);
    }
    while (true) {
        MdVItem nx = it;
        if (++nx.j == e.ng[nx.e]) {
            nx.j = 0;
            if (++nx.slice == slices) {
                nx.slice = 0;
                do {
                    ++nx.e;
                } while (nx.e < e.n && e.ng[nx.e] == 0);
            }
        }
        const bool go_on = ++item < end;
        const MdVCopy next = copy(nx, go_on);
        const int cb = it.slice * (MD_COLS / 128) + warp, rows = e.rows[it.e];
        if (cb < blocks) {
            float* mine = part + warp * (MD_ENTRY * MD_PART);
            if (rows <= 4) md_v_compute<1>(xv, mine, next);
            else md_v_compute<2>(xv, mine, next);
        } else {
            next.sides(lane);
#pragma unroll
            for (int mt = 0; mt < 8; ++mt) next.tile(mt);
        }
        if (next.codes) md_v_x(p, e, nx, nx.slice * (MD_COLS / 128) + warp, xv);
        __syncthreads();
        const int warps = min(8, blocks - it.slice * (MD_COLS / 128));
        for (int i = tid; i < rows * 128; i += MD_THREADS) {
            const int r = i >> 7, k = i & 127;
            float s = 0.f;
#pragma unroll
            for (int w = 0; w < 8; ++w) s += w < warps ? part[(w * MD_ENTRY + r) * MD_PART + k] : 0.f;
            p.h[(static_cast<size_t>(it.slice) * p.T + e.row[it.e][r]) * MD_H + it.j * 128 + k] = s;
        }
        if (!go_on) return;
        __syncthreads();
        it = nx;
    }
}

// ------------------------------------------------------------------ out = y + U h
// A tile is MD_TILE rows of one entry's U: a warp multiplies them, 16 at a time, with the entry's columns of h, a rank group at a step,
// and adds us (sum - uz sum h) to its float32 results.  `us`, `usz`: scale, and scale times zero-point, of rows `lane` and lane + 32 of
// the tile; `hsum`: for each rank group and row of the entry what an integer of lower bytes counts, and the sum of h.
template <int N>
struct MdTiles {
    static constexpr int value = N;
};

template <int NT, typename Refill>
__device__ __forceinline__ void md_u_step(uint32_t codes, const uint8_t* hcol, const float2* hsum, int j, const float (&us)[2], const float (&usz)[2],
                                          float (&acc)[NT][8], Refill refill) {
    const int lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
    int base[4] = {0, 0, 0, 0};
    uint4 b[NT][2];
    float2 s[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        s[n] = hsum[j * 8 + n * 4 + tig];
#pragma unroll
        for (int h = 0; h < 2; ++h) b[n][h] = *reinterpret_cast<const uint4*>(hcol + (n * 8 + gid) * MD_HCOL + j * 128 + (h * 4 + tig) * 16);
    }
    constexpr int PAIR = 2 / NT;                                        // blocks of 16 rows at a time: two chains of products in flight
#pragma unroll
    for (int m0 = 0; m0 < 4; m0 += PAIR) {
        uint4 q0[PAIR], q1[PAIR];
#pragma unroll
        for (int k = 0; k < PAIR; ++k) {
            q0[k] = lds16(codes + ((m0 + k) * 2) * MD_THREADS * 16);
            q1[k] = lds16(codes + ((m0 + k) * 2 + 1) * MD_THREADS * 16);
        }
        int d[PAIR][NT][4];
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int k = 0; k < PAIR; ++k) {
                const uint32_t w0 = w == 0 ? q0[k].x : w == 1 ? q0[k].y : w == 2 ? q0[k].z : q0[k].w;
                const uint32_t w1 = w == 0 ? q1[k].x : w == 1 ? q1[k].y : w == 2 ? q1[k].z : q1[k].w;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const uint4& c = b[n][w >> 1];
                    md_mma_word(d[k][n], w0, w1, w & 1 ? c.z : c.x, w & 1 ? c.w : c.y, w == 0 ? base : d[k][n]);
                }
            }
#pragma unroll
        for (int k = 0; k < PAIR; ++k) refill(m0 + k);
#pragma unroll
        for (int k = 0; k < PAIR; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i) {                               // rows gid + 8 (2 m + i) of the tile
                const int m = m0 + k, from = gid + 8 * (m * 2 + i & 3);
                const float f = __shfl_sync(0xFFFFFFFFu, us[m >> 1], from), z = __shfl_sync(0xFFFFFFFFu, usz[m >> 1], from);
#pragma unroll
                for (int n = 0; n < NT; ++n) acc[n][m * 2 + i] += f * md_join(d[k][n][i * 2], d[k][n][i * 2 + 1], s[n].x) - z * s[n].y;
            }
    }
}

// Tiles go entry by entry, and a CTA has a run of them that costs about what the others' runs cost; h of an entry is brought into shared
// memory once for the tiles of a run, which the warps take in turn.
__global__ void __launch_bounds__(MD_THREADS, 2) multi_delta_u_kernel(const MultiDeltaParams p, int slices) {
    extern __shared__ __align__(16) uint8_t md_smem[];
    __shared__ MdEntries e;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gid = lane >> 2, tig = lane & 3;
    const uint32_t fifo = smem_u32(md_smem) + tid * 16;
    uint8_t* hcol = md_smem + MD_UDEPTH * 8 * MD_THREADS * 16;                   // [16 columns][MD_HCOL]
    float2* hsum = reinterpret_cast<float2*>(hcol + 16 * MD_HCOL);               // [MD_MAX_GROUPS][MD_ENTRY]
    uint8_t* own = reinterpret_cast<uint8_t*>(hsum + MD_MAX_GROUPS * MD_ENTRY) + warp * (4 * MD_STAGE * sizeof(float) + MD_UDEPTH * MD_SIDE);
    float* stage = reinterpret_cast<float*>(own);                                // [4][MD_STAGE] results of the warp's tile, four rows and 32 outputs at a time
    const uint8_t* side = own + 4 * MD_STAGE * sizeof(float);                    // scales and zero-points of the steps in the queue
    // Of a step's scales (and zero-points) the aligned pieces of 16 bytes that hold them are copied, nine and five, a piece per lane.
    const bool is_scale = lane < 9;
    const uint8_t* side_base = is_scale ? reinterpret_cast<const uint8_t*>(p.us) : p.uz;
    const int side_log = is_scale ? 1 : 0, side_piece = is_scale ? lane : lane - 9;
    const size_t side_size = (static_cast<size_t>(p.G) * p.M) << side_log;
    md_entries(p, e);
    const int tiles = (p.M + MD_TILE - 1) / MD_TILE;
    struct Place {
        int en, tile;
    };
    // first tile that begins at or behind `cost`
    auto place = [&](int cost) {
        const int lo = md_count(e.cost_end, e.n, tiles, cost);                   // the entry that ends behind `cost`
        if (lo == e.n) return Place{lo, 0};
        const int before = lo ? e.cost_end[lo - 1] : 0, per = e.cost_end[lo] - before, tile = (cost - before * tiles + per - 1) / per;
        return tile < tiles ? Place{lo, tile} : Place{lo + 1, 0};
    };
    const int all = e.cost_end[e.n - 1] * tiles;
    const Place first = place(md_share(all, blockIdx.x)), last = place(md_share(all, blockIdx.x + 1));
    if (first.en == last.en && first.tile == last.tile) return;
    auto tile_end = [&](int en) { return en < last.en ? tiles : en == last.en ? last.tile : 0; };
    // the warp's stream of codes: 16 rows of a step make room for 16 rows of the step MD_UDEPTH behind it as soon as they have been used
    const size_t pitch = static_cast<size_t>(p.M) * 64;
    // The warps take the tiles of the run in turn.  Entries without rank groups have tiles too (y alone), but no steps.
    auto settle = [&](Place& at) {                                               // from a place that may lie behind its entry's tiles
        while (at.en < e.n && at.tile >= tile_end(at.en)) {
            if (at.en >= last.en) at.en = e.n;                                   // the run ends here
            else at.tile -= tile_end(at.en++);
        }
    };
    Place ahead = {first.en, first.tile + warp};
    int left = 0;                                                                // steps of the tile ahead
    const uint8_t* src = nullptr;
    uint32_t side_at = 0;                                                        // place of the tile's first scale (the codes of 2^32 rows would not fit a device)
    const uint32_t side_dst = smem_u32(side) + lane * 16;
    auto aim = [&] {                                                             // at the warp's next tile with rank groups
        settle(ahead);
        while (ahead.en < e.n && e.ng[ahead.en] == 0) {
            ahead.tile += MD_THREADS / 32;
            settle(ahead);
        }
        if (ahead.en < e.n) {
            left = e.ng[ahead.en];
            src = p.uq + e.first[ahead.en] * pitch + static_cast<size_t>(ahead.tile * MD_TILE + gid) * 64 + tig * 16;
            side_at = static_cast<uint32_t>(e.first[ahead.en]) * p.M + ahead.tile * MD_TILE;
        }
    };
    // rows 16 m .. 16 m + 15 of the step ahead
    auto piece = [&](int slot, int m) {
        if (!left) return;
        const uint32_t dst = fifo + slot * (8 * MD_THREADS * 16) + m * (2 * MD_THREADS * 16);
        const int row = ahead.tile * MD_TILE + gid + 16 * m;
        if (row < p.M) md_cp16(dst, src + m * 16 * 64);
        if (row + 8 < p.M) md_cp16(dst + MD_THREADS * 16, src + m * 16 * 64 + 8 * 64);
    };
    auto rest = [&](int slot) {                                                  // its scales and zero-points; on to the next
        if (left) {
            if (lane < 14) {
                const size_t from = (static_cast<size_t>(side_at) << side_log & ~static_cast<size_t>(15)) + side_piece * 16;
                if (from + 16 <= side_size) md_cp16(side_dst + slot * MD_SIDE, side_base + from);
                else if (from < side_size) md_cp16_part(side_dst + slot * MD_SIDE, side_base + from, static_cast<int>(side_size - from));
            }
            src += pitch;
            side_at += p.M;
            if (--left == 0) {
                ahead.tile += MD_THREADS / 32;
                aim();
            }
        }
        md_commit();
    };
    aim();
#pragma unroll
    for (int s = 0; s < MD_UDEPTH; ++s) {
#pragma unroll
        for (int m = 0; m < 4; ++m) piece(s, m);
        rest(s);
    }
    int slot = 0;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // the columns of h of some entries, from rank group `at` in shared memory on: two (row, rank group) per warp and round, side by side since each is a
    // chain of waits, four ranks per lane; the slices' sums in fixed point, bytes in the order of the codes' (0 4 1 5 and 2 6 3 7 of eight, which two
    // lanes share).  Magnitudes are compared as integers: NaN lies behind infinity.
    auto bring = [&](int en, int at) {
        constexpr int W = MD_THREADS / 32;
        const int ng = e.ng[en], n = e.rows[en] * ng;
        for (int i0 = warp; i0 < n; i0 += 2 * W) {
            const int i[2] = {i0, i0 + W < n ? i0 + W : i0};                     // the last one twice where the number is odd
            int r[2], j[2];
            float v[2][4] = {};
            const float* from[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                r[k] = i[k] / ng;
                j[k] = i[k] - r[k] * ng;
                from[k] = p.h + static_cast<size_t>(e.row[en][r[k]]) * MD_H + j[k] * 128 + lane * 4;
            }
#pragma unroll 4
            for (int s = 0; s < slices; ++s)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const float4 a = *reinterpret_cast<const float4*>(from[k] + static_cast<size_t>(s) * p.T * MD_H);
                    v[k][0] += a.x;
                    v[k][1] += a.y;
                    v[k][2] += a.z;
                    v[k][3] += a.w;
                }
            uint32_t m[2], up[2], lo[2], up2[2], lo2[2];
            MdFixed fx[2];
            int su[2], sl[2];
#pragma unroll
            for (int k = 0; k < 2; ++k)
                m[k] = max(max(__float_as_uint(v[k][0]) & 0x7FFFFFFFu, __float_as_uint(v[k][1]) & 0x7FFFFFFFu),
                           max(__float_as_uint(v[k][2]) & 0x7FFFFFFFu, __float_as_uint(v[k][3]) & 0x7FFFFFFFu));
#pragma unroll
            for (int k = 0; k < 2; ++k) m[k] = __reduce_max_sync(0xFFFFFFFFu, m[k]);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                fx[k] = md_fixed(__uint_as_float(m[k]));
                uint32_t q[4], q8[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    q[x] = __float_as_uint(fmaf(v[k][x], fx[k].scale, kMdMagic));
                    q8[x] = q[x] + 128u;                                         // the upper byte is the one of v + 128
                }
                up[k] = __byte_perm(__byte_perm(q8[0], q8[1], 0x51), __byte_perm(q8[2], q8[3], 0x51), 0x5410);
                lo[k] = __byte_perm(__byte_perm(q[0], q[1], 0x40), __byte_perm(q[2], q[3], 0x40), 0x5410);
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                up2[k] = __shfl_xor_sync(0xFFFFFFFFu, up[k], 1);
                lo2[k] = __shfl_xor_sync(0xFFFFFFFFu, lo[k], 1);
                su[k] = __reduce_add_sync(0xFFFFFFFFu, __dp4a(static_cast<int>(up[k]), 0x01010101, 0));
                sl[k] = __reduce_add_sync(0xFFFFFFFFu, __dp4a(static_cast<int>(lo[k]), 0x01010101, 0));
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int c = r[k] * 2;                                          // column of the upper bytes; the lower stand behind it
                uint8_t* to = hcol + c * MD_HCOL + (at + j[k]) * 128 + (lane >> 2 & 1) * 64 + (lane >> 3) * 16 + (lane >> 1 & 1) * 8 + (lane & 1) * 4;
                *reinterpret_cast<uint32_t*>(to) = lane & 1 ? __byte_perm(up2[k], up[k], 0x7362) : __byte_perm(up[k], up2[k], 0x5140);
                *reinterpret_cast<uint32_t*>(to + MD_HCOL) = lane & 1 ? __byte_perm(lo2[k], lo[k], 0x7362) : __byte_perm(lo[k], lo2[k], 0x5140);
                if (lane == 0) hsum[(at + j[k]) * 8 + r[k]] = make_float2(fx[k].unit, fx[k].unit * (256.f * su[k] + sl[k]));
            }
        }
    };
    const bool vec = (p.M & 3) == 0;                                             // four outputs are an aligned piece of 8 bytes
    auto work = [&](int en, int tile, int h_at, auto nt) {
        constexpr int NT = decltype(nt)::value;                                  // tiles of eight columns: two parts of four rows each
        const int ng = e.ng[en], rows = e.rows[en], m0 = tile * MD_TILE;
        // y of row n * 4 + lane / 8 at outputs m0 + 32 k + lane % 8 * 4 + 0 .. 3, before anything is waited for
        const int mo = m0 + (lane & 7) * 4;
        uint2 y[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int r = n * 4 + (lane >> 3);
            const __nv_bfloat16* yp = p.y + static_cast<size_t>(e.row[en][r < rows ? r : 0]) * p.M + mo;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                y[n][k] = make_uint2(0u, 0u);
                if (r < rows && mo + 32 * k < p.M) {
                    if (vec) {
                        y[n][k] = *reinterpret_cast<const uint2*>(yp + 32 * k);
                    } else {
                        uint32_t v[4] = {};
                        for (int i = 0; i < 4; ++i)
                            if (mo + 32 * k + i < p.M) v[i] = __bfloat16_as_ushort(yp[32 * k + i]);
                        y[n][k] = make_uint2(v[0] | v[1] << 16, v[2] | v[3] << 16);
                    }
                }
            }
        }
        uint32_t at = static_cast<uint32_t>(e.first[en]) * p.M + m0;              // place of the step's first scale
        float acc[NT][8] = {};
        for (int j = 0; j < ng; ++j) {
            md_wait<MD_UDEPTH - 1>();
            __syncwarp();
            const uint8_t* sz = side + slot * MD_SIDE;
            float us[2], usz[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                us[k] = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(sz + (at * 2 & 15) + (lane + 32 * k) * 2));
                usz[k] = us[k] * sz[144 + (at & 15) + lane + 32 * k];
            }
            at += p.M;
            __syncwarp();                                                        // every lane has read the scales and zero-points
            md_u_step<NT>(fifo + slot * (8 * MD_THREADS * 16), hcol, hsum, h_at + j, us, usz, acc, [&](int m) { piece(slot, m); });
            rest(slot);
            slot ^= 1;
        }
        // lane (gid, tig) has row n * 4 + tig of the entry at outputs gid + 8 i, which go through shared memory into the order in which they are stored
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int r = n * 4 + (lane >> 3);
            __nv_bfloat16* o = p.out + static_cast<size_t>(e.row[en][r < rows ? r : 0]) * p.M + mo;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
#pragma unroll
                for (int i = 0; i < 4; ++i) stage[tig * MD_STAGE + gid + 8 * i] = acc[n][4 * k + i];
                __syncwarp();
                const float4 v = *reinterpret_cast<const float4*>(stage + (lane >> 3) * MD_STAGE + (lane & 7) * 4);
                __syncwarp();
                if (r < rows && mo + 32 * k < p.M) {
                    const uint2 w = make_uint2(md_pack(md_lo(y[n][k].x) + v.x, md_hi(y[n][k].x) + v.y), md_pack(md_lo(y[n][k].y) + v.z, md_hi(y[n][k].y) + v.w));
                    if (vec) {
                        *reinterpret_cast<uint2*>(o + 32 * k) = w;
                    } else {
                        const uint32_t b[4] = {w.x & 0xFFFFu, w.x >> 16, w.y & 0xFFFFu, w.y >> 16};
                        for (int i = 0; i < 4; ++i)
                            if (mo + 32 * k + i < p.M) o[32 * k + i] = __ushort_as_bfloat16(static_cast<unsigned short>(b[i]));
                    }
                }
            }
        }
    };
    // entries by the batch: as many as have room for their rank groups in shared memory
    Place at = {first.en, first.tile + warp};
    for (int b0 = first.en; b0 < e.n && tile_end(b0) > 0;) {
        const int g0 = e.groups_end[b0] - e.ng[b0];
        int b1 = b0;
        __syncthreads();                                                         // nobody reads the columns in place any more
        for (; b1 < e.n && tile_end(b1) > 0 && e.groups_end[b1] - g0 <= MD_MAX_GROUPS; ++b1) bring(b1, e.groups_end[b1] - e.ng[b1] - g0);
        __syncthreads();
        for (settle(at); at.en < b1; settle(at)) {
            const int h_at = e.groups_end[at.en] - e.ng[at.en] - g0;
            if (e.rows[at.en] <= 4) work(at.en, at.tile, h_at, MdTiles<1>{});
            else work(at.en, at.tile, h_at, MdTiles<2>{});
            at.tile += MD_THREADS / 32;
        }
        b0 = b1;
    }
}

}  // namespace ade
