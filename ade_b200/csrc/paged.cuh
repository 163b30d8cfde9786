// Paged key-value cache: page allocation and slot maps, the write of new keys and values (paged_attn.cuh reads them).
//
// A cache layer is two arrays k_pages, v_pages [pages][kv_heads][page_size][head_dim] of bfloat16.  A request owns an
// ordered list of pages, its row of block_table [B][width]; token i of the request lives in page block_table[b][i / page_size]
// at offset i % page_size, and slot = page * page_size + offset names that place for all layers.  No counterpart in the reference,
// which keeps one contiguous cache per batch inside transformers (src/evaluate.py:241 calls model.generate).
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "ptx.cuh"

namespace ade {

__device__ __forceinline__ float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
__device__ __forceinline__ uint32_t pack_bf2(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// ------------------------------------------------------------------ page allocation, block tables, slot maps
struct ExtendParams {
    const int* lengths;          // [B] tokens each request has
    const int* fresh;            // [B] tokens to add; negative: the request ends and its pages go back
    int* table;                  // [B][width], rows table_stride apart
    int* free_pages;             // [pages] stack of free pages
    const int* free_count;       // its height
    int *lengths_out, *count_out, *status;
    long long *slots, *positions;    // [total]
    int* requests;                   // [total]
    int* work;                       // [4 + 4 B] scalars and sums, from the first launch of two to the second
    int B, width, pages, page_size, total;
    long long table_stride;
};

enum { PX_OK = 0, PX_NO_PAGE = 1, PX_TABLE_FULL = 2, PX_NO_ROW = 3, PX_BAD_LENGTH = 4 };

// pages of n tokens; n + page_size may pass 31 bits
__device__ __forceinline__ int px_pages(int n, int page_size) { return static_cast<int>((static_cast<uint32_t>(n) + page_size - 1u) / page_size); }

// What the requests come to, in shared memory: inclusive sums over the requests of the rows of the packed batch, the pages handed back and
// the pages taken, and each request's old length (-1: it has no rows).
struct PxSums {
    int *row_end, *back_end, *need_end, *len;
    int count, available, used;          // height of the stack before, with the pages handed back, and pages taken from it
};
inline size_t px_smem_bytes(int B) { return 4 * static_cast<size_t>(B) * sizeof(int); }

// smallest b with sums[b] > i, for ascending sums
__device__ __forceinline__ int px_find(const int* sums, int n, int i) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (sums[mid] > i) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

// Inclusive prefix sums over a CTA of NT threads; `ws`: a word per warp that nothing else uses.
template <int NT>
__device__ __forceinline__ long long px_scan(long long v, long long* ws) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xFFFFFFFFu, v, o);
        if (lane >= o) v += u;
    }
    if (lane == 31) ws[warp] = v;
    __syncthreads();
    long long base = lane < warp ? ws[lane] : 0;                 // at most 32 warps
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) base += __shfl_xor_sync(0xFFFFFFFFu, base, o);
    return v + base;
}

// The sums, the new lengths and the states, by one CTA.  Sums are kept in 64 bits until they are compared with `total` and the number
// of pages, and saturated to 31 bits behind that.  Every thread has read lengths and free_count before any writes them: the outputs may be
// the same arrays.
template <int NT, int ITEMS>
__device__ __forceinline__ PxSums px_sum(const ExtendParams& p, int* smem) {
    __shared__ long long ws[3][NT / 32];
    __shared__ int s_used, s_back;
    PxSums r = {smem, smem + p.B, smem + 2 * p.B, smem + 3 * p.B, 0, 0, 0};
    const int tid = threadIdx.x, b0 = tid * ITEMS;
    const long long kSat = 0x7FFFFFFF;
    if (tid == 0) s_used = 0;
    int len[ITEMS], grow[ITEMS], have[ITEMS], last[ITEMS], st[ITEMS];
    bool rel[ITEMS];
    r.count = min(max(*p.free_count, 0), p.pages);
    long long rows = 0, back = 0;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int b = b0 + i;
        len[i] = grow[i] = have[i] = last[i] = 0;
        st[i] = PX_OK;
        rel[i] = false;
        if (b < p.B) {
            len[i] = p.lengths[b];
            const int f = p.fresh[b];
            if (len[i] < 0 || len[i] > p.width * p.page_size) {
                st[i] = PX_BAD_LENGTH;
            } else {
                have[i] = px_pages(len[i], p.page_size);
                rel[i] = f < 0;
                grow[i] = max(f, 0);
                const long long end = (static_cast<long long>(len[i]) + grow[i] + p.page_size - 1) / p.page_size;
                if (end > p.width) st[i] = PX_TABLE_FULL;
                last[i] = static_cast<int>(end);
            }
        }
        rows += grow[i];
        back += rel[i] ? have[i] : 0;
    }
    long long row_at = px_scan<NT>(rows, ws[0]) - rows, back_at = px_scan<NT>(back, ws[1]) - back, need = 0;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int b = b0 + i;
        row_at += grow[i];
        back_at += rel[i] ? have[i] : 0;
        if (b < p.B) {
            if (row_at > p.total && !rel[i] && st[i] != PX_BAD_LENGTH) st[i] = PX_NO_ROW;
            r.row_end[b] = static_cast<int>(min(row_at, kSat));
            r.back_end[b] = static_cast<int>(min(back_at, kSat));
            if (b == p.B - 1) s_back = r.back_end[b];
            if (st[i] == PX_OK && !rel[i]) need += last[i] - have[i];
        }
    }
    long long need_at = px_scan<NT>(need, ws[2]) - need;
    r.available = static_cast<int>(min(static_cast<long long>(r.count) + s_back, static_cast<long long>(p.pages)));
    int used = 0;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int b = b0 + i;
        if (b < p.B) {
            if (st[i] == PX_OK && !rel[i] && last[i] > have[i]) {
                need_at += last[i] - have[i];
                if (need_at > r.available) st[i] = PX_NO_PAGE;
                else used = static_cast<int>(need_at);
            }
            const bool grows = st[i] == PX_OK && !rel[i];
            r.need_end[b] = static_cast<int>(min(need_at, kSat));
            r.len[b] = grows ? len[i] : -1;
            p.status[b] = st[i];
            p.lengths_out[b] = rel[i] ? 0 : grows ? len[i] + grow[i] : len[i];
        }
    }
    if (used) atomicMax(&s_used, used);
    __syncthreads();
    r.used = s_used;
    if (tid == 0) *p.count_out = r.available - r.used;
    return r;
}

// Stack, table and rows from the sums, by `threads` threads of which this is number `at`; all of it independent.  What is read of the stack lies
// below its old height and what is read of the table belongs to requests that end or to pages that a request had, and neither is
// written here.
__device__ __forceinline__ void px_place(const ExtendParams& p, const PxSums& r, int at, int threads) {
    // entry i of the stack once the pages handed back lie on it
    auto stack = [&](int i) {
        if (i < r.count) return p.free_pages[i];
        const int b = px_find(r.back_end, p.B, i - r.count);
        return p.table[b * p.table_stride + (i - r.count - (b ? r.back_end[b - 1] : 0))];
    };
    for (int i = r.count + at; i < r.available; i += threads) p.free_pages[i] = stack(i);
    // the i-th page of all that are taken comes from the i-th place below the top
    for (int i = at; i < r.used; i += threads) {
        const int b = px_find(r.need_end, p.B, i);
        const int col = px_pages(r.len[b], p.page_size) + i - (b ? r.need_end[b - 1] : 0);
        p.table[b * p.table_stride + col] = stack(r.available - 1 - i);
    }
    for (int row = at; row < p.total; row += threads) {
        long long slot = -1, pos = 0;
        int req = -1;
        const int b = px_find(r.row_end, p.B, row);
        if (b < p.B && r.len[b] >= 0) {
            const int len = r.len[b], to = len + row - (b ? r.row_end[b - 1] : 0), col = to / p.page_size;
            const int have = px_pages(len, p.page_size);
            const int page = col < have ? p.table[b * p.table_stride + col] : stack(r.available - 1 - ((b ? r.need_end[b - 1] : 0) + col - have));
            if (page >= 0 && page < p.pages) {
                slot = static_cast<long long>(page) * p.page_size + to - col * p.page_size;
                pos = to;
                req = b;
            }
        }
        p.slots[row] = slot;
        p.positions[row] = pos;
        p.requests[row] = req;
    }
}

// The reads depend on one another (lengths, sums, table, stack), a launch long and little else: 3.7 us for 64 requests on one CTA, and 10.8
// for 45 000 rows of 1001 requests, whose 2 MB would take 0.3; with one CTA for all of them it took 105.
// One CTA for all of it (a decode step), or, with `split`, for the sums alone, which paged_place_kernel takes from `work`.
template <int NT, int ITEMS>
__global__ void __launch_bounds__(NT) paged_extend_kernel(const ExtendParams p, bool split) {
    extern __shared__ int px_smem[];
    const PxSums r = px_sum<NT, ITEMS>(p, px_smem);
    if (!split) return px_place(p, r, threadIdx.x, NT);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 0) *reinterpret_cast<int4*>(p.work) = make_int4(r.count, r.available, r.used, 0);
    for (int i = threadIdx.x; i < 4 * p.B; i += NT) p.work[4 + i] = px_smem[i];
}

// The second of two launches for many rows.
__global__ void __launch_bounds__(256) paged_place_kernel(const ExtendParams p) {
    extern __shared__ int px_smem[];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (int i = threadIdx.x; i < 4 * p.B; i += 256) px_smem[i] = p.work[4 + i];
    const int4 s = *reinterpret_cast<const int4*>(p.work);
    __syncthreads();
    px_place(p, {px_smem, px_smem + p.B, px_smem + 2 * p.B, px_smem + 3 * p.B, s.x, s.y, s.z}, blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
}

// ------------------------------------------------------------------ keys and values of new tokens into their pages
struct WriteParams {
    const __nv_bfloat16 *k, *v, *cs, *sn;      // k, v [T][heads][dim] by strides; cs, sn [T][dim] or nullptr: k is stored as it is
    const long long* slots;
    __nv_bfloat16 *kp, *vp;
    long long k_row, k_head, v_row, v_head, cs_row;
    uint32_t slot_count;
    int T, heads, dim, page_size;
};

// A thread moves sixteen dimensions of one head: eight of the first half and the eight they are rotated with.  k cos + rotate_half(k) sin
// is formed in float32 and rounded once, to the bfloat16 that the cache stores.  2050 rows of 32 heads of 128: 13.3 us (67 MB, 5.0 TB/s); what keeps
// it from the copy rate is the pages, 256 bytes of a head's 4 KB at a time.  Through the read-only path, which lets the compiler request
// all eight pieces first, it takes 16 us.
constexpr int PW_THREADS = 256;

template <bool VEC>
__global__ void __launch_bounds__(PW_THREADS) paged_write_kernel(const WriteParams p) {
    constexpr int E = VEC ? 8 : 1;
    const int half = p.dim >> 1, pieces = half / E, per = p.heads * pieces, total = p.T * per;         // below 2^31, see the launch
    for (int i = blockIdx.x * PW_THREADS + threadIdx.x; i < total; i += gridDim.x * PW_THREADS) {
        const int t = i / per, u = i - t * per, h = u / pieces, d = (u - h * pieces) * E;
        const long long slot = p.slots[t];
        const __nv_bfloat16 *kr = p.k + t * p.k_row + h * p.k_head + d, *vr = p.v + t * p.v_row + h * p.v_head + d;
        const __nv_bfloat16 *c = p.cs + t * p.cs_row + d, *s = p.sn + t * p.cs_row + d;
        const bool on = slot >= 0 && slot < p.slot_count;
        const uint32_t at = on ? static_cast<uint32_t>(slot) : 0u, page = at / static_cast<uint32_t>(p.page_size);
        const size_t row = (page * static_cast<uint32_t>(p.heads) + h) * static_cast<uint32_t>(p.page_size) + (at - page * p.page_size);
        __nv_bfloat16 *kt = p.kp + row * p.dim + d, *vt = p.vp + row * p.dim + d;
        if constexpr (VEC) {
            uint4 a = *reinterpret_cast<const uint4*>(kr), b = *reinterpret_cast<const uint4*>(kr + half);
            const uint4 v0 = *reinterpret_cast<const uint4*>(vr), v1 = *reinterpret_cast<const uint4*>(vr + half);
            if (p.cs) {
                const uint4 c0 = *reinterpret_cast<const uint4*>(c), c1 = *reinterpret_cast<const uint4*>(c + half);
                const uint4 s0 = *reinterpret_cast<const uint4*>(s), s1 = *reinterpret_cast<const uint4*>(s + half);
                uint32_t *aw = reinterpret_cast<uint32_t*>(&a), *bw = reinterpret_cast<uint32_t*>(&b);
                const uint32_t *c0w = reinterpret_cast<const uint32_t*>(&c0), *c1w = reinterpret_cast<const uint32_t*>(&c1),
                               *s0w = reinterpret_cast<const uint32_t*>(&s0), *s1w = reinterpret_cast<const uint32_t*>(&s1);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float al = bf_lo(aw[j]), ah = bf_hi(aw[j]), bl = bf_lo(bw[j]), bh = bf_hi(bw[j]);
                    aw[j] = pack_bf2(al * bf_lo(c0w[j]) - bl * bf_lo(s0w[j]), ah * bf_hi(c0w[j]) - bh * bf_hi(s0w[j]));
                    bw[j] = pack_bf2(bl * bf_lo(c1w[j]) + al * bf_lo(s1w[j]), bh * bf_hi(c1w[j]) + ah * bf_hi(s1w[j]));
                }
            }
            if (on) {
                *reinterpret_cast<uint4*>(kt) = a;
                *reinterpret_cast<uint4*>(kt + half) = b;
                *reinterpret_cast<uint4*>(vt) = v0;
                *reinterpret_cast<uint4*>(vt + half) = v1;
            }
        } else {
            float a = __bfloat162float(kr[0]), b = __bfloat162float(kr[half]);
            if (p.cs) {
                const float ra = a * __bfloat162float(c[0]) - b * __bfloat162float(s[0]);
                b = b * __bfloat162float(c[half]) + a * __bfloat162float(s[half]);
                a = ra;
            }
            if (on) {
                kt[0] = __float2bfloat16_rn(a);
                kt[half] = __float2bfloat16_rn(b);
                vt[0] = vr[0];
                vt[half] = vr[half];
            }
        }
    }
}

}  // namespace ade
