// Attention of single token rows over the pages of their requests, split over the cache's length and joined.
//
//   out[t][h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q~ . k_j - m),   j = 0 .. positions[t],   m the largest score
//
// A (row, key-value head) pair reads its keys and values once for up to eight query heads.  Both products run on the warp matrix
// instruction m16n8k16 with the heads as its 16 rows: rows 0-7 hold the bfloat16 rounding of an operand, rows 8-15 what that
// rounding left over, so queries and probabilities enter with 16 bits of mantissa at no cost (one to eight heads leave those rows
// free) and the two halves of a result are added in float32.  The running maximum and sum of the softmax stay in registers.
//
// The cache is cut into tiles of 16 positions (32 up to 64 dimensions); the tiles of all pairs, one pair behind the other, are shared out evenly over the
// CTAs and there over the warps, whatever the lengths.  On that line of tiles every pair has PA_GAP places more in front of its tiles, for what
// a pair costs besides them (its queries, its result): without them the warps that meet the short pairs of a ragged batch end last.  A warp streams its tiles through cp.async stages of its own and never waits
// for another; what it has of a pair that others share goes to the workspace as (maximum, sum, weighted sum), and a second
// launch joins those parts in the order of the tiles.  A CTA whose tiles all belong to one pair joins its warps' parts itself.
//
// Long rows are bound by memory: 32 rows of 16 to 4000 positions, 32 heads of 128 (0.41 GB) take 81 us, 3 rows of up to 60 000 positions on 8 heads for 32
// queries (0.47 GB) 87 us, 5.0 and 5.3 TB/s, of which 4 us are set-up and 3 the join.  At 256 dimensions four warps of a CTA have registers for the sums
// and spill 232 bytes: the first case with 16 heads of 256, the same bytes, takes 131 us (3.4 TB/s).  Short rows are bound by two launches and what depends on
// what in them: lengths, table, keys, parts.
#pragma once
#include "paged.cuh"
#include "ptx.cuh"

namespace ade {

constexpr int PA_MAX_CTAS = 160;           // one CTA per SM; bounds the workspace
constexpr int PA_MAX_ROWS = 1024;          // rows of one launch (their prefix sums lie in shared memory); the places of a launch fit 31 bits
constexpr int PA_HEADS = 8;                // query heads that share one pass over the keys and values
// Places of the line in front of a pair's tiles.  With 0, 2, 3, 5, 8 of them, us: 32 rows of 16 to 4000 positions, 32 heads of 128: 103, 81.5, 82.2, 81.6, 83.4;
// 64 rows of 100 to 2000, 8 heads of 64: 27.0, 25.8, 26.1, 26.2, 27.0; 16 rows of 100 to 8000, 8 heads of 128 for 32 queries: 37.0, 37.2, 37.1, 36.9,
// 36.6; 24 rows of 50 to 3000, 2 heads of 256 for 16: 34.2, 31.6, 31.1, 31.3, 30.8; 48 rows of 16 to 2000, 3 heads of 96 for 48: 27.7, 22.1, 22.2, 22.2, 22.5;
// 8 rows of 20 to 200, 32 heads of 128: 14.7, 12.4, 12.8, 12.8, 13.6.
constexpr int PA_GAP = 3;

struct PagedAttnParams {
    const __nv_bfloat16 *q, *cs, *sn;          // q [T][q_heads][dim] by strides; cs, sn [T][dim] or nullptr: q is used as it is
    const int* table;
    const int* requests;                       // [T] row of the block table, outside 0 .. B - 1: the row has no request
    const long long* positions;                // [T] the row sees positions 0 .. positions[t] of its request
    const __nv_bfloat16 *kp, *vp;
    __nv_bfloat16* out;                        // [T][q_heads][dim]
    float* part;                               // [warps][2][PA_HEADS][dim] weighted sums
    float2* stat;                              // [warps][2][PA_HEADS] (maximum in powers of two, sum)
    int4* meta;                                // [warps] (row + 1 or 0, pair, last warp, flags) of a pair that begins there and goes on
    long long table_stride, q_row, q_head, cs_row;
    int T, B, width, pages, page_size, q_heads, kv_heads;
    float scale2;                              // scale * log2(e)
    uint32_t page_mul, page_shift;             // n / page_size = (mulhi(n, page_mul) + n) >> page_shift for n below 2^31
    bool pairs;                                // q, cs and sn begin every row and head at an even element of 4-byte aligned memory
};

template <int HD>
struct PaShape {
    static constexpr int kWarps = HD <= 128 ? 8 : 4;
    // positions of a tile: 32 up to 64 dimensions (32 rows of 100 to 2000 positions, 8 heads of 64: 19.2 us, 21.0 with 16), 16 where 32 would leave a warp
    // fewer than three stages
    static constexpr int kTile = HD <= 64 ? 32 : 16;
    static constexpr int kChunks = HD / 8;                               // 16-byte pieces of a row
    static constexpr int kTileBytes = kTile * HD * 2;
    static constexpr int kStages = 192 * 1024 / (kWarps * 2 * kTileBytes) < 8 ? 192 * 1024 / (kWarps * 2 * kTileBytes) : 8;
    static constexpr size_t kRing = static_cast<size_t>(kWarps) * kStages * 2 * kTileBytes;
    // where piece c of row r lies in a tile: the eight rows that a matrix load reads at one piece are spread over the banks
    __device__ static __forceinline__ uint32_t at(int r, int c) {
        return static_cast<uint32_t>(r * kChunks + (kChunks % 8 == 0 ? c ^ (r & 7) : c ^ (r >> 1 & 3))) * 16u;
    }
};
inline size_t pa_smem_bytes(size_t ring, int warps, int stages, int T) {
    return ring + (static_cast<size_t>(T) * 3 + 4) * 4 + static_cast<size_t>(warps) * stages * 4 + static_cast<size_t>(warps) * PA_HEADS * 8;
}

__device__ __forceinline__ void pa_ldm4(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void pa_ldm4t(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
// 16 bytes global -> shared; nothing is read and zeros are written where `live` is false
__device__ __forceinline__ void pa_cp16(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
template <int N>
__device__ __forceinline__ void pa_cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// bfloat16 pair of (a, b), and the pair of what that rounding left over
__device__ __forceinline__ uint32_t pa_split(float a, float b, uint32_t& rest) {
    const uint32_t hi = pack_bf2(a, b);
    rest = pack_bf2(a - bf_lo(hi), b - bf_hi(hi));
    return hi;
}

template <int HD>
__global__ void __launch_bounds__(PaShape<HD>::kWarps * 32, 1) paged_attn_kernel(const PagedAttnParams p) {
    using S = PaShape<HD>;
    constexpr int KS = HD / 16, NW = S::kWarps, NT = NW * 32, TILE = S::kTile;
    extern __shared__ __align__(128) uint8_t pa_smem[];
    float2* mstat = reinterpret_cast<float2*>(pa_smem + S::kRing);                 // [NW][PA_HEADS]
    uint32_t* masks = reinterpret_cast<uint32_t*>(mstat + NW * PA_HEADS);          // [NW][stages] positions of a tile that count
    int* prefix = reinterpret_cast<int*>(masks + NW * S::kStages);                 // [T + 1] places of the rows before, of all their pairs
    int* rown = prefix + p.T + 1;                                                  // [T] positions the row sees
    int* rowreq = rown + p.T;                                                      // [T] its request
    __shared__ int ws[NW];
    __shared__ int wmax[NW], wrows[NW];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gid = lane >> 2, tig = lane & 3;
    const int group = p.q_heads / p.kv_heads, sets = (group + PA_HEADS - 1) / PA_HEADS, H = p.kv_heads * sets;

    // places of every row, summed, the longest row and the rows that have any
    auto places = [](int n) { return n ? (n + TILE - 1) / TILE + PA_GAP : 0; };              // of one pair
    const int per = (p.T + NT - 1) / NT, ta = min(tid * per, p.T), tb = min(ta + per, p.T);
    int mine = 0, longest = 0, live = 0;
    for (int t = ta; t < tb; ++t) {
        const int req = p.requests[t];
        const long long pos = p.positions[t];
        const int n = req < 0 || req >= p.B || pos < 0 ? 0 : static_cast<int>(min(pos, static_cast<long long>(p.width) * p.page_size - 1)) + 1;
        rown[t] = n;
        rowreq[t] = req;
        mine += places(n) * H;
        longest = max(longest, places(n));
        live += n > 0;
    }
    int run = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xFFFFFFFFu, run, o);
        if (lane >= o) run += u;
    }
    longest = __reduce_max_sync(0xFFFFFFFFu, longest);
    live = __reduce_add_sync(0xFFFFFFFFu, live);
    if (lane == 31) {
        ws[warp] = run;
        wmax[warp] = longest;
        wrows[warp] = live;
    }
    __syncthreads();
    run -= mine;
    live = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        longest = max(longest, wmax[w]);
        live += wrows[w];
        if (w < warp) run += ws[w];
    }
    for (int t = ta; t < tb; ++t) {
        prefix[t] = run;
        run += places(rown[t]) * H;
    }
    if (tid == NT - 1) prefix[p.T] = run;
    __syncthreads();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    // rows that see nothing are zero
    for (int t = blockIdx.x; t < p.T; t += gridDim.x)
        if (rown[t] == 0)
            for (int i = tid; i < p.q_heads * HD / 8; i += NT)
                reinterpret_cast<uint4*>(p.out + static_cast<long long>(t) * p.q_heads * HD)[i] = make_uint4(0u, 0u, 0u, 0u);

    // This warp's places f .. f_end - 1 of all, and whether its whole CTA works on one pair.  Where every warp would have two tiles at most and the pairs
    // are of one length, a pair gets as many CTAs of its own as it takes: for short rows one, which then needs nobody else (100 positions, 32 heads of
    // 128: 8.4 us, 10.1 with all CTAs; 4 rows of 20 to 200 positions: 11.6 so, 11.1 with all CTAs, since the cuts do not fall between the pairs).
    const int total = prefix[p.T], cta = blockIdx.x, pairs = live * H;
    int most = gridDim.x;
    if (total <= most * NW * 2 && pairs > 0 && pairs <= most && total == pairs * longest) most = pairs * min(most / pairs, (longest + 2 * NW - 1) / (2 * NW));
    const int ctas = min(most, total), each = ctas ? total / ctas : 0, more = total - each * ctas;
    auto cta_begin = [&](int c) { return each * c + min(c, more); };
    const int wid = cta * NW + warp;
    auto no_work = [&] {
        if (lane == 0) p.meta[wid] = make_int4(0, 0, 0, 0);
    };
    if (cta >= ctas) return no_work();
    const int F0 = cta_begin(cta), F1 = cta_begin(cta + 1);
    auto warp_begin = [](int f0, int f1, int w) { return f0 + static_cast<int>(static_cast<unsigned>(f1 - f0) * w / NW); };
    struct Cursor {
        int at, t, pair, tile, nt;                                      // place of the tile, row, pair of the row, tile of the pair and their number
    };
    // the first tile at or behind a place, by the whole warp: the last row whose places begin at or before it, 32 rows at a time
    auto locate = [&](int g) {
        const int hi = 32 * lane < p.T && prefix[32 * lane] <= g;
        const int from = 32 * (__popc(__ballot_sync(0xFFFFFFFFu, hi)) - 1) + lane;
        const int row = from < p.T && prefix[from] <= g;
        Cursor c;
        c.t = from - lane + __popc(__ballot_sync(0xFFFFFFFFu, row)) - 1;
        const int nv = places(rown[c.t]), rest = g - prefix[c.t];
        c.nt = nv - PA_GAP;
        c.pair = static_cast<unsigned>(rest) / static_cast<unsigned>(nv);
        c.tile = max(rest - c.pair * nv - PA_GAP, 0);
        c.at = prefix[c.t] + c.pair * nv + PA_GAP + c.tile;
        return c;
    };
    auto advance = [&](Cursor& c) {
        ++c.at;
        if (++c.tile < c.nt) return;
        c.tile = 0;
        c.at += PA_GAP;
        if (++c.pair < H) return;
        c.pair = 0;
        do {
            ++c.t;
        } while (c.t < p.T && rown[c.t] == 0);
        c.nt = c.t < p.T ? places(rown[c.t]) - PA_GAP : 1;
    };
    auto pair_begin = [&](const Cursor& c) { return c.at - c.tile; };     // its first tile
    const Cursor c0 = locate(F0);
    if (c0.at >= F1) return no_work();                                  // nothing but places in front of a pair's tiles
    const bool merged = F1 <= pair_begin(c0) + c0.nt + PA_GAP;            // the CTA's tiles are all of pair c0
    int4 meta = make_int4(0, 0, 0, 0);
    // (last warp, flags) of the pair of c, which goes on behind this CTA or this warp
    auto chain = [&](const Cursor& c) {
        const int fe = pair_begin(c) + c.nt, cut = more * (each + 1);     // the CTA and the warp that its last tile falls to
        const int last = fe <= cut ? (fe - 1) / (each + 1) : more + (fe - 1 - cut) / each;
        const int L0 = cta_begin(last), L1 = cta_begin(last + 1);
        const int lw = static_cast<int>((static_cast<unsigned>(fe - L0) * NW - 1) / (L1 - L0));
        const bool last_merged = L1 <= fe + PA_GAP;
        return make_int4(c.t + 1, c.pair, last * NW + min(lw, NW - 1), (merged ? 1 : 0) | (last_merged ? 2 : 0));
    };

    const uint32_t ring = smem_u32(pa_smem) + static_cast<uint32_t>(warp) * (S::kStages * 2 * S::kTileBytes);
    uint32_t* mk = masks + warp * S::kStages;
    // ---- the copies, STAGES - 1 tiles ahead of the arithmetic, the look at the block table one more
    const int f_end = warp_begin(F0, F1, warp + 1);
    Cursor cur = warp == 0 ? c0 : locate(warp_begin(F0, F1, warp)), ahead = cur;
    struct Look {
        bool on;                                                        // the tile is one of this warp's
        int page, off, kvh;
    };
    auto look = [&] {
        Look l = {ahead.at < f_end, -1, 0, 0};
        if (l.on) {
            const int pos = ahead.tile * TILE + (lane & (TILE - 1));
            l.kvh = sets == 1 ? ahead.pair : ahead.pair / sets;
            if (pos < rown[ahead.t]) {
                const int col = static_cast<int>((__umulhi(static_cast<uint32_t>(pos), p.page_mul) + static_cast<uint32_t>(pos)) >> p.page_shift);
                l.off = pos - col * p.page_size;
                l.page = p.table[rowreq[ahead.t] * p.table_stride + col];
            }
            advance(ahead);
        }
        return l;
    };
    auto issue = [&](int stage, const Look& l) {
        const bool ok = l.page >= 0 && l.page < p.pages;
        const uint32_t row = ok ? (static_cast<uint32_t>(l.page) * p.kv_heads + l.kvh) * p.page_size + l.off : 0u;
        const uint32_t mask = __ballot_sync(0xFFFFFFFFu, ok) & (TILE == 32 ? 0xFFFFFFFFu : 0xFFFFu);
        if (lane == 0) mk[stage] = mask;
        const uint32_t dst = ring + static_cast<uint32_t>(stage) * (2 * S::kTileBytes);
        if (l.on) {
#pragma unroll
            for (int j = 0; j < S::kChunks * TILE / 32; ++j) {
                const int i = j * 32 + lane, r = i / S::kChunks, c = i - r * S::kChunks;
                const size_t at = static_cast<size_t>(__shfl_sync(0xFFFFFFFFu, row, r)) * HD + c * 8;
                const bool live = mask >> r & 1u;
                pa_cp16(dst + S::at(r, c), p.kp + at, live);
                pa_cp16(dst + S::kTileBytes + S::at(r, c), p.vp + at, live);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // the first tiles are looked up together, and the queries of the first pair requested, before anything is waited for
    Look seen[S::kStages];
#pragma unroll
    for (int s = 0; s < S::kStages; ++s) seen[s] = look();
    uint32_t qa[KS][4];
    float acc[HD / 8][4], m = -INFINITY, l = 0.f;
    const bool any = cur.at < f_end;
    bool fresh = true, from_start = false;
    int stage = 0, fill = S::kStages - 1;
    const int pair_heads = min(PA_HEADS, group);
    auto heads_of = [&](int pair) { return sets == 1 ? group : min(pair_heads, group - pair % sets * PA_HEADS); };
    auto first_head = [&](int pair) { return sets == 1 ? pair * group : pair / sets * group + pair % sets * PA_HEADS; };
    if (!any && !merged && lane < PA_HEADS) p.stat[(wid * 2) * PA_HEADS + lane] = make_float2(-INFINITY, 0.f);   // a warp without tiles
    // Queries of a pair, heads by lanes (gid): dimensions d and d + HD / 2, d + 1 beside each, and the angles they are rotated by, for step ks of
    // the first half.
    auto ask = [&](const Cursor& c, int ks, uint32_t (&raw)[2][6]) {
        const bool on = gid < heads_of(c.pair);
        const __nv_bfloat16* qr = p.q + c.t * p.q_row + (first_head(c.pair) + (on ? gid : 0)) * p.q_head;
        // two neighbours at once where every row begins at an even element
        auto two = [&](const __nv_bfloat16* a) {
            return p.pairs ? *reinterpret_cast<const uint32_t*>(a) : static_cast<uint32_t>(__bfloat16_as_ushort(a[0])) | static_cast<uint32_t>(__bfloat16_as_ushort(a[1])) << 16;
        };
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int d = ks * 16 + tig * 2 + i * 8;
            uint32_t(&r)[6] = raw[i];
            r[0] = on ? two(qr + d) : 0u;
            r[1] = on ? two(qr + d + HD / 2) : 0u;
            if (p.cs) {
                const __nv_bfloat16 *cr = p.cs + c.t * p.cs_row + d, *sr = p.sn + c.t * p.cs_row + d;
                r[2] = two(cr);
                r[3] = two(cr + HD / 2);
                r[4] = two(sr);
                r[5] = two(sr + HD / 2);
            }
        }
    };
    auto rotate = [&](int ks, const uint32_t (&raw)[2][6]) {            // rotated, in two bfloat16 parts
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t(&r)[6] = raw[i];
            float a0 = bf_lo(r[0]), a1 = bf_hi(r[0]), b0 = bf_lo(r[1]), b1 = bf_hi(r[1]);
            if (p.cs) {
                const float x0 = a0, x1 = a1;
                a0 = x0 * bf_lo(r[2]) - b0 * bf_lo(r[4]);
                a1 = x1 * bf_hi(r[2]) - b1 * bf_hi(r[4]);
                b0 = b0 * bf_lo(r[3]) + x0 * bf_lo(r[5]);
                b1 = b1 * bf_hi(r[3]) + x1 * bf_hi(r[5]);
            }
            qa[ks][2 * i] = pa_split(a0, a1, qa[ks][2 * i + 1]);
            qa[ks + KS / 2][2 * i] = pa_split(b0, b1, qa[ks + KS / 2][2 * i + 1]);
        }
    };
    auto queries = [&](const Cursor& c) {
        constexpr int B = KS / 2 < 4 ? KS / 2 : 4;                      // steps under way at once, as registers allow
#pragma unroll
        for (int k0 = 0; k0 < KS / 2; k0 += B) {
            uint32_t raw[B][2][6];
#pragma unroll
            for (int k = 0; k < B; ++k)
                if (k0 + k < KS / 2) ask(c, k0 + k, raw[k]);
#pragma unroll
            for (int k = 0; k < B; ++k)
                if (k0 + k < KS / 2) rotate(k0 + k, raw[k]);
        }
    };
    if constexpr (HD <= 128) {                                          // asked for in front of the first tiles
        uint32_t raw[KS / 2][2][6];
        if (any)
#pragma unroll
            for (int ks = 0; ks < KS / 2; ++ks) ask(cur, ks, raw[ks]);
#pragma unroll
        for (int s = 0; s < S::kStages - 1; ++s) issue(s, seen[s]);
        if (any)
#pragma unroll
            for (int ks = 0; ks < KS / 2; ++ks) rotate(ks, raw[ks]);
    } else {
#pragma unroll
        for (int s = 0; s < S::kStages - 1; ++s) issue(s, seen[s]);
        if (any) queries(cur);
    }
    Look next = seen[S::kStages - 1];
    bool have = true;
#pragma unroll 1
    while (cur.at < f_end) {
        if (fresh) {                                                    // a new pair
            fresh = false;
            from_start = cur.tile == 0;
            m = -INFINITY;
            l = 0.f;
#pragma unroll
            for (int j = 0; j < HD / 8; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
            if (!have) queries(cur);
            have = false;
        }
        pa_cp_wait<S::kStages - 2>();
        __syncwarp();                                                   // the tile is there, and the stage before it has been read by all lanes
        issue(fill, next);
        next = look();
        const uint32_t mask = mk[stage];
        if (mask) {
            const uint32_t kt = ring + static_cast<uint32_t>(stage) * (2 * S::kTileBytes), vt = kt + S::kTileBytes;
            // head gid at positions 8 j + 2 tig and the one behind it, j = 0 .. TILE / 8 - 1
            float w[TILE / 4];
            float mx = -INFINITY;
#pragma unroll
            for (int t = 0; t < TILE / 16; ++t) {
                float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    uint32_t b[4];
                    pa_ldm4(kt + S::at(t * 16 + (lane >> 4) * 8 + (lane & 7), 2 * ks + (lane >> 3 & 1)), b);
                    mma_bf16(s0, qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3], b[0], b[1]);
                    mma_bf16(s1, qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3], b[2], b[3]);
                }
                const float v[4] = {s0[0] + s0[2], s0[1] + s0[3], s1[0] + s1[2], s1[1] + s1[3]};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    w[t * 4 + i] = mask >> (t * 16 + tig * 2 + (i & 1) + (i >> 1) * 8) & 1u ? v[i] * p.scale2 : -INFINITY;
                    mx = fmaxf(mx, w[t * 4 + i]);
                }
            }
            mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 2));
            if (__any_sync(0xFFFFFFFFu, mx > m)) {
                const float mn = fmaxf(m, mx), fac = exp2f(m - mn);
                m = mn;
                l *= fac;
#pragma unroll
                for (int j = 0; j < HD / 8; ++j) {
                    acc[j][0] *= fac;
                    acc[j][1] *= fac;
                    acc[j][2] *= fac;
                    acc[j][3] *= fac;
                }
            }
#pragma unroll
            for (int i = 0; i < TILE / 4; ++i) {
                w[i] = exp2f(w[i] - m);
                l += w[i];
            }
#pragma unroll
            for (int t = 0; t < TILE / 16; ++t) {
                uint32_t pa[4];
                pa[0] = pa_split(w[t * 4], w[t * 4 + 1], pa[1]);
                pa[2] = pa_split(w[t * 4 + 2], w[t * 4 + 3], pa[3]);
#pragma unroll
                for (int j = 0; j < HD / 16; ++j) {
                    uint32_t b[4];
                    pa_ldm4t(vt + S::at(t * 16 + (lane >> 3 & 1) * 8 + (lane & 7), 2 * j + (lane >> 4)), b);
                    mma_bf16(acc[2 * j], pa[0], pa[1], pa[2], pa[3], b[0], b[1]);
                    mma_bf16(acc[2 * j + 1], pa[0], pa[1], pa[2], pa[3], b[2], b[3]);
                }
            }
        }
        stage = stage + 1 == S::kStages ? 0 : stage + 1;
        fill = fill + 1 == S::kStages ? 0 : fill + 1;
        const bool pair_ends = cur.tile + 1 == cur.nt;
        if (pair_ends || cur.at + 1 >= f_end) {
            l += __shfl_xor_sync(0xFFFFFFFFu, l, 1);
            l += __shfl_xor_sync(0xFFFFFFFFu, l, 2);
            const int heads = heads_of(cur.pair);
            if (!merged) {
                if (from_start && pair_ends) {
                    const float inv = l == 0.f ? 0.f : 1.f / l;
                    if (gid < heads) {
                        __nv_bfloat16* o = p.out + (static_cast<long long>(cur.t) * p.q_heads + first_head(cur.pair) + gid) * HD + tig * 2;
#pragma unroll
                        for (int j = 0; j < HD / 8; ++j)
                            *reinterpret_cast<uint32_t*>(o + j * 8) = pack_bf2((acc[j][0] + acc[j][2]) * inv, (acc[j][1] + acc[j][3]) * inv);
                    }
                } else {
                    const int slot = wid * 2 + (from_start ? 1 : 0);
                    if (gid < heads) {
                        float* o = p.part + (static_cast<size_t>(slot) * PA_HEADS + gid) * HD + tig * 2;
#pragma unroll
                        for (int j = 0; j < HD / 8; ++j)
                            *reinterpret_cast<float2*>(o + j * 8) = make_float2(acc[j][0] + acc[j][2], acc[j][1] + acc[j][3]);
                        if (tig == 0) p.stat[slot * PA_HEADS + gid] = make_float2(m, l);
                    }
                    if (from_start) meta = chain(cur);
                }
            }
            fresh = true;
        }
        advance(cur);
    }
    if (merged) {
        // the warps' parts through shared memory (the ring is free: every copy has arrived), added in the order of the warps
        pa_cp_wait<0>();
        __syncwarp();
        float* mine_acc = reinterpret_cast<float*>(pa_smem) + static_cast<size_t>(warp) * (S::kStages * 2 * S::kTileBytes / 4);
        const int heads = heads_of(c0.pair), h0 = first_head(c0.pair);
        if (any && gid < heads) {
#pragma unroll
            for (int j = 0; j < HD / 8; ++j)
                *reinterpret_cast<float2*>(mine_acc + gid * HD + j * 8 + tig * 2) = make_float2(acc[j][0] + acc[j][2], acc[j][1] + acc[j][3]);
        }
        if (tig == 0) mstat[warp * PA_HEADS + gid] = any ? make_float2(m, l) : make_float2(-INFINITY, 0.f);
        __syncthreads();
        const bool begins = F0 <= pair_begin(c0), whole = begins && F1 >= pair_begin(c0) + c0.nt;
        const int slot = cta * NW * 2 + (begins ? 1 : 0);
        for (int i = tid; i < heads * HD; i += NT) {
            const int h = i / HD, d = i - h * HD;
            float mm = -INFINITY, num = 0.f, den = 0.f;
#pragma unroll
            for (int w = 0; w < NW; ++w) mm = fmaxf(mm, mstat[w * PA_HEADS + h].x);
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float2 st = mstat[w * PA_HEADS + h];
                if (st.x == -INFINITY) continue;
                const float fac = exp2f(st.x - mm);
                num += fac * reinterpret_cast<const float*>(pa_smem)[static_cast<size_t>(w) * (S::kStages * 2 * S::kTileBytes / 4) + i];
                den += fac * st.y;
            }
            if (whole) {
                p.out[(static_cast<long long>(c0.t) * p.q_heads + h0 + h) * HD + d] = __float2bfloat16_rn(den == 0.f ? 0.f : num / den);
            } else {
                p.part[(static_cast<size_t>(slot) * PA_HEADS + h) * HD + d] = num;
                if (d == 0) p.stat[slot * PA_HEADS + h] = make_float2(mm, den);
            }
        }
        if (warp == 0 && begins && !whole) meta = chain(c0);
    }
    if (lane == 0) p.meta[wid] = meta;
}

// Joins the parts of the pairs that begin in warps PA_JOIN blockIdx.x .. of the first launch and go on in others: the warp's second slot, then the first
// slots of the warps behind it (one per CTA where the CTA has joined its warps).  Up to eight heads, the parts of a head over as many warps as are
// left.  Most blocks find nothing to do, so all of them are resident at once: two warps of the first launch each, 40 registers (one warp each with 111: 9.4 instead of 8.6 us for 100 positions).
constexpr int PA_JOIN = 2;

template <int HD>
__global__ void __launch_bounds__(256, 6) paged_attn_join_kernel(const PagedAttnParams p) {
    constexpr int NW = PaShape<HD>::kWarps;
    __shared__ float sums[8][HD + 1];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    int4 metas[PA_JOIN];
#pragma unroll
    for (int k = 0; k < PA_JOIN; ++k) metas[k] = p.meta[blockIdx.x * PA_JOIN + k];
#pragma unroll 1
    for (int k = 0; k < PA_JOIN; ++k) {
        const int w0 = blockIdx.x * PA_JOIN + k;
        const int4 meta = k == 0 ? metas[0] : metas[PA_JOIN - 1];
        if (meta.x == 0) continue;
        const int t = meta.x - 1, pair = meta.y, last = meta.z;
        const int group = p.q_heads / p.kv_heads, sets = (group + PA_HEADS - 1) / PA_HEADS;
        const int heads = min(PA_HEADS, group - pair % sets * PA_HEADS), h0 = pair / sets * group + pair % sets * PA_HEADS;
        const int ca = w0 / NW, cb = last / NW;
        const int own = meta.w & 1 ? 0 : min(last, ca * NW + NW - 1) - w0;                       // further warps of the first CTA
        const int middle = max(cb - ca - 1, 0);
        const int n = 1 + own + (cb > ca ? middle + (meta.w & 2 ? 1 : last - cb * NW + 1) : 0);
        auto slot = [&](int i) {
            if (i == 0) return w0 * 2 + 1;
            if (i <= own) return (w0 + i) * 2;
            i -= own + 1;
            return i < middle ? (ca + 1 + i) * NW * 2 : (cb * NW + i - middle) * 2;
        };
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        const int share = heads > 4 ? 1 : heads > 2 ? 2 : heads > 1 ? 4 : 8, h = warp / share, part = warp % share;
        constexpr int V = (HD + 127) / 128;                                                       // 16-byte pieces of a head per lane
        float4 acc[V];
        float den = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (h < heads) {
            // the largest maximum, and a part's sum relative to it; the weighted sums do not wait for either.  A part of no positions (its maximum is
            // -inf) has no weighted sum: what is read there is not used.
            float mm = -INFINITY;
            for (int i = lane; i < n; i += 32) mm = fmaxf(mm, p.stat[slot(i) * PA_HEADS + h].x);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xFFFFFFFFu, mm, o));
            constexpr int U = V == 1 ? 4 : 2;
            for (int i0 = part; i0 < n; i0 += U * share) {
                float2 st[U];
                float4 a[U][V];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    st[u] = make_float2(-INFINITY, 0.f);
                    if (i0 + u * share < n) {
                        const int s = slot(i0 + u * share);
                        st[u] = p.stat[s * PA_HEADS + h];
#pragma unroll
                        for (int v = 0; v < V; ++v)
                            if (lane * 4 + v * 128 < HD)
                                a[u][v] = *reinterpret_cast<const float4*>(p.part + (static_cast<size_t>(s) * PA_HEADS + h) * HD + lane * 4 + v * 128);
                    }
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (st[u].x == -INFINITY) continue;
                    const float fac = exp2f(st[u].x - mm);
                    den += fac * st[u].y;
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        acc[v].x += fac * a[u][v].x;
                        acc[v].y += fac * a[u][v].y;
                        acc[v].z += fac * a[u][v].z;
                        acc[v].w += fac * a[u][v].w;
                    }
                }
            }
            if (share > 1) {
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const int d = lane * 4 + v * 128;
                    if (d < HD) {
                        sums[warp][d] = acc[v].x;
                        sums[warp][d + 1] = acc[v].y;
                        sums[warp][d + 2] = acc[v].z;
                        sums[warp][d + 3] = acc[v].w;
                    }
                }
                if (lane == 0) sums[warp][HD] = den;
            }
        }
        __syncthreads();
        if (h < heads && part == 0) {
            if (share > 1) {
                den = 0.f;
                for (int w = warp; w < warp + share; ++w) den += sums[w][HD];
            }
            const float inv = den == 0.f ? 0.f : 1.f / den;
            __nv_bfloat16* o = p.out + (static_cast<long long>(t) * p.q_heads + h0 + h) * HD;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int d = lane * 4 + v * 128;
                if (d >= HD) continue;
                float a[4] = {acc[v].x, acc[v].y, acc[v].z, acc[v].w};
                if (share > 1) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        a[i] = 0.f;
                        for (int w = warp; w < warp + share; ++w) a[i] += sums[w][d + i];
                    }
                }
                *reinterpret_cast<uint2*>(o + d) = make_uint2(pack_bf2(a[0] * inv, a[1] * inv), pack_bf2(a[2] * inv, a[3] * inv));
            }
        }
        __syncthreads();                                                                              // the next pair's sums may be written
    }
}

}  // namespace ade
