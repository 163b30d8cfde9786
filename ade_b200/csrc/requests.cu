// C ABI of the operators of a serving step over a batch of independent requests (declared in include/ade_b200.h): paged key-value cache,
// attention over it, deltas of many fine-tuned models, log probabilities.  Host side only validates arguments and launches.
#include "../../include/ade_b200.h"

#include "host.h"
#include "logprobs.cuh"
#include "multi_delta.cuh"
#include "paged.cuh"
#include "paged_attn.cuh"

using ade_host::aligned16;
using ade_host::cuda_ok;

namespace {

// Dynamic shared memory of a kernel beyond 48 KB, asked for once per device.
template <auto Kernel>
bool allow_smem(size_t bytes) {
    static bool done[64];
    int dev = 0;
    if (!cuda_ok(cudaGetDevice(&dev))) return false;
    if (dev < 64 && done[dev]) return true;
    if (!cuda_ok(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)))) return false;
    if (dev < 64) done[dev] = true;
    return true;
}

int launched() { return cuda_ok(cudaGetLastError()) ? ADE_OK : ADE_ERR_CUDA; }

bool dim_ok(int head_dim) { return head_dim >= 32 && head_dim <= 256 && head_dim % 32 == 0; }

// A launch whose blocks may start while the kernel before it still runs; the kernel waits for that one's results itself.
template <typename... Params, typename... Args>
int launch_early(void (*kernel)(Params...), int grid, int threads, size_t smem, cudaStream_t st, Args... args) {
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    return cuda_ok(cudaLaunchKernelEx(&cfg, kernel, args...)) ? ADE_OK : ADE_ERR_CUDA;
}

// Threads of the page allocation's CTA: few, for short sums, as long as a thread has two requests at most (64 requests with a row each: 3.7 us, 7.6 with
// 1024 threads; 512 requests: 5.4, 6.8 with 1024; 1000 requests: 6.8 either way).  It places up to four rows a thread itself (64 requests: 64 rows 3.7 us,
// 5.8 with a second launch; 512 rows 6.4, 6.1; 1024 rows 9.5, 6.0; 1000 requests, 2048 rows: 8.9 either way).
int extend_threads(int B) { return B <= 128 ? 128 : B <= 1024 ? 512 : 1024; }
bool extend_split(int B, int total) { return total > 4 * extend_threads(B); }

template <int NT, int ITEMS>
int launch_extend(const ade::ExtendParams& p, bool split, cudaStream_t st) {
    if (!allow_smem<ade::paged_extend_kernel<NT, ITEMS>>(ade::px_smem_bytes(NT * ITEMS))) return ADE_ERR_CUDA;
    ade::paged_extend_kernel<NT, ITEMS><<<1, NT, ade::px_smem_bytes(p.B), st>>>(p, split);
    return launched();
}

constexpr size_t kAttnWarps = static_cast<size_t>(ade::PA_MAX_CTAS) * 8;

// Both launches of the attention for up to PA_MAX_ROWS rows.  The second begins while the first runs and waits for its end.
template <int HD>
int launch_attn(ade::PagedAttnParams p, int sms, cudaStream_t st) {
    using S = ade::PaShape<HD>;
    const int ctas = sms < ade::PA_MAX_CTAS ? sms : ade::PA_MAX_CTAS;
    const size_t smem = ade::pa_smem_bytes(S::kRing, S::kWarps, S::kStages, p.T);
    if (!allow_smem<ade::paged_attn_kernel<HD>>(ade::pa_smem_bytes(S::kRing, S::kWarps, S::kStages, ade::PA_MAX_ROWS))) return ADE_ERR_CUDA;
    ade::paged_attn_kernel<HD><<<ctas, S::kWarps * 32, smem, st>>>(p);
    if (!cuda_ok(cudaGetLastError())) return ADE_ERR_CUDA;
    return launch_early(ade::paged_attn_join_kernel<HD>, ctas * S::kWarps / ade::PA_JOIN, 256, 0, st, p);
}

int launch_attn_dim(int head_dim, const ade::PagedAttnParams& p, int sms, cudaStream_t st) {
    switch (head_dim) {
        case 32: return launch_attn<32>(p, sms, st);
        case 64: return launch_attn<64>(p, sms, st);
        case 96: return launch_attn<96>(p, sms, st);
        case 128: return launch_attn<128>(p, sms, st);
        case 160: return launch_attn<160>(p, sms, st);
        case 192: return launch_attn<192>(p, sms, st);
        case 224: return launch_attn<224>(p, sms, st);
        default: return launch_attn<256>(p, sms, st);
    }
}

// Rows of a cache layer (page, head, offset) are counted in 32 bits; a cache with more of them would not fit a device.
bool rows_fit(int pages, int kv_heads, int page_size) { return static_cast<unsigned long long>(pages) * kv_heads <= 0xFFFFFFFFull / page_size; }

}  // namespace

extern "C" {

size_t ade_b200_paged_extend_workspace_bytes(int B, int total) {
    return B < 1 || B > ADE_B200_MAX_REQUESTS || !extend_split(B, total) ? 0 : 16 + ade::px_smem_bytes(B);
}

int ade_b200_paged_extend(const int32_t* lengths, const int32_t* new_tokens, int32_t* block_table, int32_t* free_pages, const int32_t* free_count,
                          int32_t* lengths_out, int32_t* free_count_out, int32_t* status, long long* slots, long long* positions, int32_t* requests,
                          void* work, size_t work_bytes, int B, int width, long long table_row_stride, int pages, int page_size, int total,
                          void* stream) {
    if (!lengths || !new_tokens || !block_table || !free_pages || !free_count || !lengths_out || !free_count_out || !status) return ADE_ERR_NULL;
    if (total > 0 && (!slots || !positions || !requests)) return ADE_ERR_NULL;
    if (B < 1 || B > ADE_B200_MAX_REQUESTS || width < 1 || table_row_stride < width || pages < 1 || page_size < 1 || total < 0) return ADE_ERR_SHAPE;
    if (static_cast<long long>(width) * page_size > 0x7FFFFFFFll || total > (1 << 30)) return ADE_ERR_SHAPE;
    const bool split = extend_split(B, total);
    if (split && !work) return ADE_ERR_NULL;
    if (!aligned16(work)) return ADE_ERR_ALIGN;
    if (work_bytes < ade_b200_paged_extend_workspace_bytes(B, total)) return ADE_ERR_SCRATCH;
    int sms = 0;
    const int rc = ade_host::sm_count(&sms);
    if (rc) return rc;
    const ade::ExtendParams p = {lengths, new_tokens, block_table, free_pages, free_count, lengths_out, free_count_out, status, slots, positions,
                                 requests, static_cast<int*>(work), B, width, pages, page_size, total, table_row_stride};
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int threads = extend_threads(B);
    const int rc_launch = threads == 128 ? launch_extend<128, 1>(p, split, st) : threads == 512 ? launch_extend<512, 2>(p, split, st) : launch_extend<1024, 4>(p, split, st);
    if (rc_launch || !split) return rc_launch;
    if (!allow_smem<ade::paged_place_kernel>(ade::px_smem_bytes(ADE_B200_MAX_REQUESTS))) return ADE_ERR_CUDA;
    const int ctas = (total + 511) / 512;
    return launch_early(ade::paged_place_kernel, ctas < 2 * sms ? ctas : 2 * sms, 256, ade::px_smem_bytes(B), st, p);
}

int ade_b200_paged_write(const void* k, const void* v, const void* cos_t, const void* sin_t, const long long* slots, void* k_pages, void* v_pages,
                         int T, int kv_heads, int head_dim, int pages, int page_size, long long k_row_stride, long long k_head_stride,
                         long long v_row_stride, long long v_head_stride, long long cs_row_stride, void* stream) {
    if (!k || !v || !slots || !k_pages || !v_pages || !cos_t != !sin_t) return ADE_ERR_NULL;
    if (T < 1 || kv_heads < 1 || !dim_ok(head_dim) || pages < 1 || page_size < 1) return ADE_ERR_SHAPE;
    if (k_row_stride < 0 || k_head_stride < 0 || v_row_stride < 0 || v_head_stride < 0 || cs_row_stride < 0) return ADE_ERR_SHAPE;
    if (!rows_fit(pages, kv_heads, page_size)) return ADE_ERR_SHAPE;
    if (!aligned16(k_pages) || !aligned16(v_pages)) return ADE_ERR_ALIGN;
    int sms = 0;
    const int rc = ade_host::sm_count(&sms);
    if (rc) return rc;
    using bf = __nv_bfloat16;
    const bool vec = aligned16(k) && aligned16(v) && (!cos_t || (aligned16(cos_t) && aligned16(sin_t))) &&
                     ((k_row_stride | k_head_stride | v_row_stride | v_head_stride | (cos_t ? cs_row_stride : 0)) & 7) == 0;
    // pieces are counted in 31 bits, with room for a step of the grid behind them
    const long long per = static_cast<long long>(kv_heads) * (head_dim / 2 / (vec ? 8 : 1)), most = 0x70000000ll / per;
    if (most < 1) return ADE_ERR_SHAPE;
    for (long long t0 = 0; t0 < T; t0 += most) {
        const int rows = static_cast<int>(T - t0 < most ? T - t0 : most);
        const bf *cs = static_cast<const bf*>(cos_t), *sn = static_cast<const bf*>(sin_t);
        const ade::WriteParams p = {static_cast<const bf*>(k) + t0 * k_row_stride, static_cast<const bf*>(v) + t0 * v_row_stride,
                                    cs ? cs + t0 * cs_row_stride : nullptr, sn ? sn + t0 * cs_row_stride : nullptr, slots + t0,
                                    static_cast<bf*>(k_pages), static_cast<bf*>(v_pages), k_row_stride, k_head_stride, v_row_stride, v_head_stride,
                                    cs_row_stride, static_cast<uint32_t>(pages) * static_cast<uint32_t>(page_size), rows, kv_heads, head_dim, page_size};
        const long long want = (rows * per + ade::PW_THREADS - 1) / ade::PW_THREADS;
        const int grid = static_cast<int>(want < 16ll * sms ? want : 16ll * sms);
        (vec ? ade::paged_write_kernel<true> : ade::paged_write_kernel<false>)<<<grid, ade::PW_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(p);
        if (!cuda_ok(cudaGetLastError())) return ADE_ERR_CUDA;
    }
    return ADE_OK;
}

size_t ade_b200_paged_attn_workspace_bytes(int T, int q_heads, int kv_heads, int head_dim) {
    if (T < 1 || q_heads < 1 || kv_heads < 1 || q_heads % kv_heads || !dim_ok(head_dim)) return 0;
    return kAttnWarps * (2 * ade::PA_HEADS * (head_dim * sizeof(float) + sizeof(float2)) + sizeof(int4));
}

int ade_b200_paged_attn(const void* q, const void* cos_t, const void* sin_t, const int32_t* block_table, const int32_t* requests,
                        const long long* positions, const void* k_pages, const void* v_pages, void* out, void* work, size_t work_bytes, int T, int B,
                        int width, long long table_row_stride, int q_heads, int kv_heads, int head_dim, int pages, int page_size,
                        long long q_row_stride, long long q_head_stride, long long cs_row_stride, float scale, void* stream) {
    if (!q || !block_table || !requests || !positions || !k_pages || !v_pages || !out || !cos_t != !sin_t) return ADE_ERR_NULL;
    if (T < 1 || B < 1 || width < 1 || table_row_stride < width || q_heads < 1 || kv_heads < 1 || q_heads % kv_heads || !dim_ok(head_dim) ||
        pages < 1 || page_size < 1 || q_row_stride < 0 || q_head_stride < 0 || cs_row_stride < 0)
        return ADE_ERR_SHAPE;
    if (!work) return ADE_ERR_NULL;
    if (!aligned16(k_pages) || !aligned16(v_pages) || !aligned16(out) || !aligned16(work)) return ADE_ERR_ALIGN;
    if (work_bytes < ade_b200_paged_attn_workspace_bytes(T, q_heads, kv_heads, head_dim)) return ADE_ERR_SCRATCH;
    if (static_cast<long long>(width) * page_size > 0x7FFFFFFFll || !rows_fit(pages, kv_heads, page_size)) return ADE_ERR_SHAPE;
    int sms = 0;
    const int rc = ade_host::sm_count(&sms);
    if (rc) return rc;
    using bf = __nv_bfloat16;
    float* part = static_cast<float*>(work);
    float2* stat = reinterpret_cast<float2*>(part + kAttnWarps * 2 * ade::PA_HEADS * head_dim);
    int4* meta = reinterpret_cast<int4*>(stat + kAttnWarps * 2 * ade::PA_HEADS);
    const bool pairs = ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(cos_t) | reinterpret_cast<uintptr_t>(sin_t)) & 3) == 0 &&
                       ((q_row_stride | q_head_stride | (cos_t ? cs_row_stride : 0)) & 1) == 0;
    // division by page_size as a multiplication: the shift is its logarithm rounded up, the factor 2^32 (2^shift - page_size) / page_size + 1
    uint32_t page_shift = 0;
    while ((1ull << page_shift) < static_cast<unsigned long long>(page_size)) ++page_shift;
    const uint32_t page_mul = static_cast<uint32_t>((((1ull << page_shift) - page_size) << 32) / page_size + 1);
    // rows of one launch: PA_MAX_ROWS, fewer where the places of that many full rows would not fit 31 bits
    const long long heads = static_cast<long long>(kv_heads) * ((q_heads / kv_heads + ade::PA_HEADS - 1) / ade::PA_HEADS);
    const long long fit = 0x7FFFFFFFll / (heads * (static_cast<long long>(width) * page_size / 16 + 1 + ade::PA_GAP));
    if (fit < 1) return ADE_ERR_SHAPE;
    const int chunk = fit < ade::PA_MAX_ROWS ? static_cast<int>(fit) : ade::PA_MAX_ROWS;
    for (int t0 = 0; t0 < T; t0 += chunk) {
        const bf *cs = static_cast<const bf*>(cos_t), *sn = static_cast<const bf*>(sin_t);
        const long long o = t0;
        const ade::PagedAttnParams p = {static_cast<const bf*>(q) + o * q_row_stride, cs ? cs + o * cs_row_stride : nullptr,
                                        sn ? sn + o * cs_row_stride : nullptr, block_table, requests + o, positions + o, static_cast<const bf*>(k_pages),
                                        static_cast<const bf*>(v_pages), static_cast<bf*>(out) + o * q_heads * head_dim, part, stat, meta,
                                        table_row_stride, q_row_stride, q_head_stride, cs_row_stride, T - t0 < chunk ? T - t0 : chunk, B,
                                        width, pages, page_size, q_heads, kv_heads, scale * 1.44269504088896340736f, page_mul, page_shift, pairs};
        const int rc_launch = launch_attn_dim(head_dim, p, sms, static_cast<cudaStream_t>(stream));
        if (rc_launch) return rc_launch;
    }
    return ADE_OK;
}

size_t ade_b200_multi_delta_workspace_bytes(int T, int N) {
    return T < 1 || T > ADE_B200_MAX_TOKENS || N < 1 ? 0 : static_cast<size_t>(ade::md_slices(N)) * T * ade::MD_H * sizeof(float);
}

int ade_b200_multi_delta(const void* x, const void* y_dense, const ade_delta_bank_t* bank, const int32_t* ids, void* out, void* work, size_t work_bytes,
                         int T, void* stream) {
    if (!x || !y_dense || !bank || !ids || !out) return ADE_ERR_NULL;
    const ade_delta_bank_t& d = *bank;
    if (!d.uq || !d.us || !d.uz || !d.vt || !d.vs || !d.vz || !d.start) return ADE_ERR_NULL;
    if (T < 1 || T > ADE_B200_MAX_TOKENS || d.M < 1 || d.M > (1 << 21) || d.N < 128 || d.N > (1 << 21) || d.N % 128 || d.groups < 1 || d.deltas < 1)
        return ADE_ERR_SHAPE;
    if (static_cast<unsigned long long>(d.groups) * d.M > 0xFFFFFFFFull) return ADE_ERR_SHAPE;          // rows of U are counted in 32 bits
    if (!work) return ADE_ERR_NULL;
    const void* all[] = {x, y_dense, out, work, d.uq, d.us, d.uz, d.vt, d.vs, d.vz};
    for (const void* a : all)
        if (!aligned16(a)) return ADE_ERR_ALIGN;
    if (work_bytes < ade_b200_multi_delta_workspace_bytes(T, d.N)) return ADE_ERR_SCRATCH;
    int sms = 0;
    const int rc = ade_host::sm_count(&sms);
    if (rc) return rc;
    using bf = __nv_bfloat16;
    ade::MultiDeltaParams p = {static_cast<const bf*>(x), static_cast<const bf*>(y_dense), static_cast<bf*>(out), d.uq, d.uz, d.vt, d.vz,
                               reinterpret_cast<const bf*>(d.us), reinterpret_cast<const bf*>(d.vs), d.start, ids, static_cast<float*>(work),
                               d.M, d.N, d.groups, d.deltas, T};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (!allow_smem<ade::multi_delta_v_kernel>(ade::md_v_smem()) || !allow_smem<ade::multi_delta_u_kernel>(ade::md_u_smem())) return ADE_ERR_CUDA;
    const int slices = ade::md_slices(d.N);
    ade::multi_delta_v_kernel<<<2 * sms, ade::MD_THREADS, ade::md_v_smem(), st>>>(p, slices);
    if (!cuda_ok(cudaGetLastError())) return ADE_ERR_CUDA;
    // One CTA per SM for the second launch where that gives a warp one tile at most: it is set up beside the first one's CTAs then, instead of behind
    // them.  4096 x 4096: 13.2 us for 16 rows of 12 deltas, 13.7 with two CTAs; 19.3 for 40 rows of 30 deltas (two tiles), 17.2 with two.
    const long long entries = T < d.deltas + 1 + T / ade::MD_ENTRY ? T : d.deltas + 1 + T / ade::MD_ENTRY;
    const bool few = entries * ((d.M + ade::MD_TILE - 1) / ade::MD_TILE) <= 1ll * sms * (ade::MD_THREADS / 32);
    return launch_early(ade::multi_delta_u_kernel, few ? sms : 2 * sms, ade::MD_THREADS, ade::md_u_smem(), st, p, slices);
}

int ade_b200_token_logprobs(const void* logits, int dtype, const long long* tokens, float* logprobs, float* entropy, float* top_logprobs,
                            long long* top_tokens, int rows, int vocab, long long row_stride, int top, void* stream) {
    if (!logits || !entropy || !tokens != !logprobs || (top > 0 && (!top_logprobs || !top_tokens))) return ADE_ERR_NULL;
    if (rows < 1 || vocab < 1 || row_stride < 0 || top < 0 || top > ade::LP_MAX_TOP || top > vocab || dtype < ADE_DTYPE_F32 || dtype > ADE_DTYPE_F16) return ADE_ERR_SHAPE;
    int sms = 0;
    const int rc = ade_host::sm_count(&sms);
    if (rc) return rc;
    const ade::LogprobParams p = {logits, tokens, logprobs, entropy, top_logprobs, top_tokens, row_stride, rows, vocab, top};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case ADE_DTYPE_F32: ade::logprob_kernel<float><<<rows, ade::LP_THREADS, 0, st>>>(p); break;
        case ADE_DTYPE_BF16: ade::logprob_kernel<__nv_bfloat16><<<rows, ade::LP_THREADS, 0, st>>>(p); break;
        default: ade::logprob_kernel<__half><<<rows, ade::LP_THREADS, 0, st>>>(p);
    }
    return launched();
}

}  // extern "C"
