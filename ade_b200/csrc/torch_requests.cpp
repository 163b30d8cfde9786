// Torch binding of the operators of a serving step over independent requests (csrc/requests.cu): tensors in, outputs and workspaces from
// torch's caching allocator, the launch on torch's current stream of the tensors' device.  No kernel of its own; see torch_shim.cpp.
//
//   torch.ops.ade_b200.paged_extend(lengths, new_tokens, block_table, free_pages, free_count, total, page_size, in_place)
//       -> (slots, positions, requests, lengths, free_count, status); in place: lengths and free_count are empty
//   torch.ops.ade_b200.paged_write(k, v, slots, k_pages, v_pages, cos?, sin?)
//   torch.ops.ade_b200.paged_attn(q, block_table, requests, positions, k_pages, v_pages, scale, cos?, sin?) -> out
//   torch.ops.ade_b200.multi_delta(x, y_dense, uq, us, uz, vt, vs, vz, start, M, N, ids) -> out
//   torch.ops.ade_b200.token_logprobs(logits, tokens?, top) -> (logprobs, entropy, top_logprobs, top_tokens)
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <array>

#include "../../include/ade_b200.h"

namespace {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;

void check_rc(int rc, const char* entry) {
    if (rc == ADE_OK) return;
    const char* why = rc == ADE_ERR_NULL      ? "ADE_ERR_NULL: a required pointer is NULL"
                      : rc == ADE_ERR_SHAPE   ? "ADE_ERR_SHAPE: a dimension is outside the supported set"
                      : rc == ADE_ERR_ALIGN   ? "ADE_ERR_ALIGN: a pointer is not 16-byte aligned"
                      : rc == ADE_ERR_SCRATCH ? "ADE_ERR_SCRATCH: scratch buffer too small"
                      : rc == ADE_ERR_DEVICE  ? "ADE_ERR_DEVICE: the current device is not compute capability 10.x"
                                              : "ADE_ERR_CUDA: a CUDA runtime call failed";
    TORCH_CHECK(false, entry, ": ", why, rc == ADE_ERR_CUDA ? " (cudaError " + std::to_string(ade_b200_last_cuda_error()) + ")" : std::string());
}

// A CUDA tensor of this type on the device of `like`; the operators have no backward pass, so a tensor that records one is refused.
void check(const Tensor& t, const char* name, at::ScalarType type, int64_t dim, const Tensor& like) {
    TORCH_CHECK(t.is_cuda() && t.device() == like.device() && t.scalar_type() == type && t.dim() == dim, name, " must be a ", dim, "-dimensional CUDA tensor of ",
                type, " on the device of the others; got ", t.sizes(), " ", t.scalar_type(), " on ", t.device());
    TORCH_CHECK(!(t.requires_grad() && at::GradMode::is_enabled()), name, " requires a gradient: this operator has no backward pass");
}

void check_whole(const Tensor& t, const char* name, at::ScalarType type, at::IntArrayRef sizes, const Tensor& like) {
    check(t, name, type, static_cast<int64_t>(sizes.size()), like);
    TORCH_CHECK(t.sizes() == sizes && t.is_contiguous(), name, " must be contiguous with sizes ", sizes, "; got ", t.sizes(), " with strides ", t.strides());
}

int as_int(int64_t v, const char* name) {
    TORCH_CHECK(v >= 0 && v <= 0x7FFFFFFF, name, " is out of range: ", v);
    return static_cast<int>(v);
}

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// A fresh contiguous tensor on the device of `like`, without the dispatcher (about a microsecond of host time for each output).
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) { return at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt); }

// Several fresh contiguous tensors on the device of `like` in one allocation: they share a storage (and nothing else), which halves the host
// time of an operator with six outputs.
struct Out {
    at::DimVector sizes;
    at::ScalarType type;
};
template <size_t N>
std::array<Tensor, N> fresh_all(const std::array<Out, N>& want, const Tensor& like) {
    std::array<int64_t, N + 1> at_byte;
    at_byte[0] = 0;
    for (size_t i = 0; i < N; ++i) {
        int64_t n = static_cast<int64_t>(c10::elementSize(want[i].type));
        for (int64_t d : want[i].sizes) n *= d;
        at_byte[i + 1] = at_byte[i] + (n + 15) / 16 * 16;
    }
    const Tensor all = fresh({at_byte[N]}, at::kByte, like);
    std::array<Tensor, N> out;
    for (size_t i = 0; i < N; ++i) {
        out[i] = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), c10::DispatchKeySet(c10::DispatchKey::CUDA),
                                                          c10::scalarTypeToTypeMeta(want[i].type));
        out[i].unsafeGetTensorImpl()->set_storage_offset(at_byte[i] / static_cast<int64_t>(c10::elementSize(want[i].type)));
        out[i].unsafeGetTensorImpl()->set_sizes_contiguous(want[i].sizes);
    }
    return out;
}

// stride of dimension `d`, or 0 where the tensor has a single entry there (torch gives such a dimension any stride)
int64_t stride_of(const Tensor& t, int64_t d) { return t.size(d) > 1 ? t.stride(d) : 0; }

void check_pages(const Tensor& k_pages, const Tensor& v_pages, const Tensor& like) {
    check(k_pages, "k_pages", at::kBFloat16, 4, like);
    check(v_pages, "v_pages", at::kBFloat16, 4, like);
    TORCH_CHECK(k_pages.is_contiguous() && v_pages.is_contiguous() && k_pages.sizes() == v_pages.sizes(),
                "k_pages and v_pages must be contiguous and of the same sizes (pages, kv_heads, page_size, head_dim)");
}

void check_angles(const OptTensor& cos, const OptTensor& sin, int64_t T, int64_t dim, const Tensor& like) {
    TORCH_CHECK(cos.has_value() == sin.has_value(), "cos and sin come together");
    if (!cos.has_value()) return;
    check(*cos, "cos", at::kBFloat16, 2, like);
    check(*sin, "sin", at::kBFloat16, 2, like);
    TORCH_CHECK(cos->size(0) == T && cos->size(1) == dim && cos->stride(1) == 1 && sin->sizes() == cos->sizes() && sin->strides() == cos->strides(),
                "cos and sin must be (rows, head_dim) = (", T, ", ", dim, ") with a contiguous last dimension and the same strides");
}

void check_table(const Tensor& table, const Tensor& like) {
    check(table, "block_table", at::kInt, 2, like);
    TORCH_CHECK(table.size(0) >= 1 && table.size(1) >= 1 && table.stride(1) == 1 && (table.size(0) == 1 || table.stride(0) >= table.size(1)),
                "block_table must be (requests, width) with a contiguous last dimension and rows that do not overlap");
}

int64_t table_stride(const Tensor& table) { return table.size(0) > 1 ? table.stride(0) : table.size(1); }

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> paged_extend(const Tensor& lengths, const Tensor& new_tokens, const Tensor& table,
                                                                        const Tensor& free_pages, const Tensor& free_count, int64_t total,
                                                                        int64_t page_size, bool in_place) {
    check_table(table, lengths);
    const int64_t B = table.size(0);
    check_whole(lengths, "lengths", at::kInt, {B}, table);
    check_whole(new_tokens, "new_tokens", at::kInt, {B}, table);
    check(free_pages, "free_pages", at::kInt, 1, table);
    TORCH_CHECK(free_pages.is_contiguous(), "free_pages must be contiguous");
    check_whole(free_count, "free_count", at::kInt, {1}, table);
    const c10::cuda::CUDAGuard guard(table.device());
    const int n = as_int(total, "total");
    auto [slots, positions, requests, len_out, count_out, status] =             // in place: an operator may not return an argument
        fresh_all<6>({{{{total}, at::kLong}, {{total}, at::kLong}, {{total}, at::kInt}, {{in_place ? 0 : B}, at::kInt}, {{in_place ? 0 : 1}, at::kInt},
                       {{B}, at::kInt}}}, table);
    const size_t bytes = ade_b200_paged_extend_workspace_bytes(as_int(B, "requests"), n);
    const Tensor work = bytes ? fresh({static_cast<int64_t>(bytes)}, at::kByte, table) : Tensor();
    auto i = [](const Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); };
    auto l = [](const Tensor& t) { return static_cast<long long*>(t.data_ptr()); };
    check_rc(ade_b200_paged_extend(i(lengths), i(new_tokens), i(table), i(free_pages), i(free_count), i(in_place ? lengths : len_out),
                                   i(in_place ? free_count : count_out), i(status), l(slots),
                                   l(positions), i(requests), bytes ? work.data_ptr() : nullptr, bytes, as_int(B, "requests"), as_int(table.size(1), "width"),
                                   table_stride(table),
                                   as_int(free_pages.size(0), "pages"), as_int(page_size, "page_size"), n, stream_of(table)),
             "ade_b200_paged_extend");
    return {slots, positions, requests, len_out, count_out, status};
}

void paged_write(const Tensor& k, const Tensor& v, const Tensor& slots, const Tensor& k_pages, const Tensor& v_pages, const OptTensor& cos,
                 const OptTensor& sin) {
    check_pages(k_pages, v_pages, k);
    check(k, "k", at::kBFloat16, 3, k_pages);
    check(v, "v", at::kBFloat16, 3, k_pages);
    const int64_t T = k.size(0), heads = k_pages.size(1), dim = k_pages.size(3);
    TORCH_CHECK(k.size(1) == heads && k.size(2) == dim && v.sizes() == k.sizes() && k.stride(2) == 1 && v.stride(2) == 1,
                "k and v must be (rows, kv_heads, head_dim) = (rows, ", heads, ", ", dim, ") with a contiguous last dimension");
    check_whole(slots, "slots", at::kLong, {T}, k_pages);
    check_angles(cos, sin, T, dim, k_pages);
    if (T == 0) return;
    const c10::cuda::CUDAGuard guard(k_pages.device());
    check_rc(ade_b200_paged_write(k.data_ptr(), v.data_ptr(), cos ? cos->data_ptr() : nullptr, sin ? sin->data_ptr() : nullptr,
                                  static_cast<const long long*>(slots.data_ptr()), k_pages.data_ptr(), v_pages.data_ptr(), as_int(T, "rows"),
                                  as_int(heads, "kv_heads"), as_int(dim, "head_dim"), as_int(k_pages.size(0), "pages"),
                                  as_int(k_pages.size(2), "page_size"), stride_of(k, 0), stride_of(k, 1), stride_of(v, 0), stride_of(v, 1),
                                  cos ? stride_of(*cos, 0) : 0, stream_of(k_pages)),
             "ade_b200_paged_write");
}

Tensor paged_attn(const Tensor& q, const Tensor& table, const Tensor& requests, const Tensor& positions, const Tensor& k_pages, const Tensor& v_pages,
                  double scale, const OptTensor& cos, const OptTensor& sin) {
    check_pages(k_pages, v_pages, q);
    check(q, "q", at::kBFloat16, 3, k_pages);
    const int64_t T = q.size(0), hq = q.size(1), hk = k_pages.size(1), dim = k_pages.size(3);
    TORCH_CHECK(q.size(2) == dim && q.stride(2) == 1 && hk > 0 && hq > 0 && hq % hk == 0,
                "q must be (rows, q_heads, head_dim) with a contiguous last dimension, the cache's head_dim and a multiple of its heads; got ", q.sizes(),
                " for pages ", k_pages.sizes());
    check_table(table, k_pages);
    check_whole(requests, "requests", at::kInt, {T}, k_pages);
    check_whole(positions, "positions", at::kLong, {T}, k_pages);
    check_angles(cos, sin, T, dim, k_pages);
    const c10::cuda::CUDAGuard guard(k_pages.device());
    Tensor out = fresh({T, hq * dim}, at::kBFloat16, q);
    if (T == 0) return out;
    const int t = as_int(T, "rows"), h = as_int(hq, "q_heads"), g = as_int(hk, "kv_heads"), d = as_int(dim, "head_dim");
    const size_t bytes = ade_b200_paged_attn_workspace_bytes(t, h, g, d);
    const Tensor work = fresh({static_cast<int64_t>(bytes)}, at::kByte, q);
    check_rc(ade_b200_paged_attn(q.data_ptr(), cos ? cos->data_ptr() : nullptr, sin ? sin->data_ptr() : nullptr, static_cast<const int32_t*>(table.data_ptr()),
                                 static_cast<const int32_t*>(requests.data_ptr()), static_cast<const long long*>(positions.data_ptr()), k_pages.data_ptr(),
                                 v_pages.data_ptr(), out.data_ptr(), work.data_ptr(), bytes, t, as_int(table.size(0), "requests"),
                                 as_int(table.size(1), "width"), table_stride(table), h, g, d, as_int(k_pages.size(0), "pages"),
                                 as_int(k_pages.size(2), "page_size"), stride_of(q, 0), stride_of(q, 1), cos ? stride_of(*cos, 0) : 0,
                                 static_cast<float>(scale), stream_of(k_pages)),
             "ade_b200_paged_attn");
    return out;
}

Tensor multi_delta(const Tensor& x, const Tensor& y, const Tensor& uq, const Tensor& us, const Tensor& uz, const Tensor& vt, const Tensor& vs,
                   const Tensor& vz, const Tensor& start, int64_t M, int64_t N, const Tensor& ids) {
    check(x, "x", at::kBFloat16, 2, ids);
    const int64_t T = x.size(0), G = uq.dim() ? uq.size(0) : 0;
    check_whole(x, "x", at::kBFloat16, {T, N}, ids);
    check_whole(y, "y_dense", at::kBFloat16, {T, M}, x);
    check_whole(ids, "ids", at::kInt, {T}, x);
    check_whole(uq, "bank tensor uq", at::kByte, {G, M, ADE_B200_GROUP / 2}, x);
    check_whole(us, "bank tensor us", at::kBFloat16, {G, M}, x);
    check_whole(uz, "bank tensor uz", at::kByte, {G, M}, x);
    check_whole(vt, "bank tensor vt", at::kByte, {G, ADE_B200_GROUP, N / 2}, x);
    check_whole(vs, "bank tensor vs", at::kBFloat16, {G, N}, x);
    check_whole(vz, "bank tensor vz", at::kByte, {G, N}, x);
    check(start, "bank tensor start", at::kInt, 1, x);
    TORCH_CHECK(start.is_contiguous() && start.size(0) >= 2, "bank tensor start must be contiguous with an entry for each delta and one behind");
    const c10::cuda::CUDAGuard guard(x.device());
    Tensor out = fresh({T, M}, at::kBFloat16, x);
    if (T == 0) return out;
    const int t = as_int(T, "rows");
    const ade_delta_bank_t bank = {static_cast<const uint8_t*>(uq.data_ptr()), static_cast<const uint16_t*>(us.data_ptr()),
                                   static_cast<const uint8_t*>(uz.data_ptr()), static_cast<const uint8_t*>(vt.data_ptr()),
                                   static_cast<const uint16_t*>(vs.data_ptr()), static_cast<const uint8_t*>(vz.data_ptr()),
                                   static_cast<const int32_t*>(start.data_ptr()), as_int(M, "M"), as_int(N, "N"), as_int(G, "groups"),
                                   as_int(start.size(0) - 1, "deltas")};
    const size_t bytes = ade_b200_multi_delta_workspace_bytes(t, bank.N);
    const Tensor work = fresh({static_cast<int64_t>(bytes)}, at::kByte, x);
    check_rc(ade_b200_multi_delta(x.data_ptr(), y.data_ptr(), &bank, static_cast<const int32_t*>(ids.data_ptr()), out.data_ptr(), work.data_ptr(), bytes, t,
                                  stream_of(x)),
             "ade_b200_multi_delta");
    return out;
}

std::tuple<Tensor, Tensor, Tensor, Tensor> token_logprobs(const Tensor& logits, const OptTensor& tokens, int64_t top) {
    const auto type = logits.scalar_type();
    TORCH_CHECK(type == at::kFloat || type == at::kBFloat16 || type == at::kHalf, "logits must be float32, bfloat16 or float16; got ", type);
    check(logits, "logits", type, 2, logits);
    const int64_t rows = logits.size(0), vocab = logits.size(1);
    TORCH_CHECK(vocab >= 1 && (vocab == 1 || logits.stride(1) == 1), "logits must be (rows, vocabulary) with a contiguous last dimension");
    TORCH_CHECK(top >= 0 && top <= 32 && top <= vocab, "top must be in 0 .. 32 and at most the vocabulary; got ", top);
    if (tokens) check_whole(*tokens, "tokens", at::kLong, {rows}, logits);
    const c10::cuda::CUDAGuard guard(logits.device());
    auto [logp, entropy, tl, tt] = fresh_all<4>({{{{tokens ? rows : 0}, at::kFloat}, {{rows}, at::kFloat}, {{rows, top}, at::kFloat}, {{rows, top}, at::kLong}}}, logits);
    if (rows == 0) return {logp, entropy, tl, tt};
    check_rc(ade_b200_token_logprobs(logits.data_ptr(), type == at::kFloat ? ADE_DTYPE_F32 : type == at::kHalf ? ADE_DTYPE_F16 : ADE_DTYPE_BF16,
                                     tokens ? static_cast<const long long*>(tokens->data_ptr()) : nullptr, tokens ? logp.data_ptr<float>() : nullptr,
                                     entropy.data_ptr<float>(), tl.data_ptr<float>(), static_cast<long long*>(tt.data_ptr()), as_int(rows, "rows"),
                                     as_int(vocab, "vocabulary"), stride_of(logits, 0), static_cast<int>(top), stream_of(logits)),
             "ade_b200_token_logprobs");
    return {logp, entropy, tl, tt};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(ade_b200, m) {
    m.def("paged_extend(Tensor(a!) lengths, Tensor new_tokens, Tensor(b!) block_table, Tensor(c!) free_pages, Tensor(d!) free_count, int total, "
          "int page_size, bool in_place) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
    m.def("paged_write(Tensor k, Tensor v, Tensor slots, Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor? cos, Tensor? sin) -> ()");
    m.def("paged_attn(Tensor q, Tensor block_table, Tensor requests, Tensor positions, Tensor k_pages, Tensor v_pages, float scale, Tensor? cos, "
          "Tensor? sin) -> Tensor");
    m.def("multi_delta(Tensor x, Tensor y_dense, Tensor uq, Tensor us, Tensor uz, Tensor vt, Tensor vs, Tensor vz, Tensor start, int M, int N, "
          "Tensor ids) -> Tensor");
    m.def("token_logprobs(Tensor logits, Tensor? tokens, int top) -> (Tensor, Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(ade_b200, CUDA, m) {
    m.impl("paged_extend", &paged_extend);
    m.impl("paged_write", &paged_write);
    m.impl("paged_attn", &paged_attn);
    m.impl("multi_delta", &multi_delta);
    m.impl("token_logprobs", &token_logprobs);
}
