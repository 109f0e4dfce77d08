// Operators of the paged key-value cache: argument checks, outputs, and the calls of the C ABI (paged_append.cu,
// paged_attention.cu, paged_select.cu).  They serve: operands that require gradients or have tangents are refused.
#include "iex_torch_ops.h"

#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/core/grad_mode.h>
#include <ATen/core/stack.h>
#include <torch/library.h>

#include <algorithm>
#include <cmath>
#include <limits>

namespace iex_torch {
namespace {

constexpr int64_t kMostInt = std::numeric_limits<int>::max();

// Without a derivative an output that has none of its own would say that it is zero.
void check_not_differentiated(const char* name, const at::Tensor& t) {
  TORCH_CHECK(!(t.requires_grad() && at::GradMode::is_enabled()), name,
              " requires a gradient: the operators of the paged cache have no backward pass");
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(/*level=*/0).defined(), name,
                              " has a tangent: the operators of the paged cache have no forward derivatives");
}

void check_on(const at::Tensor& first, std::initializer_list<std::pair<const char*, const at::Tensor*>> named) {
  TORCH_CHECK(first.is_cuda(), "the operators of the paged cache take CUDA tensors");
  for (const auto& [name, t] : named) {
    TORCH_CHECK(t->device() == first.device(), name, " should be in the same device as the first argument");
    TORCH_CHECK(!t->is_sparse(), name, " must be a dense tensor");
    check_not_differentiated(name, *t);
  }
}

// q, k or v as the kernels read it: itself, or a contiguous copy of one whose rows they could not load in 16-byte pieces.
struct Operand {
  at::Tensor t;
  int64_t row, head;
  Operand(const at::Tensor& x) : t(x) {
    const auto stride = [&](int dim) { return x.size(dim) > 1 ? x.stride(dim) : 0; };
    row = stride(0);
    head = stride(1);
    if ((x.size(2) > 1 && x.stride(2) != 1) || row % 8 != 0 || head % 8 != 0 || row < 0 || head < 0 ||
        (reinterpret_cast<uintptr_t>(x.data_ptr()) & 15u) != 0) {
      t = x.clone(at::MemoryFormat::Contiguous);
      row = x.size(1) * x.size(2);
      head = x.size(2);
    }
  }
};

struct Cache {
  int64_t pages, kv_heads, page_size, dim, page_stride;
};

Cache check_cache(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.dim() == 4, name, " must be [pages, kv_heads, page_size, head_dim]");
  Cache c{t.size(0), t.size(1), t.size(2), t.size(3), t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2) * t.size(3)};
  const auto dense = [&](int dim, int64_t stride) { return t.size(dim) <= 1 || t.stride(dim) == stride; };
  TORCH_CHECK(dense(3, 1) && dense(2, c.dim) && dense(1, c.page_size * c.dim), "each page of ", name, " must be contiguous");
  TORCH_CHECK(c.page_stride >= c.kv_heads * c.page_size * c.dim && c.page_stride % 8 == 0 &&
                  (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0,
              "the pages of ", name, " must not overlap and must begin on 16-byte boundaries");
  TORCH_CHECK(c.pages <= kMostInt, name, " has too many pages");
  return c;
}

void check_q(const at::Tensor& q, int64_t kv_heads, int64_t dim, int64_t page_size, at::ScalarType type) {
  TORCH_CHECK(q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16, "q must be float16 or bfloat16");
  TORCH_CHECK(q.scalar_type() == type, "q and the cache must have one type");
  TORCH_CHECK(q.dim() == 3 && q.size(2) == dim, "q must be [rows, heads, head_dim], with the cache's head_dim");
  TORCH_CHECK(kv_heads > 0 && q.size(1) > 0 && q.size(1) % kv_heads == 0, "heads must be a multiple of kv_heads");
  // no other sizes by their lower 32 bits
  TORCH_CHECK(page_size > 0 && std::max({q.size(1), dim, page_size}) <= kMostInt &&
                  iex_paged_attention_supported(q.size(1), kv_heads, dim, page_size),
              "head_dim must be a multiple of 8 up to 128 and page_size 16, 32, 64, 128 or 256; got ", dim, " and ", page_size);
  TORCH_CHECK(q.size(0) * q.size(1) <= kMostInt, "q has too many rows");
}

void check_table(const at::Tensor& block_table, const at::Tensor& lengths) {
  TORCH_CHECK(block_table.scalar_type() == at::kInt && lengths.scalar_type() == at::kInt,
              "block_table and lengths must be int32");
  TORCH_CHECK(block_table.dim() == 2 && lengths.dim() == 1 && block_table.size(0) == lengths.size(0),
              "block_table must be [rows, pages] and lengths [rows]");
  TORCH_CHECK(block_table.is_contiguous() && lengths.is_contiguous(), "block_table and lengths must be contiguous tensors");
  TORCH_CHECK(block_table.size(0) <= kMostInt && block_table.size(1) <= kMostInt, "block_table is too large");
}

// A cache that is written: what was saved of it before is seen to have changed.
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// Calls through the dispatcher, ahead of the kernels: a function transform (torch.func.jvp, torch.func.grad) hands these a tensor
// without what it is differentiated by.
void refuse_derivatives(const c10::OperatorHandle& op, c10::DispatchKeySet keys, torch::jit::Stack* stack) {
  const auto& arguments = op.schema().arguments();
  const auto operands = torch::jit::last(stack, arguments.size());
  for (size_t i = 0; i < arguments.size(); ++i)
    if (operands[i].isTensor() && operands[i].toTensor().defined())
      check_not_differentiated(arguments[i].name().c_str(), operands[i].toTensor());
  at::AutoDispatchBelowAutograd below;
  op.redispatchBoxed(keys & c10::after_autograd_keyset, stack);
}

const int32_t* ints(const at::Tensor& t) { return t.data_ptr<int>(); }
int is_bf16(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16; }

}  // namespace

at::Tensor paged_append(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_cache,
                        const at::Tensor& v_cache, const at::Tensor& block_table, const at::Tensor& lengths,
                        const std::optional<at::Tensor>& cu_tokens, const std::optional<at::Tensor>& cos,
                        const std::optional<at::Tensor>& sin, bool interleaved, const std::optional<at::Tensor>& boxes) {
  check_on(q, {{"q", &q}, {"k", &k}, {"v", &v}, {"k_cache", &k_cache}, {"v_cache", &v_cache}, {"block_table", &block_table},
               {"lengths", &lengths}});
  const Cache kc = check_cache(k_cache, "k_cache"), vc = check_cache(v_cache, "v_cache");
  TORCH_CHECK(k_cache.sizes() == v_cache.sizes() && k_cache.scalar_type() == v_cache.scalar_type(),
              "k_cache and v_cache must be alike");
  check_q(q, kc.kv_heads, kc.dim, kc.page_size, k_cache.scalar_type());
  check_table(block_table, lengths);
  const int64_t tokens = q.size(0), batch = lengths.size(0);
  for (const at::Tensor* t : {&k, &v})
    TORCH_CHECK(t->dim() == 3 && t->size(0) == tokens && t->size(1) == kc.kv_heads && t->size(2) == kc.dim &&
                    t->scalar_type() == q.scalar_type(),
                "k and v must be [tokens, kv_heads, head_dim] of q's type");
  if (cu_tokens.has_value()) {
    check_on(q, {{"cu_tokens", &*cu_tokens}});
    TORCH_CHECK(cu_tokens->scalar_type() == at::kInt && cu_tokens->dim() == 1 && cu_tokens->size(0) == batch + 1 &&
                    cu_tokens->is_contiguous(),
                "cu_tokens must be a contiguous int32 [sequences + 1]");
  } else {
    TORCH_CHECK(tokens == batch, "without cu_tokens there is one token for each sequence; got ", tokens, " for ", batch);
  }
  TORCH_CHECK(cos.has_value() == sin.has_value(), "cos and sin go together");
  int64_t rotary = 0, rope_rows = 0;
  if (cos.has_value()) {
    check_on(q, {{"cos", &*cos}, {"sin", &*sin}});
    TORCH_CHECK(cos->dim() == 2 && cos->sizes() == sin->sizes() && cos->is_contiguous() && sin->is_contiguous() &&
                    cos->scalar_type() == at::kFloat && sin->scalar_type() == at::kFloat,
                "cos and sin must be contiguous float32 [positions, rotary_dim / 2]");
    rotary = 2 * cos->size(1);
    rope_rows = std::min(cos->size(0), kMostInt);
    TORCH_CHECK(rotary <= kc.dim, "cos and sin are for ", rotary, " elements of a head, which has ", kc.dim);
  }
  if (boxes.has_value()) {
    check_on(q, {{"boxes", &*boxes}});
    TORCH_CHECK(boxes->dim() == 4 && boxes->size(0) == kc.pages && boxes->size(1) == kc.kv_heads && boxes->size(2) == 2 &&
                    boxes->size(3) == kc.dim && boxes->is_contiguous() && boxes->scalar_type() == q.scalar_type(),
                "boxes must be a contiguous [pages, kv_heads, 2, head_dim] of the cache's type");
  }
  c10::cuda::CUDAGuard guard(q.device());
  at::Tensor out = empty(q, q.sizes());
  if (tokens == 0) return out;
  const Operand qo(q), ko(k), vo(v);
  check_status(
      iex_paged_append(tokens, batch, q.size(1), kc.kv_heads, kc.dim, is_bf16(q), qo.t.data_ptr(), qo.row, qo.head,
                       ko.t.data_ptr(), ko.row, ko.head, vo.t.data_ptr(), vo.row, vo.head,
                       rotary > 0 ? cos->data_ptr<float>() : nullptr, rotary > 0 ? sin->data_ptr<float>() : nullptr, rope_rows,
                       rotary, interleaved, out.data_ptr(), k_cache.data_ptr(), kc.page_stride, v_cache.data_ptr(),
                       vc.page_stride, boxes.has_value() ? boxes->data_ptr() : nullptr, kc.pages, kc.page_size,
                       ints(block_table), block_table.size(1), ints(lengths), cu_tokens.has_value() ? ints(*cu_tokens) : nullptr,
                       stream_of(q)),
      "iex_paged_append");
  written(k_cache);
  written(v_cache);
  if (boxes.has_value()) written(*boxes);
  return out;
}

at::Tensor paged_attention(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                           const at::Tensor& block_table, const at::Tensor& lengths, const std::optional<at::Tensor>& pages,
                           std::optional<double> scale) {
  check_on(q, {{"q", &q}, {"k_cache", &k_cache}, {"v_cache", &v_cache}, {"block_table", &block_table}, {"lengths", &lengths}});
  const Cache kc = check_cache(k_cache, "k_cache"), vc = check_cache(v_cache, "v_cache");
  TORCH_CHECK(k_cache.sizes() == v_cache.sizes() && k_cache.scalar_type() == v_cache.scalar_type(),
              "k_cache and v_cache must be alike");
  check_q(q, kc.kv_heads, kc.dim, kc.page_size, k_cache.scalar_type());
  check_table(block_table, lengths);
  const int64_t rows = q.size(0), heads = q.size(1);
  TORCH_CHECK(lengths.size(0) == rows, "block_table and lengths must have a row for each of q's");
  int64_t count = 0;
  if (pages.has_value()) {
    check_on(q, {{"pages", &*pages}});
    TORCH_CHECK(pages->scalar_type() == at::kInt && pages->dim() == 3 && pages->size(0) == rows &&
                    pages->size(1) == kc.kv_heads && pages->is_contiguous() && pages->size(2) <= kMostInt,
                "pages must be a contiguous int32 [rows, kv_heads, count]");
    count = pages->size(2);
  }
  const double factor = scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(kc.dim));
  // the kernels' factor, of exponents of 2
  TORCH_CHECK(std::isfinite(static_cast<float>(static_cast<float>(factor) * 1.4426950408889634)),
              "scale * log2(e) must be finite in 32 bits");
  c10::cuda::CUDAGuard guard(q.device());
  at::Tensor out = empty(q, {rows, heads, kc.dim});
  if (rows == 0) return out;
  const Operand qo(q);
  const size_t bytes = iex_paged_attention_workspace_bytes(rows, heads, kc.kv_heads, kc.dim, kc.pages, kc.page_size, block_table.size(1),
                                                           pages.has_value(), count);
  at::Tensor workspace;
  if (bytes > 0) workspace = empty_bytes(q, bytes);
  // a list of no pages is a list all the same
  const int32_t* listed = pages.has_value() ? (count > 0 ? ints(*pages) : ints(lengths)) : nullptr;
  check_status(iex_paged_attention(rows, heads, kc.kv_heads, kc.dim, is_bf16(q), qo.t.data_ptr(), qo.row, qo.head,
                                   k_cache.data_ptr(), kc.page_stride, v_cache.data_ptr(), vc.page_stride, kc.pages,
                                   kc.page_size, ints(block_table), block_table.size(1), ints(lengths), listed, count,
                                   static_cast<float>(factor), out.data_ptr(), bytes > 0 ? workspace.data_ptr() : nullptr, bytes, stream_of(q)),
               "iex_paged_attention");
  return out;
}

at::Tensor paged_select(const at::Tensor& q, const at::Tensor& boxes, const at::Tensor& block_table, const at::Tensor& lengths,
                        int64_t page_size, int64_t count, int64_t first, int64_t last) {
  check_on(q, {{"q", &q}, {"boxes", &boxes}, {"block_table", &block_table}, {"lengths", &lengths}});
  TORCH_CHECK(boxes.dim() == 4 && boxes.size(2) == 2 && boxes.is_contiguous() && boxes.size(0) <= kMostInt &&
                  (reinterpret_cast<uintptr_t>(boxes.data_ptr()) & 15u) == 0,
              "boxes must be a contiguous [pages, kv_heads, 2, head_dim]");
  const int64_t kv_heads = boxes.size(1), rows = q.size(0);
  check_q(q, kv_heads, boxes.size(3), page_size, boxes.scalar_type());
  check_table(block_table, lengths);
  TORCH_CHECK(lengths.size(0) == rows, "block_table and lengths must have a row for each of q's");
  TORCH_CHECK(count >= 1 && count <= kMostInt && first >= 0 && last >= 0 && first <= count && last <= count - first,
              "count must be positive, and first + last at most that; got ", count, ", ", first, " and ", last);
  TORCH_CHECK(block_table.size(1) <= iex_paged_select_max_pages(), "block_table has more than ", iex_paged_select_max_pages(),
              " columns");
  c10::cuda::CUDAGuard guard(q.device());
  at::Tensor pages = empty(lengths, {rows, kv_heads, count});
  if (rows == 0) return pages;
  const Operand qo(q);
  check_status(iex_paged_select(rows, q.size(1), kv_heads, boxes.size(3), is_bf16(q), qo.t.data_ptr(), qo.row, qo.head,
                                boxes.data_ptr(), boxes.size(0), page_size, ints(block_table), block_table.size(1),
                                ints(lengths), count, first, last, pages.data_ptr<int>(), stream_of(q)),
               "iex_paged_select");
  return pages;
}

}  // namespace iex_torch

TORCH_LIBRARY_FRAGMENT(iex_ops, m) {
  m.def("paged_append(Tensor q, Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor block_table, Tensor lengths, Tensor? cu_tokens=None, Tensor? cos=None, Tensor? sin=None, bool interleaved=False, Tensor(c!)? boxes=None) -> Tensor");
  m.def("paged_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, Tensor lengths, Tensor? pages=None, float? scale=None) -> Tensor");
  m.def("paged_select(Tensor q, Tensor boxes, Tensor block_table, Tensor lengths, int page_size, int count, int first=1, int last=1) -> Tensor");
}

TORCH_LIBRARY_IMPL(iex_ops, CUDA, m) {
  m.impl("paged_append", &iex_torch::paged_append);
  m.impl("paged_attention", &iex_torch::paged_attention);
  m.impl("paged_select", &iex_torch::paged_select);
}

TORCH_LIBRARY_IMPL(iex_ops, Autograd, m) {
  for (const char* name : {"paged_append", "paged_attention", "paged_select"})
    m.impl(name, torch::CppFunction::makeFromBoxedFunction<&iex_torch::refuse_derivatives>());
}
