// Attention of one new token per row over a paged key-value cache (paged.cuh):
//
//   out[r, h] = sum_t softmax_t(scale * q[r, h] . k[t]) v[t],   t over the positions that row r holds,
//
// with heads / kv_heads query heads to a key head, or over the positions of the pages that pages[r, kv_head] lists.
#include <cmath>

#include "paged.cuh"

namespace iex {
namespace paged {
namespace {

struct AttentionParams {
  int rows, heads, kv_heads, dim, num_pages, page_shift, table_width, count;
  Rows q;
  const void *k_cache, *v_cache;
  long long k_page, v_page;
  const int32_t *table, *lengths, *pages;
  float scale;
  void* out;
};

// A warp per row and query head, a lane per 32nd element.
template <typename T>
__global__ void __launch_bounds__(32) attention_kernel(const __grid_constant__ AttentionParams p) {
  grid_dependency_wait();
  const int row = blockIdx.x / p.heads, head = blockIdx.x % p.heads, kv = head / (p.heads / p.kv_heads), lane = threadIdx.x;
  const int page = 1 << p.page_shift, held_here = held(p.lengths, row, p.table_width, p.page_shift);
  const int held_pages = (held_here + page - 1) >> p.page_shift, entries = p.pages ? min(p.count, held_pages) : held_pages;
  const T* q = static_cast<const T*>(p.q.data) + row * p.q.row + head * p.q.head;
  float mine[4], acc[4] = {0.f, 0.f, 0.f, 0.f}, top = -INFINITY, total = 0.f;
  for (int i = 0; i < 4; ++i) mine[i] = lane + 32 * i < p.dim ? as_float(q[lane + 32 * i]) * p.scale : 0.f;
  for (int e = 0; e < entries; ++e) {
    const int nth = p.pages ? p.pages[(static_cast<long long>(row) * p.kv_heads + kv) * p.count + e] : e;
    if (nth < 0 || nth >= held_pages) continue;
    const int at = p.table[static_cast<long long>(row) * p.table_width + nth];
    if (at < 0 || at >= p.num_pages) continue;
    const T* k = static_cast<const T*>(p.k_cache) + at * p.k_page + static_cast<long long>(kv) * page * p.dim;
    const T* v = static_cast<const T*>(p.v_cache) + at * p.v_page + static_cast<long long>(kv) * page * p.dim;
    const int here = min(page, held_here - (nth << p.page_shift));
    for (int t = 0; t < here; ++t, k += p.dim, v += p.dim) {
      float s = 0.f;
      for (int i = 0; i < 4; ++i)
        if (lane + 32 * i < p.dim) s = fmaf(mine[i], as_float(k[lane + 32 * i]), s);
      for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
      const float now = fmaxf(top, s), base = now == -INFINITY ? 0.f : now;
      const float old = __expf(top - base), weight = __expf(s - base);
      top = now;
      total = total * old + weight;
      for (int i = 0; i < 4; ++i)
        if (lane + 32 * i < p.dim) acc[i] = acc[i] * old + weight * as_float(v[lane + 32 * i]);
    }
  }
  T* out = static_cast<T*>(p.out) + (static_cast<long long>(row) * p.heads + head) * p.dim;
  for (int i = 0; i < 4; ++i)
    if (lane + 32 * i < p.dim) out[lane + 32 * i] = rounded<T>(total == 0.f ? 0.f : acc[i] / total);
}

}  // namespace
}  // namespace paged
}  // namespace iex

extern "C" int iex_paged_attention_supported(int heads, int kv_heads, int head_dim, int page_size) {
  return iex::paged::heads_ok(heads, kv_heads, head_dim) && iex::paged::page_size_ok(page_size) ? 1 : 0;
}

extern "C" size_t iex_paged_attention_workspace_bytes(int rows, int heads, int kv_heads, int head_dim) { return 0; }

extern "C" int iex_paged_attention(int rows, int heads, int kv_heads, int head_dim, int bf16, const void* q, long long q_row,
                                   long long q_head, const void* k_cache, long long k_page, const void* v_cache,
                                   long long v_page, int num_pages, int page_size, const int32_t* block_table,
                                   int table_width, const int32_t* lengths, const int32_t* pages, int count, float scale,
                                   void* out, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace iex::paged;
  if (rows < 0 || num_pages < 0 || table_width < 0 || count < 0) return IEX_ERR_BAD_ARG;
  if (!iex_paged_attention_supported(heads, kv_heads, head_dim, page_size)) return IEX_ERR_UNSUPPORTED;
  if (rows == 0) return IEX_OK;
  if (!q || !out || !lengths || (table_width > 0 && !block_table) || (num_pages > 0 && (!k_cache || !v_cache)))
    return IEX_ERR_BAD_ARG;
  if (q_row % 8 != 0 || q_head % 8 != 0 || k_page % 8 != 0 || v_page % 8 != 0 || !iex::aligned16(q) || !iex::aligned16(out) ||
      !iex::aligned16(k_cache) || !iex::aligned16(v_cache))
    return IEX_ERR_UNSUPPORTED;
  AttentionParams p{};
  p.rows = rows;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.dim = head_dim;
  p.num_pages = num_pages;
  p.page_shift = log2_of(page_size);
  p.table_width = table_width;
  p.count = count;
  p.q = {q, q_row, q_head};
  p.k_cache = k_cache;
  p.v_cache = v_cache;
  p.k_page = k_page;
  p.v_page = v_page;
  p.table = block_table;
  p.lengths = lengths;
  p.pages = pages;
  p.scale = scale;
  p.out = out;
  const auto kern = bf16 ? attention_kernel<__nv_bfloat16> : attention_kernel<__half>;
  return iex::launch_overlapped(kern, dim3(rows * heads), dim3(32), 0, static_cast<cudaStream_t>(stream), p);
}
