// Appending the keys and values of new tokens to a paged cache (paged.cuh), rotated by their positions on the way, with the
// queries rotated beside them.
//
// Sequence i has n = cu_tokens[i + 1] - cu_tokens[i] new tokens (one without cu_tokens); its j-th new token takes position
// lengths[i] - n + j.  Of every query and key the first `rotary` elements are turned in pairs by the angles of the position,
//   (a, b) -> (a cos - b sin, b cos + a sin),   pairs (i, i + rotary / 2), or (2 i, 2 i + 1) if interleaved,
// in fp32, and rounded once.  boxes (optional) holds the smallest and largest key of every page and head in each dimension: of a
// page that is written to they are formed anew from all its positions up to the last new one.
//
// A block does one page's new tokens of one key head and its query heads, so that a box has one writer.
#include "paged.cuh"

namespace iex {
namespace paged {
namespace {

constexpr int kThreads = 128;

struct AppendParams {
  int tokens, batch, heads, kv_heads, dim, rope_rows, rotary, interleaved, num_pages, page_shift, table_width;
  Rows q, k, v;
  const float *cos, *sin;
  void *q_out, *k_cache, *v_cache, *boxes;
  long long k_page, v_page;
  const int32_t *table, *lengths, *cu_tokens;
};

__device__ __forceinline__ __half smaller(__half a, __half b) { return __hmin_nan(a, b); }
__device__ __forceinline__ __half larger(__half a, __half b) { return __hmax_nan(a, b); }
__device__ __forceinline__ __nv_bfloat16 smaller(__nv_bfloat16 a, __nv_bfloat16 b) { return __hmin_nan(a, b); }
__device__ __forceinline__ __nv_bfloat16 larger(__nv_bfloat16 a, __nv_bfloat16 b) { return __hmax_nan(a, b); }

// Where the tokens of sequence i begin among the rows.
__device__ __forceinline__ int begin_of(const AppendParams& p, int i) {
  return p.cu_tokens ? min(max(p.cu_tokens[i], 0), p.tokens) : i;
}

// Blocks are laid out by what a sequence needs at most: the n tokens of a sequence touch up to n / page + 2 pages, and
// floor(begin / page) + 2 i blocks are enough for all the sequences in front.
__device__ __forceinline__ int first_block(const AppendParams& p, int i) {
  return p.cu_tokens ? (begin_of(p, i) >> p.page_shift) + 2 * i : i;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) append_kernel(const __grid_constant__ AppendParams p) {
  grid_dependency_wait();
  const int block = blockIdx.x / p.kv_heads, blocks = gridDim.x / p.kv_heads, kv = blockIdx.x % p.kv_heads;
  const int group = p.heads / p.kv_heads, page = 1 << p.page_shift, d = threadIdx.x;
  T* q_out = static_cast<T*>(p.q_out) + static_cast<long long>(kv) * group * p.dim;
  const auto clear = [&](int row) {
    for (int g = 0; g < group; ++g)
      if (d < p.dim) q_out[(static_cast<long long>(row) * p.heads + g) * p.dim + d] = rounded<T>(0.f);
  };
  for (int row = begin_of(p, p.batch) + block; row < p.tokens; row += blocks) clear(row);
  if (p.batch == 0) return;

  int i = 0;
  for (int beyond = p.batch; beyond - i > 1;) {  // the last sequence whose blocks begin here or in front
    const int mid = (i + beyond) / 2;
    if (first_block(p, mid) <= block) i = mid; else beyond = mid;
  }
  const int begin = begin_of(p, i), n = begin_of(p, i + 1) - begin;
  if (n <= 0) return;
  const int length = p.lengths[i], start = length - n;  // the first new token's position
  const int nth = (max(start, 0) >> p.page_shift) + block - first_block(p, i);
  const long long page_begin = static_cast<long long>(nth) << p.page_shift;
  const int from = static_cast<int>(max(static_cast<long long>(start), page_begin));
  const int to = static_cast<int>(min(static_cast<long long>(length), page_begin + page));
  if (block == first_block(p, i))
    for (int j = 0; j < min(n, -start); ++j) clear(begin + j);
  if (from >= to) return;
  const int at = nth < p.table_width ? p.table[static_cast<long long>(i) * p.table_width + nth] : -1;
  const bool known = at >= 0 && at < p.num_pages;
  const int half = p.rotary / 2;
  const int other = d >= p.rotary ? d : p.interleaved ? d ^ 1 : d < half ? d + half : d - half;  // the pair's other element
  const bool second = d < p.rotary && (p.interleaved ? d & 1 : d >= half);
  const int angle = p.interleaved ? d / 2 : d % max(half, 1);
  T lo, hi;
  bool any = false;
  for (int position = from; position < to; ++position) {
    const int row = begin + position - start;
    if (!known || (p.rotary > 0 && position >= p.rope_rows)) {
      clear(row);
      continue;
    }
    if (d >= p.dim) continue;
    float c = 1.f, s = 0.f;
    if (d < p.rotary) {
      c = p.cos[static_cast<long long>(position) * half + angle];
      s = p.sin[static_cast<long long>(position) * half + angle];
      if (!second) s = -s;
    }
    const auto turned = [&](const Rows& x, int head) {
      const T* v = static_cast<const T*>(x.data) + row * x.row + head * x.head;
      return d < p.rotary ? rounded<T>(fmaf(as_float(v[d]), c, as_float(v[other]) * s)) : v[d];
    };
    for (int g = 0; g < group; ++g)
      q_out[(static_cast<long long>(row) * p.heads + g) * p.dim + d] = turned(p.q, kv * group + g);
    const long long slot = (static_cast<long long>(kv) * page + position % page) * p.dim + d;
    const T key = turned(p.k, kv);
    static_cast<T*>(p.k_cache)[at * p.k_page + slot] = key;
    static_cast<T*>(p.v_cache)[at * p.v_page + slot] = (static_cast<const T*>(p.v.data) + row * p.v.row + kv * p.v.head)[d];
    lo = any ? smaller(lo, key) : key;
    hi = any ? larger(hi, key) : key;
    any = true;
  }
  if (p.boxes != nullptr && any) {
    const T* held_keys = static_cast<const T*>(p.k_cache) + at * p.k_page + static_cast<long long>(kv) * page * p.dim + d;
    for (int slot = 0; slot < from % page; ++slot) {
      lo = smaller(lo, held_keys[slot * p.dim]);
      hi = larger(hi, held_keys[slot * p.dim]);
    }
    T* box = static_cast<T*>(p.boxes) + (static_cast<long long>(at) * p.kv_heads + kv) * 2 * p.dim + d;
    box[0] = lo;
    box[p.dim] = hi;
  }
}

}  // namespace
}  // namespace paged
}  // namespace iex

extern "C" int iex_paged_append(int tokens, int batch, int heads, int kv_heads, int head_dim, int bf16, const void* q,
                                long long q_row, long long q_head, const void* k, long long k_row, long long k_head,
                                const void* v, long long v_row, long long v_head, const float* cos, const float* sin,
                                int rope_rows, int rotary, int interleaved, void* q_out, void* k_cache, long long k_page,
                                void* v_cache, long long v_page, void* boxes, int num_pages, int page_size,
                                const int32_t* block_table, int table_width, const int32_t* lengths,
                                const int32_t* cu_tokens, void* stream) {
  using namespace iex::paged;
  if (tokens < 0 || batch < 0 || num_pages < 0 || table_width < 0 || rope_rows < 0 || rotary < 0) return IEX_ERR_BAD_ARG;
  if (!heads_ok(heads, kv_heads, head_dim) || !page_size_ok(page_size) || rotary % 2 != 0 || rotary > head_dim)
    return IEX_ERR_UNSUPPORTED;
  if (tokens == 0) return IEX_OK;
  if (!q || !k || !v || !q_out || (batch > 0 && !lengths) || (rotary > 0 && (!cos || !sin)) ||
      (batch > 0 && table_width > 0 && !block_table) || (num_pages > 0 && (!k_cache || !v_cache)) ||
      (!cu_tokens && tokens != batch))
    return IEX_ERR_BAD_ARG;
  for (const long long stride : {q_row, q_head, k_row, k_head, v_row, v_head, k_page, v_page})
    if (stride % 8 != 0) return IEX_ERR_UNSUPPORTED;
  for (const void* address : {q, k, v, static_cast<const void*>(q_out), static_cast<const void*>(k_cache),
                              static_cast<const void*>(v_cache), static_cast<const void*>(boxes)})
    if (!iex::aligned16(address)) return IEX_ERR_UNSUPPORTED;
  AppendParams p{};
  p.tokens = tokens;
  p.batch = batch;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.dim = head_dim;
  p.rope_rows = rope_rows;
  p.rotary = rotary;
  p.interleaved = interleaved;
  p.num_pages = num_pages;
  p.page_shift = log2_of(page_size);
  p.table_width = table_width;
  p.q = {q, q_row, q_head};
  p.k = {k, k_row, k_head};
  p.v = {v, v_row, v_head};
  p.cos = cos;
  p.sin = sin;
  p.q_out = q_out;
  p.k_cache = k_cache;
  p.v_cache = v_cache;
  p.boxes = boxes;
  p.k_page = k_page;
  p.v_page = v_page;
  p.table = block_table;
  p.lengths = lengths;
  p.cu_tokens = cu_tokens;
  const long long blocks = (cu_tokens ? (tokens >> p.page_shift) + 2ll * batch + 1 : batch) * kv_heads;
  if (blocks > 0x7fffffffll) return IEX_ERR_TOO_LARGE;
  const auto kern = bf16 ? append_kernel<__nv_bfloat16> : append_kernel<__half>;
  return iex::launch_overlapped(kern, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0,
                                static_cast<cudaStream_t>(stream), p);
}
