// Choosing the pages of a cache (paged.cuh) that a query attends to, from a box per page and key head: the smallest and the
// largest key in each dimension.  A page's score is the most that any key in its box could give, summed over the query
// heads of the key head,
//
//   sum_g sum_d max(q[g, d] lo[d], q[g, d] hi[d]) = sum_d hi[d] sum_g max(q[g, d], 0) + lo[d] sum_g min(q[g, d], 0):
//
// two products a dimension however many query heads there are.  The `first` first and `last` last pages are always taken, then
// those with the largest scores (NaN above all, ties to the lower page).  Scores are summed in 64 bits: which of two pages is
// taken depends on their difference.
#include "paged.cuh"

namespace iex {
namespace paged {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPages = 16384;  // keys of 8 bytes in shared memory

struct SelectParams {
  int rows, heads, kv_heads, dim, num_pages, page_shift, table_width, count, first, last;
  Rows q;
  const void* boxes;
  const int32_t *table, *lengths;
  int32_t* chosen;
};

// Doubles as unsigned numbers of the same order, 1 and above; both zeros are one number, NaN is above all.
__device__ __forceinline__ unsigned long long ordered(double score) {
  if (score != score) return ~0ull - 1;
  const long long bits = __double_as_longlong(score + 0.0);
  const unsigned long long key = static_cast<unsigned long long>(bits) ^ (bits < 0 ? ~0ull : 1ull << 63);
  return key;
}

// A block per row and key head.
template <typename T>
__global__ void __launch_bounds__(kThreads) select_kernel(const __grid_constant__ SelectParams p) {
  extern __shared__ unsigned long long keys[];
  grid_dependency_wait();
  const int row = blockIdx.x / p.kv_heads, kv = blockIdx.x % p.kv_heads, group = p.heads / p.kv_heads;
  const int page = 1 << p.page_shift, length = held(p.lengths, row, p.table_width, p.page_shift);
  const int pages = (length + page - 1) >> p.page_shift;
  int32_t* chosen = p.chosen + (static_cast<long long>(row) * p.kv_heads + kv) * p.count;
  for (int i = threadIdx.x; i < p.count; i += kThreads) chosen[i] = i < pages && pages <= p.count ? i : -1;
  if (pages <= p.count) return;
  const T* q = static_cast<const T*>(p.q.data) + row * p.q.row + kv * group * p.q.head;
  for (int i = threadIdx.x; i < pages; i += kThreads) {
    const int at = p.table[static_cast<long long>(row) * p.table_width + i];
    unsigned long long key = 0;
    if (i < p.first || i >= pages - p.last) {
      key = ~0ull;
    } else if (at >= 0 && at < p.num_pages) {
      const T* box = static_cast<const T*>(p.boxes) + (static_cast<long long>(at) * p.kv_heads + kv) * 2 * p.dim;
      double score = 0.0;
      for (int d = 0; d < p.dim; ++d) {
        double up = 0.0, down = 0.0;
        for (int g = 0; g < group; ++g) {
          const float x = as_float(q[g * p.q.head + d]);
          if (!(x <= 0.f)) up += x;
          if (!(x >= 0.f)) down += x;
        }
        score += as_float(box[p.dim + d]) * up + as_float(box[d]) * down;
      }
      key = ordered(score);
    }
    keys[i] = key;
  }
  __syncthreads();
  // taken: fewer than `count` pages come before it
  uint32_t taken[kMaxPages / kThreads / 32] = {};
  for (int i = threadIdx.x, n = 0; i < pages; i += kThreads, ++n) {
    int before = 0;
    for (int j = 0; j < pages; ++j) before += keys[j] > keys[i] || (keys[j] == keys[i] && j < i);
    if (before < p.count) taken[n / 32] |= 1u << n % 32;
  }
  __syncthreads();
  for (int i = threadIdx.x, n = 0; i < pages; i += kThreads, ++n) keys[i] = taken[n / 32] >> n % 32 & 1u;
  __syncthreads();
  for (int i = threadIdx.x; i < pages; i += kThreads) {
    if (!keys[i]) continue;
    int before = 0;
    for (int j = 0; j < i; ++j) before += static_cast<int>(keys[j]);
    chosen[before] = i;
  }
}

}  // namespace
}  // namespace paged
}  // namespace iex

extern "C" int iex_paged_select_max_pages(void) { return iex::paged::kMaxPages; }

extern "C" int iex_paged_select(int rows, int heads, int kv_heads, int head_dim, int bf16, const void* q, long long q_row,
                                long long q_head, const void* boxes, int num_pages, int page_size,
                                const int32_t* block_table, int table_width, const int32_t* lengths, int count, int first,
                                int last, int32_t* pages, void* stream) {
  using namespace iex::paged;
  if (rows < 0 || num_pages < 0 || table_width < 0 || count <= 0 || first < 0 || last < 0 ||
      static_cast<long long>(first) + last > count)
    return IEX_ERR_BAD_ARG;
  if (!heads_ok(heads, kv_heads, head_dim) || !page_size_ok(page_size)) return IEX_ERR_UNSUPPORTED;
  if (table_width > kMaxPages) return IEX_ERR_TOO_LARGE;
  if (rows == 0) return IEX_OK;
  if (!q || !pages || !lengths || (table_width > 0 && !block_table) || (num_pages > 0 && !boxes)) return IEX_ERR_BAD_ARG;
  if (q_row % 8 != 0 || q_head % 8 != 0 || !iex::aligned16(q) || !iex::aligned16(boxes)) return IEX_ERR_UNSUPPORTED;
  SelectParams p{};
  p.rows = rows;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.dim = head_dim;
  p.num_pages = num_pages;
  p.page_shift = log2_of(page_size);
  p.table_width = table_width;
  p.count = count;
  p.first = first;
  p.last = last;
  p.q = {q, q_row, q_head};
  p.boxes = boxes;
  p.table = block_table;
  p.lengths = lengths;
  p.chosen = pages;
  const auto kern = bf16 ? select_kernel<__nv_bfloat16> : select_kernel<__half>;
  const size_t smem = static_cast<size_t>(table_width) * 8;
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  return iex::launch_overlapped(kern, dim3(rows * kv_heads), dim3(kThreads), smem, static_cast<cudaStream_t>(stream), p);
}
