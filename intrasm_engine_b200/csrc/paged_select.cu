// Choosing the pages of a cache (paged.cuh) that a query attends to, from a box per page and key head: the smallest and the
// largest key in each dimension.  A page's score is the most that any key in its box could give, summed over the query
// heads of the key head,
//
//   sum_g sum_d max(q[g, d] lo[d], q[g, d] hi[d]) = sum_d hi[d] sum_g max(q[g, d], 0) + lo[d] sum_g min(q[g, d], 0):
//
// two products a dimension however many query heads there are.  The `first` first and `last` last pages are always taken, then
// those with the largest scores (NaN above all, ties to the lower page).  Scores are summed in 64 bits: which of two pages is
// taken depends on their difference.  The terms of all pages are added in one order, so equal boxes have equal scores.
//
// A cluster of blocks per row and key head: each scores a part of the pages (lanes side by side on a box, eight boxes in flight
// a lane) and stores the scores, as whole numbers of the same order, in the first block's shared memory, which selects: 8 bits at
// a time from the first one in which the largest and the smallest differ, until a digit's pages are all taken (two rounds as
// a rule).  So many blocks that they fill the GPU, or one each where rows and key heads do.
#include <algorithm>

#include <cooperative_groups.h>

#include "paged.cuh"

namespace iex {
namespace paged {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kAhead = 8;         // boxes that a lane has on their way
constexpr int kMaxPages = 16384;  // keys of 8 bytes in shared memory
constexpr int kBins = 256;

struct SelectParams {
  int rows, heads, kv_heads, dim, num_pages, page_shift, table_width, count, first, last;
  Rows q;
  const void* boxes;
  const int32_t *table, *lengths;
  int32_t* chosen;
};

using Key = unsigned long long;

// Doubles as whole numbers of the same order, all above 0; both zeros are one number, NaN is above all.
__device__ __forceinline__ Key ordered(double score) {
  if (score != score) return ~0ull;
  const long long bits = __double_as_longlong(score + 0.0);
  return static_cast<Key>(bits) ^ (bits < 0 ? ~0ull : 1ull << 63);
}

__device__ __forceinline__ uint4 load_box(const void* p) {  // may have been written by the kernel in front
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}

template <typename T>
__device__ __forceinline__ void unpack(const uint4& v, float (&to)[8]) {
  const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
  for (int i = 0; i < 8; ++i) to[i] = as_float(e[i]);
}

// The sum of v over all threads in front of this one, and over all.
__device__ __forceinline__ uint2 scan(uint32_t v, uint32_t* warps) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t sum = v;
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t other = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += other;
  }
  __syncthreads();
  if (lane == 31) warps[warp] = sum;
  __syncthreads();
  uint32_t front = 0, all = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) front += warps[w];
    all += warps[w];
  }
  return make_uint2(front + sum - v, all);
}

// LANES: side by side on a box, 8 elements each.
template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads) select_kernel(const __grid_constant__ SelectParams p) {
  extern __shared__ Key keys[];  // of all pages; the first block's are used
  __shared__ uint32_t bins[kBins], warp_sums[kWarps];
  __shared__ Key ends[2][kWarps];
  __shared__ uint32_t found[2];
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = cluster.num_blocks(), part = cluster.block_rank(), segment = blockIdx.x / parts;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = segment / p.kv_heads, kv = segment - row * p.kv_heads, group = p.heads / p.kv_heads;
  grid_dependency_wait();
  grid_launch_dependents();
  const int length = held(p.lengths, row, p.table_width, p.page_shift);
  const int pages = (length + (1 << p.page_shift) - 1) >> p.page_shift;
  int32_t* const chosen = p.chosen + static_cast<long long>(segment) * p.count;
  if (pages <= p.count) {
    if (part == 0)
      for (int i = threadIdx.x; i < p.count; i += kThreads) chosen[i] = i < pages ? i : -1;
    return;
  }
  const int from = p.first, to = pages - p.last;  // those that are chosen by their scores

  // ---- scores
  if (parts > 1) cluster.sync();  // the first block has begun: its shared memory may be written
  Key* const shared_keys = parts > 1 ? cluster.map_shared_rank(keys, 0) : keys;
  const int along = lane % LANES, side = lane / LANES;
  const bool mine = along * 8 < 2 * p.dim, high = along * 8 >= p.dim;
  const int d = along * 8 - (high ? p.dim : 0);
  double weight[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) weight[i] = 0.0;
  if (mine)
    for (int g0 = 0; g0 < group; g0 += 4) {
      uint4 some[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        some[g] = make_uint4(0, 0, 0, 0);
        if (g0 + g < group)
          some[g] = load_box(static_cast<const T*>(p.q.data) + row * p.q.row + (kv * group + g0 + g) * p.q.head + d);
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float x[8];
        unpack<T>(some[g], x);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (high ? !(x[i] <= 0.f) : !(x[i] >= 0.f)) weight[i] += x[i];
      }
    }
  constexpr int kSides = 32 / LANES, kBatch = kAhead * kSides;  // pages of a warp's turn
  const int32_t* const table = p.table + static_cast<long long>(row) * p.table_width;
  const T* const boxes = static_cast<const T*>(p.boxes) + static_cast<long long>(kv) * 2 * p.dim + along * 8;
  const long long box_stride = static_cast<long long>(p.kv_heads) * 2 * p.dim;
  const int step = parts * kWarps * kBatch;
  int base = from + (part * kWarps + warp) * kBatch;
  int at = base + lane < to && lane < kBatch ? table[base + lane] : -1;
  for (; base < to; base += step) {
    uint4 box[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int where = __shfl_sync(0xffffffffu, at, u * kSides + side);
      box[u] = make_uint4(0, 0, 0, 0);
      if (mine && where >= 0 && where < p.num_pages) box[u] = load_box(boxes + where * box_stride);
    }
    const int here = at;
    at = base + step + lane < to && lane < kBatch ? table[base + step + lane] : -1;
    double sum[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      float x[8];
      unpack<T>(box[u], x);
      sum[u] = 0.0;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[u] = fma(static_cast<double>(x[i]), weight[i], sum[u]);
    }
    // over the lanes of a box: while a lane has several boxes, it gives half of them away and adds the other lane's to its own
    int width = kAhead, which = 0;
#pragma unroll
    for (int off = LANES / 2; off > 0; off >>= 1) {
      if (width > 1) {
        width >>= 1;
        const bool upper = (lane & off) != 0;
        which = which * 2 + upper;
#pragma unroll
        for (int u = 0; u < kAhead / 2; ++u) {
          if (u >= width) break;
          const double give = upper ? sum[u] : sum[u + width];
          const double other = __shfl_xor_sync(0xffffffffu, give, off);
          sum[u] = (upper ? sum[u + width] : sum[u]) + other;
        }
      } else {
        sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], off);
      }
    }
    // LANES >= 8: one box is left
    const int nth = which * kSides + side, where = __shfl_sync(0xffffffffu, here, nth);
    if (along % (LANES / kAhead) == 0 && base + nth < to)
      shared_keys[base + nth] = where >= 0 && where < p.num_pages ? ordered(sum[0]) : 0;
  }
  if (parts > 1) cluster.sync(); else __syncthreads();
  if (part != 0) return;

  // ---- the smallest score that is taken
  uint32_t need = p.count - p.first - p.last;  // of the pages [from, to), of which there are more
  Key most = 0, least = ~0ull;
  for (int i = from + threadIdx.x; i < to; i += kThreads) {
    most = max(most, keys[i]);
    least = min(least, keys[i]);
  }
  for (int off = 16; off > 0; off >>= 1) {
    most = max(most, __shfl_xor_sync(0xffffffffu, most, off));
    least = min(least, __shfl_xor_sync(0xffffffffu, least, off));
  }
  if (lane == 0) {
    ends[0][warp] = most;
    ends[1][warp] = least;
  }
  __syncthreads();
  for (int w = 0; w < kWarps; ++w) {
    most = max(most, ends[0][w]);
    least = min(least, ends[1][w]);
  }
  // Of the keys that begin with `prefix` (all bits from shift + bits up), the next `bits` bits are looked at.
  int shift = most == least ? 0 : max(0, 56 - __clzll(most ^ least)), bits = 8;
  Key prefix = most >> shift >> 8;
  bool settled = false;  // of the keys whose bits from `shift` up are `prefix`, the first `need` are taken
  if (most == least || need == 0) {
    settled = true;
    shift = 0;
    prefix = need == 0 ? ~0ull : most;
  }
  while (!settled) {
    bins[threadIdx.x] = 0;
    __syncthreads();
    for (int i = from + threadIdx.x; i < to; i += kThreads) {
      const Key key = keys[i] >> shift;
      if (key >> bits == prefix) atomicAdd(&bins[key & ((1u << bits) - 1)], 1u);
    }
    __syncthreads();
    const int bin = kBins - 1 - threadIdx.x;  // threads from the highest bin down
    const uint32_t in_bin = bins[bin], above = scan(in_bin, warp_sums).x;
    if (above < need && need <= above + in_bin) {
      found[0] = bin;
      found[1] = above;
    }
    __syncthreads();
    prefix = prefix << bits | found[0];
    need -= found[1];
    settled = shift == 0 || bins[found[0]] == need;
    if (!settled) {
      bits = min(8, shift);
      shift -= bits;
    }
    __syncthreads();
  }

  // ---- the chosen pages in order: every thread a run of them
  const int each = (pages + kThreads - 1) / kThreads, begin = threadIdx.x * each, end = min(pages, begin + each);
  const auto above = [&](int i) { return i < from || i >= to || keys[i] >> shift > prefix; };
  const auto equal = [&](int i) { return i >= from && i < to && keys[i] >> shift == prefix; };
  uint32_t counts = 0;  // above in the lower half, equal in the upper one
  for (int i = begin; i < end; ++i) counts += above(i) ? 1u : equal(i) ? 1u << 16 : 0u;
  const uint32_t front = scan(counts, warp_sums).x;
  uint32_t higher = front & 0xffffu, same = front >> 16;
  for (int i = begin; i < end; ++i) {
    if (above(i)) {
      chosen[higher + min(same, need)] = i;
      ++higher;
    } else if (equal(i)) {
      if (same < need) chosen[higher + same] = i;
      ++same;
    }
  }
}

template <typename T, int LANES>
int launch(const SelectParams& p, cudaStream_t stream) {
  const auto kern = select_kernel<T, LANES>;
  const size_t smem = static_cast<size_t>(std::max(p.table_width, 1)) * sizeof(Key);
  if (smem > 40 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  // two blocks an SM, but a warp's turn of pages for every warp
  const long long segments = static_cast<long long>(p.rows) * p.kv_heads;
  int parts = 1;
  while (parts < 8 && segments * parts * 2 <= 2 * kNumSMs && p.table_width >= parts * 2 * kWarps * kAhead / 2) parts *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(segments * parts));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = parts;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
  return static_cast<int>(e != cudaSuccess ? e : cudaGetLastError());
}

template <typename T>
int launch(const SelectParams& p, cudaStream_t stream) {
  if (p.dim <= 32) return launch<T, 8>(p, stream);
  return p.dim <= 64 ? launch<T, 16>(p, stream) : launch<T, 32>(p, stream);
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
  if (table_width > kMaxPages || static_cast<long long>(rows) * kv_heads > (1ll << 28)) return IEX_ERR_TOO_LARGE;
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
  return bf16 ? launch<__nv_bfloat16>(p, static_cast<cudaStream_t>(stream))
              : launch<__half>(p, static_cast<cudaStream_t>(stream));
}
