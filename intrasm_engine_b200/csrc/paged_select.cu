// Choosing the pages of a cache (paged.cuh) that a query attends to, from a box per page and key head: the smallest and the
// largest key in each dimension.  A page's score is the most that any key in its box could give, summed over the query
// heads of the key head,
//
//   sum_g sum_d max(q[g, d] lo[d], q[g, d] hi[d]) = sum_d hi[d] sum_g max(q[g, d], 0) + lo[d] sum_g min(q[g, d], 0):
//
// two products a dimension however many query heads there are.  (Where lo or hi is infinite and its factor 0 the right side, which is
// what the score is, is NaN.)  The `first` first and `last` last pages are always taken, then
// those with the largest scores (NaN above all, ties to the lower page).
//
// Which of two pages is taken depends on their scores' difference, so what counts is scores in 64 bits, whose terms are added in one order
// for all pages (equal boxes have equal scores).  But converting a box to 64 bits takes longer than reading it: all pages are scored
// in 32 bits with a bound on the error, the border between taken and not is found, and only where pages lie so near to it that their
// scores in 32 bits do not tell are they scored again (any score that is not finite has all of them scored again).
//
// A cluster of blocks per row and key head: each scores a part of the pages (lanes side by side on a box, eight boxes in flight
// a lane) and stores the scores, as whole numbers of the same order, in the first block's shared memory, which selects: 10 bits at
// a time from the first one in which the largest and the smallest differ, until a digit's pages are all taken (two rounds as
// a rule).  Up to 32 pages near the border are then compared with one another in 64 bits, more of them searched like all were.  So
// many blocks that they fill the GPU, or one each where rows and key heads do.
//
// 1 row of 512 pages, 8 key heads of 128: 6.1 us, latency (lengths and queries, boxes, the cluster's barrier, the search); 16 rows:
// 10.2 us (19 MB of boxes); 256 rows of 256 pages: 37 us, issue slots (70 %; 70 instructions a box and warp, half of them the search's) and 268 MB from L2.
#include <algorithm>

#include <cooperative_groups.h>

#include "paged.cuh"

namespace iex {
namespace paged {
namespace {

namespace cg = cooperative_groups;

constexpr int kMostWarps = 8;     // of a block
constexpr int kAhead = 8;         // boxes that a lane has on their way
constexpr int kMaxPages = 16384, kPageBytes = sizeof(unsigned long long) + sizeof(uint32_t);  // shared memory of each
constexpr int kBits = 10, kBins = 1 << kBits;  // of a round
constexpr int kMostBlocks = 8;                 // of a cluster
constexpr size_t kSmallSmem = 22 * 1024;       // of which an SM has room for 6, beside what is fixed
constexpr uint32_t kFewNear = 32;              // pages near the border that are compared with one another: a lane each

struct SelectParams {
  int rows, heads, kv_heads, dim, num_pages, page_shift, table_width, count, first, last;
  Rows q;
  const void* boxes;
  const int32_t *table, *lengths;
  int32_t* chosen;
};

using Key = unsigned long long;

// Scores as whole numbers of the same order, all above 0; both zeros are one number, NaN is above all.  And the other way round, for numbers.
__device__ __forceinline__ Key ordered(double score) {
  const long long bits = __double_as_longlong(score + 0.0);
  const Key key = static_cast<Key>(bits) ^ (bits < 0 ? ~0ull : 1ull << 63);
  return score != score ? ~0ull : key;
}
__device__ __forceinline__ uint32_t ordered(float score) {
  const int bits = __float_as_int(score + 0.f);
  const uint32_t key = static_cast<uint32_t>(bits) ^ (bits < 0 ? ~0u : 1u << 31);
  return score != score ? ~0u : key;
}
__device__ __forceinline__ float number(uint32_t key) { return __uint_as_float(key >> 31 ? key ^ 1u << 31 : ~key); }

template <typename T>
__device__ __forceinline__ void unpack(const uint4& v, float (&to)[8]) {
  const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
  for (int i = 0; i < 8; ++i) to[i] = as_float(e[i]);
}

// The largest of three without their signs; not NaN where one is a number.
__device__ __forceinline__ float largest_size(float a, float b, float c) {
  float v;
  asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(v) : "f"(a), "f"(b), "f"(c));
  return v;
}

// The sums of v over all threads in front of this one and over all.  `warps` has not been read since the last barrier.
template <int THREADS>
__device__ __forceinline__ uint2 add_in_order(uint32_t v, uint32_t* warps) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t sum = v;
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t other = __shfl_up_sync(0xffffffffu, sum, d);
    sum += lane >= d ? other : 0;
  }
  if (lane == 31) warps[warp] = sum;
  __syncthreads();
  const uint32_t of_warp = lane < THREADS / 32 ? warps[lane] : 0;
  return make_uint2(sum - v + __reduce_add_sync(0xffffffffu, lane < warp ? of_warp : 0), __reduce_add_sync(0xffffffffu, of_warp));
}

// The positive part, NaN if x is.  No branches in what follows: lanes would go their own ways element by element (weighing took 6000
// cycles with them, 400 without).
__device__ __forceinline__ float positive(float x) {
  float v;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(v) : "f"(x), "f"(0.f));
  return v;
}

// What a lane's 8 elements of a box weigh: the sums of the query heads' positive (high) or negative parts.
template <typename T, typename Number>
__device__ __forceinline__ void weigh(const SelectParams& p, int row, int head0, int group, int d, bool high, bool mine,
                                      Number (&weight)[8]) {
  const float sign = high ? 1.f : -1.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) weight[i] = 0;
  for (int g0 = 0; g0 < group; g0 += 4) {
    uint4 some[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      some[g] = make_uint4(0, 0, 0, 0);
      load_if(some[g], static_cast<const T*>(p.q.data) + row * p.q.row + (head0 + g0 + g) * p.q.head + d, mine && g0 + g < group);
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float x[8];
      unpack<T>(some[g], x);
#pragma unroll
      for (int i = 0; i < 8; ++i) weight[i] += positive(sign * x[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) weight[i] *= sign;
}

// A lane's terms of kAhead boxes, added over the LANES lanes of a box: while a lane has several boxes, it gives half of them away and
// adds the other lane's to its own.  Returns which of the boxes is left, in sum[0].
template <int LANES, typename Number>
__device__ __forceinline__ int add_up(Number (&sum)[kAhead]) {
  const int lane = threadIdx.x & 31;
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
        const Number give = upper ? sum[u] : sum[u + width];
        const Number other = __shfl_xor_sync(0xffffffffu, give, off);
        sum[u] = (upper ? sum[u + width] : sum[u]) + other;
      }
    } else {
      sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], off);
    }
  }
  return which;
}

// Where the taken pages begin: all those with keys above `high`, and the first `need` of those with keys from `low` to `high`.
template <typename K>
struct Border {
  K low, high;
  uint32_t need;
};

struct Shared {
  uint32_t bins[3][kBins], groups[3][32];  // keys in a bin, in 32 bins
  // of every warp of the cluster: the most that a page's terms without their signs add up to, as bits; keys
  uint32_t bound[kMostBlocks * kMostWarps], most[kMostBlocks * kMostWarps], least[kMostBlocks * kMostWarps];
  uint32_t warps[2][kMostWarps];
  int near[kFewNear];
};

__device__ __forceinline__ int leading_zeros(uint32_t v) { return __clz(v); }
__device__ __forceinline__ int leading_zeros(Key v) { return __clzll(v); }

template <int THREADS>
__device__ __forceinline__ void clear_bins(Shared& sh, int which) {
#pragma unroll
  for (int i = 0; i < kBins; i += THREADS) sh.bins[which][i + threadIdx.x] = 0;
  if (threadIdx.x < 32) sh.groups[which][threadIdx.x] = 0;
}

// Which of 32 numbers, one a lane, the need-th key is in, counted from the last lane down; need becomes its place in there.
__device__ __forceinline__ int find_lane(uint32_t mine, uint32_t& need, uint32_t& in_lane) {
  const int lane = threadIdx.x & 31;
  uint32_t above = mine;
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t other = __shfl_down_sync(0xffffffffu, above, d);
    above += lane + d < 32 ? other : 0;
  }
  above -= mine;
  const int owner = __ffs(__ballot_sync(0xffffffffu, (above < need) & (need <= above + mine))) - 1;
  in_lane = __shfl_sync(0xffffffffu, mine, owner);
  need -= __shfl_sync(0xffffffffu, above, owner);
  return owner;
}

// The border of the `need` largest of keys [from, to), which are more than that and lie from `least` to `most`; called by all
// threads of the block, with the first bins cleared.
template <int THREADS, typename K>
__device__ __forceinline__ Border<K> find_border(const K* keys, int from, int to, K least, K most, uint32_t need, Shared& sh) {
  const int lane = threadIdx.x & 31;
  if (need == 0) return {static_cast<K>(~K(0)), static_cast<K>(~K(0)), 0};
  constexpr int kRounds = (8 * sizeof(K) + kBits - 1) / kBits;  // each leaves kBits fewer
  for (int round = 0; least != most && round < kRounds; ++round) {
    const K span = most - least;
    const int shift = max(0, static_cast<int>(8 * sizeof(K)) - kBits - leading_zeros(span));  // span >> shift is below kBins
    uint32_t* const bins = sh.bins[round % 3];
    uint32_t* const groups = sh.groups[round % 3];
    clear_bins<THREADS>(sh, (round + 1) % 3);  // last read two rounds ago
    for (int i = from + threadIdx.x; i < to; i += THREADS) {
      const K place = keys[i] - least;
      if (place <= span) {
        atomicAdd(&bins[place >> shift], 1u);
        atomicAdd(&groups[place >> shift >> 5], 1u);
      }
    }
    __syncthreads();
    // every warp for itself
    uint32_t in_bin;
    const int first = find_lane(groups[lane], need, in_bin) * 32;
    const int bin = first + find_lane(bins[first + lane], need, in_bin);
    least += static_cast<K>(bin) << shift;
    most = least + min(most - least, (K(1) << shift) - 1);  // the last bin may reach over the largest number
    if (in_bin == need) break;
  }
  return {least, most, need};
}

// LANES: side by side on a box, 8 elements each.  THREADS, BLOCKS of an SM at once: 256, 2 where there are no more blocks (all of a
// lane's boxes then find registers: 16 rows x 8 key heads x 512 pages take 11 % less than with a third block); else 128, 6 (what every warp does
// for itself counts there: 256 rows x 8 key heads x 256 pages 37 us, with 256, 3 44), or 256, 3 where the scores' shared memory leaves no
// room for 6 (the same with 4096 pages: 453 us, with 128 threads 562, with 256, 2 498).
template <typename T, int LANES, int THREADS, int BLOCKS>
__global__ void __launch_bounds__(THREADS, BLOCKS) select_kernel(const __grid_constant__ SelectParams p) {
  constexpr int kThreads = THREADS, kWarps = THREADS / 32;
  extern __shared__ Key keys64[];  // of all pages, of which the scores in 64 bits are needed; the first block's are used
  uint32_t* const keys = reinterpret_cast<uint32_t*>(keys64 + p.table_width);  // of all pages, in 32 bits
  __shared__ Shared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = cluster.num_blocks(), part = cluster.block_rank(), segment = blockIdx.x / parts;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = segment / p.kv_heads, kv = segment - row * p.kv_heads, group = p.heads / p.kv_heads;
  grid_dependency_wait();
  grid_launch_dependents();
  constexpr int kSides = 32 / LANES, kBatch = kAhead * kSides;  // pages of a warp's turn
  const int along = lane % LANES, side = lane / LANES, d0 = along * 8;
  const bool mine = d0 < 2 * p.dim, upper = d0 >= p.dim;  // upper: of the largest keys
  const int d = d0 - (upper ? p.dim : 0);
  const int32_t* const table = p.table + static_cast<long long>(row) * p.table_width;
  const int from = min(p.first, p.table_width), base0 = from + (part * kWarps + warp) * kBatch;
  // what does not depend on the length is requested beside it
  const int at0 = base0 + lane < p.table_width && lane < kBatch ? table[base0 + lane] : -1;
  const int length = held(p.lengths, row, p.table_width, p.page_shift);
  float weight[8];
  weigh<T>(p, row, kv * group, group, d, upper, mine, weight);
  const int pages = (length + (1 << p.page_shift) - 1) >> p.page_shift;
  int32_t* const chosen = p.chosen + static_cast<long long>(segment) * p.count;
  if (pages <= p.count) {
    if (part == 0)
      for (int i = threadIdx.x; i < p.count; i += kThreads) chosen[i] = i < pages ? i : -1;
    return;
  }
  if (p.num_pages == 0) {  // all are alike
    if (part == 0)
      for (int i = threadIdx.x; i < p.count; i += kThreads) chosen[i] = i < p.count - p.last ? i : pages - p.count + i;
    return;
  }
  if (parts > 1) cluster_begun();
  const int to = pages - p.last;  // [from, to): those that are chosen by their scores

  // ---- scores
  const T* const boxes = static_cast<const T*>(p.boxes) + static_cast<long long>(kv) * 2 * p.dim + d0;
  const uint32_t box_stride = static_cast<uint32_t>(p.kv_heads) * 2 * p.dim;  // kv_heads is below 2^24
  const auto box_of = [&](int where) { return boxes + static_cast<unsigned long long>(static_cast<uint32_t>(where)) * box_stride; };
  const auto real = [&](int where) { return where < p.num_pages ? where : -1; };  // negative where it is not one of the cache's
  const auto look_up = [&](int base) { return real(base + lane < to && lane < kBatch ? table[base + lane] : -1); };
  const auto request = [&](int at, uint4 (&box)[kAhead]) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int where = __shfl_sync(0xffffffffu, at, u * kSides + side);
      box[u] = make_uint4(0, 0, 0, 0);
      load_once_if(box[u], box_of(where), mine ? where : -1);
    }
  };
  const bool holder = along % (LANES / kAhead) == 0;  // one lane for each box that is added up
  {
    const int step = parts * kWarps * kBatch;
    int base = base0;
    int at = real(base + lane < to ? at0 : -1);
    float largest[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};  // of the lane's elements of all boxes, without their signs
    bool finite = true;
    uint32_t key_most = 0, key_least = ~0u;
    uint32_t* const shared_keys = parts > 1 ? cluster.map_shared_rank(keys, 0) : keys;
    bool waited = parts == 1;
    // Loads without conditions (their registers need not be set first): lanes without a piece read the first one, which weighs nothing,
    // and pages that are not the cache's are read as its first one and then not counted.  An infinite value in there makes a score that
    // is not finite, and costs no more than that the pages are scored again.
    const T* const own = boxes - (mine ? 0 : d0);
    for (; base < to; base += step) {
      uint4 box[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int where = max(__shfl_sync(0xffffffffu, at, u * kSides + side), 0);
        box[u] = load_once(own + static_cast<unsigned long long>(static_cast<uint32_t>(where)) * box_stride);
      }
      const int here = at;
      at = look_up(base + step);
      float sum[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; u += 2) {
        float x[2][8];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          unpack<T>(box[u + j], x[j]);
          float2 two = make_float2(0.f, 0.f);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            two = ffma2(make_float2(x[j][2 * i], x[j][2 * i + 1]), make_float2(weight[2 * i], weight[2 * i + 1]), two);
          sum[u + j] = two.x + two.y;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) largest[i] = largest_size(largest[i], x[0][i], x[1][i]);
      }
      const int nth = add_up<LANES>(sum) * kSides + side, where = __shfl_sync(0xffffffffu, here, nth);
      if (!waited) {
        cluster_wait_begun();
        waited = true;
      }
      const uint32_t key = where >= 0 ? ordered(sum[0]) : 0;
      const bool there = holder & (base + nth < to);
      if (there) shared_keys[base + nth] = key;
      key_most = max(key_most, there ? key : 0u);
      key_least = min(key_least, there ? key : ~0u);
      finite &= fabsf(sum[0]) < INFINITY;
    }
    if (!waited) cluster_wait_begun();
    // A sum of the largest elements' terms is no less than that of any page's.
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = fmaf(largest[i], fabsf(weight[i]), most);
    if (!finite) most = INFINITY;
    for (int off = LANES / 2; off > 0; off >>= 1) most += __shfl_xor_sync(0xffffffffu, most, off);
    const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(most));  // NaN is above infinity
    key_most = __reduce_max_sync(0xffffffffu, key_most);
    key_least = __reduce_min_sync(0xffffffffu, key_least);
    if (lane == 0) {
      Shared& first = parts > 1 ? *cluster.map_shared_rank(&sh, 0) : sh;
      first.bound[part * kWarps + warp] = bits;
      first.most[part * kWarps + warp] = key_most;
      first.least[part * kWarps + warp] = key_least;
    }
    if (part == 0) clear_bins<THREADS>(sh, 0);
  }
  if (parts > 1) cluster.sync(); else __syncthreads();
  if (part != 0) return;

  // ---- where the taken ones begin, and the pages that are too near to it
  const uint32_t wanted = p.count - p.first - p.last;  // of the pages [from, to), of which there are more
  uint32_t key_most = 0, key_least = ~0u, bound_bits = 0;
  for (int w = lane; w < parts * kWarps; w += 32) {
    key_most = max(key_most, sh.most[w]);
    key_least = min(key_least, sh.least[w]);
    bound_bits = max(bound_bits, sh.bound[w]);
  }
  key_most = __reduce_max_sync(0xffffffffu, key_most);
  key_least = __reduce_min_sync(0xffffffffu, key_least);
  const float bound = __uint_as_float(__reduce_max_sync(0xffffffffu, bound_bits));
  const Border<uint32_t> border = find_border<THREADS>(keys, from, to, key_least, key_most, wanted, sh);
  // Off by at most: a rounding for each of a lane's 4 products and sums, one for their sum, 5 over lanes and one for every query head,
  // relative to the terms without their signs; and products below the smallest numbers.  The border is off by no more than a page's score.
  const float twice = __fmaf_ru(bound, (group + 16.f) * 0x1p-23f, 1e-40f);
  const uint32_t minus = ordered(-INFINITY), plus = ordered(INFINITY);  // keys below are pages that are not the cache's
  uint32_t low = border.low <= minus ? 0 : ordered(__fsub_rd(number(border.low), twice));
  uint32_t high = border.high <= minus ? minus : border.high >= plus ? ~0u : ordered(__fadd_ru(number(border.high), twice));
  if (!(bound < INFINITY)) low = 0, high = ~0u;
  if (wanted == 0) low = high = ~0u;

  // ---- the chosen pages in order: every thread a run of them
  const int each = (pages + kThreads - 1) / kThreads, begin = threadIdx.x * each, end = min(pages, begin + each);
  {
    // keys above `high` are taken (1), those from `low` on near (1 << 16)
    const auto kind = [&](int i) {
      const uint32_t key = keys[i];
      return (i < from) | (i >= to) | (key > high) ? 1u : (key >= low) & (wanted != 0) ? 1u << 16 : 0u;
    };
    uint32_t mine_of = 0;
    for (int i = begin; i < end; ++i) mine_of += kind(i);
    const uint2 counts = add_in_order<THREADS>(mine_of, sh.warps[0]);
    const uint32_t near = counts.y >> 16, open = p.count - (counts.y & 0xffffu);  // places for the near ones
    if (near <= open || near <= kFewNear) {
      uint32_t taken = ~0u, before = counts.x >> 16;  // which of the near ones are taken; near ones in front of the thread's
      if (near > open) {
        for (int i = begin; i < end; ++i)
          if (kind(i) > 1u) sh.near[before++] = i;
        before = counts.x >> 16;
        double weight[8];
        weigh<T>(p, row, kv * group, group, d, upper, mine, weight);
        __syncthreads();
        for (uint32_t e0 = warp * kSides; e0 < near; e0 += kWarps * kSides) {
          const uint32_t e = e0 + side;
          const int where = real(e < near ? table[sh.near[e]] : -1);
          uint4 box = make_uint4(0, 0, 0, 0);
          load_once_if(box, box_of(where), mine ? where : -1);
          float x[8];
          unpack<T>(box, x);
          double sum = 0.0;
#pragma unroll
          for (int i = 0; i < 8; ++i) sum = fma(static_cast<double>(x[i]), weight[i], sum);
#pragma unroll
          for (int off = LANES / 2; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
          if (along == 0 && e < near) keys64[e] = where >= 0 ? ordered(sum) : 0;
        }
        __syncthreads();
        // every warp for itself: a lane's place among them
        const uint32_t e = lane;
        const Key key = e < near ? keys64[e] : 0;
        uint32_t place = 0;
        for (uint32_t f = 0; f < near; ++f) {
          const Key other = keys64[f];
          place += (other > key) | ((other == key) & (f < e));
        }
        taken = __ballot_sync(0xffffffffu, e < near && place < open);
      }
      const bool all = near <= open;
      uint32_t at = (counts.x & 0xffffu) + (all ? before : __popc(taken & static_cast<uint32_t>((1ull << min(before, 32u)) - 1)));
      for (int i = begin; i < end; ++i) {
        const uint32_t here = kind(i);
        if (here == 1u || (here > 1u && (all || (taken >> before & 1u)))) chosen[at++] = i;
        before += here >> 16;
      }
      return;
    }
  }
  {
    double weight[8];
    weigh<T>(p, row, kv * group, group, d, upper, mine, weight);
    for (int base = from + warp * kBatch; base < to; base += kWarps * kBatch) {
      const bool inside = lane < kBatch && base + lane < to;
      const uint32_t old = inside ? keys[base + lane] : 0;
      const bool near = inside & (old >= low) & (old <= high);
      if (__any_sync(0xffffffffu, near)) {
        const int at = look_up(base);
        uint4 box[kAhead];
        request(at, box);
        double sum[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          float x[8];
          unpack<T>(box[u], x);
          sum[u] = 0.0;
#pragma unroll
          for (int i = 0; i < 8; ++i) sum[u] = fma(static_cast<double>(x[i]), weight[i], sum[u]);
        }
        const int nth = add_up<LANES>(sum) * kSides + side, where = __shfl_sync(0xffffffffu, at, nth);
        const bool near_there = __shfl_sync(0xffffffffu, near, nth);
        if (holder && base + nth < to && near_there) keys64[base + nth] = where >= 0 ? ordered(sum[0]) : 0;
      }
      if (inside && !near) keys64[base + lane] = old > high ? ~0ull : 0;
    }
  }
  clear_bins<THREADS>(sh, 0);
  __syncthreads();
  const Border<Key> exact = find_border<THREADS>(keys64, from, to, Key(0), ~Key(0), wanted, sh);
  // above in the lower half, equal in the upper one; keys outside [from, to) are whatever they are
  const auto kind = [&](int i) {
    const Key key = keys64[i];
    const bool forced = (i < from) | (i >= to);
    return forced | (key > exact.high) ? 1u : key >= exact.low ? 1u << 16 : 0u;
  };
  uint32_t counts = 0;
  for (int i = begin; i < end; ++i) counts += kind(i);
  const uint32_t front = add_in_order<THREADS>(counts, sh.warps[1]).x;
  uint32_t higher = front & 0xffffu, same = front >> 16;
  for (int i = begin; i < end; ++i) {
    const uint32_t here = kind(i), is_above = here & 1u, is_equal = here >> 16;
    if (is_above | (is_equal & (same < exact.need))) chosen[higher + min(same, exact.need)] = i;
    higher += is_above;
    same += is_equal;
  }
}

template <typename T, int LANES, int THREADS, int BLOCKS>
int launch(const SelectParams& p, int parts, size_t smem, cudaStream_t stream) {
  const auto kern = select_kernel<T, LANES, THREADS, BLOCKS>;
  if (smem > 32 * 1024) {
    // the kernel's, not the call's: with one value for all calls, host threads that launch at the same time agree on it
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxPages * kPageBytes);
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  return launch_clusters<SelectParams>(kern, static_cast<unsigned>(p.rows) * p.kv_heads * parts, parts, THREADS, smem, stream, p);
}

template <typename T, int LANES>
int launch(const SelectParams& p, cudaStream_t stream) {
  // two blocks an SM, but a warp's turn of pages for every warp
  const long long segments = static_cast<long long>(p.rows) * p.kv_heads;
  int parts = 1;
  while (parts < kMostBlocks && segments * parts * 2 <= 2 * kNumSMs && p.table_width >= parts * kMostWarps * kAhead) parts *= 2;
  const size_t smem = static_cast<size_t>(std::max(p.table_width, 1)) * kPageBytes;
  if (segments * parts <= 2 * kNumSMs) return launch<T, LANES, 256, 2>(p, parts, smem, stream);
  return smem <= kSmallSmem ? launch<T, LANES, 128, 6>(p, parts, smem, stream) : launch<T, LANES, 256, 3>(p, parts, smem, stream);
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
