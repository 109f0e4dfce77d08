// Attention over listed pages (paged_attention.cu) where many rows list the same ones: the queries of a prompt's piece against
// one sequence, or sequences with a common beginning.
//
// Row by row, every row and key head reads its pages from L2 (256 rows x 8 heads x 16 pages of 64 x 128: 1.07 GB, 9.1 TB/s, 118 us).
// Here a page is read once for up to 64 of the (entry, query head) pairs that list it: index_kernel sorts the entries of the lists
// by page, page_kernel forms the softmax and the product of such a tile with its page, join_entries_kernel adds up each row's
// entries in the order of its list.  What is written and read between them, a product of fp32 for every entry and query head, is
// 2 G / page of the keys and values that would be read (G query heads to a key head).  83 us at the same sizes: 11 us of sorting
// (latency), 63 us of page_kernel (378 MB through L2, 6 TB/s), 18 us of joining (108 MB, 6 TB/s), with their launches overlapped; 96
// us instead of 420 where each of 32 key heads has its own query head.
//
// page_kernel: keys and values of 64 positions and the queries in shared memory (rows of 16 bytes more than they have, so that
// eight of them lie in different banks), a warp has 16 of the pairs: S = Q K^T by m16n8k16, whose accumulators are the fragments
// of P in O = P V; P enters as a 16-bit head and rest.
//
// Rows of one tile see different numbers of the page's positions.  An infinite or NaN value of v that one row sees must not
// reach the others (0 x Inf): rows whose product comes out not finite are summed again, position by position, and, as large bfloat16
// values may be the reason, handed on as averages.
#include <algorithm>

#include <cooperative_groups.h>

#include "paged_mma.cuh"
#include "paged_shared.cuh"

namespace iex {
namespace paged {
namespace {

namespace cg = cooperative_groups;

constexpr int kIndexThreads = 1024;
constexpr int kTileRows = 64, kThreads = 128, kPositions = 64;
constexpr int kMostPages = 16384, kPageBytes = 3 * sizeof(int);  // shared memory of each
constexpr int kIndexBlocks = 8;    // of a cluster, at most
constexpr int kMostGroup = 16;
constexpr size_t kMostScratch = 512u << 20;  // of a call; entries are then fewer than 2^24

struct Item {
  int page, begin, n, most;  // entries list[begin .. begin + n) of the head; positions of the page that any entry sees
};

struct Params {
  SharedCall c;
  int entries, tile_entries, most_items;  // rows x count; of a tile; a head's items at most
  int* items_of;   // [kv_heads]
  Item* items;     // [kv_heads][most_items]
  int2* seen;      // [kv_heads][entries]: page or -1, positions of it that the row sees
  int2* list;      // [kv_heads][entries], by page: entry, positions
  float2* stats;   // [kv_heads][entries][group]: base and sum; base -inf where there is nothing
  float* product;  // [kv_heads][entries][group][dim]
};

// A cluster for each key head: counts the entries of every page, and writes them page by page.  In which order a page's entries come
// makes no difference: an entry's sums depend on nothing else of its tile.  Lookups and writes go everywhere, 32 places a warp: one
// block alone takes 9 us for 4096 entries, eight take 6; 26 and 10 for 16384.
__global__ void __launch_bounds__(kIndexThreads) index_kernel(const __grid_constant__ Params p) {
  extern __shared__ int counters[];  // of the pages: entries of this block; the most positions that one sees; where the next one goes
  __shared__ unsigned long long warps[32];
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = cluster.num_blocks(), rank = cluster.block_rank();
  grid_dependency_wait();
  grid_launch_dependents();
  const SharedCall& c = p.c;
  int *const most = counters + c.num_pages, *const next = most + c.num_pages;
  const int kv = blockIdx.x / blocks, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = c.heads / c.kv_heads;
  int2* const seen = p.seen + static_cast<long long>(kv) * p.entries;
  for (int i = threadIdx.x; i < 2 * c.num_pages; i += kIndexThreads) counters[i] = 0;
  __syncthreads();
  const int each_block = (p.entries + blocks - 1) / blocks, first = rank * each_block + threadIdx.x;
  const int last = min(p.entries, (rank + 1) * each_block);
  // kAhead entries of a thread at once, in steps without branches, as they take three loads after one another
  constexpr int kAhead = 4;
  const int page = 1 << c.page_shift;
  for (int e0 = first; e0 < last; e0 += kAhead * kIndexThreads) {
    int row[kAhead], nth[kAhead], length[kAhead], at[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int e = min(e0 + u * kIndexThreads, last - 1);
      row[u] = e / c.count;
      const int i = e - row[u] * c.count;
      length[u] = held(c.lengths, row[u], c.table_width, c.page_shift);
      nth[u] = c.pages[(static_cast<long long>(row[u]) * c.kv_heads + kv) * c.count + i];
      if (i >= (length[u] + page - 1) >> c.page_shift) length[u] = 0;  // an entry that does not count
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      at[u] = c.table[static_cast<long long>(row[u]) * c.table_width + min(max(nth[u], 0), c.table_width - 1)];
      const bool there = nth[u] >= 0 && nth[u] < (length[u] + page - 1) >> c.page_shift;
      length[u] = there ? min(page, length[u] - (nth[u] << c.page_shift)) : 0;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int e = e0 + u * kIndexThreads;
      if (e >= last) break;
      const bool there = length[u] > 0 && at[u] >= 0 && at[u] < c.num_pages;
      seen[e] = make_int2(there ? at[u] : -1, length[u]);
      if (there) {
        atomicAdd(&counters[at[u]], 1);
        atomicMax(&most[at[u]], length[u]);
      } else {
        float2* const stats = p.stats + (static_cast<long long>(kv) * p.entries + e) * group;
        for (int g = 0; g < group; ++g) stats[g] = make_float2(-INFINITY, 0.f);
      }
    }
  }
  cluster.sync();
  // entries (lower half) and items (upper half) of the pages in front; a thread has a run of pages
  const int each = (c.num_pages + kIndexThreads - 1) / kIndexThreads;
  const int from = min(c.num_pages, static_cast<int>(threadIdx.x) * each), to = min(c.num_pages, from + each);
  const auto items_for = [&](int n) { return (n + p.tile_entries - 1) / p.tile_entries; };
  struct Page {
    int all, in_front, most;  // entries of all blocks, of those in front of this one
  };
  const auto count = [&](int i) {
    Page found{0, 0, 0};
    for (int b = 0; b < blocks; ++b) {
      const int* const theirs = cluster.map_shared_rank(counters, b);
      const int n = theirs[i];
      found.all += n;
      found.in_front += b < rank ? n : 0;
      found.most = max(found.most, theirs[c.num_pages + i]);
    }
    return found;
  };
  unsigned long long mine = 0;
  for (int i = from; i < to; ++i) {
    const int n = count(i).all;
    mine += static_cast<unsigned long long>(items_for(n)) << 32 | static_cast<unsigned>(n);
  }
  unsigned long long sum = mine;
  for (int d = 1; d < 32; d <<= 1) {
    const unsigned long long other = __shfl_up_sync(0xffffffffu, sum, d);
    sum += lane >= d ? other : 0;
  }
  if (lane == 31) warps[warp] = sum;
  __syncthreads();
  unsigned long long front = 0;
  for (int w = 0; w < warp; ++w) front += warps[w];
  front += sum - mine;
  int list_at = static_cast<int>(front & 0xffffffffu), item_at = static_cast<int>(front >> 32);
  Item* const items = p.items + static_cast<long long>(kv) * p.most_items;
  for (int i = from; i < to; ++i) {
    const Page here = count(i);
    if (rank == 0)
      for (int begin = 0; begin < here.all; begin += p.tile_entries)
        items[item_at++] = {i, list_at + begin, min(p.tile_entries, here.all - begin), here.most};
    next[i] = list_at + here.in_front;
    list_at += here.all;
  }
  if (rank == 0 && threadIdx.x == kIndexThreads - 1) p.items_of[kv] = item_at;
  __syncthreads();
  int2* const list = p.list + static_cast<long long>(kv) * p.entries;
  for (int e0 = first; e0 < last; e0 += kAhead * kIndexThreads) {
    int2 here[kAhead];
    int to[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int e = e0 + u * kIndexThreads;
      here[u] = e < last ? seen[e] : make_int2(-1, 0);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) to[u] = here[u].x >= 0 ? atomicAdd(&next[here[u].x], 1) : -1;
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (to[u] >= 0) list[to[u]] = make_int2(e0 + u * kIndexThreads, here[u].y);
  }
  cluster.sync();  // others may read this block's counters until then
}

__device__ __forceinline__ uint32_t smem(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t address) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(address));
}
__device__ __forceinline__ void load_transposed(uint32_t (&r)[4], uint32_t address) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(address));
}
// 16 bytes to shared memory, or zeros.
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}

// PIECES: of 64 elements of a head.
template <typename T, int PIECES>
__global__ void __launch_bounds__(kThreads) page_kernel(const __grid_constant__ Params p) {
  constexpr int kDim = 64 * PIECES, kPitch = kDim + 8, kPieces16 = kDim / 8;
  extern __shared__ __align__(16) unsigned char tiles[];
  T* const q_tile = reinterpret_cast<T*>(tiles);
  T* const k_tile = q_tile + kTileRows * kPitch;
  T* const v_tile = k_tile + kPositions * kPitch;
  __shared__ int entry_of[kTileRows], valid_of[kTileRows];
  grid_dependency_wait();
  const SharedCall& c = p.c;
  const int kv = blockIdx.y, group = c.heads / c.kv_heads, page = 1 << c.page_shift;
  const int items = p.items_of[kv];
  const Item item = p.items[static_cast<long long>(kv) * p.most_items + blockIdx.x];  // not one, behind the last
  if (static_cast<int>(blockIdx.x) >= items) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3, rows = item.n * group, most = item.most;
  const T* const k_page = static_cast<const T*>(c.k_cache) + item.page * c.k_page + static_cast<long long>(kv) * page * c.dim;
  const T* const v_page = static_cast<const T*>(c.v_cache) + item.page * c.v_page + static_cast<long long>(kv) * page * c.dim;

  const auto request_tile = [&](int begin) {
    for (int x = threadIdx.x; x < kPositions * kPieces16; x += kThreads) {
      const int t = x / kPieces16, d = x % kPieces16 * 8;
      const bool there = begin + t < most && d < c.dim;
      const long long at = there ? static_cast<long long>(begin + t) * c.dim + d : 0;
      copy16(smem(k_tile + t * kPitch + d), k_page + at, there);
      copy16(smem(v_tile + t * kPitch + d), v_page + at, there);
    }
  };
  request_tile(0);
  // pair m of the tile: entry m / group, query head m % group
  if (threadIdx.x < kTileRows) {
    const int m = threadIdx.x;
    const int2 here = m < rows ? p.list[static_cast<long long>(kv) * p.entries + item.begin + m / group] : make_int2(-1, 0);
    entry_of[m] = here.x;
    valid_of[m] = here.y;
  }
  __syncthreads();
  for (int x = threadIdx.x; x < kTileRows * kPieces16; x += kThreads) {
    const int m = x / kPieces16, d = x % kPieces16 * 8, entry = entry_of[m];
    const bool there = entry >= 0 && d < c.dim;
    const T* const from = static_cast<const T*>(c.q.data) +
                          (there ? entry / c.count * c.q.row + (kv * group + m % group) * c.q.head + d : 0);
    copy16(smem(q_tile + m * kPitch + d), from, there);
  }

  float o[kDim / 8][4], base[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
#pragma unroll
  for (int n = 0; n < kDim / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
  const bool busy = warp * 16 < rows;
  const int valid[2] = {valid_of[warp * 16 + g], valid_of[warp * 16 + g + 8]};
  for (int begin = 0; begin < most; begin += kPositions) {
    if (begin > 0) {
      __syncthreads();  // the tile in front has been read
      request_tile(begin);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    if (!busy) continue;
    float s[kPositions / 8][4];
#pragma unroll
    for (int n = 0; n < kPositions / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
    for (int k = 0; k < kDim / 16; ++k) {
      uint32_t a[4];
      load_matrices(a, smem(q_tile + (warp * 16 + lane % 16) * kPitch + k * 16 + lane / 16 * 8));
#pragma unroll
      for (int n = 0; n < kPositions / 8; n += 2) {
        uint32_t b[4];  // positions 8 n .. 8 n + 15
        load_matrices(b, smem(k_tile + (n * 8 + lane / 16 * 8 + lane % 8) * kPitch + k * 16 + lane / 8 % 2 * 8));
        mma<T>(s[n], a[0], a[1], a[2], a[3], b[0], b[1]);
        mma<T>(s[n + 1], a[0], a[1], a[2], a[3], b[2], b[3]);
      }
    }
    // s[n][e]: pair g + (e & 2) * 4 of the warp's, position 8 n + 2 q + (e & 1)
    float high[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < kPositions / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] = begin + n * 8 + 2 * q + (e & 1) < valid[e / 2] ? s[n][e] * c.scale_log2 : -INFINITY;
        high[e / 2] = fmaxf(high[e / 2], s[n][e]);
      }
    float old[2], from[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      high[r] = fmaxf(high[r], __shfl_xor_sync(0xffffffffu, high[r], 1));
      high[r] = fmaxf(base[r], fmaxf(high[r], __shfl_xor_sync(0xffffffffu, high[r], 2)));
      from[r] = high[r] == -INFINITY ? 0.f : high[r];
      old[r] = exp2f(base[r] - from[r]);
      base[r] = high[r];
      sum[r] *= old[r];
    }
#pragma unroll
    for (int n = 0; n < kDim / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][e] *= old[e / 2];
#pragma unroll
    for (int j = 0; j < kPositions / 16; ++j) {
      uint32_t head[4], rest[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // fragment i: pairs g + (i & 1) * 8, positions 16 j + (i / 2) * 8 + 2 q
        float w[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          w[e] = exp2f(s[2 * j + i / 2][(i & 1) * 2 + e] - from[i & 1] + Half2<T>::kBias);
          sum[i & 1] += w[e];
        }
        head[i] = Half2<T>::pack(w[0], w[1]);
        const float2 kept = Half2<T>::unpack(head[i]);
        rest[i] = Half2<T>::pack(w[0] - kept.x, w[1] - kept.y);
      }
#pragma unroll
      for (int n = 0; n < kDim / 8; n += 2) {
        uint32_t b[4];
        load_transposed(b, smem(v_tile + (j * 16 + lane % 16) * kPitch + n * 8 + lane / 16 * 8));
        mma<T>(o[n], head[0], head[1], head[2], head[3], b[0], b[1]);
        mma<T>(o[n], rest[0], rest[1], rest[2], rest[3], b[0], b[1]);
        mma<T>(o[n + 1], head[0], head[1], head[2], head[3], b[2], b[3]);
        mma<T>(o[n + 1], rest[0], rest[1], rest[2], rest[3], b[2], b[3]);
      }
    }
  }
  grid_launch_dependents();
  if (!busy) return;
  bool odd[2] = {false, false};
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
    sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
  }
#pragma unroll
  for (int n = 0; n < kDim / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) odd[e / 2] |= !(fabsf(o[n][e]) < INFINITY);
  const long long head_at = static_cast<long long>(kv) * p.entries;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int m = warp * 16 + g + 8 * r;
    if (m >= rows) continue;
    const long long slot = (head_at + entry_of[m]) * group + m % group;
    float* const to = p.product + slot * c.dim;
#pragma unroll
    for (int n = 0; n < kDim / 8; ++n)
      if (n * 8 < c.dim) *reinterpret_cast<float2*>(to + n * 8 + 2 * q) = make_float2(o[n][2 * r], o[n][2 * r + 1]);
    if (q == 0) p.stats[slot] = make_float2(base[r], sum[r]);
  }
  // rows that are not finite, again: of the four lanes of a row any may have seen it
#pragma unroll 1
  for (int r = 0; r < 2; ++r) {
    uint32_t found = __ballot_sync(0xffffffffu, odd[r] && warp * 16 + g + 8 * r < rows);
    while (found != 0) {
      const int row_here = (__ffs(found) - 1) / 4, m = warp * 16 + row_here + 8 * r;
      found &= ~(0xfu << row_here * 4);
      const long long slot = (head_at + entry_of[m]) * group + m % group;
      const int d = lane * 4;
      constexpr float kSmall = Half2<T>::kOverflows ? 1.f / (2 * kMaxPage) : 1.f;  // of which the page's sum does not overflow
      float top = -INFINITY, total = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
      for (int t = 0; t < valid_of[m]; ++t) {
        float score = 0.f;
        if (d < c.dim)
          for (int i = 0; i < 4; ++i) score = fmaf(as_float(q_tile[m * kPitch + d + i]), as_float(k_page[static_cast<long long>(t) * c.dim + d + i]), score);
        for (int x = 16; x > 0; x >>= 1) score += __shfl_xor_sync(0xffffffffu, score, x);
        score *= c.scale_log2;
        const float now = fmaxf(top, score), zero = now == -INFINITY ? 0.f : now;
        const float before = exp2f(top - zero), weight = exp2f(score - zero + Half2<T>::kBias);
        top = now;
        total = total * before + weight;
        if (d < c.dim)
          for (int i = 0; i < 4; ++i) acc[i] = acc[i] * before + weight * kSmall * as_float(v_page[static_cast<long long>(t) * c.dim + d + i]);
      }
      if (Half2<T>::kOverflows) {
        const float factor = to_average<T>(total);
        for (float& v : acc) v = v * factor * (1.f / kSmall);
        total = -total;
      }
      __syncwarp();
      if (d < c.dim) *reinterpret_cast<float4*>(p.product + slot * c.dim + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      if (lane == 0) p.stats[slot] = make_float2(top, total);
    }
  }
}

// Four elements of a query head's average, where an entry's are averages; total: of the weights.
template <typename T>
__device__ __noinline__ void join_averages(const Params& p, long long first, int g, int group, int d, float base, float unit, float total,
                                           float (&o)[4]) {
  const SharedCall& c = p.c;
  const float factor = to_average<T>(total);
  o[0] = o[1] = o[2] = o[3] = 0.f;
  for (int i = 0; i < c.count; ++i) {
    const long long slot = first + static_cast<long long>(i) * group + g;
    const float2 s = p.stats[slot];
    if (s.x == -INFINITY && s.y == 0.f) continue;
    const float4 v = *reinterpret_cast<const float4*>(p.product + slot * c.dim + d);
    const float weight = exp2f(s.x - base) * unit * factor * (averaged<T>(s.y) ? -s.y : 1.f);
    o[0] += v.x * weight;
    o[1] += v.y * weight;
    o[2] += v.z * weight;
    o[3] += v.w * weight;
  }
}

// A block for each row and key head; a thread has four elements of a query head.
template <typename T>
__global__ void __launch_bounds__(kThreads) join_entries_kernel(const __grid_constant__ Params p) {
  grid_dependency_wait();
  grid_launch_dependents();
  const SharedCall& c = p.c;
  const int row = blockIdx.x / c.kv_heads, kv = blockIdx.x - row * c.kv_heads, group = c.heads / c.kv_heads, vectors = c.dim / 4;
  const long long first = (static_cast<long long>(kv) * p.entries + static_cast<long long>(row) * c.count) * group;
  // products that are finite may add up to more than fp32 holds: an exact factor, no more than one over their number
  const float unit = Half2<T>::kOverflows ? __int_as_float((127 - 32 + __clz(c.count)) << 23) : 1.f;
  for (int x = threadIdx.x; x < group * vectors; x += kThreads) {
    const int g = x / vectors, d = (x - g * vectors) * 4;
    float high = -INFINITY, sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    bool any_averaged = false;
#pragma unroll 4
    for (int i = 0; i < c.count; ++i) {
      const float2 s = p.stats[first + static_cast<long long>(i) * group + g];
      high = fmaxf(high, s.x);
      any_averaged |= averaged<T>(s.y);
    }
    const float base = high == -INFINITY ? 0.f : high;
#pragma unroll 4
    for (int i = 0; i < c.count; ++i) {
      const long long slot = first + static_cast<long long>(i) * group + g;
      const float2 s = p.stats[slot];
      const float4 v = *reinterpret_cast<const float4*>(p.product + slot * c.dim + d);
      // nothing was written for an entry that is no page; a NaN maximum (of no score that is a number) is not -inf
      const bool there = s.x != -INFINITY || s.y != 0.f;
      const float weight = there ? exp2f(s.x - base) * unit : 0.f;
      sum += there ? (Half2<T>::kOverflows ? fabsf(s.y) : s.y) * weight : 0.f;
      o[0] += there ? v.x * weight : 0.f;
      o[1] += there ? v.y * weight : 0.f;
      o[2] += there ? v.z * weight : 0.f;
      o[3] += there ? v.w * weight : 0.f;
    }
    const float factor = any_averaged ? 1.f : to_average<T>(sum);
    if (any_averaged) join_averages<T>(p, first, g, group, d, base, unit, sum, o);
    T* const to = static_cast<T*>(c.out) + (static_cast<long long>(row) * c.heads + kv * group + g) * c.dim + d;
    *reinterpret_cast<uint2*>(to) = make_uint2(Half2<T>::pack(o[0] * factor, o[1] * factor), Half2<T>::pack(o[2] * factor, o[3] * factor));
  }
}

size_t rounded_up(size_t bytes) { return (bytes + 255) / 256 * 256; }

struct Sizes {
  long long entries, most_items;
  int tile_entries;
  size_t items_of, items, seen, list, stats, product, all;
};
Sizes sizes(int rows, int heads, int kv_heads, int head_dim, int num_pages, int count) {
  const int group = heads / kv_heads;
  Sizes s;
  s.entries = static_cast<long long>(rows) * count;
  s.tile_entries = kTileRows / group;
  s.most_items = s.entries / s.tile_entries + std::min<long long>(num_pages, s.entries);
  s.items_of = rounded_up(sizeof(int) * kv_heads);
  s.items = rounded_up(sizeof(Item) * kv_heads * s.most_items);
  s.seen = rounded_up(sizeof(int2) * kv_heads * s.entries);
  s.list = s.seen;
  s.stats = rounded_up(sizeof(float2) * heads * s.entries);
  s.product = rounded_up(sizeof(float) * heads * s.entries * head_dim);
  s.all = s.items_of + s.items + s.seen + s.list + s.stats + s.product;
  return s;
}

template <typename T, int PIECES>
int launch(const Params& p, cudaStream_t stream) {
  const SharedCall& c = p.c;
  constexpr int bytes = (kTileRows + 2 * kPositions) * (64 * PIECES + 8) * 2;
  const int counters = c.num_pages * kPageBytes;
  if (counters > 40 * 1024) {
    // the kernel's, not the call's: with one value for all calls, host threads that launch at the same time agree on it
    const cudaError_t e = cudaFuncSetAttribute(index_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostPages * kPageBytes);
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  if (bytes > 40 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(page_kernel<T, PIECES>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  // Together no more than half the SMs: 16 key heads with 8 blocks each take 7 us longer than with 4 (clusters wait for places).
  int blocks = 1;
  while (blocks < kIndexBlocks && p.entries > blocks * kIndexThreads / 2 && c.kv_heads * blocks * 4 <= kNumSMs) blocks *= 2;
  if (const int st = launch_clusters<Params>(index_kernel, c.kv_heads * blocks, blocks, kIndexThreads, counters, stream, p)) return st;
  if (const int st = launch_overlapped(page_kernel<T, PIECES>, dim3(p.most_items, c.kv_heads), dim3(kThreads), bytes, stream, p)) return st;
  return launch_overlapped(join_entries_kernel<T>, dim3(c.rows * c.kv_heads), dim3(kThreads), 0, stream, p);
}

}  // namespace

size_t shared_workspace_bytes(int rows, int heads, int kv_heads, int head_dim, int num_pages, int page_size, int table_width,
                              int count) {
  const int group = heads / kv_heads;
  if (group > kMostGroup || num_pages <= 0 || num_pages > kMostPages || count <= 0 || count > table_width || kv_heads > 65535) return 0;
  const double entries = static_cast<double>(rows) * count;
  if (entries * heads * head_dim * sizeof(float) > kMostScratch) return 0;
  // us of the two ways; of 30 measurements (rows 32 .. 4096, 1 .. 16 query heads to a key head, pages of 16 .. 256) all but three
  // within a quarter.  Row by row: keys and values from L2.  Here: the sort, a product to and fro for every entry and query head,
  // and a block's work.
  //   rows, key heads x G, dim, page, pages, listed    row by row   here
  //   256,   8 x 4, 128,  64,  256, 16                    118        85
  //   256,  32 x 1, 128,  64,   64, 16                    420        96
  //   512,  16 x 2,  64, 128,  128, 16                    470       120
  //   4096,  2 x 2, 128,  64,  512, 32                    836       292
  //   64,    8 x 4, 128,  64,  256, 16                     38        45
  //   1024,  2 x 8, 128,  64,  256, 16                    119       156
  //   256,   8 x 4, 128,  64, 4096, 16                    160       311
  //   16384, 1 x 1,  64,  64, 1000, 60                   1656       548
  //   20000, 1 x 1, 128,  64,  500, 33                   2105       491
  const int dim = head_dim > 64 ? 128 : 64, tiles = (page_size + kPositions - 1) / kPositions;
  const double pairs = entries * heads, blocks = kv_heads * (entries / (kTileRows / group) + 0.5 * std::min<double>(num_pages, entries));
  const double one_by_one = 12.0 + entries * kv_heads * 4 * page_size * dim * (group > 8 ? 1.25 : 1.0) / 9.7e6;
  const double shared = 15.0 + 6e-4 * entries + 1e-6 * pairs * head_dim + blocks * (6e-3 + 8.8e-5 * tiles * dim);
  if (one_by_one < 1.05 * shared) return 0;
  const Sizes s = sizes(rows, heads, kv_heads, head_dim, num_pages, count);
  return s.all <= kMostScratch ? s.all : 0;
}

int shared_attention(const SharedCall& call, bool bf16, void* workspace, cudaStream_t stream) {
  const Sizes s = sizes(call.rows, call.heads, call.kv_heads, call.dim, call.num_pages, call.count);
  Params p{};
  p.c = call;
  p.entries = static_cast<int>(s.entries);
  p.tile_entries = s.tile_entries;
  p.most_items = static_cast<int>(s.most_items);
  char* at = static_cast<char*>(workspace);
  p.items_of = reinterpret_cast<int*>(at);
  p.items = reinterpret_cast<Item*>(at += s.items_of);
  p.seen = reinterpret_cast<int2*>(at += s.items);
  p.list = reinterpret_cast<int2*>(at += s.seen);
  p.stats = reinterpret_cast<float2*>(at += s.list);
  p.product = reinterpret_cast<float*>(at += s.stats);
  if (call.dim > 64) return bf16 ? launch<__nv_bfloat16, 2>(p, stream) : launch<__half, 2>(p, stream);
  return bf16 ? launch<__nv_bfloat16, 1>(p, stream) : launch<__half, 1>(p, stream);
}

}  // namespace paged
}  // namespace iex
