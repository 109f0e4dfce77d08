// Appending the keys and values of new tokens to a paged cache (paged.cuh), rotated by their positions on the way, with the
// queries rotated beside them.
//
// Sequence i has n = cu_tokens[i + 1] - cu_tokens[i] new tokens (one without cu_tokens); its j-th new token takes position
// lengths[i] - n + j.  Of every query and key the first `rotary` elements are turned in pairs by the angles of the position,
//   (a, b) -> (a cos - b sin, b cos + a sin),   pairs (i, i + rotary / 2), or (2 i, 2 i + 1) if interleaved,
// in fp32, and rounded once.  boxes (optional) holds the smallest and largest key of every page and head in each dimension: of a
// page that is written to they are formed anew from all its positions up to the last new one.
//
// A block does one page's new tokens of one key head and its query heads, so that a box has one writer; with many tokens the query
// heads have blocks of their own.  An item is 16 bytes, or the two 16-byte pieces that are turned into each other.  What the
// page held before is requested ahead of all else; new keys pass through shared memory on their way into the box.
//
// 8 x 512 tokens, 32 query and 8 key heads of 128: 12.5 us, 4.7 TB/s with 3 us of start; 64 sequences' next tokens, 32 heads: 8.7 us (the
// latency of 2016 small blocks, and 21 MB of earlier keys for the boxes); one token: 4.1 us, four loads that wait for one another.
#include <algorithm>
#include <type_traits>

#include "paged.cuh"

namespace iex {
namespace paged {
namespace {

constexpr int kKept = 32;       // new keys that are kept in shared memory: of pages with more of them the box reads the cache
constexpr int kQueryHeads = 2;  // of a block that has nothing but query heads

enum Turn {
  kHalves,    // pairs (i, i + rotary / 2), rotary a multiple of 16: two pieces of 8 elements at once
  kNeighbors, // pairs (2 i, 2 i + 1): one piece
  kElements,  // pairs (i, i + rotary / 2) of any rotary
};

struct AppendParams {
  int tokens, batch, heads, kv_heads, dim, rope_rows, rotary, num_pages, page_shift, table_width;
  uint32_t by_items, by_pieces, by_units;  // inverses for divided()
  Rows q, k, v;
  const float *cos, *sin;
  void *q_out, *k_cache, *v_cache, *boxes;
  long long k_page, v_page;
  const int32_t *table, *lengths, *cu_tokens;
};

// x / d for x * d below 2^16, with inverse_of(d); a division takes a tenth of what such a block lives.
inline uint32_t inverse_of(int d) { return 65536u / static_cast<uint32_t>(d) + 1; }
__device__ __forceinline__ int divided(int x, uint32_t inverse) { return static_cast<int>(static_cast<uint32_t>(x) * inverse >> 16); }

template <typename T>
struct Pair;
template <>
struct Pair<__half> {
  using Type = __half2;
};
template <>
struct Pair<__nv_bfloat16> {
  using Type = __nv_bfloat162;
};
template <typename T>
__device__ __forceinline__ uint32_t smaller(uint32_t a, uint32_t b) {  // of two elements each; NaN if one is
  using P = typename Pair<T>::Type;
  const P v = __hmin2_nan(reinterpret_cast<const P&>(a), reinterpret_cast<const P&>(b));
  return reinterpret_cast<const uint32_t&>(v);
}
template <typename T>
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
  using P = typename Pair<T>::Type;
  const P v = __hmax2_nan(reinterpret_cast<const P&>(a), reinterpret_cast<const P&>(b));
  return reinterpret_cast<const uint32_t&>(v);
}
template <typename T>
__device__ __forceinline__ uint4 smaller(const uint4& a, const uint4& b) {
  return make_uint4(smaller<T>(a.x, b.x), smaller<T>(a.y, b.y), smaller<T>(a.z, b.z), smaller<T>(a.w, b.w));
}
template <typename T>
__device__ __forceinline__ uint4 larger(const uint4& a, const uint4& b) {
  return make_uint4(larger<T>(a.x, b.x), larger<T>(a.y, b.y), larger<T>(a.z, b.z), larger<T>(a.w, b.w));
}

// May have been written by the kernel in front.
__device__ __forceinline__ uint4 load16(const void* p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}

__device__ __forceinline__ float turned(float a, float b, float c, float s) { return fmaf(a, c, b * s); }

// Items of a head's row: pieces that are turned, then pieces that are copied.
template <Turn kTurn>
__host__ __device__ __forceinline__ int items_of(int dim, int rotary) {
  if (kTurn == kHalves) return rotary / 16 + (dim - rotary) / 8;
  if (kTurn == kNeighbors) return dim / 8;
  return rotary / 2 + dim - rotary;
}

// The angles of an item at a position, and what they make of it.
template <typename T, Turn kTurn>
struct Angles {
  static constexpr int kPairs = kTurn == kHalves ? 8 : kTurn == kNeighbors ? 4 : 1;
  float c[kPairs], s[kPairs];
  int pairs;  // of the item

  __device__ __forceinline__ void load(const AppendParams& p, const float* cos, const float* sin, int item) {
    const int half = p.rotary / 2;
    pairs = min(kPairs, max(0, half - item * kPairs));
    if constexpr (kTurn == kHalves) {
      uint4 v[4] = {};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        load_if(v[i], cos + item * 8 + 4 * i, pairs > 0);
        load_if(v[2 + i], sin + item * 8 + 4 * i, pairs > 0);
        c[4 * i] = __uint_as_float(v[i].x), c[4 * i + 1] = __uint_as_float(v[i].y);
        c[4 * i + 2] = __uint_as_float(v[i].z), c[4 * i + 3] = __uint_as_float(v[i].w);
        s[4 * i] = __uint_as_float(v[2 + i].x), s[4 * i + 1] = __uint_as_float(v[2 + i].y);
        s[4 * i + 2] = __uint_as_float(v[2 + i].z), s[4 * i + 3] = __uint_as_float(v[2 + i].w);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        const int pair = min(item * kPairs + i, half - 1);
        c[i] = half > 0 ? cos[pair] : 1.f;
        s[i] = half > 0 ? sin[pair] : 0.f;
      }
    }
  }
};

template <typename T, Turn kTurn>
struct Item {
  uint4 a, b;  // the piece, or both (kElements: one element each)

  // Item `item` of the row at `from`, where there is one.
  __device__ __forceinline__ void load(const AppendParams& p, const T* from, int item, int pairs, bool there) {
    const int half = p.rotary / 2;
    if constexpr (kTurn == kHalves) {
      load_if(a, from + (pairs > 0 ? item * 8 : p.rotary + (item - half / 8) * 8), there);
      load_if(b, from + half + item * 8, there && pairs > 0);
    } else if constexpr (kTurn == kNeighbors) {
      load_if(a, from + item * 8, there);
    } else if (there) {
      *reinterpret_cast<T*>(&a) = from[pairs > 0 ? item : half + item];
      if (pairs > 0) *reinterpret_cast<T*>(&b) = from[half + item];
    }
  }
  __device__ __forceinline__ void turn(const Angles<T, kTurn>& angles) {
    T *x = reinterpret_cast<T*>(&a), *y = reinterpret_cast<T*>(&b);
    if constexpr (kTurn == kNeighbors) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float one = as_float(x[2 * i]), two = as_float(x[2 * i + 1]);
        const bool turns = i < angles.pairs;
        x[2 * i] = turns ? rounded<T>(turned(one, two, angles.c[i], -angles.s[i])) : x[2 * i];
        x[2 * i + 1] = turns ? rounded<T>(turned(two, one, angles.c[i], angles.s[i])) : x[2 * i + 1];
      }
    } else if (angles.pairs > 0) {
#pragma unroll
      for (int i = 0; i < Angles<T, kTurn>::kPairs; ++i) {
        const float one = as_float(x[i]), two = as_float(y[i]);
        x[i] = rounded<T>(turned(one, two, angles.c[i], -angles.s[i]));
        y[i] = rounded<T>(turned(two, one, angles.c[i], angles.s[i]));
      }
    }
  }
  // To the row at `to`.
  __device__ __forceinline__ void store(const AppendParams& p, T* to, int item, int pairs) const {
    const int half = p.rotary / 2;
    if constexpr (kTurn == kHalves) {
      *reinterpret_cast<uint4*>(to + (pairs > 0 ? item * 8 : p.rotary + (item - half / 8) * 8)) = a;
      if (pairs > 0) *reinterpret_cast<uint4*>(to + half + item * 8) = b;
    } else if constexpr (kTurn == kNeighbors) {
      *reinterpret_cast<uint4*>(to + item * 8) = a;
    } else {
      to[pairs > 0 ? item : half + item] = *reinterpret_cast<const T*>(&a);
      if (pairs > 0) to[half + item] = *reinterpret_cast<const T*>(&b);
    }
  }
};

// `heads` heads of `tokens` rows turned, kHeads of them by one thread, which share the angles.  `thread`: which of the block's this one
// counts as; kept (or null): a second place for the first head.
template <typename T, Turn kTurn, int kThreads, int kHeads>
__device__ __forceinline__ void turn_rows(const AppendParams& p, int thread, int tokens, int heads, uint32_t by_units, const T* x, long long x_row,
                                          long long x_head, T* out, long long out_row, const float* cos, const float* sin,
                                          T (*kept)[kMaxHeadDim]) {
  const int items = items_of<kTurn>(p.dim, p.rotary), units = (heads + kHeads - 1) / kHeads * items;
  if (units == 0) return;
  const bool few = units <= kThreads;
  const int rows = few ? divided(kThreads, by_units) : 1, row = few ? divided(thread, by_units) : 0, half = p.rotary / 2;
  if (row >= rows) return;
  for (int y = thread - row * units; y < units; y += kThreads) {
    const int set = few ? divided(y, p.by_items) : y / items, item = y - set * items;
#pragma unroll 1
    for (int t = row; t < tokens; t += rows) {
      Angles<T, kTurn> angles;
      Item<T, kTurn> some[kHeads];
#pragma unroll
      for (int h = 0; h < kHeads; ++h)
        some[h].load(p, x + t * x_row + (set * kHeads + h) * x_head, item, min(1, max(0, half - item * Angles<T, kTurn>::kPairs)),
                     set * kHeads + h < heads);
      angles.load(p, cos + static_cast<long long>(t) * half, sin + static_cast<long long>(t) * half, item);
#pragma unroll
      for (int h = 0; h < kHeads; ++h) {
        some[h].turn(angles);
        if (set * kHeads + h < heads) some[h].store(p, out + t * out_row + (set * kHeads + h) * p.dim, item, angles.pairs);
      }
      if (kept != nullptr) some[0].store(p, kept[t], item, angles.pairs);
    }
  }
}

// The new tokens that a block has.
struct Span {
  int sequence, begin, n, length, nth;  // nth: of the pages that the sequence's new tokens touch
};

// Blocks in a row have the pages of one sequence after the other: n new tokens touch up to (n + page - 2) / page + 1 of them.
// False where there is no such block.  used: the rows of the sequences.
template <int kThreads>
__device__ __forceinline__ bool find_span(const AppendParams& p, int block, Span& found, int& used) {
  constexpr int kWarps = kThreads / 32;
  __shared__ Span shared;
  __shared__ int sums[kWarps], last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (p.cu_tokens == nullptr) {
    used = p.tokens;
    if (block >= p.batch) return false;
    found = {block, block, 1, max(p.lengths[block], 0), 0};
    return true;
  }
  int front = 0;
  for (int s0 = 0; s0 < p.batch; s0 += kThreads) {
    const int s = s0 + threadIdx.x;
    int begin = 0, n = 0, length = 0;
    if (s < p.batch) {
      begin = min(max(p.cu_tokens[s], 0), p.tokens);
      const int next = min(max(p.cu_tokens[s + 1], 0), p.tokens);
      n = max(0, next - begin);
      length = max(p.lengths[s], 0);
      if (s == p.batch - 1) last = next;
    }
    const int mine = n > 0 ? ((n + (1 << p.page_shift) - 2) >> p.page_shift) + 1 : 0;
    int sum = mine;
    for (int d = 1; d < 32; d <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, sum, d);
      sum += lane >= d ? other : 0;
    }
    if (lane == 31) sums[warp] = sum;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      sum += w < warp ? sums[w] : 0;
      all += sums[w];
    }
    const int first = front + sum - mine;
    if (first <= block && block < first + mine) shared = {s, begin, n, length, block - first};
    front += all;
    __syncthreads();
    const bool here = block < front;
    if (here) found = shared;
    if (here || s0 + kThreads >= p.batch) {
      used = s0 + kThreads >= p.batch ? last : min(max(p.cu_tokens[p.batch], 0), p.tokens);
      return here;
    }
  }
  used = min(max(p.cu_tokens[0], 0), p.tokens);  // no sequences
  return false;
}

// kThreads: 128, or 64 where a block has few tokens and what counts is how many blocks are under way at once.
template <typename T, Turn kTurn, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) append_kernel(const __grid_constant__ AppendParams p) {
  __shared__ alignas(16) T kept[kKept][kMaxHeadDim];
  __shared__ uint4 parts[2][kThreads];  // smallest and largest of a thread's pieces of keys
  grid_dependency_wait();
  grid_launch_dependents();
  const int block = blockIdx.x, blocks = gridDim.x, kv = blockIdx.z;
  const int group = p.heads / p.kv_heads, page = 1 << p.page_shift, pieces = p.dim / 8;
  // what this block has of the head group: keys and values, query heads [head0, head0 + heads) of it
  const bool alone = gridDim.y == 1, keys_too = blockIdx.y == 0;
  const int head0 = alone || keys_too ? 0 : (blockIdx.y - 1) * kQueryHeads;
  const int heads = alone ? group : keys_too ? 0 : min(kQueryHeads, group - head0);
  const T* const q = static_cast<const T*>(p.q.data) + (kv * group + head0) * p.q.head;
  T* const q_out = static_cast<T*>(p.q_out) + static_cast<long long>(kv * group + head0) * p.dim;
  const auto clear = [&](int row) {  // the queries of a token without a place
    uint4* to = reinterpret_cast<uint4*>(q_out + static_cast<long long>(row) * p.heads * p.dim);
    for (int x = threadIdx.x; x < heads * pieces; x += kThreads) to[x] = make_uint4(0, 0, 0, 0);
  };
  Span span;
  int used;
  const bool any_span = find_span<kThreads>(p, block, span, used);
  for (int row = used + block; row < p.tokens; row += blocks) clear(row);
  if (!any_span) return;
  const int start = span.length - span.n;  // the first new token's position
  const int nth = (max(start, 0) >> p.page_shift) + span.nth;
  const long long page_begin = static_cast<long long>(nth) << p.page_shift;
  const int from = static_cast<int>(max(static_cast<long long>(start), page_begin));
  const int to = static_cast<int>(min(static_cast<long long>(span.length), page_begin + page));
  if (span.nth == 0)
    for (int j = 0; j < min(span.n, -start); ++j) clear(span.begin + j);
  if (from >= to) return;
  const int at = nth < p.table_width ? p.table[static_cast<long long>(span.sequence) * p.table_width + nth] : -1;
  const int row0 = span.begin + from - start, half = p.rotary / 2, slot0 = from & (page - 1);
  const float* const cos = p.cos + static_cast<long long>(from) * half;
  const float* const sin = p.sin + static_cast<long long>(from) * half;
  const int positions = p.rotary > 0 ? max(0, min(to, p.rope_rows) - from) : to - from;  // that have angles

  // Queries do not wait for the page.  Where there are few, other warps have them than the keys.
  turn_rows<T, kTurn, kThreads, kQueryHeads>(p, (threadIdx.x + kThreads - 32) % kThreads, positions, heads, p.by_units, q + row0 * p.q.row, p.q.row, p.q.head,
                                   q_out + static_cast<long long>(row0) * p.heads * p.dim, static_cast<long long>(p.heads) * p.dim, cos,
                                   sin, nullptr);
  const bool known = at >= 0 && at < p.num_pages;
  const int tokens = known ? positions : 0;
  if (tokens < to - from) {
    if (!known) __syncthreads();  // they have been written
    for (int t = tokens; t < to - from; ++t) clear(row0 + t);
  }
  if (tokens == 0 || !keys_too) return;
  T* const k_page = static_cast<T*>(p.k_cache) + at * p.k_page + static_cast<long long>(kv) * page * p.dim;
  T* const v_page = static_cast<T*>(p.v_cache) + at * p.v_page + static_cast<long long>(kv) * page * p.dim;

  // what the page held before: a piece of the head to a thread
  constexpr int kOldAhead = 512 / kThreads;
  const int rows = divided(kThreads, p.by_pieces), mine = divided(threadIdx.x, p.by_pieces), piece = threadIdx.x - mine * pieces;
  const bool boxed = p.boxes != nullptr;
  const T* const old_keys = k_page + piece * 8;
  uint4 old[kOldAhead];
  const bool any_old = boxed && mine < rows && mine < slot0;
  const auto request_old = [&](int slot) {  // those behind the last one: one of the others again
#pragma unroll
    for (int u = 0; u < kOldAhead; ++u)
      load_if(old[u], old_keys + (slot + u * rows < slot0 ? slot + u * rows : mine) * p.dim, any_old);
  };
  request_old(mine);

  const bool keep = boxed && tokens <= kKept;
  turn_rows<T, kTurn, kThreads, 1>(p, threadIdx.x, tokens, 1, p.by_items, static_cast<const T*>(p.k.data) + row0 * p.k.row + kv * p.k.head, p.k.row, 0,
                         k_page + slot0 * p.dim, p.dim, cos, sin, keep ? kept : nullptr);
  const int vector = (threadIdx.x + 16) % kThreads, v_row = divided(vector, p.by_pieces), d = (vector - v_row * pieces) * 8;
  const T* const v = static_cast<const T*>(p.v.data) + row0 * p.v.row + kv * p.v.head + d;
  if (v_row < rows)
    for (int t0 = v_row; t0 < tokens; t0 += 4 * rows) {
      uint4 some[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) load_if(some[u], v + (t0 + u * rows) * p.v.row, t0 + u * rows < tokens);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (t0 + u * rows < tokens) *reinterpret_cast<uint4*>(v_page + (slot0 + t0 + u * rows) * p.dim + d) = some[u];
    }
  if (!boxed) return;
  __syncthreads();  // the new keys are in shared memory, or in the cache
  constexpr uint32_t kInfinity = std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u;  // two of them
  uint4 lo = make_uint4(kInfinity, kInfinity, kInfinity, kInfinity), hi = lo;
  hi.x = hi.y = hi.z = hi.w = kInfinity | 0x80008000u;
  if (any_old)
    for (int slot = mine;;) {
#pragma unroll
      for (int u = 0; u < kOldAhead; ++u) {
        lo = smaller<T>(lo, old[u]);
        hi = larger<T>(hi, old[u]);
      }
      slot += kOldAhead * rows;
      if (slot >= slot0) break;
      request_old(slot);
    }
  if (mine < rows)
    for (int t = mine; t < tokens; t += rows) {
      const uint4 key = keep ? *reinterpret_cast<const uint4*>(&kept[t][piece * 8]) : load16(old_keys + (slot0 + t) * p.dim);
      lo = smaller<T>(lo, key);
      hi = larger<T>(hi, key);
    }
  parts[0][threadIdx.x] = lo;
  parts[1][threadIdx.x] = hi;
  __syncthreads();
  // a thread for two elements, the smallest or the largest; rows of threads without a key are the last ones
  const int filled = min(rows, max(slot0, tokens));
  uint32_t* const box = reinterpret_cast<uint32_t*>(static_cast<T*>(p.boxes) + (static_cast<long long>(at) * p.kv_heads + kv) * 2 * p.dim);
  for (int x = threadIdx.x; x < p.dim; x += kThreads) {
    const int high = x >= p.dim / 2, word = x - high * (p.dim / 2);  // of four to a piece
    const uint32_t* const from_parts = reinterpret_cast<const uint32_t*>(parts[high]) + word;
    uint32_t value = from_parts[0];
    for (int r = 1; r < filled; ++r) {
      const uint32_t other = from_parts[r * pieces * 4];
      value = high ? larger<T>(value, other) : smaller<T>(value, other);
    }
    box[x] = value;
  }
}

template <typename T, Turn kTurn>
int launch(AppendParams p, int blocks, cudaStream_t stream) {
  const bool few = p.tokens <= 4ll * p.batch;
  const int group = p.heads / p.kv_heads, items = items_of<kTurn>(p.dim, p.rotary);
  const int heads = few ? group : std::min(group, kQueryHeads);  // of a block
  p.by_items = inverse_of(items);
  p.by_pieces = inverse_of(p.dim / 8);
  p.by_units = inverse_of((heads + kQueryHeads - 1) / kQueryHeads * items);
  const dim3 grid(blocks, few ? 1 : 1 + (group + kQueryHeads - 1) / kQueryHeads, p.kv_heads);
  return few ? launch_overlapped(append_kernel<T, kTurn, 64>, grid, dim3(64), 0, stream, p)
             : launch_overlapped(append_kernel<T, kTurn, 128>, grid, dim3(128), 0, stream, p);
}

template <typename T>
int launch(const AppendParams& p, bool interleaved, int blocks, cudaStream_t stream) {
  if (interleaved) return launch<T, kNeighbors>(p, blocks, stream);
  const bool in_pieces = p.rotary % 16 == 0 && aligned16(p.cos) && aligned16(p.sin);
  return in_pieces ? launch<T, kHalves>(p, blocks, stream) : launch<T, kElements>(p, blocks, stream);
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
  if (kv_heads > 65535 || heads / kv_heads > 65535 || !table_ok(table_width, page_size))  // a grid's second and third dimension
    return IEX_ERR_TOO_LARGE;
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
  // n tokens touch no more than n pages, nor than n / page + 2
  const long long pages = cu_tokens ? std::min<long long>(tokens, (tokens >> p.page_shift) + 2ll * batch) : batch;
  const int blocks = static_cast<int>(std::max(1ll, pages));
  return bf16 ? launch<__nv_bfloat16>(p, interleaved != 0, blocks, static_cast<cudaStream_t>(stream))
              : launch<__half>(p, interleaved != 0, blocks, static_cast<cudaStream_t>(stream));
}
