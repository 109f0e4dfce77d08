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
#include <algorithm>

#include "paged.cuh"

namespace iex {
namespace paged {
namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kKept = 32;       // new keys that are kept in shared memory: of pages with more of them the box reads the cache
constexpr int kQueryHeads = 2;  // of a block that has nothing but query heads

enum Turn {
  kHalves,    // pairs (i, i + rotary / 2), rotary a multiple of 16: two pieces of 8 elements at once
  kNeighbors, // pairs (2 i, 2 i + 1): one piece
  kElements,  // pairs (i, i + rotary / 2) of any rotary
};

struct AppendParams {
  int tokens, batch, heads, kv_heads, dim, rope_rows, rotary, num_pages, page_shift, table_width;
  Rows q, k, v;
  const float *cos, *sin;
  void *q_out, *k_cache, *v_cache, *boxes;
  long long k_page, v_page;
  const int32_t *table, *lengths, *cu_tokens;
};

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
__device__ __forceinline__ int items_of(int dim, int rotary) {
  if (kTurn == kHalves) return rotary / 16 + (dim - rotary) / 8;
  if (kTurn == kNeighbors) return dim / 8;
  return rotary / 2 + dim - rotary;
}

// An item on its way: what is loaded of it ahead of the items before it being stored.
template <typename T, Turn kTurn>
struct Item {
  uint4 a, b;  // the piece, or both (kElements: one element each)
  float c[kTurn == kHalves ? 8 : kTurn == kNeighbors ? 4 : 1], s[kTurn == kHalves ? 8 : kTurn == kNeighbors ? 4 : 1];

  __device__ __forceinline__ void load_copy(const T* from, int item) { a = load16(from + item * 8); }
  __device__ __forceinline__ void store_copy(T* to, int item) const { *reinterpret_cast<uint4*>(to + item * 8) = a; }

  // Item `item` of the row at `from`; the angles of its position at cos and sin.
  __device__ __forceinline__ void load(const AppendParams& p, const T* from, const float* cos, const float* sin, int item) {
    const int half = p.rotary / 2;
    if constexpr (kTurn == kHalves) {
      if (item < half / 8) {
        const int d = item * 8;
        a = load16(from + d);
        b = load16(from + half + d);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint4 vc = load16(cos + d + 4 * i), vs = load16(sin + d + 4 * i);
          c[4 * i] = __uint_as_float(vc.x), c[4 * i + 1] = __uint_as_float(vc.y);
          c[4 * i + 2] = __uint_as_float(vc.z), c[4 * i + 3] = __uint_as_float(vc.w);
          s[4 * i] = __uint_as_float(vs.x), s[4 * i + 1] = __uint_as_float(vs.y);
          s[4 * i + 2] = __uint_as_float(vs.z), s[4 * i + 3] = __uint_as_float(vs.w);
        }
      } else {
        a = load16(from + p.rotary + (item - half / 8) * 8);
      }
    } else if constexpr (kTurn == kNeighbors) {
      a = load16(from + item * 8);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int pair = min(item * 4 + i, max(half - 1, 0));
        c[i] = half > 0 ? cos[pair] : 1.f;
        s[i] = half > 0 ? sin[pair] : 0.f;
      }
    } else {
      T *x = reinterpret_cast<T*>(&a), *y = reinterpret_cast<T*>(&b);
      if (item < half) {
        x[0] = from[item];
        y[0] = from[half + item];
        c[0] = cos[item];
        s[0] = sin[item];
      } else {
        x[0] = from[half + item];
      }
    }
  }

  __device__ __forceinline__ void turn(const AppendParams& p, int item) {
    const int half = p.rotary / 2;
    T *x = reinterpret_cast<T*>(&a), *y = reinterpret_cast<T*>(&b);
    if constexpr (kTurn == kNeighbors) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float one = as_float(x[2 * i]), two = as_float(x[2 * i + 1]);
        const bool turns = item * 4 + i < half;
        x[2 * i] = turns ? rounded<T>(turned(one, two, c[i], -s[i])) : x[2 * i];
        x[2 * i + 1] = turns ? rounded<T>(turned(two, one, c[i], s[i])) : x[2 * i + 1];
      }
    } else {
      constexpr int kElementsOf = kTurn == kHalves ? 8 : 1;
      if (item < half / kElementsOf) {
#pragma unroll
        for (int i = 0; i < kElementsOf; ++i) {
          const float one = as_float(x[i]), two = as_float(y[i]);
          x[i] = rounded<T>(turned(one, two, c[i], -s[i]));
          y[i] = rounded<T>(turned(two, one, c[i], s[i]));
        }
      }
    }
  }

  // To the row at `to`.
  __device__ __forceinline__ void store(const AppendParams& p, T* to, int item) const {
    const int half = p.rotary / 2;
    if constexpr (kTurn == kNeighbors) {
      *reinterpret_cast<uint4*>(to + item * 8) = a;
    } else {
      constexpr int kElementsOf = kTurn == kHalves ? 8 : 1;
      const bool turns = item < half / kElementsOf;
      T* const first = turns ? to + item * kElementsOf : to + p.rotary + (item - half / kElementsOf) * kElementsOf;
      if constexpr (kTurn == kHalves) {
        *reinterpret_cast<uint4*>(first) = a;
        if (turns) *reinterpret_cast<uint4*>(first + half) = b;
      } else {
        *first = *reinterpret_cast<const T*>(&a);
        if (turns) first[half] = *reinterpret_cast<const T*>(&b);
      }
    }
  }
};

// The new tokens that a block has.
struct Span {
  int sequence, begin, n, length, nth;  // nth: of the pages that the sequence's new tokens touch
};

// Blocks in a row have the pages of one sequence after the other: n new tokens touch up to (n + page - 2) / page + 1 of them.
// False where there is no such block.
__device__ __forceinline__ bool find_span(const AppendParams& p, int block, Span& found) {
  __shared__ Span shared;
  __shared__ int sums[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (p.cu_tokens == nullptr) {
    if (block >= p.batch) return false;
    found = {block, block, 1, p.lengths[block], 0};
    return true;
  }
  int front = 0;
  for (int s0 = 0; s0 < p.batch; s0 += kThreads) {
    const int s = s0 + threadIdx.x;
    int begin = 0, n = 0, length = 0;
    if (s < p.batch) {
      begin = min(max(p.cu_tokens[s], 0), p.tokens);
      n = max(0, min(max(p.cu_tokens[s + 1], 0), p.tokens) - begin);
      length = p.lengths[s];
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
    if (block < front) {
      found = shared;
      return true;
    }
  }
  return false;
}

// kAhead: items that a thread has on their way.  With few tokens there is one for a thread and blocks side by side hide the
// latency; with many, two.
template <typename T, Turn kTurn, int kAhead>
__global__ void __launch_bounds__(kThreads, kAhead == 1 ? 8 : 4) append_kernel(const __grid_constant__ AppendParams p) {
  __shared__ alignas(16) T kept[kKept][kMaxHeadDim];
  __shared__ uint4 parts[2][kThreads];  // smallest and largest of a thread's pieces of keys
  grid_dependency_wait();
  grid_launch_dependents();
  const int block = blockIdx.x / p.kv_heads, blocks = gridDim.x / p.kv_heads, kv = blockIdx.x % p.kv_heads;
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
  const int used = p.cu_tokens ? min(max(p.cu_tokens[p.batch], 0), p.tokens) : p.tokens;  // rows of some sequence

  Span span;
  const bool any_span = find_span(p, block, span);
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
  const int row0 = span.begin + from - start, half = p.rotary / 2, items = items_of<kTurn>(p.dim, p.rotary), slot0 = from % page;
  const float* const cos = p.cos + static_cast<long long>(from) * half;
  const float* const sin = p.sin + static_cast<long long>(from) * half;

  // a token's items: of the key, the value, the queries
  const int of_keys = keys_too ? items : 0, of_values = keys_too ? pieces : 0, of_token = of_keys + of_values + heads * items;
  const T* const k = static_cast<const T*>(p.k.data) + kv * p.k.head;
  const T* const v = static_cast<const T*>(p.v.data) + kv * p.v.head;
  struct Place {
    int t, head, item;  // head: -2 the key's, -1 the value's
  };
  const auto place_of = [&](int x) {
    Place w;
    w.t = x / of_token;
    int y = x - w.t * of_token;
    w.head = y < of_keys ? -2 : y < of_keys + of_values ? -1 : (y - of_keys - of_values) / items;
    w.item = w.head == -2 ? y : w.head == -1 ? y - of_keys : y - of_keys - of_values - w.head * items;
    return w;
  };
  Item<T, kTurn> some[kAhead];
  Place place[kAhead];
  const int positions = p.rotary > 0 ? max(0, min(to, p.rope_rows) - from) : to - from;  // that have angles
  const auto request = [&](int x0) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int x = x0 + u * kThreads;
      if (x >= positions * of_token) break;
      place[u] = place_of(x);
      const long long row = row0 + place[u].t, angles = static_cast<long long>(place[u].t) * half;
      if (place[u].head == -1) some[u].load_copy(v + row * p.v.row, place[u].item);
      else some[u].load(p, place[u].head == -2 ? k + row * p.k.row : q + row * p.q.row + place[u].head * p.q.head, cos + angles,
                        sin + angles, place[u].item);
    }
  };
  request(threadIdx.x);  // does not wait for the page
  const bool known = at >= 0 && at < p.num_pages;
  const int tokens = known ? positions : 0;
  for (int t = tokens; t < to - from; ++t) clear(row0 + t);
  if (tokens == 0) return;
  T* const k_page = static_cast<T*>(p.k_cache) + at * p.k_page + static_cast<long long>(kv) * page * p.dim;
  T* const v_page = static_cast<T*>(p.v_cache) + at * p.v_page + static_cast<long long>(kv) * page * p.dim;

  // what the page held before: a piece of the head to a thread
  constexpr int kOldAhead = 4;
  const int rows = kThreads / pieces, mine = threadIdx.x / pieces, piece = threadIdx.x % pieces;
  const bool boxed = p.boxes != nullptr && keys_too;
  const T* const old_keys = k_page + piece * 8;
  uint4 old[kOldAhead];
  const auto request_old = [&](int slot) {
#pragma unroll
    for (int u = 0; u < kOldAhead; ++u) {
      old[u] = make_uint4(0, 0, 0, 0);
      load_if(old[u], old_keys + (slot + u * rows) * p.dim, boxed && mine < rows && slot + u * rows < slot0);
    }
  };
  request_old(mine);

  const bool keep = boxed && tokens <= kKept;
  for (int x0 = threadIdx.x; x0 < tokens * of_token; x0 += kAhead * kThreads) {
    if (x0 != threadIdx.x) request(x0);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (x0 + u * kThreads >= tokens * of_token) break;
      const Place& w = place[u];
      if (w.head == -1) {
        some[u].store_copy(v_page + (slot0 + w.t) * p.dim, w.item);
        continue;
      }
      some[u].turn(p, w.item);
      some[u].store(p, w.head == -2 ? k_page + (slot0 + w.t) * p.dim : q_out + (static_cast<long long>(row0 + w.t) * p.heads + w.head) * p.dim,
                    w.item);
      if (keep && w.head == -2) some[u].store(p, kept[w.t], w.item);
    }
  }
  if (!boxed) return;
  __syncthreads();  // the new keys are in shared memory, or in the cache
  uint4 lo, hi;
  bool any = false;
  const auto join = [&](const uint4& key) {
    lo = any ? smaller<T>(lo, key) : key;
    hi = any ? larger<T>(hi, key) : key;
    any = true;
  };
  if (mine < rows) {
    for (int slot = mine; slot < slot0;) {
#pragma unroll
      for (int u = 0; u < kOldAhead; ++u)
        if (slot + u * rows < slot0) join(old[u]);
      slot += kOldAhead * rows;
      if (slot < slot0) request_old(slot);
    }
    for (int t = mine; t < tokens; t += rows)
      join(keep ? *reinterpret_cast<const uint4*>(&kept[t][piece * 8]) : load16(old_keys + (slot0 + t) * p.dim));
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

template <typename T>
int launch(const AppendParams& p, bool interleaved, unsigned blocks, cudaStream_t stream) {
  const bool in_pieces = p.rotary % 16 == 0 && aligned16(p.cos) && aligned16(p.sin);
  const bool few = p.tokens <= 4ll * p.batch;
  const auto kern = interleaved ? (few ? append_kernel<T, kNeighbors, 1> : append_kernel<T, kNeighbors, 2>)
                    : in_pieces ? (few ? append_kernel<T, kHalves, 1> : append_kernel<T, kHalves, 2>)
                                : (few ? append_kernel<T, kElements, 1> : append_kernel<T, kElements, 2>);
  const int group = p.heads / p.kv_heads;
  return launch_overlapped(kern, dim3(blocks, few ? 1 : 1 + (group + kQueryHeads - 1) / kQueryHeads), dim3(kThreads), 0, stream, p);
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
  const long long blocks = std::max(1ll, pages) * kv_heads;
  if (blocks > 0x7fffffffll) return IEX_ERR_TOO_LARGE;
  return bf16 ? launch<__nv_bfloat16>(p, interleaved != 0, static_cast<unsigned>(blocks), static_cast<cudaStream_t>(stream))
              : launch<__half>(p, interleaved != 0, static_cast<unsigned>(blocks), static_cast<cudaStream_t>(stream));
}
