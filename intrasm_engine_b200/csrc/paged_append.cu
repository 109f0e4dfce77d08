// Appending the keys and values of new tokens to a paged cache (paged.cuh), rotated by their positions on the way, with the
// queries rotated beside them.
//
// Sequence i has n = cu_tokens[i + 1] - cu_tokens[i] new tokens (one without cu_tokens); its j-th new token takes position
// lengths[i] - n + j.  Of every query and key the first `rotary` elements are turned in pairs by the angles of the position,
//   (a, b) -> (a cos - b sin, b cos + a sin),   pairs (i, i + rotary / 2), or (2 i, 2 i + 1) if interleaved,
// in fp32, and rounded once.  boxes (optional) holds the smallest and largest key of every page and head in each dimension: of a
// page that is written to they are formed anew from all its positions up to the last new one.
//
// A block does one page's new tokens of one key head and its query heads, so that a box has one writer.  A thread's item is 16
// bytes, or the two 16-byte pieces that are turned into each other; keys are done with a fixed piece of the head to a thread,
// which keeps the smallest and largest of its own, and meet those of the positions that the page held before in shared memory.
#include <algorithm>

#include "paged.cuh"

namespace iex {
namespace paged {
namespace {

constexpr int kThreads = 128;

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

// Where the tokens of sequence i begin among the rows.
__device__ __forceinline__ int begin_of(const AppendParams& p, int i) {
  return p.cu_tokens ? min(max(p.cu_tokens[i], 0), p.tokens) : i;
}

// Blocks are laid out by what a sequence needs at most: the n tokens of a sequence touch up to n / page + 2 pages, and
// floor(begin / page) + 2 i blocks are enough for all the sequences in front.
__device__ __forceinline__ int first_block(const AppendParams& p, int i) {
  return p.cu_tokens ? (begin_of(p, i) >> p.page_shift) + 2 * i : i;
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
      for (int i = 0; i < 4; ++i)
        if (item * 4 + i < half) {
          c[i] = cos[item * 4 + i];
          s[i] = sin[item * 4 + i];
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

  // Turned, to the row at `to`; a and b are what is written.
  __device__ __forceinline__ void store(const AppendParams& p, T* to, int item) {
    const int half = p.rotary / 2;
    T *x = reinterpret_cast<T*>(&a), *y = reinterpret_cast<T*>(&b);
    if constexpr (kTurn == kNeighbors) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (item * 4 + i < half) {
          const float one = as_float(x[2 * i]), two = as_float(x[2 * i + 1]);
          x[2 * i] = rounded<T>(turned(one, two, c[i], -s[i]));
          x[2 * i + 1] = rounded<T>(turned(two, one, c[i], s[i]));
        }
      *reinterpret_cast<uint4*>(to + item * 8) = a;
    } else {
      constexpr int kElementsOf = kTurn == kHalves ? 8 : 1;
      const bool turns = item < half / kElementsOf;
      if (turns) {
#pragma unroll
        for (int i = 0; i < kElementsOf; ++i) {
          const float one = as_float(x[i]), two = as_float(y[i]);
          x[i] = rounded<T>(turned(one, two, c[i], -s[i]));
          y[i] = rounded<T>(turned(two, one, c[i], s[i]));
        }
      }
      T* const first = turns ? to + item * kElementsOf : to + p.rotary + (item - half / kElementsOf) * kElementsOf;
      if constexpr (kTurn == kHalves) {
        *reinterpret_cast<uint4*>(first) = a;
        if (turns) *reinterpret_cast<uint4*>(first + half) = b;
      } else {
        *first = x[0];
        if (turns) first[half] = y[0];
      }
    }
  }
};

// kAhead: items that a thread has on their way.  With few tokens there is one for a thread and blocks side by side hide the
// latency (8 an SM); with many, two.
template <typename T, Turn kTurn, int kAhead>
__global__ void __launch_bounds__(kThreads, kAhead == 1 ? 6 : 4) append_kernel(const __grid_constant__ AppendParams p) {
  __shared__ uint4 box_parts[2][kThreads][1 + (kTurn == kHalves)];  // smallest and largest of a thread's pieces of new keys
  __shared__ uint4 old_parts[2][kThreads];                          // ... of what the page held before
  grid_dependency_wait();
  grid_launch_dependents();
  const int block = blockIdx.x / p.kv_heads, blocks = gridDim.x / p.kv_heads, kv = blockIdx.x % p.kv_heads;
  const int group = p.heads / p.kv_heads, page = 1 << p.page_shift, pieces = p.dim / 8;
  T* const q_out = static_cast<T*>(p.q_out) + static_cast<long long>(kv) * group * p.dim;
  const auto clear = [&](int row) {  // the head group's queries of a token without a place
    uint4* to = reinterpret_cast<uint4*>(q_out + static_cast<long long>(row) * p.heads * p.dim);
    for (int x = threadIdx.x; x < group * pieces; x += kThreads) to[x] = make_uint4(0, 0, 0, 0);
  };
  for (int row = begin_of(p, p.batch) + block; row < p.tokens; row += blocks) clear(row);
  if (p.batch == 0) return;

  int i = block;
  if (p.cu_tokens != nullptr) {  // the last sequence whose blocks begin here or in front
    i = -1;
    for (int s = 0; s < p.batch; s += kThreads)
      i += __syncthreads_count(s + static_cast<int>(threadIdx.x) < p.batch && first_block(p, s + threadIdx.x) <= block);
    if (i < 0) return;
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
  const int until = !known ? from : p.rotary > 0 ? max(from, min(to, p.rope_rows)) : to;  // [from, until) have a place
  const int row0 = begin + from - start;  // the row of position `from`
  for (int position = until; position < to; ++position) clear(row0 + position - from);
  if (from >= until) return;
  const int tokens = until - from, half = p.rotary / 2, items = items_of<kTurn>(p.dim, p.rotary), slot0 = from % page;
  const float* const cos = p.cos + static_cast<long long>(from) * half;
  const float* const sin = p.sin + static_cast<long long>(from) * half;
  T* const k_to = static_cast<T*>(p.k_cache) + at * p.k_page + static_cast<long long>(kv) * page * p.dim;
  T* const v_to = static_cast<T*>(p.v_cache) + at * p.v_page + (static_cast<long long>(kv) * page + slot0) * p.dim;

  // what the page held before: a piece of the head to a thread; the first ones are requested ahead of all else
  constexpr int kOldAhead = 4;
  const int old_rows = kThreads / pieces, old_row = threadIdx.x / pieces;
  const bool any_old = p.boxes != nullptr && kTurn != kElements && old_row < min(old_rows, slot0);
  const T* const old_keys = k_to + threadIdx.x % pieces * 8;
  uint4 old[kOldAhead];
  const auto request_old = [&](int slot) {
#pragma unroll
    for (int u = 0; u < kOldAhead; ++u) {
      const int mine = slot + u * old_rows;
      old[u] = load16(old_keys + (mine < slot0 ? mine : old_row) * p.dim);
    }
  };
  if (any_old) request_old(old_row);
  // keys: a piece of the head to a thread
  const int key_rows = kThreads / items, key_row = threadIdx.x / items, key_item = threadIdx.x % items;
  uint4 lo[2], hi[2];
  bool any = false;
  if (key_row < key_rows)
    for (int t0 = key_row; t0 < tokens; t0 += kAhead * key_rows) {
      Item<T, kTurn> some[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int t = t0 + u * key_rows;
        if (t < tokens)
          some[u].load(p, static_cast<const T*>(p.k.data) + (row0 + t) * p.k.row + kv * p.k.head, cos + static_cast<long long>(t) * half,
                       sin + static_cast<long long>(t) * half, key_item);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int t = t0 + u * key_rows;
        if (t >= tokens) break;
        some[u].store(p, k_to + (slot0 + t) * p.dim, key_item);
        lo[0] = any ? smaller<T>(lo[0], some[u].a) : some[u].a;
        hi[0] = any ? larger<T>(hi[0], some[u].a) : some[u].a;
        if (kTurn == kHalves) {
          lo[1] = any ? smaller<T>(lo[1], some[u].b) : some[u].b;
          hi[1] = any ? larger<T>(hi[1], some[u].b) : some[u].b;
        }
        any = true;
      }
    }
  if (kTurn != kElements && p.boxes != nullptr) {
#pragma unroll
    for (int e = 0; e < 1 + (kTurn == kHalves); ++e) {
      box_parts[0][threadIdx.x][e] = lo[e];
      box_parts[1][threadIdx.x][e] = hi[e];
    }
  }
  // queries and values; where there are few, other warps have them than the keys
  const int queries = tokens * group * items;
  for (int x0 = (threadIdx.x + kThreads - 32) % kThreads; x0 < queries; x0 += kAhead * kThreads) {
    Item<T, kTurn> some[kAhead];
    int item[kAhead];
    T* to_row[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int x = x0 + u * kThreads;
      if (x >= queries) break;
      const int head_row = x / items, t = head_row / group, g = head_row - t * group;
      item[u] = x - head_row * items;
      to_row[u] = q_out + (static_cast<long long>(row0 + t) * p.heads + g) * p.dim;
      some[u].load(p, static_cast<const T*>(p.q.data) + (row0 + t) * p.q.row + (kv * group + g) * p.q.head,
                   cos + static_cast<long long>(t) * half, sin + static_cast<long long>(t) * half, item[u]);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (x0 + u * kThreads < queries) some[u].store(p, to_row[u], item[u]);
  }
  for (int x0 = (threadIdx.x + kThreads - 96) % kThreads; x0 < tokens * pieces; x0 += 4 * kThreads) {
    uint4 some[4];
    T* to_piece[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int x = x0 + u * kThreads;
      if (x >= tokens * pieces) break;
      const int t = x / pieces, d = (x - t * pieces) * 8;
      to_piece[u] = v_to + t * p.dim + d;
      some[u] = load16(static_cast<const T*>(p.v.data) + (row0 + t) * p.v.row + kv * p.v.head + d);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (x0 + u * kThreads < tokens * pieces) *reinterpret_cast<uint4*>(to_piece[u]) = some[u];
  }
  if (p.boxes == nullptr) return;
  uint32_t* const box = reinterpret_cast<uint32_t*>(static_cast<T*>(p.boxes) + (static_cast<long long>(at) * p.kv_heads + kv) * 2 * p.dim);
  if constexpr (kTurn == kElements) {
    __syncthreads();  // the block's keys have been written
    for (int d = threadIdx.x; d < p.dim / 2; d += kThreads) {
      const uint32_t* const keys = reinterpret_cast<const uint32_t*>(k_to) + d;
      uint32_t low = *keys, high = low;
      for (int t = 1; t < slot0 + tokens; ++t) {
        const uint32_t key = keys[t * (p.dim / 2)];
        low = smaller<T>(low, key);
        high = larger<T>(high, key);
      }
      box[d] = low;
      box[p.dim / 2 + d] = high;
    }
  } else {
    if (any_old) {
      uint4 old_lo = old[0], old_hi = old[0];
      for (int slot = old_row;;) {
#pragma unroll
        for (int u = 0; u < kOldAhead; ++u) {
          old_lo = smaller<T>(old_lo, old[u]);
          old_hi = larger<T>(old_hi, old[u]);
        }
        slot += kOldAhead * old_rows;
        if (slot >= slot0) break;
        request_old(slot);
      }
      old_parts[0][threadIdx.x] = old_lo;
      old_parts[1][threadIdx.x] = old_hi;
    }
    __syncthreads();
    // a thread for two elements, the smallest or the largest
    for (int x = threadIdx.x; x < p.dim; x += kThreads) {
      const int high = x >= p.dim / 2, d = (x - high * (p.dim / 2)) * 2;
      int item = d / 8, piece = 0;
      if (kTurn == kHalves) {
        piece = d >= half && d < p.rotary;
        item = d < p.rotary ? (d - piece * half) / 8 : half / 8 + (d - p.rotary) / 8;
      }
      const auto part = [&](const uint4& v) { return (&v.x)[d % 8 / 2]; };
      uint32_t value = part(box_parts[high][item][piece]);
      for (int r = 1; r < min(key_rows, tokens); ++r) {
        const uint32_t other = part(box_parts[high][r * items + item][piece]);
        value = high ? larger<T>(value, other) : smaller<T>(value, other);
      }
      for (int r = 0; r < min(old_rows, slot0); ++r) {
        const uint32_t other = part(old_parts[high][r * pieces + d / 8]);
        value = high ? larger<T>(value, other) : smaller<T>(value, other);
      }
      box[x] = value;
    }
  }
}

template <typename T>
int launch(const AppendParams& p, bool interleaved, unsigned blocks, cudaStream_t stream) {
  const bool in_pieces = p.rotary % 16 == 0 && aligned16(p.cos) && aligned16(p.sin);
  const bool few = p.tokens <= 4ll * p.batch;
  const auto kern = interleaved ? (few ? append_kernel<T, kNeighbors, 1> : append_kernel<T, kNeighbors, 2>)
                    : in_pieces ? (few ? append_kernel<T, kHalves, 1> : append_kernel<T, kHalves, 2>)
                                : (few ? append_kernel<T, kElements, 1> : append_kernel<T, kElements, 2>);
  return launch_overlapped(kern, dim3(blocks), dim3(kThreads), 0, stream, p);
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
  const long long blocks = (cu_tokens ? (tokens >> p.page_shift) + 2ll * batch + 1 : batch) * kv_heads;
  if (blocks > 0x7fffffffll) return IEX_ERR_TOO_LARGE;
  return bf16 ? launch<__nv_bfloat16>(p, interleaved != 0, static_cast<unsigned>(blocks), static_cast<cudaStream_t>(stream))
              : launch<__half>(p, interleaved != 0, static_cast<unsigned>(blocks), static_cast<cudaStream_t>(stream));
}
