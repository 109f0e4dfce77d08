// Attention of one new token per row over a paged key-value cache (paged.cuh):
//
//   out[r, h] = sum_t softmax_t(scale * q[r, h] . k[t]) v[t],   t over the positions that row r holds,
//
// with heads / kv_heads query heads to a key head, or over the positions of the pages that pages[r, kv_head] lists.  A segment is
// what one row and one key head (up to 16 of its query heads) have to read, in chunks of 16 positions.  One to sixteen flops a byte: HBM bounds it.
// 64 rows up to 4096, 32 query and 8 key heads of 128: 104 us, 6.2 TB/s; 2 rows of 131071: 147 us, 6.5 TB/s; 1 row of 500, 32 heads: 5.8 us.
//
// Work, where segments are many or uneven (attention_kernel): the chunks of all segments, in order, are shared out evenly to the
// warps of one block per SM, whatever the rows' lengths, a segment's start counted as kStart chunks; a warp that has a whole segment
// writes its rows, the others leave maximum, sum and product, which the block joins through shared memory and, where a segment reaches over
// several blocks, join_kernel joins from the workspace, in order.  Where there are few segments (cluster_kernel): a cluster of blocks for
// each, joined through distributed shared memory, without workspace or second launch.  Where many rows list the same pages:
// paged_shared.cu.
//
// A chunk: keys and values come straight from global memory into registers, 16 bytes a lane, the next chunk's keys requested
// when this one's scores are formed and its values after the product; the lengths of what a warp has on its way (8 KB) and nothing else covers
// the latency, no barriers.  Products are m16n8k16 with the positions (scores) or the elements of v (output) as
// the 16 rows and 8 query heads as the columns, so that a key head with few query heads does not pay for 16:
//   S^T = K Q^T    a lane's 16 bytes of a key are its fragments of two instructions: the order of a sum's terms is free as
//                  long as both operands agree
//   O^T = V^T P^T  a lane's 16 bytes of four positions, bytes paired up by prmt, are its fragments of four; the scores'
//                  accumulators become P^T by movmatrix
// The running maximum, sum and O are fp32.  P enters the second product as a 16-bit head and the 16-bit rest, so that what is lost of it
// does not show beside the output's own rounding; fp16 weights carry 2^15, which keeps small ones out of the subnormals.  bfloat16 values may be
// so large that their sum leaves fp32 although their average does not: see Walk::run and join.
#include <algorithm>
#include <cmath>

#include <cooperative_groups.h>

#include "paged_mma.cuh"
#include "paged_shared.cuh"

namespace iex {
namespace paged {
namespace {

namespace cg = cooperative_groups;

constexpr int kChunk = 16;
constexpr int kStart = 2;     // what a segment's start costs, in chunks
constexpr int kMinUnits = 4;  // of a warp, starts included: with less to do, fewer warps
constexpr int kJoinThreads = 128;
constexpr int kClusterWarps = 8;
constexpr int kMostBlocks = 8;  // of a cluster

struct AttentionParams {
  int rows, heads, kv_heads, dim, num_pages, page_shift, table_width, count;
  int parts;   // segments of a key head
  int blocks;  // of a cluster, or 0
  Rows q;
  const void *k_cache, *v_cache;
  long long k_page, v_page;
  const int32_t *table, *lengths, *pages;
  float scale_log2;  // the factor of a score in an exponent of 2
  void* out;
  int2* open;      // [blocks]: the segment that begins in a block and ends in another, or -1; the block that it ends in
  float2* stats;   // [blocks][2][heads of a segment]: maximum and sum of a block's part of a segment that ...
  float* product;  // [blocks][2][heads of a segment][dim bucket]  ... 0: began in front of the block, 1: begins in it
};

// The 8 x 8 matrix of 16-bit elements that the warp holds, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t t;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(t) : "r"(v));
  return t;
}
__device__ __forceinline__ uint32_t& word(uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
__device__ __forceinline__ float max_over_positions(float v) {  // of the lanes with the same lane % 4
  for (int d = 4; d < 32; d <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}
__device__ __forceinline__ float sum_over_positions(float v) {
  for (int d = 4; d < 32; d <<= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// Chunks of a segment of row `row`.
__device__ __forceinline__ int chunks_of(const AttentionParams& p, int row) {
  const int length = held(p.lengths, row, p.table_width, p.page_shift);
  if (p.pages == nullptr) return (length + kChunk - 1) / kChunk;
  const int pages = (length + (1 << p.page_shift) - 1) >> p.page_shift;
  return min(p.count, pages) << (p.page_shift - 4);
}

// A page of a row: its place in the cache and in the row of the table.
struct PageOfLane {
  int at, nth;
};

// What a warp has of a segment: of its chunks [first, stop), for the 8 NT query heads from head0.
//   PIECES: of 64 elements of a head; NT: groups of 8 query heads
template <typename T, int PIECES, int NT>
struct Walk {
  static constexpr int kHeads = 8 * NT, kDim = 64 * PIECES, kPitch = kDim + 4;
  float o[NT][PIECES][4][4], top[NT][2], sum[NT][2];

  // Where keep() puts o[n][i][j][e].
  static __device__ __forceinline__ int place(int n, int i, int j, int e) {
    const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    return (n * 8 + 2 * q + (e & 1)) * kPitch + i * 64 + g * 8 + 2 * j + (e >> 1);
  }

  // `scratch`: kHeads x kPitch of shared memory that is this warp's; `here`: query heads that there are; `early`: the lane's page of the
  // first 32, looked up before the row's length was known
  __device__ __forceinline__ void run(const AttentionParams& p, int row, int kv, int head0, int here, int first, int stop, int chunks,
                                      float* scratch, const PageOfLane* early = nullptr) {
    const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3, page = 1 << p.page_shift, sub_shift = p.page_shift - 4;
    const long long head_stride = static_cast<long long>(page) * p.dim;
    const uint4 none = make_uint4(0, 0, 0, 0);
    uint4 qr[NT][PIECES][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < PIECES; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int d = i * 64 + h * 32 + q * 8;
          qr[n][i][h] = none;
          load_if(qr[n][i][h], static_cast<const T*>(p.q.data) + row * p.q.row + (head0 + n * 8 + g) * p.q.head + d,
                  n * 8 + g < here && d < p.dim);
        }
    const int length = held(p.lengths, row, p.table_width, p.page_shift), held_pages = (length + page - 1) >> p.page_shift;
    // a lane's places in a chunk
    const T* const k_lane = static_cast<const T*>(p.k_cache) + kv * head_stride + g * p.dim + q * 8;
    const T* const v_lane = static_cast<const T*>(p.v_cache) + kv * head_stride + 2 * q * p.dim + g * 8;

    // which pages: lane i has entry `entry0 + i`
    int entry0 = 0, page_at = -1, page_nth = 0;
    const auto look_up = [&](int entry) {
      entry0 = entry;
      const int e = entry + lane;
      page_at = -1;
      page_nth = e;
      if (e < (chunks + (1 << sub_shift) - 1) >> sub_shift) {
        if (p.pages != nullptr) page_nth = p.pages[(static_cast<long long>(row) * p.kv_heads + kv) * p.count + e];
        if (page_nth >= 0 && page_nth < held_pages) page_at = p.table[static_cast<long long>(row) * p.table_width + page_nth];
        if (page_at >= p.num_pages) page_at = -1;
      }
    };
    struct Chunk {
      int valid;       // positions
      long long k, v;  // elements from the lane's place in the first page
    };
    const auto locate = [&](int c) {
      Chunk found{0, 0, 0};
      if (c >= stop) return found;
      const int e = c >> sub_shift, slot = (c & ((1 << sub_shift) - 1)) * kChunk;
      if (e >= entry0 + 32) look_up(e);
      const int where = __shfl_sync(0xffffffffu, page_at, e - entry0), nth = __shfl_sync(0xffffffffu, page_nth, e - entry0);
      if (where >= 0) {
        found.valid = max(0, min(kChunk, length - (nth << p.page_shift) - slot));
        found.k = where * p.k_page + slot * p.dim;
        found.v = where * p.v_page + slot * p.dim;
      }
      return found;
    };
    // What lies behind the head's elements or the row's positions is zero and never read.
    uint4 kr[2][PIECES][2], vr[4][PIECES];
    const auto clear = [&](auto& regs) {
#pragma unroll
      for (auto& some : regs)
#pragma unroll
        for (auto& one : some) one = uint4{};
    };
    const auto clear_k = [&] {
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int i = 0; i < PIECES; ++i) kr[r][i][0] = kr[r][i][1] = none;
    };
    const auto request_k = [&](const Chunk& c) {
      if (c.valid < kChunk) clear_k();
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int i = 0; i < PIECES; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            load_once_if(kr[r][i][h], k_lane + c.k + 8 * r * p.dim + i * 64 + h * 32,
                         g + 8 * r < c.valid && i * 64 + h * 32 + q * 8 < p.dim ? 0 : -1);
    };
    const auto request_v = [&](const Chunk& c) {
      if (c.valid < kChunk) clear(vr);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          const int t = (r & 1) + (r & 2) * 4;
          load_once_if(vr[r][i], v_lane + c.v + t * p.dim + i * 64, 2 * q + t < c.valid && i * 64 + g * 8 < p.dim ? 0 : -1);
        }
    };

    // Where elements of the product come out not finite, either v has infinite or NaN elements, of which a rest of a weight that is
    // 0 or below makes NaN, or large elements of v add up to more than fp32 holds.  The product is formed a second time with all weights
    // above zero as one number of which no sum overflows: what is not finite then is taken from there.  What is, is formed a third
    // time, with weights made as small, and divided by the weights' sum.
    enum { kReal, kPlaces, kSmaller };
    int pass = kReal;
    for (;;) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        top[n][0] = top[n][1] = -INFINITY;
        sum[n][0] = sum[n][1] = 0.f;
#pragma unroll
        for (int i = 0; i < PIECES; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][i][j][e] = 0.f;
      }
      clear_k();
      clear(vr);
      if (early != nullptr && first >> sub_shift < 32) {
        entry0 = 0;
        page_nth = early->nth;
        page_at = lane < (chunks + (1 << sub_shift) - 1) >> sub_shift && page_nth < held_pages && early->at < p.num_pages ? early->at : -1;
      } else {
        look_up(first >> sub_shift);
      }
      Chunk now = locate(first);
      request_k(now);
      request_v(now);
#pragma unroll 1
      for (int c = first; c < stop; ++c) {
        const Chunk next = locate(c + 1);
        float s[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
          for (int i = 0; i < PIECES; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint4 a = kr[0][i][h], b = kr[1][i][h], x = qr[n][i][h];
              mma<T>(s[n], a.x, b.x, a.y, b.y, x.x, x.y);
              mma<T>(s[n], a.z, b.z, a.w, b.w, x.z, x.w);
            }
        }
        request_k(next);
        uint32_t head[NT][2], rest[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          // s[e]: position g + (e & 2) * 4, query head 2 q + (e & 1)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n][e] = g + (e & 2) * 4 < now.valid ? s[n][e] * p.scale_log2 : -INFINITY;
          float old[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float high = fmaxf(top[n][e], max_over_positions(fmaxf(s[n][e], s[n][e + 2])));
            const float base = high == -INFINITY ? 0.f : high;
            old[e] = exp2f(top[n][e] - base);
            top[n][e] = high;
            s[n][e] = exp2f(s[n][e] - base + Half2<T>::kBias);
            s[n][e + 2] = exp2f(s[n][e + 2] - base + Half2<T>::kBias);
            sum[n][e] = sum[n][e] * old[e] + (s[n][e] + s[n][e + 2]);
          }
          if (__any_sync(0xffffffffu, old[0] != 1.f || old[1] != 1.f)) {
#pragma unroll
            for (int i = 0; i < PIECES; ++i)
#pragma unroll
              for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[n][i][j][e] *= old[e & 1];
          }
          if (pass != kReal) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              s[n][e] = pass == kSmaller ? s[n][e] * Half2<T>::kSmall : s[n][e] > 0.f ? Half2<T>::kSmall : s[n][e];
          }
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const uint32_t both = Half2<T>::pack(s[n][2 * t], s[n][2 * t + 1]);
            const float2 kept = Half2<T>::unpack(both);
            head[n][t] = transposed(both);
            rest[n][t] = transposed(pass == kPlaces ? 0 : Half2<T>::pack(s[n][2 * t] - kept.x, s[n][2 * t + 1] - kept.y));
          }
        }
#pragma unroll
        for (int i = 0; i < PIECES; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            // rows g and g + 8 of the instruction: elements 2 j and 2 j + 1 of the lanes' 8
            const uint32_t v0 = word(vr[0][i], j), v1 = word(vr[1][i], j), v2 = word(vr[2][i], j), v3 = word(vr[3][i], j);
            const uint32_t a0 = __byte_perm(v0, v1, 0x5410), a1 = __byte_perm(v0, v1, 0x7632);
            const uint32_t a2 = __byte_perm(v2, v3, 0x5410), a3 = __byte_perm(v2, v3, 0x7632);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma<T>(o[n][i][j], a0, a1, a2, a3, head[n][0], head[n][1]);
              if (pass != kPlaces) mma<T>(o[n][i][j], a0, a1, a2, a3, rest[n][0], rest[n][1]);
            }
          }
        request_v(next);
        now = next;
      }
      if (pass == kSmaller) break;
      bool odd = false;  // another pass is needed
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < PIECES; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float& mine = o[n][i][j][e];
              const bool there = n * 8 + 2 * q + (e & 1) < here;
              if (pass == kReal) {
                odd |= there & !finite(mine);
              } else {
                const float before = scratch[place(n, i, j, e)];
                const bool large = Half2<T>::kOverflows && !finite(before) && finite(mine);
                odd |= there & large;
                mine = finite(before) ? before : large ? INFINITY : mine;
              }
            }
      if (!__any_sync(0xffffffffu, odd)) break;
      keep(scratch);
      pass = pass == kReal ? kPlaces : kSmaller;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) sum[n][e] = sum_over_positions(sum[n][e]);
    if (Half2<T>::kOverflows && pass == kSmaller) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float factor = to_average<T>(sum[n][e & 1]);
#pragma unroll
          for (int i = 0; i < PIECES; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float& mine = o[n][i][j][e];
              const float before = scratch[place(n, i, j, e)];
              mine = finite(before) ? before * factor : finite(mine) ? mine * factor * (1.f / Half2<T>::kSmall) : before;
            }
        }
#pragma unroll
      for (int n = 0; n < NT; ++n) sum[n][0] = -sum[n][0], sum[n][1] = -sum[n][1];
    }
  }

  // The product as it is, [kHeads][kPitch]; every lane writes what it alone reads again.
  __device__ __forceinline__ void keep(float* to) const {
    const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int i = 0; i < PIECES; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            *reinterpret_cast<float2*>(to + (n * 8 + 2 * q + e) * kPitch + i * 64 + g * 8 + 2 * j) =
                make_float2(o[n][i][j][e], o[n][i][j][e + 2]);
  }
  __device__ __forceinline__ void keep(float* to, float2* stats) const {
    const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    keep(to);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (g == 0) stats[n * 8 + 2 * q + e] = make_float2(top[n][e], sum[n][e]);
  }
  __device__ __forceinline__ void write(const AttentionParams& p, int row, int head0, int here) const {
    const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int h = n * 8 + 2 * q + e;
        const float factor = to_average<T>(sum[n][e]);
        T* const to = static_cast<T*>(p.out) + (static_cast<long long>(row) * p.heads + head0 + h) * p.dim;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          uint4 v;
#pragma unroll
          for (int j = 0; j < 4; ++j) word(v, j) = Half2<T>::pack(o[n][i][j][e] * factor, o[n][i][j][e + 2] * factor);
          if (h < here && i * 64 + g * 8 < p.dim) *reinterpret_cast<uint4*>(to + i * 64 + g * 8) = v;
        }
      }
  }
};

// Four elements of the product, and the sum, of several parts of a segment.
struct Joined {
  float high, sum, o[4];
};
// `each` calls what it gets for every part, in order; stats: its maximum and sum; product: its elements.  No more than MOST parts:
// products that are finite may add up to more than fp32 holds, so that they and the sums get a factor.
template <typename T, int MOST, typename Each, typename Stats, typename Product>
__device__ __forceinline__ Joined join(Each each, Stats stats, Product product) {
  constexpr float kUnit = Half2<T>::kOverflows ? 1.f / MOST : 1.f;
  static_assert((MOST & (MOST - 1)) == 0, "an exact factor");
  Joined j{-INFINITY, 0.f, {0.f, 0.f, 0.f, 0.f}};
  bool any_averaged = false;
  each([&](int i) {
    const float2 s = stats(i);
    j.high = fmaxf(j.high, s.x);
    any_averaged |= averaged<T>(s.y);
  });
  const float base = j.high == -INFINITY ? 0.f : j.high;
  each([&](int i) {
    const float2 s = stats(i);
    const float4 v = product(i);
    const float weight = exp2f(s.x - base) * kUnit;
    j.sum += (Half2<T>::kOverflows ? fabsf(s.y) : s.y) * weight;
    j.o[0] += v.x * weight;
    j.o[1] += v.y * weight;
    j.o[2] += v.z * weight;
    j.o[3] += v.w * weight;
  });
  if (any_averaged) {  // then this is an average, too
    const float factor = to_average<T>(j.sum);
    j.o[0] = j.o[1] = j.o[2] = j.o[3] = 0.f;
    each([&](int i) {
      const float2 s = stats(i);
      const float4 v = product(i);
      const float weight = exp2f(s.x - base) * kUnit * factor * (averaged<T>(s.y) ? -s.y : 1.f);
      j.o[0] += v.x * weight;
      j.o[1] += v.y * weight;
      j.o[2] += v.z * weight;
      j.o[3] += v.w * weight;
    });
    j.sum = -j.sum;
  }
  return j;
}
template <typename T>
__device__ __forceinline__ void write4(const AttentionParams& p, int row, int head, int d, float sum, float o0, float o1, float o2,
                                       float o3) {
  const float factor = to_average<T>(sum);
  T* const to = static_cast<T*>(p.out) + (static_cast<long long>(row) * p.heads + head) * p.dim + d;
  *reinterpret_cast<uint2*>(to) = make_uint2(Half2<T>::pack(o0 * factor, o1 * factor), Half2<T>::pack(o2 * factor, o3 * factor));
}

// Warps of a block: as many as there are registers for.
constexpr int warps_of(int pieces, int nt) { return pieces * nt == 1 ? 16 : pieces * nt == 2 ? 12 : 8; }

template <typename T, int PIECES, int NT>
__global__ void __launch_bounds__(32 * warps_of(PIECES, NT), 1) attention_kernel(const __grid_constant__ AttentionParams p) {
  using W = Walk<T, PIECES, NT>;
  constexpr int kHeads = W::kHeads, kDim = W::kDim, kPitch = W::kPitch, kWarps = warps_of(PIECES, NT), kThreads = 32 * kWarps;
  extern __shared__ float parts_of_warps[];  // [warp][2][kHeads][kPitch], then [warp][2][kHeads] float2
  __shared__ long long before[kThreads + 1];  // units (of one segment) of the rows in front of a thread's
  __shared__ long long warp_sums[kWarps];
  __shared__ int segment_of[kWarps][2], last_block[kWarps], ends[kWarps];
  __shared__ int2 place_of[kWarps][2];  // of the segment: row, part of it
  float2* const stats_of_warps = reinterpret_cast<float2*>(parts_of_warps + 2 * kWarps * kHeads * kPitch);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per_row = p.kv_heads * p.parts, group = p.heads / p.kv_heads;

  grid_dependency_wait();
  // ---- how the work is shared out: a segment is a unit for each chunk behind kStart units
  const int rows_each = (p.rows + kThreads - 1) / kThreads;
  const auto units_of = [&](int chunks) { return chunks == 0 ? 0 : chunks + kStart; };
  {
    long long mine = 0;
    for (int r = threadIdx.x * rows_each, i = 0; i < rows_each && r < p.rows; ++i, ++r) mine += units_of(chunks_of(p, r));
    long long sum = mine;
    for (int d = 1; d < 32; d <<= 1) {
      const long long other = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += other;
    }
    if (lane == 31) warp_sums[warp] = sum;
    __syncthreads();
    long long front = 0;
    for (int w = 0; w < warp; ++w) front += warp_sums[w];
    before[threadIdx.x] = front + sum - mine;
    if (threadIdx.x == kThreads - 1) before[kThreads] = front + sum;
    if (lane < 2) segment_of[warp][lane] = -1;
    __syncthreads();
  }
  const long long total = before[kThreads] * per_row;
  const int workers = static_cast<int>(min(static_cast<long long>(gridDim.x) * kWarps, (total + kMinUnits - 1) / kMinUnits));
  const int worker = blockIdx.x * kWarps + warp;
  const bool small = total < 1 << 20;  // products with numbers of workers fit 32 bits
  const auto share = [&](int w) {      // where the units of worker w begin
    return small ? static_cast<long long>(static_cast<uint32_t>(total) * static_cast<uint32_t>(w) / static_cast<uint32_t>(workers))
                 : total * w / workers;
  };
  const long long begin = worker < workers ? share(worker) : 0, end = worker < workers ? share(worker + 1) : 0;

  // rows that hold nothing
  for (int r = blockIdx.x; r < p.rows; r += gridDim.x)
    if (chunks_of(p, r) == 0) {
      uint4* to = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + static_cast<long long>(r) * p.heads * p.dim);
      for (int i = threadIdx.x; i < p.heads * p.dim / 8; i += kThreads) to[i] = make_uint4(0, 0, 0, 0);
    }

  // ---- the warp's own part
  int row = 0, part_of_row = 0, chunks = 0;  // the segment
  long long at = begin, segment_begin = begin;
  if (begin < end) {
    int lo = -1;  // the last thread whose rows begin at or in front of `begin`
#pragma unroll
    for (int t = 0; t < kThreads; t += 32) lo += __popc(__ballot_sync(0xffffffffu, before[t + lane] * per_row <= begin));
    row = lo * rows_each;
    long long rest = begin - before[lo] * per_row;
    for (chunks = chunks_of(p, row); rest >= static_cast<long long>(units_of(chunks)) * per_row; chunks = chunks_of(p, ++row))
      rest -= static_cast<long long>(units_of(chunks)) * per_row;
    part_of_row = small ? static_cast<int>(static_cast<uint32_t>(rest) / static_cast<uint32_t>(units_of(chunks)))
                        : static_cast<int>(rest / units_of(chunks));
    segment_begin = begin - (rest - static_cast<long long>(part_of_row) * units_of(chunks));
  }
  while (at < end) {
    const int first = static_cast<int>(max(0ll, at - segment_begin - kStart));
    const int stop = static_cast<int>(min(static_cast<long long>(chunks), max(0ll, end - segment_begin - kStart)));
    if (first < stop) {
      const int kv = part_of_row / p.parts, head0 = kv * group + (part_of_row - kv * p.parts) * kHeads;
      const int here = min(kHeads, (kv + 1) * group - head0);  // query heads
      W walk;
      // the warp's last part is written last: its place is free until then
      walk.run(p, row, kv, head0, here, first, stop, chunks, parts_of_warps + (warp * 2 + 1) * kHeads * kPitch);
      if (first == 0 && stop == chunks) {
        walk.write(p, row, head0, here);
      } else {
        const int slot = first == 0 ? 1 : 0;
        walk.keep(parts_of_warps + (warp * 2 + slot) * kHeads * kPitch, stats_of_warps + (warp * 2 + slot) * kHeads);
        if (lane == 0) {
          segment_of[warp][slot] = row * per_row + part_of_row;
          place_of[warp][slot] = make_int2(row, part_of_row);
          if (slot == 0) ends[warp] = stop == chunks;
          // the block whose warp has the segment's last unit
          else last_block[warp] = static_cast<int>(((segment_begin + units_of(chunks)) * workers - 1) / total) / kWarps;
        }
      }
    }
    at = segment_begin += units_of(chunks);
    if (at < end && ++part_of_row == per_row) {
      part_of_row = 0;
      do chunks = chunks_of(p, ++row);
      while (chunks == 0);
    }
  }
  __syncthreads();
  grid_launch_dependents();

  // ---- parts of one segment that several warps have; every warp for itself finds the segments, and joins some of their query heads
  static_assert(2 * kWarps <= 32, "a lane for each part");
  const int segment_here = lane < 2 * kWarps ? segment_of[lane / 2][lane % 2] : -1;
  const uint32_t parts_there = __ballot_sync(0xffffffffu, segment_here >= 0), in_front = parts_there & ((1u << lane) - 1);
  const int segment_before = __shfl_sync(0xffffffffu, segment_here, in_front != 0 ? 31 - __clz(in_front) : lane);
  uint32_t starts = __ballot_sync(0xffffffffu, segment_here >= 0 && (in_front == 0 || segment_before != segment_here));
  const int most_heads = min(kHeads, group);
  int opened = -1, opened_until = 0, turn = warp;  // the first query head that this warp joins
  while (starts != 0) {
    const int from = __ffs(starts) - 1;
    starts &= starts - 1;
    const uint32_t behind = starts != 0 ? ~0u << (__ffs(starts) - 1) : 0u;
    const uint32_t members = parts_there & (~0u << from) & ~behind;
    const int last = 31 - __clz(members);
    const bool begins = from % 2 == 1, finished = last % 2 == 0 && ends[last / 2];
    if (begins && !finished) {
      opened = segment_of[from / 2][1];
      opened_until = last_block[from / 2];
    }
    if (turn >= most_heads) {
      turn -= most_heads;
      continue;
    }
    const int2 place = place_of[from / 2][from % 2];
    const int seg_row = place.x, kv = p.parts == 1 ? place.y : place.y / p.parts, d = lane * 4;
    const int head0 = kv * group + (place.y - kv * p.parts) * kHeads, here = min(kHeads, (kv + 1) * group - head0);
    for (; turn < most_heads; turn += kWarps) {
      if (turn >= here) continue;
      const int h = turn;
      const Joined j = join<T, 32>(
          [&](auto add) {
            for (uint32_t m = members; m != 0; m &= m - 1) add(__ffs(m) - 1);
          },
          [&](int i) { return stats_of_warps[i * kHeads + h]; },
          [&](int i) { return d < p.dim ? *reinterpret_cast<const float4*>(parts_of_warps + (i * kHeads + h) * kPitch + d) : float4{}; });
      if (begins && finished) {
        if (d < p.dim) write4<T>(p, seg_row, head0 + h, d, j.sum, j.o[0], j.o[1], j.o[2], j.o[3]);
      } else {
        const long long slot = (static_cast<long long>(blockIdx.x) * 2 + begins) * kHeads + h;
        if (d < p.dim) *reinterpret_cast<float4*>(p.product + slot * kDim + d) = make_float4(j.o[0], j.o[1], j.o[2], j.o[3]);
        if (lane == 0) p.stats[slot] = make_float2(j.high, j.sum);
      }
    }
    turn -= most_heads;
  }
  if (threadIdx.x == 0) p.open[blockIdx.x] = make_int2(opened, opened_until);
}

// A cluster of p.blocks blocks per segment.  Query head h of the segment is joined by block h % p.blocks, to which the others send what
// they have of it.
template <typename T, int PIECES, int NT>
__global__ void __launch_bounds__(32 * kClusterWarps, 1) cluster_kernel(const __grid_constant__ AttentionParams p) {
  using W = Walk<T, PIECES, NT>;
  constexpr int kHeads = W::kHeads, kPitch = W::kPitch, kThreads = 32 * kClusterWarps;
  extern __shared__ float parts_of_warps[];                       // [warp][kHeads][kPitch]
  __shared__ float2 stats_of_warps[kClusterWarps][kHeads];
  __shared__ alignas(16) float received[kHeads + kMostBlocks][kPitch];  // [block][head / blocks], (blocks - 1 places stay free)
  __shared__ float2 received_stats[kHeads + kMostBlocks];
  cg::cluster_group cluster = cg::this_cluster();
  const int warp = threadIdx.x >> 5, blocks = p.blocks, rank = blocks > 1 ? static_cast<int>(cluster.block_rank()) : 0;
  const int per_row = p.kv_heads * p.parts, group = p.heads / p.kv_heads, segment = blockIdx.x / blocks;
  const int row = segment / per_row, part = segment - row * per_row, kv = part / p.parts;
  const int head0 = kv * group + (part - kv * p.parts) * kHeads, here = min(kHeads, (kv + 1) * group - head0);
  grid_dependency_wait();
  grid_launch_dependents();
  // the first 32 pages, beside the length
  const int lane = threadIdx.x & 31;
  PageOfLane early{-1, lane};
  if (p.pages != nullptr) early.nth = lane < p.count ? p.pages[(static_cast<long long>(row) * p.kv_heads + kv) * p.count + lane] : -1;
  if (early.nth >= 0 && early.nth < p.table_width) early.at = p.table[static_cast<long long>(row) * p.table_width + early.nth];
  const int chunks = chunks_of(p, row), vectors = p.dim / 4;
  if (chunks == 0) {
    for (int x = threadIdx.x; rank == 0 && x < here * vectors; x += kThreads)
      write4<T>(p, row, head0 + x / vectors, x % vectors * 4, 0.f, 0.f, 0.f, 0.f, 0.f);
    return;
  }
  if (blocks > 1) cluster_begun();
  // the warps of all blocks side by side, so that few chunks are spread over all of them
  const int workers = min(chunks, blocks * kClusterWarps), worker = warp * blocks + rank;
  if (worker < workers) {
    W walk;
    float* const mine = parts_of_warps + warp * kHeads * kPitch;
    walk.run(p, row, kv, head0, here, static_cast<int>(static_cast<long long>(chunks) * worker / workers),
             static_cast<int>(static_cast<long long>(chunks) * (worker + 1) / workers), chunks, mine, &early);
    walk.keep(mine, stats_of_warps[warp]);
  }
  __syncthreads();
  const int working = workers > rank ? (workers - rank + blocks - 1) / blocks : 0;
  const int heads_each = (kHeads + blocks - 1) / blocks;
  if (blocks > 1) cluster_wait_begun();
  for (int x = threadIdx.x; x < here * vectors; x += kThreads) {
    const int h = x / vectors, d = (x - h * vectors) * 4;
    const Joined j = join<T, kClusterWarps>(
        [&](auto add) {
          for (int i = 0; i < working; ++i) add(i);
        },
        [&](int i) { return stats_of_warps[i][h]; },
        [&](int i) { return *reinterpret_cast<const float4*>(parts_of_warps + (i * kHeads + h) * kPitch + d); });
    if (blocks == 1) {
      write4<T>(p, row, head0 + h, d, j.sum, j.o[0], j.o[1], j.o[2], j.o[3]);
    } else {
      const int place = rank * heads_each + h / blocks, owner = h % blocks;
      *cluster.map_shared_rank(reinterpret_cast<float4*>(&received[place][d]), owner) = make_float4(j.o[0], j.o[1], j.o[2], j.o[3]);
      if (d == 0) *cluster.map_shared_rank(&received_stats[place], owner) = make_float2(j.high, j.sum);
    }
  }
  if (blocks == 1) return;
  cluster.sync();
  for (int x = threadIdx.x; x < heads_each * vectors; x += kThreads) {
    const int nth = x / vectors, h = nth * blocks + rank, d = (x - nth * vectors) * 4;
    if (h >= here) break;
    const Joined j = join<T, kMostBlocks>(
        [&](auto add) {
          for (int i = 0; i < blocks; ++i) add(i);
        },
        [&](int i) { return received_stats[i * heads_each + nth]; },
        [&](int i) { return *reinterpret_cast<const float4*>(&received[i * heads_each + nth][d]); });
    write4<T>(p, row, head0 + h, d, j.sum, j.o[0], j.o[1], j.o[2], j.o[3]);
  }
}

// A block for each query head of the segment that begins in block blockIdx.x of the kernel in front and ends in another.
template <typename T, int PIECES, int NT>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const __grid_constant__ AttentionParams p) {
  constexpr int kHeads = 8 * NT, kDim = 64 * PIECES, kJoinWarps = kJoinThreads / 32;
  __shared__ float2 stats[kJoinWarps];
  __shared__ float4 products[kJoinWarps][32];
  grid_dependency_wait();
  grid_launch_dependents();
  const int2 open = p.open[blockIdx.x];
  if (open.x < 0) return;
  const int per_row = p.kv_heads * p.parts, group = p.heads / p.kv_heads, h = blockIdx.y;
  const int row = open.x / per_row, part = open.x - row * per_row, kv = part / p.parts;
  const int head0 = kv * group + (part - kv * p.parts) * kHeads;
  if (head0 + h >= (kv + 1) * group) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = lane * 4;
  const int n = open.y - static_cast<int>(blockIdx.x) + 1;
  // every warp joins a quarter of the parts, and the first one the quarters
  static_assert(kNumSMs <= 256 * kJoinWarps, "parts of a warp");
  constexpr float kUnit = Half2<T>::kOverflows ? 1.f / 256 : 1.f;  // as in join()
  float high = -INFINITY, sum = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  bool any_averaged = false;
  const auto slot_of = [&](int i) { return (static_cast<long long>(blockIdx.x + i) * 2 + (i == 0)) * kHeads + h; };
  const auto product_of = [&](long long slot) { return *reinterpret_cast<const float4*>(p.product + slot * kDim + (d < p.dim ? d : 0)); };
  for (int i = warp; i < n; i += kJoinWarps) {
    const long long slot = slot_of(i);
    const float2 s = p.stats[slot];
    const float4 v = product_of(slot);
    const float next = fmaxf(high, s.x), base = next == -INFINITY ? 0.f : next;
    const float old = exp2f(high - base), weight = exp2f(s.x - base) * kUnit;
    high = next;
    any_averaged |= averaged<T>(s.y);
    sum = sum * old + (Half2<T>::kOverflows ? fabsf(s.y) : s.y) * weight;
    o.x = o.x * old + v.x * weight;
    o.y = o.y * old + v.y * weight;
    o.z = o.z * old + v.z * weight;
    o.w = o.w * old + v.w * weight;
  }
  if (any_averaged) {
    const float factor = to_average<T>(sum), base = high == -INFINITY ? 0.f : high;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = warp; i < n; i += kJoinWarps) {
      const long long slot = slot_of(i);
      const float2 s = p.stats[slot];
      const float4 v = product_of(slot);
      const float weight = exp2f(s.x - base) * kUnit * factor * (averaged<T>(s.y) ? -s.y : 1.f);
      o.x += v.x * weight;
      o.y += v.y * weight;
      o.z += v.z * weight;
      o.w += v.w * weight;
    }
    sum = -sum;
  }
  if (lane == 0) stats[warp] = make_float2(high, sum);
  products[warp][lane] = o;
  __syncthreads();
  if (warp != 0 || d >= p.dim) return;
  const Joined j = join<T, kJoinWarps>(
      [&](auto add) {
        for (int i = 0; i < kJoinWarps; ++i) add(i);
      },
      [&](int i) { return stats[i]; }, [&](int i) { return products[i][lane]; });
  write4<T>(p, row, head0 + h, d, j.sum, j.o[0], j.o[1], j.o[2], j.o[3]);
}

// Query heads of a segment: 8, or 16 where a key head has more than 8.
int segment_heads(int heads, int kv_heads) { return heads / kv_heads > 8 ? 16 : 8; }

size_t open_bytes() { return (kNumSMs * sizeof(int2) + 255) / 256 * 256; }
size_t stats_bytes(int heads) { return static_cast<size_t>(kNumSMs) * 2 * heads * sizeof(float2); }
size_t product_bytes(int heads, int head_dim) {
  return static_cast<size_t>(kNumSMs) * 2 * heads * (head_dim > 64 ? 128 : 64) * sizeof(float);
}

// Blocks of a cluster for each segment, or 0 for attention_kernel; from the most that the rows could hold.
//
// attention_kernel with join_kernel behind it takes 13 us before anything is read (how the work is shared out, joining twice), a
// cluster 6; but it keeps all SMs busy until the end, where clusters leave some idle and last as long as the longest row.
// Rows are taken to hold kFill of the most on average, with listed pages all: a short row in a wide table is taken for a long one (1 row of
// 500, 32 heads: 5.8 us up to 85 columns of 64, 14.4 above).  Measured, attention_kernel / clusters, us: 1 row of 500, 32
// heads 14.4 / 5.8; 4 rows up to 4096, 8 key heads 17.4 / 15.9; 16 rows of 32 listed pages of 64 29.0 / 27.7; 1 row of 16384, 8 key heads
// 20.1 / 26.2; 32 rows up to 8192, one key head 27.2 / 33.0.
int cluster_blocks(long long segments, long long most_chunks, int head_dim, bool listed) {
  constexpr double kSaved = 7.0, kFill = 0.65, kRate = 6.5e6;  // us, -, bytes a us
  if (segments > kNumSMs) return 0;
  int blocks = 1;
  while (blocks < kMostBlocks && segments * blocks * 2 <= kNumSMs && most_chunks > blocks * kClusterWarps) blocks *= 2;
  const double us = segments * static_cast<double>(most_chunks) * kChunk * head_dim * 4 / kRate;
  return us * (static_cast<double>(kNumSMs) / (segments * blocks) - (listed ? 1.0 : kFill)) < kSaved ? blocks : 0;
}

template <typename Kernel>
int allow_shared(Kernel kern, int smem) {
  return smem > 40 * 1024 ? static_cast<int>(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) : 0;
}

template <typename T, int PIECES, int NT>
int launch(const AttentionParams& p, double chunks, cudaStream_t stream) {
  using W = Walk<T, PIECES, NT>;
  if (p.blocks > 0) {
    const auto kern = cluster_kernel<T, PIECES, NT>;
    constexpr int smem = kClusterWarps * W::kHeads * W::kPitch * 4;
    if (const int st = allow_shared(kern, smem)) return st;
    return launch_clusters<AttentionParams>(kern, p.rows * p.kv_heads * p.parts * p.blocks, p.blocks, 32 * kClusterWarps, smem, stream, p);
  }
  constexpr int kWarps = warps_of(PIECES, NT), smem = 2 * kWarps * W::kHeads * (W::kPitch * 4 + 8);
  const int blocks = static_cast<int>(std::min<double>(kNumSMs, std::max(1.0, std::ceil(chunks / (2 * kWarps)))));
  const auto kern = attention_kernel<T, PIECES, NT>;
  if (const int st = allow_shared(kern, smem)) return st;
  if (const int st = launch_overlapped(kern, dim3(blocks), dim3(32 * kWarps), smem, stream, p)) return st;
  return launch_overlapped(join_kernel<T, PIECES, NT>, dim3(blocks, std::min(W::kHeads, p.heads / p.kv_heads)), dim3(kJoinThreads), 0,
                           stream, p);
}

template <typename T>
int launch(const AttentionParams& p, double chunks, cudaStream_t stream) {
  const bool wide = p.dim > 64, many = segment_heads(p.heads, p.kv_heads) > 8;
  if (wide) return many ? launch<T, 2, 2>(p, chunks, stream) : launch<T, 2, 1>(p, chunks, stream);
  return many ? launch<T, 1, 2>(p, chunks, stream) : launch<T, 1, 1>(p, chunks, stream);
}

// Segments of a call, and the chunks that each could have.
struct Extent {
  long long segments, chunks;
};
Extent extent(int rows, int heads, int kv_heads, int page_size, int table_width, bool listed, int count) {
  const int n = segment_heads(heads, kv_heads);
  return {static_cast<long long>(rows) * kv_heads * ((heads / kv_heads + n - 1) / n),
          static_cast<long long>(listed ? std::min(count, table_width) : table_width) * (page_size / kChunk)};
}

}  // namespace
}  // namespace paged
}  // namespace iex

extern "C" int iex_paged_attention_supported(int heads, int kv_heads, int head_dim, int page_size) {
  return iex::paged::heads_ok(heads, kv_heads, head_dim) && iex::paged::page_size_ok(page_size) ? 1 : 0;
}

extern "C" size_t iex_paged_attention_workspace_bytes(int rows, int heads, int kv_heads, int head_dim, int num_pages, int page_size,
                                                      int table_width, int listed, int count) {
  using namespace iex::paged;
  if (rows <= 0 || num_pages < 0 || table_width < 0 || count < 0 || !iex_paged_attention_supported(heads, kv_heads, head_dim, page_size)) return 0;
  if (listed)
    if (const size_t bytes = shared_workspace_bytes(rows, heads, kv_heads, head_dim, num_pages, page_size, table_width, count)) return bytes;
  const Extent e = extent(rows, heads, kv_heads, page_size, table_width, listed != 0, count);
  if (cluster_blocks(e.segments, e.chunks, head_dim, listed != 0) > 0) return 0;
  const int n = segment_heads(heads, kv_heads);
  return open_bytes() + stats_bytes(n) + product_bytes(n, head_dim);
}

extern "C" int iex_paged_attention(int rows, int heads, int kv_heads, int head_dim, int bf16, const void* q, long long q_row,
                                   long long q_head, const void* k_cache, long long k_page, const void* v_cache,
                                   long long v_page, int num_pages, int page_size, const int32_t* block_table,
                                   int table_width, const int32_t* lengths, const int32_t* pages, int count, float scale,
                                   void* out, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace iex::paged;
  if (rows < 0 || num_pages < 0 || table_width < 0 || count < 0) return IEX_ERR_BAD_ARG;
  if (!iex_paged_attention_supported(heads, kv_heads, head_dim, page_size)) return IEX_ERR_UNSUPPORTED;
  const float scale_log2 = static_cast<float>(scale * 1.4426950408889634);  // of a score, in an exponent of 2
  if (!std::isfinite(scale_log2)) return IEX_ERR_BAD_ARG;
  if (rows == 0) return IEX_OK;
  if (!q || !out || !lengths || (table_width > 0 && !block_table) || (num_pages > 0 && (!k_cache || !v_cache)))
    return IEX_ERR_BAD_ARG;
  if (q_row % 8 != 0 || q_head % 8 != 0 || k_page % 8 != 0 || v_page % 8 != 0 || !iex::aligned16(q) || !iex::aligned16(out) ||
      !iex::aligned16(k_cache) || !iex::aligned16(v_cache) || !iex::aligned16(workspace))
    return IEX_ERR_UNSUPPORTED;
  if (static_cast<long long>(rows) * heads > 0x7fffffffll || !table_ok(table_width, page_size)) return IEX_ERR_TOO_LARGE;
  const size_t need =
      iex_paged_attention_workspace_bytes(rows, heads, kv_heads, head_dim, num_pages, page_size, table_width, pages != nullptr, count);
  if (need > 0 && (!workspace || workspace_bytes < need)) return IEX_ERR_BAD_ARG;
  if (pages != nullptr && shared_workspace_bytes(rows, heads, kv_heads, head_dim, num_pages, page_size, table_width, count) > 0) {
    SharedCall c{rows, heads, kv_heads, head_dim, num_pages, log2_of(page_size), table_width, count, {q, q_row, q_head},
                 k_cache, v_cache, k_page, v_page, block_table, lengths, pages, scale_log2, out};
    return shared_attention(c, bf16 != 0, workspace, static_cast<cudaStream_t>(stream));
  }
  const int segment = segment_heads(heads, kv_heads);
  const Extent e = extent(rows, heads, kv_heads, page_size, table_width, pages != nullptr, count);
  AttentionParams p{};
  p.rows = rows;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.dim = head_dim;
  p.num_pages = num_pages;
  p.page_shift = log2_of(page_size);
  p.table_width = table_width;
  p.count = count;
  p.parts = (heads / kv_heads + segment - 1) / segment;
  p.blocks = cluster_blocks(e.segments, e.chunks, head_dim, pages != nullptr);
  p.q = {q, q_row, q_head};
  p.k_cache = k_cache;
  p.v_cache = v_cache;
  p.k_page = k_page;
  p.v_page = v_page;
  p.table = block_table;
  p.lengths = lengths;
  p.pages = pages;
  p.scale_log2 = scale_log2;
  p.out = out;
  if (need > 0) {
    char* const ws = static_cast<char*>(workspace);
    p.open = reinterpret_cast<int2*>(ws);
    p.stats = reinterpret_cast<float2*>(ws + open_bytes());
    p.product = reinterpret_cast<float*>(ws + open_bytes() + stats_bytes(segment));
  }
  const double chunks = static_cast<double>(e.segments) * static_cast<double>(e.chunks);
  return bf16 ? launch<__nv_bfloat16>(p, chunks, static_cast<cudaStream_t>(stream))
              : launch<__half>(p, chunks, static_cast<cudaStream_t>(stream));
}
