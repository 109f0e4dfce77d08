// What the kernels of the paged key-value cache share (paged_append.cu, paged_attention.cu, paged_select.cu).
//
// The cache: keys and values [pages, kv_heads, page_size, head_dim], one contiguous slab per page and head, pages at any
// distance.  Row r of the block table names the pages of a sequence in order, lengths[r] says how many positions it holds.
// Both come from the device and are not trusted: attention and selection read a length as one between 0 and what the row of the table
// can hold (held()), appending drops tokens behind the table, and positions of a page that is not one of the cache's are as if they
// were not held.
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"

namespace iex {
namespace paged {

constexpr int kMaxHeadDim = 128;
constexpr int kMinPage = 16, kMaxPage = 256;

inline bool page_size_ok(int page_size) {
  return page_size >= kMinPage && page_size <= kMaxPage && (page_size & (page_size - 1)) == 0;
}
inline bool heads_ok(int heads, int kv_heads, int head_dim) {
  return kv_heads > 0 && heads > 0 && heads % kv_heads == 0 && head_dim > 0 && head_dim % 8 == 0 && head_dim <= kMaxHeadDim &&
         heads <= (1 << 24) - 1;  // a row's elements are counted in 32 bits
}
// Positions, rounded up to whole pages, are counted in 32 bits.
inline bool table_ok(int table_width, int page_size) { return static_cast<long long>(table_width) * page_size <= 0x7fffff00ll; }
inline int log2_of(int power_of_two) {
  int bits = 0;
  while ((1 << bits) < power_of_two) ++bits;
  return bits;
}

// Positions that row `row` holds.
__device__ __forceinline__ int held(const int32_t* lengths, int row, int table_width, int page_shift) {
  const long long most = static_cast<long long>(table_width) << page_shift;
  const int length = lengths[row];
  return length <= 0 ? 0 : static_cast<int>(length < most ? length : most);
}

// This block has begun, and so have the others of its cluster: from then on their shared memory may be written.  Nothing that was
// written before is seen by them (ordering that takes half a microsecond).
__device__ __forceinline__ void cluster_begun() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait_begun() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// A launch in clusters of `cluster` blocks, that may begin while the kernel in front runs (launch_overlapped).
template <typename P>
int launch_clusters(void (*kern)(P), unsigned blocks, int cluster, int threads, size_t smem, cudaStream_t stream, const P& p) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
  return static_cast<int>(e != cudaSuccess ? e : cudaGetLastError());
}

// A matrix of rows and heads whose innermost dimension is contiguous, in elements.
struct Rows {
  const void* data;
  long long row, head;
};

// 16 bytes, where `there`; else v stays as it is.  Not invariant (".nc"): the kernel in front, which may still run when this one
// starts, can have written what is read, and loads that claim otherwise may be moved ahead of the wait for it.  A predicate, so
// that a row of such loads has no branches between them.
__device__ __forceinline__ void load_if(uint4& v, const void* p, bool there) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "@p ld.global.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
      : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w)
      : "l"(p), "r"(static_cast<int>(there))
      : "memory");
}
// The same for what this SM reads once, where `index` is not negative.
__device__ __forceinline__ void load_once_if(uint4& v, const void* p, int index) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ge.s32 p, %5, 0;\n\t"
      "@p ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
      : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w)
      : "l"(p), "r"(index)
      : "memory");
}
__device__ __forceinline__ uint4 load_once(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}

__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T rounded(float v);
template <>
__device__ __forceinline__ __half rounded<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 rounded<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

}  // namespace paged
}  // namespace iex
