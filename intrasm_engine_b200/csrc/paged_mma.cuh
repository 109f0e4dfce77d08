// Pairs of 16-bit elements and the matrix instructions on them, for the attention kernels of the paged cache.
#pragma once
#include "paged.cuh"

namespace iex {
namespace paged {

template <typename T>
struct Half2;
template <>
struct Half2<__half> {
  static constexpr float kBias = 15.f;  // weights are 2^15 times as large
  static constexpr bool kOverflows = false;  // whether sums of weights times values may leave fp32 where their average does not
  static constexpr float kSmall = 1.f;       // a weight of which no sum of fewer than 2^31 values overflows
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return reinterpret_cast<const uint32_t&>(v);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t v) { return __half22float2(reinterpret_cast<const __half2&>(v)); }
};
template <>
struct Half2<__nv_bfloat16> {
  static constexpr float kBias = 0.f;
  static constexpr bool kOverflows = true;
  static constexpr float kSmall = 0x1p-32f;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return reinterpret_cast<const uint32_t&>(v);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return __bfloat1622float2(reinterpret_cast<const __nv_bfloat162&>(v));
  }
};

// Parts of a softmax are handed on as maximum, sum of weights and product, or, where elements of the product would leave fp32, as
// maximum, the negative sum and the average: what a part's sum says of its elements.
template <typename T>
__device__ __forceinline__ bool averaged(float sum) { return Half2<T>::kOverflows && sum < 0.f; }
// What makes an element of the product the average.
template <typename T>
__device__ __forceinline__ float to_average(float sum) { return sum == 0.f ? 0.f : averaged<T>(sum) ? 1.f : 1.f / sum; }
__device__ __forceinline__ bool finite(float v) { return fabsf(v) < INFINITY; }

template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma<__half>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                            uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                   uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

}  // namespace paged
}  // namespace iex
