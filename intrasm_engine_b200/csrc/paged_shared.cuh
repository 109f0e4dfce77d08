// Attention over listed pages that many rows have in common (paged_shared.cu), as paged_attention.cu calls it.
#pragma once
#include "paged.cuh"

namespace iex {
namespace paged {

struct SharedCall {
  int rows, heads, kv_heads, dim, num_pages, page_shift, table_width, count;
  Rows q;
  const void *k_cache, *v_cache;
  long long k_page, v_page;
  const int32_t *table, *lengths, *pages;
  float scale_log2;
  void* out;
};

// Scratch of a call; 0 where rows one by one are expected to be as fast.
size_t shared_workspace_bytes(int rows, int heads, int kv_heads, int head_dim, int num_pages, int page_size, int table_width,
                              int count);
int shared_attention(const SharedCall& call, bool bf16, void* workspace, cudaStream_t stream);

}  // namespace paged
}  // namespace iex
