// Launchers of the page cache's kernels (page_cache.cu).
#pragma once

#include "ia_common.cuh"

namespace ia {

int64_t page_cache_scratch_bytes(int64_t n_rows, int64_t n_pages);
int launch_pages_extend(const ia_page_cache& c, const int32_t* rows, const int32_t* n_tokens, int n, cudaStream_t stream);
int launch_pages_fork(const ia_page_cache& c, const int32_t* parents, const int32_t* children, int n, int share,
                      cudaStream_t stream);
int launch_pages_free(const ia_page_cache& c, const int32_t* rows, int n, cudaStream_t stream);
int launch_pages_compact(const ia_page_cache& c, cudaStream_t stream);
struct PagesWrite {
  const void *k, *v;
  void *k_pool, *v_pool;
  int64_t k_tok_stride, k_head_stride, v_tok_stride, v_head_stride;  // elements
  int n_tokens;
};
int launch_pages_write(const ia_page_cache& c, const int32_t* rows, const int32_t* starts, int n, const PagesWrite& w,
                       cudaStream_t stream);

}  // namespace ia
