// Internal C++ interface of what stands around the block and its paged cache: norms, projections with 4-bit weights, the cache's pages (the C ABI in
// efa_b200.h forwards to it).
#pragma once

#include <cuda_runtime.h>
#include "../../include/efa_b200.h"

namespace efa {

const char* block_norm_check(const efa_block_norm_params& p, int rows);
int block_norm(const void* x, const void* y, const void* gate, const void* post_w, const void* post_b, const void* pre_w, const void* pre_b, void* x_out, void* h,
               int rows, const efa_block_norm_params& p, cudaStream_t stream);

const char* w4_check(const efa_w4& w);
int project_w4(const void* X, long long x_stride, const efa_w4& w, void* out, int out_dtype, long long out_stride, int rows, cudaStream_t stream);

const char* page_pool_check(const efa_page_pool& p);
size_t pages_bytes(const efa_page_pool& p);
int pages_take(const efa_page_pool& p, const int* q_start, void* workspace, size_t workspace_bytes, cudaStream_t stream);
int pages_fork(const efa_page_pool& p, const efa_paged_cache& c, const int* parents, const int* children, int n, void* workspace, size_t workspace_bytes, cudaStream_t stream);
int pages_free(const efa_page_pool& p, const int* seqs, int n, cudaStream_t stream);
int pages_compact(const efa_page_pool& p, const efa_paged_cache& c, int* pages_out, int* refs_out, int* moved, void* workspace, size_t workspace_bytes, cudaStream_t stream);
int pages_copy(const efa_paged_cache& c, const int* src, const int* dst, int n, cudaStream_t stream);

}  // namespace efa
