// Internal C++ interface of the paged key/value cache (the C ABI in efa_b200.h forwards to it).
#pragma once

#include <cuda_runtime.h>
#include "../../include/efa_b200.h"

namespace efa {

const char* paged_check(const efa_paged_cache& c, const efa_paged_batch& b);
const char* paged_attention_check(const efa_paged_cache& c, const efa_paged_batch& b, const efa_paged_attention_params& p);
size_t paged_attention_bytes(const efa_paged_cache& c, const efa_paged_batch& b, const efa_paged_attention_params& p);

int cache_write(const void* K, const void* V, long long head_stride, long long token_stride, const efa_paged_cache& c, const efa_paged_batch& b, cudaStream_t stream);
int cache_read(void* K, void* V, long long head_stride, long long token_stride, const efa_paged_cache& c, const efa_paged_batch& b, cudaStream_t stream);
int paged_attention(const void* Q, void* O, const efa_paged_cache& c, const efa_paged_batch& b, const efa_paged_attention_params& p,
                    void* workspace, size_t workspace_bytes, cudaStream_t stream);

}  // namespace efa
