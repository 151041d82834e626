// Internal interface of the attention kernels over pages.
#pragma once

#include "fmha.cuh"
#include "paged.cuh"

namespace dli_sm100 {

// Tensor maps over the K and V pages of the model's type with boxes of box_rows rows x
// 128 bytes of one (page, head).
dli_status make_page_maps(const PagedAttnArgs& a, dli_dtype dtype, int d, int box_rows, CUtensorMap* tk, CUtensorMap* tv);

// Few query rows per KV head, and every float32 call (k_paged_decode.cu): head_dim 64
// or 128, 16-byte aligned tensors.
bool paged_decode_serves(const PagedAttnArgs& a, dli_dtype dtype);
size_t paged_decode_workspace(int64_t batch, int64_t hkv, int64_t group, int64_t max_new, int64_t head_dim,
                              int64_t max_keys, dli_dtype dtype);
dli_status run_paged_decode(const PagedAttnArgs& a, dli_dtype dtype, dli_dtype kv_dtype, void* workspace,
                            size_t workspace_bytes, cudaStream_t stream);

// Many query rows (k_paged_prefill.cu): bf16/f16, head_dim 64 or 128, at most 128 query heads per KV head, 16-byte aligned tensors.
bool paged_prefill_serves(const PagedAttnArgs& a, dli_dtype dtype, dli_dtype kv_dtype);
size_t paged_prefill_workspace(int64_t batch, int64_t hkv, int64_t group, int64_t max_new, int64_t head_dim,
                               int64_t max_keys);
dli_status run_paged_prefill(const PagedAttnArgs& a, dli_dtype dtype, dli_dtype kv_dtype, void* workspace,
                             size_t workspace_bytes, cudaStream_t stream);

}  // namespace dli_sm100
