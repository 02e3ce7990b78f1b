// vw_attention.h -- launch parameters of the attention operators over a paged key/value cache (vw_rope.cu,
// vw_prompt.cu, vw_decode.cu), shared with their C-ABI host code (vw_attention.cpp).  Not part of the public ABI.
#pragma once

#include <cstddef>
#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_runtime.h>

namespace vw {

struct KvCacheDev {             // vw_kv_cache
    __nv_bfloat16* k;
    __nv_bfloat16* v;
    int64_t page_stride, token_stride, head_stride;   // elements
    int32_t n_pages, page_size, page_shift, n_kv_heads, head_dim;
};

struct KvBatchDev {             // vw_kv_batch (and the page tables of vw_kv_prefix)
    const int32_t* page_table;
    int64_t page_table_stride;
    int32_t max_pages, n_seqs;
    const int32_t* kv_lens;
    const int32_t* q_offsets;   // nullable: one row per sequence
    int32_t n_rows;
};

struct KvPrefixDev {            // vw_kv_prefix; n_groups == 0: none
    const int32_t* page_table;
    int64_t page_table_stride;
    int32_t max_pages, n_groups;
    const int32_t* lens;
    const int32_t* group_offsets;
};

struct AttnRowsDev {            // vw_attn_rows
    const __nv_bfloat16* q;
    int64_t q_row, q_head;
    __nv_bfloat16* out;
    int64_t out_row, out_head;
    float* lse;                 // nullable, [n_rows, n_q_heads]
    int32_t n_q_heads;
    float scale;
};

struct RopeParams {
    const void* q;
    const void* k;
    const void* v;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head;   // elements
    __nv_bfloat16* q_out;
    int64_t q_out_row, q_out_head;
    const float* q_norm;        // nullable [head_dim]
    const float* k_norm;
    const float* cos_table;     // [n_positions, half]
    const float* sin_table;
    const int32_t* positions;   // nullable: a row's position is its key index
    float eps;
    int32_t n_positions, half, interleaved, f32, n_q_heads;
    KvCacheDev cache;
    KvBatchDev batch;
    unsigned* err;
};
cudaError_t launch_rope_append(const RopeParams& p, cudaStream_t stream);

struct AttnParams {
    AttnRowsDev rows;
    KvCacheDev cache;
    KvBatchDev batch;
    KvPrefixDev prefix;         // decode only
    unsigned* err;
};
cudaError_t launch_prompt_attention(const AttnParams& p, cudaStream_t stream);
cudaError_t launch_decode_attention(const AttnParams& p, cudaStream_t stream);

#ifdef __CUDACC__
// A sequence's key count, held inside its page table; a count outside it is reported and clamped.
__device__ __forceinline__ int checked_len(int len, int max_pages, int page_shift, unsigned* err, unsigned bit) {
    const int cap = static_cast<int>(min(static_cast<int64_t>(max_pages) << page_shift, static_cast<int64_t>(INT32_MAX)));
    if (len < 0 || len > cap) {
        atomicOr(err, bit);
        return len < 0 ? 0 : cap;
    }
    return len;
}
#endif

}  // namespace vw
