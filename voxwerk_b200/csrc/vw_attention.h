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

// ---- the tile kernel (vw_prompt.cu): how a call runs, and its part of the handle's workspace
constexpr int kPartRows = 256;  // rows of a block, and what one more CTA adds to the partial rows
struct TilePlan {
    int32_t split;              // pieces of blocks, joined afterwards
    int32_t grid;
    int32_t dim;                // head_dim padded to 64 or 128
    int64_t part_rows;          // partial rows
    int64_t unit_ends;
};
struct TileWork {
    int32_t* counters;          // [2] tickets taken, CTAs done; both 0 between calls
    int64_t* units_per_cta;
    int64_t* unit_end;          // [sequences or groups] units up to and including each
    float* part_lse;            // [part_rows] log2 of each partial row's sum, -inf: no key
    float* part_o;              // [part_rows, dim] its softmax-weighted values
};
TilePlan plan_prompt(const AttnParams& p, int sms);
cudaError_t launch_prompt_attention(const AttnParams& p, const TilePlan& plan, const TileWork& w, cudaStream_t stream);
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

// The sequence whose rows hold `row`: the last s with offsets[s] <= row (-1: none), found 32 probes at a time by a warp.
__device__ __forceinline__ int find_sequence(const int32_t* offsets, int n_seqs, int row, int lane) {
    int lo = 0, n = n_seqs;   // the answer is in [lo, lo + n)
    while (n > 1) {
        const int step = (n + 31) / 32;
        const int at = lo + lane * step;
        const bool le = lane * step < n && offsets[at] <= row;
        const unsigned m = __ballot_sync(0xffffffffu, le);
        if (!m) return -1;
        const int last = 31 - __clz(m);
        n = min(step, n - last * step);
        lo += last * step;
    }
    return lo;
}

// A row's partial results weighed together by one warp, DIM / 32 dims a lane: o = sum_i 2^(lse_i - m) o_i / l,
// l = sum_i 2^(lse_i - m).
template <int DIM>
struct PartSum {
    static constexpr int kDims = DIM / 32;
    float m = -INFINITY, l = 0.0f, o[kDims] = {};

    // pieces c0 .. c1 of the row whose piece c is at partial row base + c * kPartRows
    __device__ void add(const TileWork& w, int64_t base, int c0, int c1, int lane) {
        for (int c = c0; c <= c1; c += 32) {
            const int n = min(32, c1 - c + 1);
            const float lse = lane < n ? w.part_lse[base + static_cast<int64_t>(c + lane) * kPartRows] : -INFINITY;
            float top = lse;
#pragma unroll
            for (int i = 16; i > 0; i >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
            raise(top);
            const float mine = m == -INFINITY ? 0.0f : exp2f(lse - m);
#pragma unroll 4
            for (int i = 0; i < n; ++i) {
                const float f = __shfl_sync(0xffffffffu, mine, i);
                const float* src = w.part_o + (base + static_cast<int64_t>(c + i) * kPartRows) * DIM + lane * kDims;
                float x[kDims];
                if constexpr (kDims == 4) {
                    const float4 v = *reinterpret_cast<const float4*>(src);
                    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
                } else {
                    const float2 v = *reinterpret_cast<const float2*>(src);
                    x[0] = v.x, x[1] = v.y;
                }
                l += f;
#pragma unroll
                for (int d = 0; d < kDims; ++d) o[d] = __fmaf_rn(f, x[d], o[d]);
            }
        }
    }
    __device__ void raise(float top) {
        if (top > m) {
            const float f = m == -INFINITY ? 0.0f : exp2f(m - top);
            l *= f;
#pragma unroll
            for (int d = 0; d < kDims; ++d) o[d] *= f;
            m = top;
        }
    }
    __device__ void write(const AttnParams& p, int64_t row, int head, int lane) {
        const float r = l == 0.0f ? 0.0f : 1.0f / l;
        __nv_bfloat16* out = p.rows.out + row * p.rows.out_row + head * p.rows.out_head + lane * kDims;
        if (lane * kDims < p.cache.head_dim)
#pragma unroll
            for (int d = 0; d < kDims; d += 2)
                *reinterpret_cast<__nv_bfloat162*>(out + d) = __floats2bfloat162_rn(o[d] * r, o[d + 1] * r);
        if (p.rows.lse && lane == 0)
            p.rows.lse[row * p.rows.n_q_heads + head] = (m + log2f(l)) * 0.693147180559945309f;
    }
};
#endif

}  // namespace vw
