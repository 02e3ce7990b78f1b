// vw_decode.cu -- single-token attention over a paged key/value cache (include/vwsampler.h, vw_decode_attention): softmax(scale q k^T) v of each row over the keys it sees.
//
// One warp per (row, query head), each lane four dims of the head, one pass over the keys with the running maximum m
// and sum l of the softmax in fp32: o and l are scaled by exp(m - m') when the maximum rises to m'.

#include <cuda_runtime.h>

#include <algorithm>

#include "vw_attention.h"
#include "vw_internal.h"

namespace vw {
namespace {

struct Softmax {
    float m = -INFINITY, l = 0.0f, o[4] = {};
};

__device__ void attend(const AttnParams& p, const int32_t* table, int keys, int kv_head, int d0, const float* q,
                       Softmax& s) {
    const KvCacheDev& c = p.cache;
    for (int j = 0; j < keys; ++j) {
        const int page = table[j >> c.page_shift];
        if (static_cast<unsigned>(page) >= static_cast<unsigned>(c.n_pages)) {
            atomicOr(p.err, kErrPageRange);
            continue;
        }
        const int64_t at = page * c.page_stride + (j & (c.page_size - 1)) * c.token_stride + kv_head * c.head_stride + d0;
        float x = 0.0f;
        if (d0 < c.head_dim)
            for (int i = 0; i < 4; ++i) x = __fmaf_rn(q[i], __bfloat162float(c.k[at + i]), x);
        for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        const float m = fmaxf(s.m, x);
        const float w = expf(x - m), f = expf(s.m - m);
        s.m = m;
        s.l = __fmaf_rn(s.l, f, w);
        if (d0 < c.head_dim)
            for (int i = 0; i < 4; ++i) s.o[i] = __fmaf_rn(s.o[i], f, w * __bfloat162float(c.v[at + i]));
    }
}

__global__ void __launch_bounds__(128) attention_kernel(const AttnParams p, int decode) {
    const int lane = threadIdx.x & 31, d0 = 4 * lane;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
    const int heads = p.rows.n_q_heads, D = p.cache.head_dim;
    const int64_t row = item / heads;
    if (item == 0 && lane == 0) {   // the offsets ascend within the rows
        const int32_t* o = decode ? p.prefix.group_offsets : p.batch.q_offsets;
        const int n = decode ? p.prefix.n_groups : p.batch.n_seqs, end = decode ? p.batch.n_seqs : p.batch.n_rows;
        for (int i = 0; o && i < n; ++i)
            if (o[i] < 0 || o[i + 1] < o[i] || o[i + 1] > end) atomicOr(p.err, kErrKvLens);
    }
    const int head = static_cast<int>(item % heads);
    if (row >= p.batch.n_rows) return;
    const KvBatchDev& b = p.batch;
    int seq = static_cast<int>(row), behind = 0;
    if (b.q_offsets) {
        for (seq = 0; seq < b.n_seqs && row >= b.q_offsets[seq + 1]; ++seq) {}
        if (seq < b.n_seqs) behind = max(0, b.q_offsets[seq + 1] - 1 - static_cast<int>(row));
    }
    if (seq >= b.n_seqs) return;
    const int keys = checked_len(b.kv_lens[seq], b.max_pages, p.cache.page_shift, p.err, kErrKvLens) - behind;
    const int kv_head = head / (heads / p.cache.n_kv_heads);
    float q[4] = {};
    if (d0 < D)
        for (int i = 0; i < 4; ++i)
            q[i] = __bfloat162float(p.rows.q[row * p.rows.q_row + head * p.rows.q_head + d0 + i]) * p.rows.scale;
    Softmax s;
    for (int g = 0; decode && g < p.prefix.n_groups; ++g)
        if (seq >= p.prefix.group_offsets[g] && seq < p.prefix.group_offsets[g + 1])
            attend(p, p.prefix.page_table + g * p.prefix.page_table_stride,
                   checked_len(p.prefix.lens[g], p.prefix.max_pages, p.cache.page_shift, p.err, kErrKvLens), kv_head, d0,
                   q, s);
    attend(p, b.page_table + seq * b.page_table_stride, keys, kv_head, d0, q, s);
    const float r = s.l > 0.0f ? 1.0f / s.l : 0.0f;
    if (d0 < D)
        for (int i = 0; i < 4; ++i)
            p.rows.out[row * p.rows.out_row + head * p.rows.out_head + d0 + i] = __float2bfloat16_rn(s.o[i] * r);
    if (p.rows.lse && lane == 0) p.rows.lse[row * heads + head] = s.m + logf(s.l);
}

cudaError_t launch(const AttnParams& p, int decode, cudaStream_t stream) {
    const int64_t items = static_cast<int64_t>(p.batch.n_rows) * p.rows.n_q_heads;
    attention_kernel<<<static_cast<unsigned>((items + 3) / 4), 128, 0, stream>>>(p, decode);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_decode_attention(const AttnParams& p, cudaStream_t stream) { return launch(p, 1, stream); }

}  // namespace vw
