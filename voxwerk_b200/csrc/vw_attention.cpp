// vw_attention.cpp -- C ABI of the attention operators over a paged key/value cache (include/vwsampler.h): argument
// checks, workspace and stream ordering.  No C++ exception crosses the boundary.

#include <cmath>
#include <cstdint>
#include <string>

#include <cuda_runtime.h>

#include "../../include/vwsampler.h"
#include "vw_attention.h"
#include "vw_handle.h"
#include "vw_internal.h"

namespace {

constexpr int kMaxQueryHeadsPerKey = 64;

vw_status check_cache(vw_handle* h, const vw_kv_cache* c, int max_dim, int dim_unit) {
    if (!c || !c->k || !c->v) return fail(h, VW_ERR_INVALID_ARG, "cache: k and v are required");
    if (c->n_pages < 1 || c->n_kv_heads < 1) return fail(h, VW_ERR_INVALID_ARG, "cache: n_pages and n_kv_heads >= 1");
    if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)))
        return fail(h, VW_ERR_INVALID_ARG, "cache: page_size must be a power of two from 16 to 256");
    if (c->head_dim < dim_unit || c->head_dim > max_dim || c->head_dim % dim_unit)
        return fail(h, VW_ERR_INVALID_ARG, "cache: head_dim must be a multiple of " + std::to_string(dim_unit) +
                                               ", at most " + std::to_string(max_dim));
    const int64_t strides[3] = {c->page_stride, c->token_stride, c->head_stride};
    for (int64_t s : strides)
        if (s < 8 || s % 8 || s >= (int64_t{1} << 38))
            return fail(h, VW_ERR_INVALID_ARG, "cache: strides must be positive multiples of 8 elements");
    if (!aligned(c->k, 16) || !aligned(c->v, 16))
        return fail(h, VW_ERR_INVALID_ARG, "cache: k and v must be 16-byte aligned");
    return VW_OK;
}

vw_status check_batch(vw_handle* h, const vw_kv_batch* b) {
    if (!b) return fail(h, VW_ERR_INVALID_ARG, "a batch is required");
    if (b->n_seqs < 0 || b->n_rows < 0) return fail(h, VW_ERR_INVALID_ARG, "batch: n_seqs and n_rows >= 0");
    if (b->n_seqs == 0 || b->n_rows == 0) return VW_OK;
    if (!b->page_table || !b->kv_lens || b->max_pages < 1 || b->page_table_stride < b->max_pages)
        return fail(h, VW_ERR_INVALID_ARG, "batch: page_table, kv_lens and 1 <= max_pages <= page_table_stride");
    return VW_OK;
}

vw::KvCacheDev cache_dev(const vw_kv_cache& c) {
    int shift = 0;
    while ((1 << shift) < c.page_size) ++shift;
    return {static_cast<__nv_bfloat16*>(c.k), static_cast<__nv_bfloat16*>(c.v), c.page_stride, c.token_stride,
            c.head_stride, c.n_pages, c.page_size, shift, c.n_kv_heads, c.head_dim};
}
vw::KvBatchDev batch_dev(const vw_kv_batch& b) {
    return {b.page_table, b.page_table_stride, b.max_pages, b.n_seqs, b.kv_lens, b.q_offsets, b.n_rows};
}

vw_status check_rows(vw_handle* h, const vw_attn_rows* r, const vw_kv_cache& c) {
    if (!r || !r->q || !r->out) return fail(h, VW_ERR_INVALID_ARG, "rows: q and out are required");
    if (r->n_q_heads < 1 || r->n_q_heads % c.n_kv_heads || r->n_q_heads / c.n_kv_heads > kMaxQueryHeadsPerKey)
        return fail(h, VW_ERR_INVALID_ARG, "rows: n_q_heads must be a multiple of n_kv_heads, at most 64 times it");
    const int64_t strides[4] = {r->q_row_stride, r->q_head_stride, r->out_row_stride, r->out_head_stride};
    for (int64_t s : strides)
        if (s < 8 || s % 8 || s >= (int64_t{1} << 38))
            return fail(h, VW_ERR_INVALID_ARG, "rows: strides must be positive multiples of 8 elements");
    if (!aligned(r->q, 16) || !aligned(r->out, 16))
        return fail(h, VW_ERR_INVALID_ARG, "rows: q and out must be 16-byte aligned");
    if (!std::isfinite(r->scale)) return fail(h, VW_ERR_INVALID_ARG, "rows: scale must be finite");
    return VW_OK;
}
vw::AttnRowsDev rows_dev(const vw_attn_rows& r) {
    return {static_cast<const __nv_bfloat16*>(r.q), r.q_row_stride, r.q_head_stride,
            static_cast<__nv_bfloat16*>(r.out), r.out_row_stride, r.out_head_stride, r.lse, r.n_q_heads, r.scale};
}

// The attention workspace is one buffer of the handle: a call waits for the one before it, whose stream may be another
// though its handle is the same (a new stream can have a destroyed one's; one handle names every thread's default
// stream).  Inside a stream capture no order is added (an event of uncaptured work cannot be waited for there): the caller
// orders its graphs.
cudaError_t enter_workspace(vw_handle* h, cudaStream_t st, bool* capturing) {
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    cudaError_t e = cudaStreamIsCapturing(st, &cap);
    *capturing = cap != cudaStreamCaptureStatusNone;
    if (e == cudaSuccess && !*capturing) e = cudaStreamWaitEvent(st, h->attn_done, 0);   // (no call yet: nothing to wait for)
    return e;
}
// `e` is how the call's launches went: what they enqueued is recorded in either case.
cudaError_t leave_workspace(vw_handle* h, cudaStream_t st, bool capturing, cudaError_t e) {
    const cudaError_t r = capturing ? cudaSuccess : cudaEventRecord(h->attn_done, st);
    return e != cudaSuccess ? e : r;
}

// Grows one of the two attention buffers (clear: the one whose contents are zero between calls).  Not inside a capture:
// neither the wait nor the allocation is allowed there.
vw_status reserve(vw_handle* h, DeviceBuffer* b, size_t need, bool clear, cudaStream_t st, bool capturing) {
    if (need <= b->bytes) {
        b->captured = b->captured || capturing;
        return VW_OK;
    }
    if (capturing)
        return fail(h, VW_ERR_INVALID_ARG, "attention workspace: run a call of this size once before one is captured");
    constexpr const char* kWhat = "attention workspace";
    cudaError_t e = cudaDeviceSynchronize();   // an earlier call, on any stream, may still use the old buffer
    if (e != cudaSuccess) return cuda_fail(h, e, kWhat);
    const vw_status r = let_go(h, b, clear ? &h->old_attn_counts : &h->old_buffers, kWhat);
    if (r != VW_OK) return r;
    const size_t bytes = round_up(need + need / 4, 1 << 16);
    e = cudaMalloc(reinterpret_cast<void**>(&b->p), bytes);
    if (e == cudaSuccess && clear) e = cudaMemsetAsync(b->p, 0, bytes, st);
    if (e == cudaSuccess && clear) e = cudaStreamSynchronize(st);   // whatever stream the next call is on
    if (e != cudaSuccess) return cuda_fail(h, e, kWhat);
    b->bytes = bytes;
    return VW_OK;
}

constexpr size_t kCountsHeader = 256;   // the tile kernel's counters, then the decode kernel's tickets

vw_status reserve_counts(vw_handle* h, int64_t tickets, cudaStream_t st, bool capturing) {
    return reserve(h, &h->attn_counts, kCountsHeader + static_cast<size_t>(tickets) * 4, true, st, capturing);
}
// The parts buffer, carved twice: without a base for its size, then for the pointers.
template <typename F>
vw_status reserve_parts(vw_handle* h, cudaStream_t st, bool capturing, F carve) {
    size_t size = 0;
    const auto take = [&size](char* base, int64_t bytes) {
        char* p = base ? base + size : nullptr;
        size += round_up(static_cast<size_t>(bytes), 256);
        return p;
    };
    carve([&](int64_t bytes) { return take(nullptr, bytes); });
    const vw_status r = reserve(h, &h->attn, size, false, st, capturing);
    if (r != VW_OK) return r;
    size = 0;
    carve([&](int64_t bytes) { return take(h->attn.p, bytes); });
    return VW_OK;
}
template <typename Take>
void carve_tiles(vw_handle* h, const vw::TilePlan& plan, Take take, vw::TileWork* w) {
    w->counters = reinterpret_cast<int32_t*>(h->attn_counts.p);
    w->units_per_cta = reinterpret_cast<int64_t*>(take(8));
    w->unit_end = reinterpret_cast<int64_t*>(take(plan.unit_ends * 8));
    w->part_lse = reinterpret_cast<float*>(take(plan.part_rows * 4));
    w->part_o = reinterpret_cast<float*>(take(plan.part_rows * plan.dim * 4));
}

}  // namespace

VW_EXPORT vw_status vw_rope_append(vw_handle* h, const vw_kv_cache* cache, const vw_kv_batch* batch,
                                   const vw_rope_rows* rows, void* stream) {
    if (!h) return VW_ERR_INVALID_ARG;
    h->last_error.clear();
    vw_status r = check_cache(h, cache, 256, 2);
    if (r == VW_OK) r = check_batch(h, batch);
    if (r != VW_OK || batch->n_seqs == 0 || batch->n_rows == 0) return r;
    if (!rows || !rows->q || !rows->k || !rows->v || !rows->q_out)
        return fail(h, VW_ERR_INVALID_ARG, "rows: q, k, v and q_out are required");
    if (rows->dtype != VW_F32 && rows->dtype != VW_BF16)
        return fail(h, VW_ERR_INVALID_ARG, "rows: dtype must be VW_F32 or VW_BF16");
    if (rows->n_q_heads < 1) return fail(h, VW_ERR_INVALID_ARG, "rows: n_q_heads >= 1");
    if (rows->rotary_dim < 0 || rows->rotary_dim % 2 || rows->rotary_dim > cache->head_dim)
        return fail(h, VW_ERR_INVALID_ARG, "rows: rotary_dim must be even, from 0 to head_dim");
    if (rows->rotary_dim > 0 && (!rows->cos_table || !rows->sin_table || rows->n_positions < 1))
        return fail(h, VW_ERR_INVALID_ARG, "rows: cos_table, sin_table and n_positions are required");
    if (!(rows->eps >= 0.0f)) return fail(h, VW_ERR_INVALID_ARG, "rows: eps must be >= 0");
    const int64_t strides[8] = {rows->q_row_stride, rows->q_head_stride, rows->k_row_stride, rows->k_head_stride,
                                rows->v_row_stride, rows->v_head_stride, rows->q_out_row_stride,
                                rows->q_out_head_stride};
    for (int64_t s : strides)
        if (s < 0) return fail(h, VW_ERR_INVALID_ARG, "rows: strides must not be negative");
    const size_t es = rows->dtype == VW_F32 ? 4 : 2;
    if (!aligned(rows->q, es) || !aligned(rows->k, es) || !aligned(rows->v, es) || !aligned(rows->q_out, 2))
        return fail(h, VW_ERR_INVALID_ARG, "rows: pointers must be aligned to their elements");
    if (!batch->q_offsets && batch->n_rows > batch->n_seqs)
        return fail(h, VW_ERR_INVALID_ARG, "batch: n_rows exceeds n_seqs without q_offsets");
    DeviceGuard guard(h->device);
    if (!guard.ok()) return fail(h, VW_ERR_CUDA, "cudaSetDevice failed");
    cudaStream_t st = stream ? static_cast<cudaStream_t>(stream) : h->stream;
    vw::RopeParams p{};
    p.q = rows->q;
    p.k = rows->k;
    p.v = rows->v;
    p.q_row = rows->q_row_stride;
    p.q_head = rows->q_head_stride;
    p.k_row = rows->k_row_stride;
    p.k_head = rows->k_head_stride;
    p.v_row = rows->v_row_stride;
    p.v_head = rows->v_head_stride;
    p.q_out = static_cast<__nv_bfloat16*>(rows->q_out);
    p.q_out_row = rows->q_out_row_stride;
    p.q_out_head = rows->q_out_head_stride;
    p.q_norm = rows->q_norm;
    p.k_norm = rows->k_norm;
    p.cos_table = rows->cos_table;
    p.sin_table = rows->sin_table;
    p.positions = rows->positions;
    p.eps = rows->eps;
    p.inv_dim = 1.0f / static_cast<float>(cache->head_dim);
    p.half = rows->rotary_dim / 2;
    p.n_positions = p.half ? rows->n_positions : INT32_MAX;   // no table: any position
    p.interleaved = rows->interleaved != 0;
    p.f32 = rows->dtype == VW_F32;
    p.n_q_heads = rows->n_q_heads;
    p.cache = cache_dev(*cache);
    p.batch = batch_dev(*batch);
    p.err = h->d_err;
    const cudaError_t e = vw::launch_rope_append(p, h->sm_count, st);
    if (e != cudaSuccess) return cuda_fail(h, e, "rope append");
    if (!stream) return read_device_error(h, st);
    return VW_OK;
}

VW_EXPORT vw_status vw_prompt_attention(vw_handle* h, const vw_kv_cache* cache, const vw_kv_batch* batch,
                                        const vw_attn_rows* rows, void* stream) {
    if (!h) return VW_ERR_INVALID_ARG;
    h->last_error.clear();
    vw_status r = check_cache(h, cache, 128, 8);
    if (r == VW_OK) r = check_batch(h, batch);
    if (r != VW_OK || batch->n_seqs == 0 || batch->n_rows == 0) return r;
    r = check_rows(h, rows, *cache);
    if (r != VW_OK) return r;
    if (!batch->q_offsets && batch->n_rows > batch->n_seqs)
        return fail(h, VW_ERR_INVALID_ARG, "batch: n_rows exceeds n_seqs without q_offsets");
    DeviceGuard guard(h->device);
    if (!guard.ok()) return fail(h, VW_ERR_CUDA, "cudaSetDevice failed");
    cudaStream_t st = stream ? static_cast<cudaStream_t>(stream) : h->stream;
    vw::AttnParams p{rows_dev(*rows), cache_dev(*cache), batch_dev(*batch), vw::KvPrefixDev{}, h->d_err};
    bool capturing = false;
    cudaError_t e = enter_workspace(h, st, &capturing);
    if (e != cudaSuccess) return cuda_fail(h, e, "prompt attention");
    const vw::TilePlan plan = vw::plan_prompt(p, h->sm_count);
    vw::TileWork w{};
    r = reserve_counts(h, 0, st, capturing);
    if (r == VW_OK) r = reserve_parts(h, st, capturing, [&](auto take) { carve_tiles(h, plan, take, &w); });
    if (r != VW_OK) return r;
    e = vw::launch_prompt_attention(p, plan, w, st);
    e = leave_workspace(h, st, capturing, e);
    if (e != cudaSuccess) return cuda_fail(h, e, "prompt attention");
    if (!stream) return read_device_error(h, st);
    return VW_OK;
}

VW_EXPORT vw_status vw_decode_attention(vw_handle* h, const vw_kv_cache* cache, const vw_kv_batch* batch,
                                        const vw_kv_prefix* prefix, const vw_attn_rows* rows, void* stream) {
    if (!h) return VW_ERR_INVALID_ARG;
    h->last_error.clear();
    vw_status r = check_cache(h, cache, 128, 8);
    if (r == VW_OK) r = check_batch(h, batch);
    if (r != VW_OK || batch->n_seqs == 0 || batch->n_rows == 0) return r;
    r = check_rows(h, rows, *cache);
    if (r != VW_OK) return r;
    if (batch->n_rows < batch->n_seqs) return fail(h, VW_ERR_INVALID_ARG, "batch: n_rows must cover every sequence");
    if (prefix) {
        if (prefix->n_groups < 0) return fail(h, VW_ERR_INVALID_ARG, "prefix: n_groups >= 0");
        if (prefix->n_groups > 0 && (!prefix->page_table || !prefix->lens || !prefix->group_offsets ||
                                     prefix->max_pages < 1 || prefix->page_table_stride < prefix->max_pages))
            return fail(h, VW_ERR_INVALID_ARG,
                        "prefix: page_table, lens, group_offsets and 1 <= max_pages <= page_table_stride");
    }
    DeviceGuard guard(h->device);
    if (!guard.ok()) return fail(h, VW_ERR_CUDA, "cudaSetDevice failed");
    cudaStream_t st = stream ? static_cast<cudaStream_t>(stream) : h->stream;
    vw::AttnParams p{rows_dev(*rows), cache_dev(*cache), batch_dev(*batch), vw::KvPrefixDev{}, h->d_err};
    p.batch.q_offsets = nullptr;
    if (prefix && prefix->n_groups > 0)
        p.prefix = {prefix->page_table, prefix->page_table_stride, prefix->max_pages, prefix->n_groups, prefix->lens,
                    prefix->group_offsets};
    bool capturing = false;
    cudaError_t e = enter_workspace(h, st, &capturing);
    if (e != cudaSuccess) return cuda_fail(h, e, "decode attention");
    const vw::DecodePlan plan = vw::plan_decode(p, h->sm_count);
    vw::TilePlan prefix_plan{};
    if (p.prefix.n_groups > 0) prefix_plan = vw::plan_prefix(p, h->sm_count);
    vw::DecodeWork w{};
    r = reserve_counts(h, plan.items, st, capturing);
    if (r == VW_OK)
        r = reserve_parts(h, st, capturing, [&](auto take) {
            w.tickets = reinterpret_cast<int32_t*>(h->attn_counts.p + kCountsHeader);
            w.units_per_cta = reinterpret_cast<int64_t*>(take(8));
            w.chunk = reinterpret_cast<int32_t*>(take(4));
            w.unit_end = reinterpret_cast<int64_t*>(take(static_cast<int64_t>(p.batch.n_seqs) * 8));
            w.part_lse = reinterpret_cast<float*>(take(plan.part_rows * 4));
            w.part_o = reinterpret_cast<float*>(take(plan.part_rows * plan.dim * 4));
            if (p.prefix.n_groups > 0) carve_tiles(h, prefix_plan, take, &w.prefix);
        });
    if (r != VW_OK) return r;
    if (p.prefix.n_groups > 0) e = vw::launch_prefix_attention(p, prefix_plan, w.prefix, st);
    if (e == cudaSuccess) e = vw::launch_decode_attention(p, plan, w, st);
    if (e != cudaSuccess) cudaMemsetAsync(h->attn_counts.p, 0, h->attn_counts.bytes, st);   // the join would have
    e = leave_workspace(h, st, capturing, e);
    if (e != cudaSuccess) return cuda_fail(h, e, "decode attention");
    if (!stream) return read_device_error(h, st);
    return VW_OK;
}
