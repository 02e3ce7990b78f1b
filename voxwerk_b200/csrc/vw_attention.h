// vw_attention.h -- launch parameters of the attention operators over a paged key/value cache (vw_rope.cu,
// vw_prompt.cu, vw_decode.cu), shared with their C-ABI host code (vw_attention.cpp).  Not part of the public ABI.
#pragma once

#include <cstddef>
#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "vw_internal.h"

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
    float eps, inv_dim;         // 1 / head_dim
    int32_t n_positions, half, interleaved, f32, n_q_heads;
    KvCacheDev cache;
    KvBatchDev batch;
    unsigned* err;
};
cudaError_t launch_rope_append(const RopeParams& p, int sms, cudaStream_t stream);

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
    int32_t* counters;          // [3] tickets taken, CTAs done, CTAs of the decode kernel with units; 0 between calls
    int64_t* units_per_cta;
    int64_t* unit_end;          // [sequences or groups] units up to and including each
    float* part_lse;            // [part_rows] log2 of each partial row's sum, -inf: no key
    float* part_o;              // [part_rows, dim] its softmax-weighted values
};
constexpr int kTileKeys = 128, kTileRows = 128;
struct Geometry {
    int32_t group;              // query heads per key head
    int32_t tile_tokens;        // tokens of a row tile; a block has two
};
inline Geometry geometry(const AttnParams& a) {
    const int group = a.rows.n_q_heads / a.cache.n_kv_heads;
    return {group, kTileRows / group};
}
// scale as the kernels use it, for powers of two; 0 becomes a factor that leaves every probability the same
inline float exp2_scale(float scale) {
    const float c = (scale < 0.0f ? -scale : scale) * 1.44269504088896341f;
    return c > 1e-30f ? c : 1e-30f;
}
TilePlan plan_prompt(const AttnParams& p, int sms);
TilePlan plan_prefix(const AttnParams& p, int sms);
cudaError_t launch_prefix_attention(const AttnParams& p, const TilePlan& plan, const TileWork& w, cudaStream_t stream);
cudaError_t launch_prompt_attention(const AttnParams& p, const TilePlan& plan, const TileWork& w, cudaStream_t stream);

// ---- the decode kernel (vw_decode.cu)
struct DecodePlan {
    int32_t grid, sms;
    int32_t rows;               // query heads an item takes: min(group, 16)
    int32_t row_blocks;         // items per key head
    int32_t dim;
    int64_t items;              // sequences x key heads x row_blocks
    int64_t part_rows;
};
struct DecodeWork {
    int32_t* tickets;           // [items] pieces done, 0 between calls
    int64_t* units_per_cta;
    int64_t* unit_end;          // [sequences] units up to and including each
    int32_t* chunk;             // tiles of a unit
    float* part_lse;
    float* part_o;
    TileWork prefix;            // the prefixes' partial results
};
DecodePlan plan_decode(const AttnParams& p, int sms);
cudaError_t launch_decode_attention(const AttnParams& p, const DecodePlan& plan, const DecodeWork& w, cudaStream_t stream);

// Threads of a join block: one for every four dims of the query heads of a key head, at most 256 at a time
inline int join_threads(int group, int dim) {
    const int n = (group * dim / 4 + 31) / 32 * 32;
    return n < 256 ? n : 256;
}

#ifdef __CUDACC__
// A sequence's key count, held inside its page table; a count outside it is reported and clamped.
__device__ __forceinline__ int checked_len(int len, int max_pages, int page_shift, unsigned* err, unsigned bit) {
    const int cap = static_cast<int>(min(static_cast<int64_t>(max_pages) << page_shift, int64_t{1} << 30));
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
        const bool le = lane * step < n && __ldg(offsets + at) <= row;
        const unsigned m = __ballot_sync(0xffffffffu, le);
        if (!m) return -1;
        const int last = 31 - __clz(m);
        n = min(step, n - last * step);
        lo += last * step;
    }
    return lo;
}

// ---- the tile kernel's units: key tiles of blocks, in the order sequence, block, key head
struct Seq {
    int32_t row0, n, kv, past;   // first row, tokens, keys, keys before the first token's own
};

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

template <bool kPrefix>
__device__ __forceinline__ Seq load_seq(const AttnParams& a, int s) {
    Seq q{0, 0, 0, 0};
    const int shift = a.cache.page_shift;
    const int32_t* o = kPrefix ? a.prefix.group_offsets : a.batch.q_offsets;
    const int limit = kPrefix ? a.batch.n_seqs : a.batch.n_rows;
    int begin = min(s, limit), end = min(s + 1, limit);   // (fewer rows than sequences: the later ones have none)
    if (o) {
        begin = __ldg(o + s);
        end = __ldg(o + s + 1);
    }
    q.kv = kPrefix ? checked_len(__ldg(a.prefix.lens + s), a.prefix.max_pages, shift, a.err, kErrKvLens)
                   : checked_len(__ldg(a.batch.kv_lens + s), a.batch.max_pages, shift, a.err, kErrKvLens);
    if (begin < 0 || end < begin || end > limit) {
        atomicOr(a.err, kErrKvLens);
        return q;
    }
    q.row0 = begin;
    q.n = end - begin;
    q.past = q.kv - q.n;
    return q;
}

// Keys that tokens [.., t) of a sequence see together
template <bool kPrefix>
__device__ __forceinline__ int keys_seen(const Seq& q, int t) {
    return kPrefix ? q.kv : min(max(q.past + min(q.n, t), 0), q.kv);
}
// Units of a sequence's block i (split): its key tiles, at least one for a prompt's block (its rows are written)
template <bool kPrefix>
__device__ __forceinline__ int block_units(const Seq& q, int i, int block_tokens) {
    return max(ceil_div(keys_seen<kPrefix>(q, (i + 1) * block_tokens), kTileKeys), kPrefix ? 0 : 1);
}
template <bool kPrefix>
__device__ __forceinline__ int64_t seq_units(const Seq& q, int block_tokens, int kv_heads) {
    const int blocks = ceil_div(q.n, block_tokens);
    int64_t u = 0;
    if (kPrefix)
        u = static_cast<int64_t>(blocks) * block_units<kPrefix>(q, 0, block_tokens);
    else
        for (int i = 0; i < blocks; ++i) u += block_units<kPrefix>(q, i, block_tokens);
    return u * kv_heads;
}

// a / b, by 32-bit division where both fit (the 64-bit one takes some hundred instructions)
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {
    if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
    return a / b;
}
template <typename T>
__device__ __forceinline__ T warp_scan(T x, int lane) {   // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    return x;
}

// The lengths that a CTA's schedule begins with, asked for while it still sets up
__device__ __forceinline__ void prefetch_lengths(const AttnParams& a, int lane) {
    for (int s = 32 * lane; s < a.batch.n_seqs; s += 32 * 32)   // (a line holds 32)
        asm volatile("prefetch.global.L1 [%0];" ::"l"(a.batch.kv_lens + s));
    if (lane == 0 && a.prefix.n_groups > 0) {
        asm volatile("prefetch.global.L1 [%0];" ::"l"(a.prefix.lens));
        asm volatile("prefetch.global.L1 [%0];" ::"l"(a.prefix.group_offsets));
    }
}
// 64-key tiles of the sequences' own keys, one at least of each, for one key head.  (Together they fit 32 bits: 2^31 of
// them would be 2^37 keys.)
__device__ __forceinline__ int own_tiles(const AttnParams& a, int lane) {
    int tiles = 0;
    for (int s0 = lane; s0 < a.batch.n_seqs; s0 += 4 * 32) {
        int len[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) len[i] = s0 + 32 * i < a.batch.n_seqs ? __ldg(a.batch.kv_lens + s0 + 32 * i) : -1;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (s0 + 32 * i < a.batch.n_seqs)
                tiles += max(ceil_div(checked_len(len[i], a.batch.max_pages, a.cache.page_shift, a.err, kErrKvLens), 64), 1);
    }
    return __reduce_add_sync(0xffffffffu, tiles);
}

// SMs for the prefixes' tile kernel; the decode kernel, launched behind it, takes the others at once (all when this is
// all, after the prefixes).  It is bound by HBM and reaches that rate with some 80 of 148 SMs, the prefixes by the SMs, so
// the two overlap well.  Of 32 counts the one whose later end comes first, by what was measured of each: 10 us and then
// 1.7 us a unit for a prefix CTA (16 us and 2.3 us where the mean group fills two row tiles: 50 sequences in four groups
// 23.6 us, 27.4 us with the latter); 7 us, then 64-key tiles at 6.5 TB/s or 0.45 us each on an SM, an item's end counted
// as two, for the sequences' own keys.  Every CTA of both kernels comes to the same count.  With 0.42 and 0.5 us in place of
// 0.45 (16 query heads on 8 of 128 dims): 256 sequences on a prefix of 16001 153 and 155 us against 142, 64 on one of 4099
// 33.8 and 34.5 against 34.5.  The times are those of three batches (these two, and the 50 sequences of 32 heads on 4 of 64);
// for others the count is as good as the model: a unit's cost does not follow head_dim, and groups of very different sizes
// count as their mean.
__device__ __forceinline__ int prefix_ctas(const AttnParams& a, int64_t units, int tiles, int sms, int lane) {
    const int group = a.rows.n_q_heads / a.cache.n_kv_heads;
    const float items = static_cast<float>(a.cache.n_kv_heads * ((group + 15) / 16));   // of a sequence
    const float own_tiles = static_cast<float>(tiles) * items;
    const float own_units = own_tiles + 2.0f * items * static_cast<float>(a.batch.n_seqs);
    const int mine = (sms * (lane + 1)) >> 5;
    const bool two = static_cast<int64_t>(a.batch.n_seqs) * group > int64_t{kTileRows} * a.prefix.n_groups;
    const float prefix_us = (two ? 16.0f : 10.0f) + static_cast<float>(units) * (two ? 2.3f : 1.7f) / static_cast<float>(mine);
    const float hbm_us = own_tiles * (256.0f * a.cache.head_dim) / 6.5e6f;
    const int rest = mine < sms ? sms - mine : sms;
    const float own_us = 7.0f + fmaxf(hbm_us, own_units * 0.45f / static_cast<float>(rest));
    const float us = mine == 0 ? 1e30f : mine < sms ? fmaxf(prefix_us, own_us) : prefix_us + own_us;
    const unsigned best = __reduce_min_sync(0xffffffffu, __float_as_uint(us));   // (positive floats order as integers)
    const unsigned m = __ballot_sync(0xffffffffu, __float_as_uint(us) == best);
    return (sms * (32 - __clz(m))) >> 5;
}

// Where the pieces of one row's block are: piece c (of CTA c) at partial row base + c * kPartRows, c0 <= c <= c1; c0 > c1
// where the row has none.
struct PieceSpan {
    int64_t base;
    int32_t c0, c1;
};
template <bool kPrefix>
__device__ PieceSpan piece_span(const AttnParams& a, const TileWork& w, int s, int row, int head, int tile_tokens) {
    PieceSpan at{0, 1, 0};
    const Seq q = load_seq<kPrefix>(a, s);
    if (row < q.row0 || row >= q.row0 + q.n) return at;
    const int kv_heads = a.cache.n_kv_heads, heads = a.rows.n_q_heads, group = heads / kv_heads;
    const int block_tokens = 2 * tile_tokens, i = (row - q.row0) / block_tokens, kv_head = head / group;
    const int cost = block_units<kPrefix>(q, i, block_tokens);
    if (cost == 0) return at;
    int64_t first = s > 0 ? w.unit_end[s - 1] : 0;
    if (kPrefix)
        first += static_cast<int64_t>(i) * kv_heads * cost;
    else
        for (int j = 0; j < i; ++j) first += static_cast<int64_t>(kv_heads) * block_units<kPrefix>(q, j, block_tokens);
    first += static_cast<int64_t>(kv_head) * cost;
    const int64_t per = *w.units_per_cta;
    at.c0 = static_cast<int>(divide(first, per));
    at.c1 = static_cast<int>(divide(first + cost - 1, per));
    const int tokens = min(block_tokens, q.n - i * block_tokens);
    at.base = static_cast<int64_t>(q.row0) * heads + static_cast<int64_t>(i) * kv_heads * block_tokens * group +
              static_cast<int64_t>(kv_head) * tokens * group + (row - q.row0 - i * block_tokens) * group + head % group;
    return at;
}

// Four dims of a row's partial results weighed together by one thread: o = sum_i 2^(lse_i - m) o_i / l,
// l = sum_i 2^(lse_i - m).  The pieces' loads do not wait for one another.
template <int DIM>
struct PartSum {
    float m = -INFINITY, l = 0.0f;
    float4 o = {0.0f, 0.0f, 0.0f, 0.0f};

    // pieces c0 .. c1, piece c at partial row base + c * stride, of it dims d .. d + 3
    __device__ void add(const float* part_lse, const float* part_o, int64_t base, int stride, int c0, int c1, int d) {
        float top = m;
#pragma unroll 4
        for (int c = c0; c <= c1; ++c) top = fmaxf(top, part_lse[base + static_cast<int64_t>(c) * stride]);
        const float f = m == -INFINITY ? 0.0f : exp2f(m - top);
        m = top;
        l *= f;
        o.x *= f, o.y *= f, o.z *= f, o.w *= f;
#pragma unroll 4
        for (int c = c0; c <= c1; ++c) {
            const int64_t row = base + static_cast<int64_t>(c) * stride;
            const float lse = part_lse[row];
            const float4 v = *reinterpret_cast<const float4*>(part_o + row * DIM + d);
            const float w = lse == -INFINITY ? 0.0f : exp2f(lse - top);   // (not a number stays one)
            l += w;
            o.x = __fmaf_rn(w, v.x, o.x);
            o.y = __fmaf_rn(w, v.y, o.y);
            o.z = __fmaf_rn(w, v.z, o.z);
            o.w = __fmaf_rn(w, v.w, o.w);
        }
    }
    __device__ void write(const AttnParams& p, int64_t row, int head, int d) {
        const float r = l == 0.0f ? 0.0f : 1.0f / l;
        if (d < p.cache.head_dim) {
            __nv_bfloat162 v[2] = {__floats2bfloat162_rn(o.x * r, o.y * r), __floats2bfloat162_rn(o.z * r, o.w * r)};
            *reinterpret_cast<uint2*>(p.rows.out + row * p.rows.out_row + head * p.rows.out_head + d) =
                *reinterpret_cast<const uint2*>(v);
        }
        if (p.rows.lse && d == 0)
            p.rows.lse[row * p.rows.n_q_heads + head] = (m + log2f(l)) * 0.693147180559945309f;
    }
};
#endif

}  // namespace vw
