// vw_rope.cu -- norm, rotary positions and cache append of a decoder layer's queries, keys and values
// (include/vwsampler.h, vw_rope_append): DecoderStack.ForwardSegments (src/Voxwerk/Talker/DecoderStack.cs:144-228)
// between the projections and the attention, over a paged cache.
//
// Per row r and head: x' = x rsqrt(mean(x^2) + eps) w (queries and keys with a norm weight), then each pair (a, b) of
// the first 2 * half dims turns by the angle of the row's position: (a cos - b sin, b cos + a sin); pairs are
// (i, i + half) or, interleaved, (2 i, 2 i + 1).  All in fp32, rounded to bf16 once, when written.  Queries go to
// q_out, keys and values into the page that holds the row's key index.
//
// Bound: HBM (one read of q, k, v, one write of q_out and the cache rows); a handful of rows: latency.  So one pass: a
// lane holds the two chunks of CH elements that hold its pairs' both halves, a group of GS lanes holds one head, and
// the norm's sum is the only exchange between lanes.  The loads of a block's rows are issued before the row's sequence
// is looked up, so the lookup's latency (sequence, page, table row) overlaps theirs.

#include <cuda_runtime.h>

#include <algorithm>

#include "vw_attention.h"
#include "vw_internal.h"

namespace vw {
namespace {

constexpr int kMaxRowsPerBlock = 32;

struct RowPlace {
    int64_t slot;   // element offset of the row's (page, token) in the cache, or -1: the row is left alone
    int32_t pos;
};

__device__ RowPlace place_row(const RopeParams& p, int row, int lane) {
    RowPlace r{-1, 0};
    const KvBatchDev& b = p.batch;
    int seq = row, end = row + 1, begin = row;
    if (b.q_offsets) {
        seq = find_sequence(b.q_offsets, b.n_seqs, row, lane);
        if (seq < 0) return r;
        begin = b.q_offsets[seq];
        end = b.q_offsets[seq + 1];
    }
    if (row < begin || row >= end) return r;   // a padding row
    const int len = b.kv_lens[seq];
    const int index = len - (end - row);
    if (index < 0 || (index >> p.cache.page_shift) >= b.max_pages) {
        if (lane == 0) atomicOr(p.err, kErrKvLens);
        return r;
    }
    const int page = b.page_table[seq * b.page_table_stride + (index >> p.cache.page_shift)];
    const int pos = p.positions ? p.positions[row] : index;
    if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.cache.n_pages)) {
        if (lane == 0) atomicOr(p.err, kErrPageRange);
        return r;
    }
    if (static_cast<unsigned>(pos) >= static_cast<unsigned>(p.n_positions)) {
        if (lane == 0) atomicOr(p.err, kErrPosition);
        return r;
    }
    r.slot = page * p.cache.page_stride + (index & (p.cache.page_size - 1)) * p.cache.token_stride;
    r.pos = pos;
    return r;
}

template <int CH>
__device__ __forceinline__ void load_chunk(const __nv_bfloat16* s, float* x) {
    if constexpr (CH == 8) {
        const uint4 u = __ldcs(reinterpret_cast<const uint4*>(s));
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    } else if constexpr (CH == 4) {
        const uint2 u = __ldcs(reinterpret_cast<const uint2*>(s));
        const uint32_t w[2] = {u.x, u.y};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    } else {
        x[0] = __bfloat162float(*s);
    }
}
template <int CH>
__device__ __forceinline__ void load_chunk(const float* s, float* x) {
    if constexpr (CH == 1) {
        x[0] = *s;
    } else {
#pragma unroll
        for (int i = 0; i < CH; i += 4) {
            const float4 f = __ldcs(reinterpret_cast<const float4*>(s + i));
            x[i] = f.x;
            x[i + 1] = f.y;
            x[i + 2] = f.z;
            x[i + 3] = f.w;
        }
    }
}
// fp32 table or weight values; they are shared by many rows, so they stay cached
template <int N>
__device__ __forceinline__ void load_f32(const float* s, float* x) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 f = __ldg(reinterpret_cast<const float4*>(s + i));
            x[i] = f.x;
            x[i + 1] = f.y;
            x[i + 2] = f.z;
            x[i + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = __ldg(s + i);
    }
}
template <int CH>
__device__ __forceinline__ void store_chunk(__nv_bfloat16* d, const float* x) {
    if constexpr (CH == 1) {
        *d = __float2bfloat16_rn(x[0]);
    } else {
        uint32_t w[CH / 2];
#pragma unroll
        for (int i = 0; i < CH / 2; ++i) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&b);
        }
        if constexpr (CH == 8)
            *reinterpret_cast<uint4*>(d) = make_uint4(w[0], w[1], w[2], w[3]);
        else
            *reinterpret_cast<uint2*>(d) = make_uint2(w[0], w[1]);
    }
}

// The two chunks of pair slot j, and whether they turn.  Half layout: (j CH, half + j CH) while j CH < half, then the
// dims that pass, two chunks at a time; interleaved: two neighbouring chunks.
template <int CH, bool kInterleaved>
__device__ __forceinline__ void slot_dims(int j, int half, int& a, int& b, bool& turns) {
    if (kInterleaved) {
        a = 2 * CH * j;
        b = a + CH;
        turns = a < 2 * half;
    } else {
        const int n = half / CH;
        turns = j < n;
        a = turns ? j * CH : 2 * half + (j - n) * 2 * CH;
        b = turns ? half + a : a + CH;
    }
}

// x[0..CH) and x[CH..2 CH): the slot's chunks
template <int CH, bool kInterleaved>
__device__ __forceinline__ void turn(const RopeParams& p, int pos, int a, float* x) {
    const float* c = p.cos_table + static_cast<int64_t>(pos) * p.half;
    const float* s = p.sin_table + static_cast<int64_t>(pos) * p.half;
    float cs[CH], sn[CH];
    if constexpr (kInterleaved && CH > 1) {   // chunk elements (2 e, 2 e + 1) are pair a / 2 + e of the head
        load_f32<CH>(c + a / 2, cs);
        load_f32<CH>(s + a / 2, sn);
#pragma unroll
        for (int e = 0; e < CH; ++e) {
            const float u = x[2 * e], v = x[2 * e + 1];
            x[2 * e] = u * cs[e] - v * sn[e];
            x[2 * e + 1] = v * cs[e] + u * sn[e];
        }
    } else {
        const int i = kInterleaved ? a / 2 : a;
        load_f32<CH>(c + i, cs);
        load_f32<CH>(s + i, sn);
#pragma unroll
        for (int e = 0; e < CH; ++e) {
            const float u = x[e], v = x[CH + e];
            x[e] = u * cs[e] - v * sn[e];
            x[CH + e] = v * cs[e] + u * sn[e];
        }
    }
}

// NP pair slots per lane (1 unless a head has more slots than a warp has lanes)
template <typename T, int CH, bool kInterleaved, int NP>
__global__ void __launch_bounds__(512) rope_append_kernel(const RopeParams p, int rows_per_block, int group_shift) {
    __shared__ RowPlace places[kMaxRowsPerBlock];
    const int heads = p.n_q_heads + 2 * p.cache.n_kv_heads;
    const int D = p.cache.head_dim, slots = D / (2 * CH);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row0 = blockIdx.x * rows_per_block;
    const int rows = min(rows_per_block, p.batch.n_rows - row0);
    const int groups = blockDim.x >> group_shift, gs = 1 << group_shift;
    const int j0 = threadIdx.x & (gs - 1);
    const int tasks = rows * heads;

    // head `t` of the block's rows: its source and kind (0 query, 1 key, 2 value)
    auto source = [&](int t, int& row, int& head, int& kind) -> const T* {
        row = row0 + t / heads;
        head = t % heads;
        kind = head < p.n_q_heads ? 0 : head < p.n_q_heads + p.cache.n_kv_heads ? 1 : 2;
        head -= kind == 0 ? 0 : kind == 1 ? p.n_q_heads : p.n_q_heads + p.cache.n_kv_heads;
        return kind == 0   ? static_cast<const T*>(p.q) + row * p.q_row + head * p.q_head
               : kind == 1 ? static_cast<const T*>(p.k) + row * p.k_row + head * p.k_head
                           : static_cast<const T*>(p.v) + row * p.v_row + head * p.v_head;
    };
    auto load_task = [&](int t, float (&x)[NP][2 * CH]) {
        if (t >= tasks) return;
        int row, head, kind;
        const T* s = source(t, row, head, kind);
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            const int j = j0 + n * gs;
            if (j >= slots) break;
            int a, b;
            bool turns;
            slot_dims<CH, kInterleaved>(j, p.half, a, b, turns);
            load_chunk<CH>(s + a, x[n]);
            load_chunk<CH>(s + b, x[n] + CH);
        }
    };

    float x[NP][2 * CH] = {};
    load_task(threadIdx.x >> group_shift, x);
    for (int r = warp; r < rows; r += blockDim.x >> 5) {
        const RowPlace pl = place_row(p, row0 + r, lane);
        if (lane == 0) places[r] = pl;
    }
    __syncthreads();

    for (int t0 = 0; t0 < tasks; t0 += groups) {
        const int t = t0 + (threadIdx.x >> group_shift);
        if (t0 > 0) load_task(t, x);
        const bool live = t < tasks;
        int row = 0, head = 0, kind = 0;
        RowPlace pl{-1, 0};
        if (live) {
            source(t, row, head, kind);
            pl = places[row - row0];
        }
        const float* weight = kind == 0 ? p.q_norm : kind == 1 ? p.k_norm : nullptr;
        float sum = 0.0f;
        if (live && weight) {
#pragma unroll
            for (int n = 0; n < NP; ++n)
                if (j0 + n * gs < slots)
#pragma unroll
                    for (int e = 0; e < 2 * CH; ++e) sum = __fmaf_rn(x[n][e], x[n][e], sum);
        }
        for (int o = gs >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (!live || pl.slot < 0) continue;
        const float rs = __frsqrt_rn(sum / static_cast<float>(D) + p.eps);
        __nv_bfloat16* dst = kind == 0   ? p.q_out + row * p.q_out_row + head * p.q_out_head
                             : kind == 1 ? p.cache.k + pl.slot + head * p.cache.head_stride
                                         : p.cache.v + pl.slot + head * p.cache.head_stride;
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            const int j = j0 + n * gs;
            if (j >= slots) break;
            int a, b;
            bool turns;
            slot_dims<CH, kInterleaved>(j, p.half, a, b, turns);
            if (weight) {
                float w[2 * CH];
                load_f32<CH>(weight + a, w);
                load_f32<CH>(weight + b, w + CH);
#pragma unroll
                for (int e = 0; e < 2 * CH; ++e) x[n][e] = x[n][e] * rs * w[e];
            }
            if (kind != 2 && turns) turn<CH, kInterleaved>(p, pl.pos, a, x[n]);
            store_chunk<CH>(dst + a, x[n]);
            store_chunk<CH>(dst + b, x[n] + CH);
        }
    }
}

bool multiple(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Whether every chunk of `ch` elements starts on a boundary its load or store needs, and no chunk straddles the end of
// the part that turns.
bool chunks_fit(const RopeParams& p, int ch) {
    const int64_t in = ch * (p.f32 ? 4 : 2) < 16 ? ch * (p.f32 ? 4 : 2) : 16, out = ch * 2;
    const int64_t es = p.f32 ? 4 : 2;
    const int64_t in_strides[6] = {p.q_row, p.q_head, p.k_row, p.k_head, p.v_row, p.v_head};
    for (int64_t s : in_strides)
        if (s * es % in) return false;
    const int64_t out_strides[5] = {p.q_out_row, p.q_out_head, p.cache.page_stride, p.cache.token_stride,
                                    p.cache.head_stride};
    for (int64_t s : out_strides)
        if (s * 2 % out) return false;
    return multiple(p.q, in) && multiple(p.k, in) && multiple(p.v, in) && multiple(p.q_out, out) &&
           multiple(p.cache.k, out) && multiple(p.cache.v, out) && multiple(p.cos_table, 16) &&
           multiple(p.sin_table, 16) && multiple(p.q_norm, 16) && multiple(p.k_norm, 16) &&
           p.cache.head_dim % (2 * ch) == 0 && p.half % 4 == 0 &&
           (p.interleaved ? 2 * p.half % (2 * ch) == 0 : p.half % ch == 0);
}

template <typename T, int CH, int NP>
cudaError_t launch_ch(const RopeParams& p, cudaStream_t stream) {
    const int heads = p.n_q_heads + 2 * p.cache.n_kv_heads;
    const int slots = p.cache.head_dim / (2 * CH);
    int shift = 0;
    while ((1 << shift) < slots && shift < 5) ++shift;
    const int per_row = heads << shift;
    const int threads = std::clamp((per_row + 31) / 32 * 32, 128, 512);
    const int rows = std::clamp(threads / per_row, 1, kMaxRowsPerBlock);
    const int grid = (p.batch.n_rows + rows - 1) / rows;
    if (p.interleaved)
        rope_append_kernel<T, CH, true, NP><<<grid, threads, 0, stream>>>(p, rows, shift);
    else
        rope_append_kernel<T, CH, false, NP><<<grid, threads, 0, stream>>>(p, rows, shift);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_type(const RopeParams& p, cudaStream_t stream) {
    if (chunks_fit(p, 8)) return launch_ch<T, 8, 1>(p, stream);
    if (chunks_fit(p, 4)) return launch_ch<T, 4, 1>(p, stream);
    return launch_ch<T, 1, 4>(p, stream);   // any alignment, any even head_dim <= 256
}

}  // namespace

cudaError_t launch_rope_append(const RopeParams& p, cudaStream_t stream) {
    return p.f32 ? launch_type<float>(p, stream) : launch_type<__nv_bfloat16>(p, stream);
}

}  // namespace vw
