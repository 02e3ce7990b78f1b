// vw_rope.cu -- norm, rotary positions and cache append of a decoder layer's queries, keys and values
// (include/vwsampler.h, vw_rope_append): DecoderStack.ForwardSegments (src/Voxwerk/Talker/DecoderStack.cs:144-228)
// between the projections and the attention, over a paged cache.
//
// Per row r and head: x' = x rsqrt(mean(x^2) + eps) w (queries and keys with a norm weight), then each pair (a, b) of
// the first 2 * half dims turns by the angle of the row's position: (a cos - b sin, b cos + a sin); pairs are
// (i, i + half) or, interleaved, (2 i, 2 i + 1).  All in fp32, rounded to bf16 once, when written.  Queries go to
// q_out, keys and values into the page that holds the row's key index.
//
// Bound: HBM (one read of q, k, v, one write of q_out and the cache rows); a handful of rows: latency.  So one pass, a
// warp to a row (several where rows are few): a lane holds the two chunks of CH elements that hold its pairs' both
// halves, a group of GS lanes holds one head, and the norm's sum is the only exchange between lanes.  A lane meets the
// same dims in every head of a row, so its part of the cos / sin row is read once, and the weights once for queries and
// once for keys.  The first heads' loads are issued before the row's place is looked up (a chain of four dependent
// loads: sequence, its length, its page, table row), four at a time after that.

#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "vw_attention.h"
#include "vw_internal.h"

namespace vw {
namespace {

constexpr int kThreads = 128;
constexpr int kWarpsPerSm = 16;   // all resident at once (a second wave of such long-lived warps would double the time);
                                  // 14 595 rows: 52.3 us with 12, 51.7 with 16, 63 with 20 (fewer registers)

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
        if (begin < 0 || end > b.n_rows) return r;   // (offsets_fit reports it)
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

// Reports row offsets that are negative, descend or pass the rows, of every thread's share of the sequences.
__device__ __forceinline__ void offsets_fit(const RopeParams& p) {
    const KvBatchDev& b = p.batch;
    if (!b.q_offsets) return;
    const int threads = gridDim.x * kThreads;
    for (int s = blockIdx.x * kThreads + threadIdx.x; s < b.n_seqs; s += threads) {
        const int begin = b.q_offsets[s], end = b.q_offsets[s + 1];
        if (begin < 0 || end < begin || end > b.n_rows) atomicOr(p.err, kErrKvLens);
    }
}

// CH elements as they were loaded
template <typename T, int CH>
struct Chunk {
    static constexpr int kBytes = CH * static_cast<int>(sizeof(T));
    uint32_t w[kBytes < 4 ? 1 : kBytes / 4];

    __device__ __forceinline__ void load(const T* s) {
        if constexpr (kBytes >= 16) {
#pragma unroll
            for (int i = 0; i < kBytes / 16; ++i) {
                const uint4 u = __ldcs(reinterpret_cast<const uint4*>(s) + i);
                w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
            }
        } else if constexpr (kBytes == 8) {
            const uint2 u = __ldcs(reinterpret_cast<const uint2*>(s));
            w[0] = u.x, w[1] = u.y;
        } else if constexpr (kBytes == 4) {
            w[0] = *reinterpret_cast<const uint32_t*>(s);
        } else {
            w[0] = *reinterpret_cast<const uint16_t*>(s);
        }
    }
    __device__ __forceinline__ void widen(float* x) const {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < CH; ++i) x[i] = __uint_as_float(w[i]);
        } else if constexpr (CH == 1) {
            x[0] = __uint_as_float(w[0] << 16);
        } else {
#pragma unroll
            for (int i = 0; i < CH / 2; ++i) {
                x[2 * i] = __uint_as_float(w[i] << 16);
                x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        }
    }
};
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

// two fp32 products, or products and sums, per instruction
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
template <int N>
__device__ __forceinline__ void scale(float* x, const float* w) {   // x[i] *= w[i]
    if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 y = mul2(make_float2(x[i], x[i + 1]), make_float2(w[i], w[i + 1]));
            x[i] = y.x, x[i + 1] = y.y;
        }
    } else {
        x[0] *= w[0];
    }
}

// The row of the tables a slot turns by, and x[0..CH) and x[CH..2 CH), the slot's chunks, turned
template <int CH, bool kInterleaved>
struct Turn {
    float cs[CH], sn[CH];

    __device__ __forceinline__ void load(const RopeParams& p, int pos, int a) {
        // interleaved chunks: elements (2 e, 2 e + 1) of a slot are pair a / 2 + e of the head
        const int64_t at = static_cast<int64_t>(pos) * p.half + (kInterleaved ? a / 2 : a);
        load_f32<CH>(p.cos_table + at, cs);
        load_f32<CH>(p.sin_table + at, sn);
    }
    __device__ __forceinline__ void apply(float* x) const {
        if constexpr (!kInterleaved && CH > 1) {   // two pairs at a time
#pragma unroll
            for (int e = 0; e < CH; e += 2) {
                const float2 u = make_float2(x[e], x[e + 1]), v = make_float2(x[CH + e], x[CH + e + 1]);
                const float2 c = make_float2(cs[e], cs[e + 1]), s = make_float2(sn[e], sn[e + 1]);
                const float2 a = fma2(make_float2(-v.x, -v.y), s, mul2(u, c)), b = fma2(u, s, mul2(v, c));
                x[e] = a.x, x[e + 1] = a.y, x[CH + e] = b.x, x[CH + e + 1] = b.y;
            }
        } else {
#pragma unroll
            for (int e = 0; e < CH; ++e) {
                float& first = CH > 1 ? x[2 * e] : x[e];
                float& second = CH > 1 ? x[2 * e + 1] : x[CH + e];
                const float u = first, v = second;
                first = __fmaf_rn(-v, sn[e], u * cs[e]);
                second = __fmaf_rn(u, sn[e], v * cs[e]);
            }
        }
    }
};

// Asks the L2 for a kind's heads of a row (14 595 rows of 32 heads of 128: 51.7 us, 53.9 without)
template <typename T>
__device__ __forceinline__ void prefetch_heads(const T* src, int64_t stride, int heads, int dim, int lane) {
    constexpr int kLine = 128 / sizeof(T);
    for (int h = lane; h < heads; h += 32)
        for (int d = 0; d < dim; d += kLine)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(src + h * stride + d));
}

// NP pair slots per lane (1 unless a head has more slots than a warp has lanes); teams of 2^team_shift warps to a row,
// 2^group_shift lanes to a head
// U heads of a lane on their way at once.  kFew (rows): the first head of every kind is loaded up front, in registers of
// its own, since the row's latency counts; else the kinds follow each other in the same registers, so that more warps fit
// (14 595 rows of 16 + 2 * 8 heads of 128: 66 us with all of a row's loads up front, 52 us so, 239 MB at 4.6 TB/s).
template <typename T, int CH, bool kInterleaved, int NP, int U, bool kFew>
__global__ void __launch_bounds__(kThreads, kFew ? 1 : kWarpsPerSm * 32 / kThreads)
rope_append_kernel(const __grid_constant__ RopeParams p, int team_shift, int group_shift) {
    const int lane = threadIdx.x & 31;
    const int warp = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    const int teams = (gridDim.x * (kThreads / 32)) >> team_shift, member = warp & ((1 << team_shift) - 1);
    const int D = p.cache.head_dim, slots = D / (2 * CH), gs = 1 << group_shift;
    const int sub = lane >> group_shift, j0 = lane & (gs - 1);
    const int step = 32 >> group_shift;   // heads of a warp at a time
    int da[NP], db[NP];                   // the lane's chunks of every head
    bool has[NP], turns[NP];
#pragma unroll
    for (int n = 0; n < NP; ++n) {
        slot_dims<CH, kInterleaved>(j0 + n * gs, p.half, da[n], db[n], turns[n]);
        has[n] = j0 + n * gs < slots;
        turns[n] = turns[n] && has[n];
    }
    const int first = member * step + sub, next = step << team_shift;

    for (int row = warp >> team_shift; row < p.batch.n_rows; row += teams) {
        Turn<CH, kInterleaved> turn[NP];
        Chunk<T, CH> raw_q[U][NP][2], own_k[1][NP][2], own_v[1][NP][2];
        const auto load_batch = [&](auto& raw, const T* src, int64_t stride, int h0, int heads) {
            constexpr int kCount = sizeof(raw) / sizeof(raw[0]);
#pragma unroll
            for (int u = 0; u < kCount; ++u)
                if (h0 + u * next < heads) {
                    const T* s = src + (h0 + u * next) * stride;
#pragma unroll
                    for (int n = 0; n < NP; ++n)
                        if (has[n]) {
                            raw[u][n][0].load(s + da[n]);
                            raw[u][n][1].load(s + db[n]);
                        }
                }
        };
        // the heads of one kind (values are copied only)
        const auto heads_of = [&](auto value, auto& raw, const T* src, int64_t stride, int heads, const float* w,
                                  __nv_bfloat16* dst, int64_t dst_stride, bool loaded) {
            constexpr bool kValue = decltype(value)::value;
            constexpr int kCount = sizeof(raw) / sizeof(raw[0]);
            float weight[NP][2 * CH];
            if (!kValue && w) {
#pragma unroll
                for (int n = 0; n < NP; ++n)
                    if (has[n]) {
                        load_f32<CH>(w + da[n], weight[n]);
                        load_f32<CH>(w + db[n], weight[n] + CH);
                    }
            }
            // (a warp's lanes leave together: the norm's sum takes all of them)
            for (int base = member * step; base < heads; base += kCount * next, loaded = false) {
                if (!loaded) load_batch(raw, src, stride, base + sub, heads);
#pragma unroll
                for (int u = 0; u < kCount; ++u) {
                    if (base + u * next >= heads) break;
                    const int h = base + u * next + sub;
                    const bool live = h < heads;
                    float x[NP][2 * CH];
#pragma unroll
                    for (int n = 0; n < NP; ++n) {
                        raw[u][n][0].widen(x[n]);
                        raw[u][n][1].widen(x[n] + CH);
                    }
                    if (!kValue && w) {
                        float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
                        for (int n = 0; n < NP; ++n)
                            if (live && has[n])
#pragma unroll
                                for (int e = 0; e < 2 * CH; e += 2) {
                                    const float2 y = make_float2(x[n][e], x[n][e + 1]);
                                    sum = fma2(y, y, sum);
                                }
                        float all = sum.x + sum.y;
                        for (int o = gs >> 1; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
                        const float rs = rsqrtf(__fmaf_rn(all, p.inv_dim, p.eps));
#pragma unroll
                        for (int n = 0; n < NP; ++n) {
                            scale<2 * CH>(x[n], weight[n]);
                            float r[2 * CH];
#pragma unroll
                            for (int e = 0; e < 2 * CH; ++e) r[e] = rs;
                            scale<2 * CH>(x[n], r);
                        }
                    }
                    if (!live) continue;
                    __nv_bfloat16* to = dst + h * dst_stride;
#pragma unroll
                    for (int n = 0; n < NP; ++n) {
                        if (!has[n]) continue;
                        if (!kValue && turns[n]) turn[n].apply(x[n]);
                        store_chunk<CH>(to + da[n], x[n]);
                        store_chunk<CH>(to + db[n], x[n] + CH);
                    }
                }
            }
        };
        const T* q = static_cast<const T*>(p.q) + row * p.q_row;
        const T* k = static_cast<const T*>(p.k) + row * p.k_row;
        const T* v = static_cast<const T*>(p.v) + row * p.v_row;
        const int n_kv = p.cache.n_kv_heads;
        load_batch(raw_q, q, p.q_head, first, p.n_q_heads);
        if (!kFew && row + teams < p.batch.n_rows) {   // the warp's next row
            prefetch_heads(q + teams * p.q_row, p.q_head, p.n_q_heads, D, lane);
            prefetch_heads(k + teams * p.k_row, p.k_head, n_kv, D, lane);
            prefetch_heads(v + teams * p.v_row, p.v_head, n_kv, D, lane);
        }
        if (kFew) {
            load_batch(own_k, k, p.k_head, first, n_kv);
            load_batch(own_v, v, p.v_head, first, n_kv);
        }
        const RowPlace at = place_row(p, row, lane);
        if (at.slot < 0) continue;   // the warp's one row
#pragma unroll
        for (int n = 0; n < NP; ++n)
            if (turns[n]) turn[n].load(p, at.pos, da[n]);
        heads_of(std::false_type{}, raw_q, q, p.q_head, p.n_q_heads, p.q_norm, p.q_out + row * p.q_out_row, p.q_out_head,
                 true);
        __nv_bfloat16 *k_to = p.cache.k + at.slot, *v_to = p.cache.v + at.slot;
        if constexpr (kFew) {
            heads_of(std::false_type{}, own_k, k, p.k_head, n_kv, p.k_norm, k_to, p.cache.head_stride, true);
            heads_of(std::true_type{}, own_v, v, p.v_head, n_kv, nullptr, v_to, p.cache.head_stride, true);
        } else {
            heads_of(std::false_type{}, raw_q, k, p.k_head, n_kv, p.k_norm, k_to, p.cache.head_stride, false);
            heads_of(std::true_type{}, raw_q, v, p.v_head, n_kv, nullptr, v_to, p.cache.head_stride, false);
        }
    }
    offsets_fit(p);   // last: what it reads was read for the rows before, so that it costs them nothing
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
cudaError_t launch_ch(const RopeParams& p, int sms, cudaStream_t stream) {
    const int slots = p.cache.head_dim / (2 * CH);
    int group_shift = 0;
    while ((1 << group_shift) < slots && group_shift < 5) ++group_shift;
    const int passes = (p.n_q_heads + (32 >> group_shift) - 1) / (32 >> group_shift);
    // warps to a row: more while some would have nothing to do otherwise
    const int64_t room = static_cast<int64_t>(sms) * kWarpsPerSm;
    int team_shift = 0;
    while (team_shift < 3 && (2 << team_shift) <= passes && (static_cast<int64_t>(p.batch.n_rows) << (team_shift + 1)) <= room)
        ++team_shift;
    const int64_t warps = std::min(static_cast<int64_t>(p.batch.n_rows) << team_shift, room);
    const int grid = static_cast<int>((warps + kThreads / 32 - 1) / (kThreads / 32));
    constexpr int kMany = NP > 1 ? 1 : 4;
    const bool few = team_shift > 0 || NP > 1;
    if (p.interleaved && few)
        rope_append_kernel<T, CH, true, NP, 1, true><<<grid, kThreads, 0, stream>>>(p, team_shift, group_shift);
    else if (p.interleaved)
        rope_append_kernel<T, CH, true, NP, kMany, false><<<grid, kThreads, 0, stream>>>(p, team_shift, group_shift);
    else if (few)
        rope_append_kernel<T, CH, false, NP, 1, true><<<grid, kThreads, 0, stream>>>(p, team_shift, group_shift);
    else
        rope_append_kernel<T, CH, false, NP, kMany, false><<<grid, kThreads, 0, stream>>>(p, team_shift, group_shift);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_type(const RopeParams& p, int sms, cudaStream_t stream) {
    if (chunks_fit(p, 8)) return launch_ch<T, 8, 1>(p, sms, stream);
    if (chunks_fit(p, 4)) return launch_ch<T, 4, 1>(p, sms, stream);
    return launch_ch<T, 1, 4>(p, sms, stream);   // any alignment, any even head_dim <= 256
}

}  // namespace

cudaError_t launch_rope_append(const RopeParams& p, int sms, cudaStream_t stream) {
    return p.f32 ? launch_type<float>(p, sms, stream) : launch_type<__nv_bfloat16>(p, sms, stream);
}

}  // namespace vw
