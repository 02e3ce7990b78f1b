// vw_prompt.cu -- attention of many rows over a paged key/value cache on the tensor cores (include/vwsampler.h):
// vw_prompt_attention, and the shared prefixes of vw_decode_attention.
//
// out = softmax(scale Q K^T) V in one pass over the keys: a block of query rows keeps a reference m and the sum l of its
// probabilities in registers and its output O in tensor memory; a tile of 128 keys adds P V with P = exp2(c S - c m),
// c = scale log2(e).  m is the maximum of the first keys a row sees.  It need not follow the running maximum: any m gives
// the same O / l as long as nothing overflows, so m is raised, O and l brought to it and the tile done again only when
// the tile's probabilities sum to more than 2^16.  That saves a pass over the scores in nearly every tile.
//
// A block is two tiles of up to 128 rows of one key head: the rows of a tile are (token, query head) pairs, so grouped
// heads share every key and value read.  One CTA per SM, 12 warps:
//   warp 0     schedules the blocks and loads by TMA: Q once per block, K and V tiles (page boxes) into two rings;
//   warps 1, 3 issue the tcgen05.mma: S = Q K^T (operands in shared memory) and O += P V (P from tensor memory);
//   warp 2     clears the rows past a sequence's last key in its last V tile (pages end inside a tile, and what lies
//              there may be anything: 0 * NaN would reach every row);
//   warps 4-7, 8-11   one warpgroup per row tile, one thread per row: S from tensor memory into registers, exponentials,
//              P back to tensor memory as bf16, and at the end O / l to the output.
// Tensor memory (512 columns): one S (128 fp32 columns) that both row tiles use in turn, since the softmax warps read it
// as soon as it is there; P0 P1 (64 each); O0 O1 (128 each).  So S of the next tile is computed while the softmax of this
// one runs, and a row tile's time per key tile is its softmax alone.
//
// Schedule.  Blocks in order of decreasing key count from a ticket counter, so that the last ones are short.  Where
// there are too few blocks for the SMs, the (block, tile) units are dealt evenly instead, a block's pieces leave
// partial results (O / l and log2-sum in fp32), and a join kernel, or the decode kernel, weighs them together.
//
// Rounding.  P is rounded to bf16 for its product with V (scores, sums and O stay fp32): one tcgen05.mma takes two
// operands of one 16-bit type, and V is bf16.  Outputs are then 0.0017-0.0023 (relative) from the 64-bit values, where
// their own rounding to bf16 makes 0.0016-0.0017.  tf32 for both would halve the rate and double V's space; P in two
// bf16 terms would take 1.5 times the products and 128 columns of tensor memory more than there are.
//
// Measured (16 query heads on 8 of 128 dims; device time, CUDA graphs one after the other): one prompt of 7937 214-219 us
// = 1.18-1.21 PFLOP/s for the first 25 ms, then the power limit takes the clock from 1965 to 1620-1710 MHz and it takes
// 242-254 us = 1.02-1.07 PFLOP/s (bound: a row tile's exponentials and its two products take turns, half of the time
// each); 12 prompts of 170-1300 tokens 43.4 us = 0.42 PFLOP/s (bound: three short blocks an SM, each with 5-8 us before
// its first product and after its last); one of 37 10.3 us (latency of one block).  32 heads on 4 of 64: pieces of 130-250
// on 9001 cached keys 56-57 us = 0.42 PFLOP/s (bound: exponentials, twice as many a flop as with 128).
//
// Every mbarrier wait is bounded; on expiry an error bit is set, every role stops and drains, tensor memory is freed.

#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>

#include "vw_attention.h"
#include "vw_internal.h"
#include "vw_tc.cuh"

namespace vw {
namespace {

constexpr int kThreads384 = 384;
constexpr int kKeys = kTileKeys;  // keys per tile
constexpr int kRows = kTileRows;  // rows per row tile
constexpr int kWholeKeys = 512;   // sequences of at most this many keys are never split
constexpr int kMinPromptUnits = 2, kMinPrefixUnits = 1;   // fewest units a CTA takes
constexpr int kFeedRegs = 72, kSoftmaxRegs = 208;   // registers per thread of warps 0-3 and 4-11
// a tile whose probabilities sum to more is done again with its own maximum: far from what overflows in fp32 or bf16
constexpr float kMaxTileSum = 65536.0f;
constexpr uint32_t kColS = 0, kColP = 128, kColO = 256;   // tensor memory columns: S; P0 P1, 64 each; O0 O1, 128 each
constexpr float kLn2 = 0.693147180559945309f;
constexpr int kItemSlots = 3;
constexpr int kItemReaders = 11;  // warps 1 to 11

template <int DP>   // head_dim padded to 64 or 128 (the TMA fills the rest with zeros)
struct TileCfg {
    static constexpr int kHalves = DP / 64;
    static constexpr uint32_t kHalfBytes = 128 * 128;   // 128 rows of 64 bf16, 128-byte swizzle
    static constexpr uint32_t kTileBytes = kHalves * kHalfBytes;
    static constexpr int kStages = DP == 128 ? 2 : 4;   // of K, and of V
    static constexpr uint32_t kOffKv = 2 * kTileBytes;   // after the two Q tiles
    static constexpr uint32_t kOffBar = kOffKv + 2 * kStages * kTileBytes;
    // k_full[S] k_empty[S] v_full[S] v_empty[S] q_full q_empty s_full[2] s_free p_full[2] o_full[2] v_tail v_fixed
    // item_full[3] item_empty[3] done[2]
    static constexpr uint32_t kBars = 4 * kStages + 19;
    static constexpr uint32_t kOffItems = kOffBar + 8 * kBars;
    static constexpr uint32_t kOffMisc = kOffItems + kItemSlots * 64;
    static constexpr uint32_t kBytes = kOffMisc + 16;
    static_assert(kBytes + 1024 <= 232448, "shared memory");
};

struct Item {            // a block, or a piece of one
    int32_t valid;
    int32_t row0, tokens;        // first row of the call, tokens (rows per query head) of the block
    int32_t pos0, kv;            // index of the first token among the sequence's keys; keys of the sequence
    int32_t seq, kv_head;
    int32_t tile0, end[2];       // key tiles [tile0, end[q]) of row tile q
    int32_t part_row;            // first partial row, or -1: the result goes to the output
};
static_assert(sizeof(Item) <= 64, "item slots");

struct TileParams {
    AttnParams a;
    int32_t group;               // query heads per key head
    int32_t tile_tokens;         // tokens per row tile: floor(128 / group)
    int32_t split;               // units dealt evenly (pieces) instead of whole blocks by ticket
    int32_t min_units;           // fewest units a CTA takes (split)
    uint32_t kv_inverse;         // (2^32 - 1) / n_kv_heads
    float c;                     // |scale| log2(e), not 0
    int32_t negate;              // scale < 0
    int32_t wide_out;            // output rows start on 32-byte boundaries
    TileWork w;
};

// The whole warp fills an item from block i of sequence s, key tiles [t0, t1) of it.
template <bool kPrefix>
__device__ Item make_item(const TileParams& p, const Seq& q, int s, int i, int kv_head, int t0, int t1, bool whole,
                          int cta) {
    const int tt = p.tile_tokens, first = 2 * tt * i;
    Item it;
    it.valid = 1;
    it.row0 = q.row0 + first;
    it.tokens = min(2 * tt, q.n - first);
    it.pos0 = q.past + first;
    it.kv = q.kv;
    it.seq = s;
    it.kv_head = kv_head;
    it.tile0 = t0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int n = min(max(it.tokens - h * tt, 0), tt);
        const int end = n ? ceil_div(keys_seen<kPrefix>(q, first + h * tt + n), kKeys) : 0;
        it.end[h] = max(min(end, t1), t0);
    }
    const int rows = it.tokens * p.group;
    it.part_row = whole && !kPrefix ? -1
                                    : q.row0 * p.a.rows.n_q_heads + i * p.a.cache.n_kv_heads * 2 * tt * p.group +
                                          kv_head * rows + cta * kPartRows;
    return it;
}

// The schedule, walked by the 32 lanes of warp 0 together.
template <bool kPrefix>
struct Scheduler {
    const TileParams& p;
    int lane, n_seqs, block_tokens, kv_heads;
    // by ticket
    int ticket, level, base;
    int below;                           // of this lane's sequences so far: the highest level below `level` with a block
    int32_t before;
    Seq own;                             // sequence `lane`, its lowest level and blocks
    int own_level, own_blocks;
    bool taken = false;                  // the first ticket is the CTA's number
    // split
    int64_t unit, unit_end, seq_first;   // the CTA's units; the first unit of sequence `seq`
    int seq;

    __device__ Scheduler(const TileParams& params, int l) : p(params), lane(l) {
        n_seqs = kPrefix ? p.a.prefix.n_groups : p.a.batch.n_seqs;
        block_tokens = 2 * p.tile_tokens;
        kv_heads = p.a.cache.n_kv_heads;
        if (p.split) {
            const auto units_of = [&](int s) {
                return s < n_seqs ? seq_units<kPrefix>(load_seq<kPrefix>(p.a, s), block_tokens, kv_heads) : 0;
            };
            const int tiles = kPrefix ? own_tiles(p.a, lane) : 0;
            int64_t total = 0, u = 0, sum = 0;
            for (int s0 = 0; s0 < n_seqs; s0 += 32) {
                const int s = s0 + lane;
                u = units_of(s);
                sum = warp_scan(u, lane);
                if (blockIdx.x == 0 && s < n_seqs) p.w.unit_end[s] = total + sum;   // for the kernels that join
                total += __shfl_sync(0xffffffffu, sum, 31);
            }
            const int ctas = kPrefix ? prefix_ctas(p.a, total, tiles, gridDim.x, lane) : gridDim.x;
            const int64_t per = max(divide(total + ctas - 1, ctas), static_cast<int64_t>(p.min_units));
            if (blockIdx.x == 0 && lane == 0) *p.w.units_per_cta = per;
            unit = min(per * blockIdx.x, total);
            unit_end = min(unit + per, total);
            seq = 0;
            seq_first = 0;
            for (int s0 = 0; unit < unit_end && s0 < n_seqs; s0 += 32) {   // the sequence that holds `unit`
                if (n_seqs > 32) {   // (else the values above)
                    u = units_of(s0 + lane);
                    sum = warp_scan(u, lane);
                }
                const unsigned m = __ballot_sync(0xffffffffu, seq_first + sum > unit);
                if (m) {
                    const int at = __ffs(m) - 1;
                    seq = s0 + at;
                    seq_first += __shfl_sync(0xffffffffu, sum - u, at);
                    break;
                }
                seq_first += __shfl_sync(0xffffffffu, sum, 31);
            }
        } else {
            ticket = blockIdx.x;
            own = lane < n_seqs ? load_seq<kPrefix>(p.a, lane) : Seq{0, 0, 0, 0};
            own_level = first_level(own);
            own_blocks = ceil_div(own.n, block_tokens);
            int top = own_blocks > 0 ? own_level + own_blocks - 1 : -1;
            for (int s = lane + 32; s < n_seqs; s += 32) {
                const Seq q = load_seq<kPrefix>(p.a, s);
                if (q.n > 0) top = max(top, first_level(q) + ceil_div(q.n, block_tokens) - 1);
            }
            level = __reduce_max_sync(0xffffffffu, top);
            base = 0;
            below = -1;
            before = 0;
        }
    }
    // Blocks are taken level by level from the highest: a block's level is its key count in units of block tokens.  A walk
    // over a level's sequences finds the next one down that has a block, so that empty levels cost nothing (256 short
    // prompts, one behind 8000 keys, 8 query heads to a key head: 102 us, 684 level by level; 4096 of them, 64 heads: 271
    // us, 80.7 ms).
    __device__ int first_level(const Seq& q) const { return max(q.past, 0) / block_tokens; }

    __device__ Item next() {
        Item none;
        none.valid = 0;
        if (p.split) return unit < unit_end ? next_piece() : none;
        if (taken) {
            if (lane == 0) ticket = gridDim.x + atomicAdd(p.w.counters, 1);
            ticket = __shfl_sync(0xffffffffu, ticket, 0);
        }
        taken = true;
        // The (sequence, block) pair wanted and its key head: ticket / kv_heads and the rest.  The product with the inverse
        // is at most one too small; a division's 20 instructions, cold each time, take longer than the walk that follows (a
        // prompt of 7937: 220.6 us, 223).
        int wanted = static_cast<int>(__umulhi(ticket, p.kv_inverse)), kv_head = ticket - wanted * kv_heads;
        if (kv_head >= kv_heads) {
            ++wanted;
            kv_head -= kv_heads;
        }
        while (level >= 0) {
            Seq q = own;
            int i = level - own_level, blocks = own_blocks;
            if (base > 0) {
                q = base + lane < n_seqs ? load_seq<kPrefix>(p.a, base + lane) : Seq{0, 0, 0, 0};
                i = level - first_level(q);
                blocks = ceil_div(q.n, block_tokens);
            }
            if (i > 0 && blocks > 0) below = max(below, level - 1 - max(i - blocks, 0));
            if (i >= blocks) i = -1;
            const unsigned m = __ballot_sync(0xffffffffu, i >= 0);
            const int slot = wanted - before;
            if (slot < __popc(m)) {
                const int at =
                    __ffs(__ballot_sync(0xffffffffu, i >= 0 && __popc(m & ((1u << lane) - 1)) == slot)) - 1;
                q.row0 = __shfl_sync(0xffffffffu, q.row0, at);
                q.n = __shfl_sync(0xffffffffu, q.n, at);
                q.kv = __shfl_sync(0xffffffffu, q.kv, at);
                q.past = __shfl_sync(0xffffffffu, q.past, at);
                i = __shfl_sync(0xffffffffu, i, at);
                const Item it = make_item<kPrefix>(p, q, base + at, i, kv_head, 0, INT32_MAX, true, 0);
                return it;
            }
            before += __popc(m);
            base += 32;
            if (base >= n_seqs) {
                base = 0;
                level = __reduce_max_sync(0xffffffffu, below);
                below = -1;
            }
        }
        return none;
    }

    __device__ Item next_piece() {
        Seq q = load_seq<kPrefix>(p.a, seq);   // every lane the same
        int64_t units = seq_units<kPrefix>(q, block_tokens, kv_heads);
        while (unit >= seq_first + units) {   // on to the sequence that holds `unit`
            seq_first += units;
            q = load_seq<kPrefix>(p.a, ++seq);
            units = seq_units<kPrefix>(q, block_tokens, kv_heads);
        }
        int64_t first = seq_first;
        int i = 0, cost;
        if (kPrefix) {
            cost = block_units<kPrefix>(q, 0, block_tokens);
            i = static_cast<int>(divide(unit - first, static_cast<int64_t>(cost) * kv_heads));
            first += static_cast<int64_t>(i) * cost * kv_heads;
        } else {
            for (;; ++i) {
                cost = block_units<kPrefix>(q, i, block_tokens);
                if (unit < first + static_cast<int64_t>(cost) * kv_heads) break;
                first += static_cast<int64_t>(cost) * kv_heads;
            }
        }
        const int kv_head = static_cast<int>(divide(unit - first, cost));
        first += static_cast<int64_t>(kv_head) * cost;
        const int t0 = static_cast<int>(unit - first);
        const int t1 = static_cast<int>(min(unit_end - first, static_cast<int64_t>(cost)));
        unit = first + t1;
        return make_item<kPrefix>(p, q, seq, i, kv_head, t0, t1, t0 == 0 && t1 == cost, blockIdx.x);
    }
};

// value matrix descriptor: N-major (64 head dims contiguous), 128-byte swizzle; 64-dim halves kHalfBytes apart (LBO),
// 8-key groups 1024 bytes apart (SBO)
__device__ __forceinline__ uint64_t value_desc(uint32_t saddr) {
    return static_cast<uint64_t>((saddr >> 4) & 0x3fffu) | (static_cast<uint64_t>((128 * 128) >> 4) << 16) |
           (64ull << 32) | (1ull << 46) | (2ull << 61);
}

__device__ __forceinline__ void tmem_load32(uint32_t addr, float* f) {
    uint32_t* v = reinterpret_cast<uint32_t*>(f);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
        "%13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, "
        "[%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_load16(uint32_t addr, float* f) {
    uint32_t* v = reinterpret_cast<uint32_t*>(f);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
        "[%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16};" ::"r"(addr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// two fp32 operations per instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {   // NaN if one is
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
// an item read by the whole warp, in a form the compiler knows to be uniform
__device__ __forceinline__ Item uniform_item(const Item& m) {
    Item it = m;
    constexpr unsigned kAll = 0xffffffffu;
    it.valid = __shfl_sync(kAll, it.valid, 0);
    it.tokens = __shfl_sync(kAll, it.tokens, 0);
    it.pos0 = __shfl_sync(kAll, it.pos0, 0);
    it.kv = __shfl_sync(kAll, it.kv, 0);
    it.tile0 = __shfl_sync(kAll, it.tile0, 0);
    it.end[0] = __shfl_sync(kAll, it.end[0], 0);
    it.end[1] = __shfl_sync(kAll, it.end[1], 0);
    return it;
}
// products of bf16 operands into fp32 tensor memory: left operand from shared memory, or from tensor memory
__device__ __forceinline__ void mma_ss(bool pred, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(pred ? 1 : 0)
        : "memory");
}
__device__ __forceinline__ void mma_ts(bool pred, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(pred ? 1 : 0)
        : "memory");
}

__device__ __forceinline__ void store_sector(void* to, const uint32_t* v) {   // 32 bytes, 32-byte aligned
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                 "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

template <int DP, bool kPrefix>
__global__ void __launch_bounds__(kThreads384, 1)
attention_tile_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                      const __grid_constant__ CUtensorMap map_v, const __grid_constant__ TileParams p) {
    using C = TileCfg<DP>;
    constexpr int S = C::kStages;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = s32(sm);
    const uint32_t k_full = sbase + C::kOffBar, k_empty = k_full + 8 * S, v_full = k_empty + 8 * S, v_empty = v_full + 8 * S;
    const uint32_t q_full = v_empty + 8 * S, q_empty = q_full + 8, s_full = q_empty + 8, s_free = s_full + 16,
                   p_full = s_free + 8, o_full = p_full + 16, v_tail = o_full + 16, v_fixed = v_tail + 8,
                   item_full = v_fixed + 8, item_empty = item_full + 8 * kItemSlots, done = item_empty + 8 * kItemSlots;
    const uint32_t k_smem = sbase + C::kOffKv, v_smem = k_smem + S * C::kTileBytes;
    Item* items = reinterpret_cast<Item*>(sm + C::kOffItems);   // 64 bytes apart
    auto item_slot = [&](uint32_t n) { return reinterpret_cast<Item*>(reinterpret_cast<uint8_t*>(items) + 64 * (n % kItemSlots)); };
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + C::kOffMisc);
    volatile int32_t* abort = reinterpret_cast<volatile int32_t*>(sm + C::kOffMisc + 4);
    unsigned* err = p.a.err;
    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;

    // the kernel that follows (the decode kernel behind the prefixes', the join) may take the SMs as they come free; it
    // waits before it reads here
    if (p.split) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (kPrefix && warp == 3) prefetch_lengths(p.a, lane);
    if (threadIdx.x == 0) {
        auto init = [](uint32_t bar, int n) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(n)); };
        for (int s = 0; s < 4 * S; ++s) init(k_full + 8 * s, 1);
        init(q_full, 1);
        init(q_empty, 1);
        for (int q = 0; q < 2; ++q) {
            init(s_full + 8 * q, 1);
            init(p_full + 8 * q, 4);
            init(o_full + 8 * q, 1);
        }
        init(s_free, 4);
        init(v_tail, 1);
        init(v_fixed, 1);
        for (int s = 0; s < kItemSlots; ++s) {
            init(item_full + 8 * s, 1);
            init(item_empty + 8 * s, kItemReaders);
        }
        init(done, 1);
        init(done + 8, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        *abort = 0;
    }
    if (warp == 0 && lane == 0)
        for (const CUtensorMap* m : {&map_q, &map_k, &map_v})
            asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory");
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(s32(tmem_slot)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;

    // one setmaxnreg for each warpgroup
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFeedRegs));
        if (warp == 0) {
            // ---------------- schedule and loads
            const KvCacheDev& cache = p.a.cache;
            const int shift = cache.page_shift;
            const int boxes = cache.page_size >= kKeys ? 1 : kKeys >> shift;      // page boxes of a key tile
            const int box_rows = min(cache.page_size, kKeys);
            const int32_t* tables = kPrefix ? p.a.prefix.page_table : p.a.batch.page_table;
            const int64_t table_stride = kPrefix ? p.a.prefix.page_table_stride : p.a.batch.page_table_stride;
            Scheduler<kPrefix> sched(p, lane);
            uint32_t n_items = 0, n_q = 0, st = 0, loaded_k = 0, loaded_v = 0;
            bool stop = false;
            Item it = sched.next(), following = it;
            for (; !stop; it = following) {
                if (n_items >= kItemSlots &&
                    !wait_warp(item_empty + 8 * (n_items % kItemSlots), (n_items / kItemSlots - 1) & 1, abort, err))
                    break;
                if (lane == 0) {
                    *item_slot(n_items) = it;
                    arrive(item_full + 8 * (n_items % kItemSlots));
                }
                __syncwarp();
                ++n_items;
                if (!it.valid) break;
                const int end = max(it.end[0], it.end[1]);
                if (end <= it.tile0) {
                    following = sched.next();
                    continue;
                }
                // page of this lane's box of a key tile; past the block's last key: no box
                const int seen = kPrefix ? it.kv : min(max(it.pos0 + it.tokens, 0), it.kv);
                const int32_t* table = tables + it.seq * table_stride;
                auto page_of = [&](int t) {
                    const int key = t * kKeys + lane * box_rows;
                    if (lane >= boxes || key >= seen || t >= end) return -1;
                    const int page = __ldg(table + (key >> shift));
                    if (static_cast<unsigned>(page) >= static_cast<unsigned>(cache.n_pages)) {
                        atomicOr(err, kErrPageRange);
                        return cache.n_pages;   // past the map's end: zeros
                    }
                    return page;
                };
                int page = page_of(it.tile0);
                if (n_q > 0 && !wait_warp(q_empty, (n_q - 1) & 1, abort, err)) break;
                ++n_q;
                if (lane == 0) {
                    const int tiles = it.end[1] > it.tile0 ? 2 : 1;   // row tile 1 sees at least row tile 0's keys
                    const uint32_t box = C::kHalves * 128 * p.tile_tokens * p.group;
                    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(q_full), "r"(tiles * box)
                                 : "memory");
                    for (int q = 0; q < tiles; ++q)
                        for (int h = 0; h < C::kHalves; ++h)
                            tma_load_3d(sbase + q * C::kTileBytes + h * C::kHalfBytes, &map_q, 64 * h, it.kv_head * p.group,
                                        it.row0 + q * p.tile_tokens, q_full);
                }
                for (int t = it.tile0; t < end && !stop; ++t, ++st) {
                    const int next = page_of(t + 1);
                    const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, page >= 0)) * box_rows * 128 * C::kHalves;
                    const uint32_t s = st % S;
#pragma unroll
                    for (int kv = 0; kv < 2; ++kv) {
                        const uint32_t full = (kv ? v_full : k_full) + 8 * s, empty = (kv ? v_empty : k_empty) + 8 * s;
                        if (st >= S && !wait_warp(empty, (st / S - 1) & 1, abort, err)) {
                            stop = true;
                            break;
                        }
                        if (lane == 0)
                            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(full), "r"(bytes)
                                         : "memory");
                        __syncwarp();
                        if (page >= 0) {
                            const int token = (t * kKeys) & (cache.page_size - 1);
#pragma unroll
                            for (int h = 0; h < C::kHalves; ++h)
                                tma_load_4d((kv ? v_smem : k_smem) + s * C::kTileBytes + h * C::kHalfBytes +
                                                lane * box_rows * 128,
                                            kv ? &map_v : &map_k, 64 * h, token, it.kv_head, page, full);
                        }
                        if (kv) loaded_v = st + 1;
                        else loaded_k = st + 1;
                    }
                    page = next;
                    // the next block is taken when this one's loads are issued: early tickets would deal the blocks out as by
                    // turns, and before its last tile the search delayed that (a prompt of 7937: 217 us, 219 a tile before)
                    if (t == end - 1) following = sched.next();
                }
            }
            // teardown: the copies in flight land before the CTA may exit
            if (lane == 0) {
                if (n_q > 0) drain_wait(q_full, (n_q - 1) & 1);
                for (uint32_t j = loaded_k > S ? loaded_k - S : 0; j < loaded_k; ++j) drain_wait(k_full + 8 * (j % S), (j / S) & 1);
                for (uint32_t j = loaded_v > S ? loaded_v - S : 0; j < loaded_v; ++j) drain_wait(v_full + 8 * (j % S), (j / S) & 1);
            }
            __syncwarp();
        } else if (warp & 1) {
            // ---------------- matrix products: warp 1 issues S = Q K^T, warp 3 O += P V, one thread of each.  The whole warp
            // walks the loop, so that descriptors and addresses stay in uniform registers (computed in a divergent thread
            // they cost ten cycles apiece to move there, and the issue takes longer than the products).
            const bool leader = lane == 0, scores = warp == 1;
            const int k_steps = (p.a.cache.head_dim + 15) / 16;       // of Q K^T
            const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((kRows >> 4) << 24);   // fp32 += bf16 x bf16
            const uint32_t idesc_pv = idesc | (1u << 16) | (static_cast<uint32_t>(2 * k_steps) << 17);   // V is N-major
            const uint32_t t0 = __shfl_sync(0xffffffffu, tmem, 0);
            uint32_t st = 0, n_q = 0, n_s = 0, n_p[2] = {0, 0}, n_fixed = 0;
            bool ok = true;
            for (uint32_t n = 0; ok; ++n) {
                ok = wait_warp(item_full + 8 * (n % kItemSlots), (n / kItemSlots) & 1, abort, err);
                if (!ok) break;
                const Item it = uniform_item(*item_slot(n));
                arrive_if(leader, item_empty + 8 * (n % kItemSlots));
                if (!it.valid) break;
                const int end = max(it.end[0], it.end[1]);
                if (end <= it.tile0) continue;
                int seen[2];   // keys the row tile's last row sees
#pragma unroll
                for (int q = 0; q < 2; ++q)
                    seen[q] = kPrefix ? it.kv : min(max(it.pos0 + min(it.tokens, (q + 1) * p.tile_tokens), 0), it.kv);
                if (scores) {
                    ok = wait_warp(q_full, n_q++ & 1, abort, err);
                    for (int t = it.tile0; t < end && ok; ++t, ++st) {
                        const uint32_t s = st % S;
                        ok = wait_warp(k_full + 8 * s, (st / S) & 1, abort, err);
                        const uint64_t bd = umma_desc(k_smem + s * C::kTileBytes);
#pragma unroll
                        for (int q = 0; q < 2; ++q)
                            if (t < it.end[q]) {
                                // the softmax warps have read the S before this one
                                if (n_s > 0) ok = ok && wait_warp(s_free, (n_s - 1) & 1, abort, err);
                                ++n_s;
                                fence_after();
                                const int n16 = (min(seen[q] - t * kKeys, kKeys) + 15) / 16;
                                const uint32_t id = idesc | (static_cast<uint32_t>(2 * n16) << 17);
                                const uint64_t ad = umma_desc(sbase + q * C::kTileBytes);
#pragma unroll
                                for (int k = 0; k < DP / 16; ++k) {   // 16 dims: 32 bytes along a row of 64
                                    const uint32_t off = ((k >> 2) * C::kHalfBytes + 32 * (k & 3)) >> 4;
                                    mma_ss(leader && ok && k < k_steps, t0 + kColS, ad + off, bd + off, id, k > 0 ? 1u : 0u);
                                }
                                mma_commit_if(leader && ok, s_full + 8 * q);
                            }
                        mma_commit_if(leader && ok, k_empty + 8 * s);
                        mma_commit_if(leader && ok && t == end - 1, q_empty);
                    }
                } else {
                    const int all = max(seen[0], seen[1]);
                    const bool fix = ((all + 15) & ~15) > it.kv;   // the last tile's value rows past it.kv are cleared
                    for (int t = it.tile0; t < end && ok; ++t, ++st) {
                        const uint32_t s = st % S;
                        ok = wait_warp(v_full + 8 * s, (st / S) & 1, abort, err);
                        if (ok && fix && t == (all - 1) / kKeys) {
                            arrive_if(leader, v_tail);   // V(t) has landed: warp 2 may clear its tail
                            ok = wait_warp(v_fixed, n_fixed++ & 1, abort, err);
                        }
                        const uint64_t vd = value_desc(v_smem + s * C::kTileBytes);
                        const uint32_t later = t > it.tile0 ? 1u : 0u;
#pragma unroll
                        for (int q = 0; q < 2; ++q)
                            if (t < it.end[q]) {
                                ok = ok && wait_warp(p_full + 8 * q, n_p[q]++ & 1, abort, err);
                                fence_after();
                                const int steps = (min(seen[q] - t * kKeys, kKeys) + 15) / 16;
#pragma unroll
                                for (int k = 0; k < kKeys / 16; ++k)   // 16 keys: 16 rows of 128 bytes, 8 columns of P
                                    mma_ts(leader && ok && k < steps, t0 + kColO + 128 * q, t0 + kColP + 64 * q + 8 * k,
                                           vd + k * (2048 >> 4), idesc_pv, k > 0 ? 1u : later);
                                mma_commit_if(leader && ok, o_full + 8 * q);
                            }
                        mma_commit_if(leader && ok, v_empty + 8 * s);
                    }
                }
            }
            // teardown: every product issued has completed before the tensor memory is freed
            if (leader) {
                mma_commit(done + 8 * (warp >> 1));
                drain_wait(done + 8 * (warp >> 1), 0);
            }
            __syncwarp();
        } else if (warp == 2) {
            // ---------------- clears value rows past a sequence's last key
            uint32_t st = 0, n_fixed = 0;
            for (uint32_t n = 0;; ++n) {
                if (!wait_warp(item_full + 8 * (n % kItemSlots), (n / kItemSlots) & 1, abort, err)) break;
                const Item it = *item_slot(n);
                __syncwarp();
                if (lane == 0) arrive(item_empty + 8 * (n % kItemSlots));
                if (!it.valid) break;
                const int end = max(it.end[0], it.end[1]);
                if (end <= it.tile0) continue;
                const int all = kPrefix ? it.kv : min(max(it.pos0 + it.tokens, 0), it.kv);
                const int upto = (all + 15) & ~15;
                if (upto > it.kv && end == (all + kKeys - 1) / kKeys) {
                    const uint32_t j = st + (end - 1 - it.tile0), s = j % S;   // the stage of V(end - 1)
                    // (its own phase of v_full: the stage is not released before v_fixed)
                    if (!wait_warp(v_tail, n_fixed++ & 1, abort, err) || !wait_warp(v_full + 8 * s, (j / S) & 1, abort, err))
                        break;
                    const int r0 = it.kv - (end - 1) * kKeys, rows = upto - it.kv;
                    for (int h = 0; h < C::kHalves; ++h)
                        for (int i = lane; i < rows * 8; i += 32)
                            *reinterpret_cast<uint4*>(sm + (v_smem - sbase) + s * C::kTileBytes + h * C::kHalfBytes + r0 * 128 +
                                                      16 * i) = make_uint4(0, 0, 0, 0);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // visible to the products
                    __syncwarp();
                    if (lane == 0) arrive(v_fixed);
                }
                st += end - it.tile0;
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        // ---------------- softmax: warps 4-7 row tile 0, warps 8-11 row tile 1, a thread per row
        const int q = (warp - 4) >> 2;
        const int row = 32 * (warp & 3) + lane;
        const uint32_t quarter = static_cast<uint32_t>(32 * (warp & 3)) << 16;
        const uint32_t t_s = tmem + quarter + kColS, t_p = tmem + quarter + kColP + 64 * q,
                       t_o = tmem + quarter + kColO + 128 * q;
        const int token = q * p.tile_tokens + row / p.group, sub = row % p.group;
        const bool in_tile = row < p.tile_tokens * p.group;
        const float c = p.c;
        const float2 c2 = make_float2(c, c);
        uint32_t n_s = 0, n_o = 0;
        bool stop = false;
        for (uint32_t n = 0; !stop; ++n) {
            if (!wait_warp(item_full + 8 * (n % kItemSlots), (n / kItemSlots) & 1, abort, err)) break;
            const Item it = *item_slot(n);
            __syncwarp();
            if (lane == 0) arrive(item_empty + 8 * (n % kItemSlots));
            if (!it.valid) break;
            bool ok = true;
            const bool live = in_tile && token < it.tokens;
            const int limit = !live ? 0 : kPrefix ? it.kv : min(it.pos0 + token + 1, it.kv);   // keys this row sees
            const bool any_live = __any_sync(0xffffffffu, live);
            float m = -INFINITY, l = 0.0f;
            for (int t = it.tile0; t < it.end[q]; ++t, ++n_s) {
                if (!wait_warp(s_full + 8 * q, n_s & 1, abort, err)) {
                    stop = true;
                    break;
                }
                fence_after();
                float s[kKeys];
                if (any_live) {
#pragma unroll
                    for (int i = 0; i < kKeys; i += 32) tmem_load32(t_s + i, s + i);
                    tmem_wait_load();
                }
                fence_before();
                __syncwarp();
                arrive_if(lane == 0, s_free);   // the next S may be written
                if (any_live) {
                    if (p.negate) {
#pragma unroll
                        for (int i = 0; i < kKeys; ++i) s[i] = -s[i];
                    }
                    const int columns = limit - t * kKeys;
                    if (!__all_sync(0xffffffffu, columns >= kKeys || !live)) {
#pragma unroll
                        for (int i = 0; i < kKeys; ++i) s[i] = i < columns ? s[i] : -INFINITY;
                    }
                    const auto row_max = [&] {   // NaN if a score is
                        float top[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) top[j] = max3(s[j], s[4 + j], s[8 + j]);
#pragma unroll
                        for (int i = 12; i + 8 <= kKeys; i += 8)
#pragma unroll
                            for (int j = 0; j < 4; ++j) top[j] = max3(top[j], s[i + j], s[i + 4 + j]);
                        static_assert((kKeys - 12) % 8 == 4, "the last four scores are left");
                        return max3(max3(top[0], s[kKeys - 4], s[kKeys - 3]), max3(top[1], s[kKeys - 2], s[kKeys - 1]),
                                    max3(top[2], top[3], top[3]));
                    };
                    // The first keys a row sees set m to their maximum; later ones are taken relative to it as it is, and m
                    // is raised (and the tile done again) only when their sum shows that they are far above it.
                    if (__any_sync(0xffffffffu, m == -INFINITY)) {
                        const float top = row_max();
                        if (m == -INFINITY) m = top;
                    }
                    // P V(t - 1) is done: P may be written, and O brought to a new maximum
                    if (t > it.tile0) ok = spin_warp(o_full + 8 * q, n_o++ & 1, abort, err);
                    fence_after();
                    float tile_sum;
                    for (bool again = false;; again = true) {
                        const float mc = m == -INFINITY ? 0.0f : -m * c;
                        const float2 mc2 = make_float2(mc, mc);
                        float2 sum[4] = {};
#pragma unroll
                        for (int i = 0; i < kKeys; i += 32) {
                            uint32_t pk[16];   // the product's operand; the sum keeps fp32
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                const float2 x = fma2(make_float2(s[i + 2 * j], s[i + 2 * j + 1]), c2, mc2);
                                const float2 e = make_float2(exp2_fast(x.x), exp2_fast(x.y));
                                sum[j & 3] = add2(sum[j & 3], e);
                                pk[j] = pack_bf16(e.x, e.y);
                            }
                            tmem_store16(t_p + (i >> 1), pk);
                        }
                        const float2 both = add2(add2(sum[0], sum[1]), add2(sum[2], sum[3]));
                        tile_sum = both.x + both.y;
                        const bool rise = live && !(tile_sum <= kMaxTileSum);   // (or not a number)
                        if (again || !__any_sync(0xffffffffu, rise)) break;
                        float f = 1.0f;
                        if (rise) {
                            const float top = row_max();
                            f = exp2_fast((m - top) * c);
                            m = top;
                        }
                        l *= f;
                        if (t > it.tile0) {
#pragma unroll 1
                            for (int d = 0; d < DP; d += 16) {
                                float o[16];
                                tmem_load16(t_o + d, o);
                                tmem_wait_load();
#pragma unroll
                                for (int j = 0; j < 16; ++j) o[j] *= f;
                                tmem_store16(t_o + d, reinterpret_cast<const uint32_t*>(o));
                            }
                        }
                    }
                    l += tile_sum;
                    tmem_wait_store();
                } else if (t > it.tile0) {
                    ok = wait_warp(o_full + 8 * q, n_o++ & 1, abort, err);
                    fence_after();
                }
                if (!ok) {
                    stop = true;
                    break;
                }
                fence_before();
                __syncwarp();
                arrive_if(lane == 0, p_full + 8 * q);
            }
            if (stop) break;
            const bool some = it.end[q] > it.tile0;
            if (some) {
                if (!wait_warp(o_full + 8 * q, n_o++ & 1, abort, err)) break;
                fence_after();
            }
            if (!any_live) continue;
            const float r = l > 0.0f || l != l ? 1.0f / l : 0.0f;   // no key seen: 0 (a NaN stays one)
            const int D = p.a.cache.head_dim;
            const int64_t call_row = it.row0 + token;
            const int head = it.kv_head * p.group + sub;
            const bool part = it.part_row >= 0;
            const int tile_rows = p.tile_tokens * p.group;
            const int64_t part0 = static_cast<int64_t>(it.part_row) + q * tile_rows;     // the tile's first partial row
            if (live) {
                const float lse = m * p.c + log2f(l);   // no key seen: -inf
                if (part)
                    p.w.part_lse[part0 + row] = lse;
                else if (p.a.rows.lse)
                    p.a.rows.lse[call_row * p.a.rows.n_q_heads + head] = lse * kLn2;
            }
            // O / l to the row, a lane its own, whole 32-byte sectors where the rows' alignment allows (through shared
            // memory, so that lanes share lines, it takes longer: the loop is bound by its latencies, not by the stores)
            __nv_bfloat16* out = p.a.rows.out + call_row * p.a.rows.out_row + head * p.a.rows.out_head;
            float* to_part = p.w.part_o + (part0 + row) * DP;
            const bool wide = p.wide_out;
#pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += 32) {
                float o[32];
                tmem_load32(t_o + c0, o);
                tmem_wait_load();
#pragma unroll
                for (int j = 0; j < 32; ++j) o[j] = some ? o[j] * r : 0.0f;
                if (!live) {
                } else if (part) {
#pragma unroll
                    for (int j = 0; j < 32; j += 8)
                        store_sector(to_part + c0 + j, reinterpret_cast<const uint32_t*>(o + j));
                } else {
                    uint32_t v[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] = pack_bf16(o[2 * j], o[2 * j + 1]);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int col = c0 + 16 * j;
                        if (wide && col + 16 <= D) {
                            store_sector(out + col, v + 8 * j);
                        } else {
                            if (col < D)
                                *reinterpret_cast<uint4*>(out + col) = make_uint4(v[8 * j], v[8 * j + 1], v[8 * j + 2], v[8 * j + 3]);
                            if (col + 8 < D)
                                *reinterpret_cast<uint4*>(out + col + 8) =
                                    make_uint4(v[8 * j + 4], v[8 * j + 5], v[8 * j + 6], v[8 * j + 7]);
                        }
                    }
                }
                __syncwarp();
            }
            fence_before();   // the next block's products may overwrite O once its P is handed over
        }
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == 1) {
        __syncwarp();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
    if (!p.split && threadIdx.x == 0) {   // the last CTA leaves the ticket counter ready for the next call
        __threadfence();
        if (atomicAdd(p.w.counters + 1, 1) == static_cast<int>(gridDim.x) - 1) {
            p.w.counters[0] = 0;
            p.w.counters[1] = 0;
        }
    }
}

// Joins the pieces of the blocks that were split: a block for each row and key head.
template <int DP>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ TileParams p) {
    const int lane = threadIdx.x & 31, kv_heads = p.a.cache.n_kv_heads;
    const int row = blockIdx.x / kv_heads, head0 = (blockIdx.x % kv_heads) * p.group;
    const int s = p.a.batch.q_offsets ? find_sequence(p.a.batch.q_offsets, p.a.batch.n_seqs, row, lane) : row;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (s < 0 || s >= p.a.batch.n_seqs) return;
    const PieceSpan at = piece_span<false>(p.a, p.w, s, row, head0, p.tile_tokens);
    if (at.c0 >= at.c1) return;   // whole (written by the tile kernel), or no row of the sequence
    for (int i = threadIdx.x; i < p.group * (DP / 4); i += blockDim.x) {
        const int r = i / (DP / 4), d = 4 * (i % (DP / 4));
        PartSum<DP> sum;
        sum.add(p.w.part_lse, p.w.part_o, at.base + r, kPartRows, at.c0, at.c1, d);
        sum.write(p.a, row, head0 + r, d);
    }
}

template <int DP, bool kPrefix>
cudaError_t launch_tiles(const TileParams& p, const Geometry& g, int grid, cudaStream_t stream) {
    CUtensorMap q, k, v;
    if (!make_row_map(&q, p.a, g.tile_tokens) || !make_cache_map(&k, p.a.cache, p.a.cache.k, kKeys) ||
        !make_cache_map(&v, p.a.cache, p.a.cache.v, kKeys))
        return cudaErrorInvalidValue;
    const int smem = static_cast<int>(TileCfg<DP>::kBytes) + 1024;
    static std::atomic<uint64_t> attr_set{0};   // one bit per device ordinal whose attribute is set
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (!(attr_set.load(std::memory_order_acquire) & bit)) {
        cudaFuncAttributes fa;
        e = cudaFuncGetAttributes(&fa, attention_tile_kernel<DP, kPrefix>);
        // the warpgroups' register shares must fit what the block is launched with
        if (e == cudaSuccess && fa.numRegs * kThreads384 < 128 * kFeedRegs + 256 * kSoftmaxRegs)
            e = cudaErrorInvalidConfiguration;
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(attention_tile_kernel<DP, kPrefix>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        attr_set.fetch_or(bit, std::memory_order_acq_rel);
    }
    attention_tile_kernel<DP, kPrefix><<<grid, kThreads384, smem, stream>>>(q, k, v, p);
    return cudaGetLastError();
}

bool wide_rows(const AttnParams& a) {
    return reinterpret_cast<uintptr_t>(a.rows.out) % 32 == 0 && a.rows.out_row % 16 == 0 && a.rows.out_head % 16 == 0;
}

}  // namespace

// Whole blocks by ticket when there are at least two for each SM, or when no sequence can have more keys than
// kWholeKeys; otherwise pieces of equal length.
TilePlan plan_prompt(const AttnParams& a, int sms) {
    const Geometry g = geometry(a);
    const int block_tokens = 2 * g.tile_tokens;
    const int64_t whole = a.batch.n_rows / block_tokens;
    const int64_t blocks = (a.batch.n_seqs == 1 ? (a.batch.n_rows + block_tokens - 1) / block_tokens
                                                : std::min<int64_t>(whole + a.batch.n_seqs, a.batch.n_rows)) *
                           a.cache.n_kv_heads;
    const int64_t keys = static_cast<int64_t>(a.batch.max_pages) * a.cache.page_size;
    TilePlan plan{};
    plan.split = blocks < 2 * sms && keys > kWholeKeys;
    plan.grid = static_cast<int>(plan.split ? sms : std::min<int64_t>(blocks, sms));
    if (plan.split) plan.part_rows = static_cast<int64_t>(a.batch.n_rows) * a.rows.n_q_heads + kPartRows * plan.grid;
    plan.unit_ends = plan.split ? a.batch.n_seqs : 0;
    plan.dim = a.cache.head_dim <= 64 ? 64 : 128;
    return plan;
}

// The prefixes: their units are dealt evenly whatever their number; every piece leaves a partial result.
TilePlan plan_prefix(const AttnParams& a, int sms) {
    TilePlan plan{};
    plan.split = 1;
    plan.grid = sms;
    plan.part_rows = static_cast<int64_t>(a.batch.n_seqs) * a.rows.n_q_heads + kPartRows * plan.grid;
    plan.unit_ends = a.prefix.n_groups;
    plan.dim = a.cache.head_dim <= 64 ? 64 : 128;
    return plan;
}

cudaError_t launch_prefix_attention(const AttnParams& a, const TilePlan& plan, const TileWork& w, cudaStream_t stream) {
    const Geometry g = geometry(a);
    TileParams p{a, g.group, g.tile_tokens, 1, kMinPrefixUnits, UINT32_MAX / a.cache.n_kv_heads,
                 exp2_scale(a.rows.scale), a.rows.scale < 0.0f, wide_rows(a), w};
    return plan.dim == 64 ? launch_tiles<64, true>(p, g, plan.grid, stream) : launch_tiles<128, true>(p, g, plan.grid, stream);
}

cudaError_t launch_prompt_attention(const AttnParams& a, const TilePlan& plan, const TileWork& w, cudaStream_t stream) {
    const Geometry g = geometry(a);
    TileParams p{a, g.group, g.tile_tokens, plan.split, kMinPromptUnits, UINT32_MAX / a.cache.n_kv_heads,
                 exp2_scale(a.rows.scale), a.rows.scale < 0.0f, wide_rows(a), w};
    cudaError_t e = plan.dim == 64 ? launch_tiles<64, false>(p, g, plan.grid, stream)
                                   : launch_tiles<128, false>(p, g, plan.grid, stream);
    if (e != cudaSuccess || !plan.split) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(static_cast<int64_t>(a.batch.n_rows) * a.cache.n_kv_heads));
    cfg.blockDim = dim3(join_threads(g.group, plan.dim));
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // its blocks are there when the tile kernel ends
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return plan.dim == 64 ? cudaLaunchKernelEx(&cfg, join_kernel<64>, p) : cudaLaunchKernelEx(&cfg, join_kernel<128>, p);
}

}  // namespace vw
