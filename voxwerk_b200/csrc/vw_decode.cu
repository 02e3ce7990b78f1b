// vw_decode.cu -- single-token attention over a paged key/value cache (include/vwsampler.h, vw_decode_attention).
//
// out = softmax(scale q K^T) v for one row per sequence, over its own keys here; the keys of a shared prefix are read
// once for their whole group by the tile kernel (vw_prompt.cu), whose partial results are weighed in at the end.
//
// Bound: HBM (each key and value is read once, for the few query heads of its key head).  So the kernel is a stream: an
// item is (sequence, key head, block of at most 16 of its query heads), its units are tiles of 64 keys, and all units
// are dealt evenly to two CTAs per SM, whatever the sequences' lengths.  A CTA's producer warp loads its units' K and V
// by TMA (a lane per page box) into a ring and runs ahead across items; four warps each take 16 keys of a tile:
// S = Q K^T and O += P V by mma.sync m16n8k16 from shared memory (rows are the query heads; the tensor cores idle most
// of the time either way, a tile of 32 KB takes an SM about 1400 cycles to fetch), with a running maximum and sum of
// their own, raised only past 2^8.  At an item's end the four are joined in shared memory, a warp per row.  An item cut
// by a CTA boundary leaves its pieces in the workspace, and the CTA that finishes last joins them in order; with
// prefixes every item leaves its result there, and a join kernel weighs it with the prefix's.
//
// P is rounded to bf16 for its product with V, as in vw_prompt.cu (an mma's operands are of one 16-bit type).
//
// Measured (16 query heads on 8 of 128 dims, prefixes included; device time, CUDA graphs one after the other): 256
// sequences of 100-2000 keys on a prefix of 16001 142-146 us = 5.0-5.1 TB/s; 64 of 20-600 on one of 4099 33-35 us, 50 of
// 60-900 on four prefixes (32 heads on 4 of 64) 24-25 us, one of 700 12.3 us (of the 64's: the prefix kernel's other CTAs
// leave after 3 us, a schedule takes 4, the first tile is there 2 us later, an item's end costs 0.9 and the join 4).
// Without a prefix: the 256 120 us = 5.5 TB/s, the 64 20.5 us, the 50 14.4 us, 16 of 200-4000 27 us, 512 of 1-900 86 us.
//
// Every mbarrier wait is bounded.

#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>

#include "vw_attention.h"
#include "vw_internal.h"
#include "vw_tc.cuh"

namespace vw {
namespace {

constexpr int kThreads = 160;     // producer warp, four warps of 16 keys
constexpr int kKeys = 64;         // keys per tile
constexpr int kMaxRows = 16;      // query heads per item: the rows of an mma
constexpr int kItemSlots = 2;
constexpr int kItemUnits = 2;     // an item's end costs about what two tiles do (64 sequences: 36 us, 40 without)
constexpr float kLn2 = 0.693147180559945309f;
constexpr uint32_t kSmemBudget = 113 * 1024;   // two CTAs per SM

template <int DP>
struct DecodeCfg {
    static constexpr int kHalves = DP / 64;
    static constexpr uint32_t kHalfBytes = kKeys * 128;
    static constexpr uint32_t kTileBytes = kHalves * kHalfBytes;   // K or V
    static constexpr uint32_t kStageBytes = 2 * kTileBytes;
    static constexpr uint32_t kQueryHalf = kMaxRows * 128;
    static constexpr uint32_t kQueryBytes = kHalves * kQueryHalf;
    static constexpr int kMaxStages = 6;
    // barriers full[6] empty[6] item_full[2] item_empty[2], item slots, flags
    static constexpr uint32_t kBarBytes = 8 * (2 * kMaxStages + 2 * kItemSlots);
    static constexpr uint32_t kTail = kBarBytes + kItemSlots * 64 + 16;
    // joining four warps: O of `rows` rows each, and (m, l)
    __host__ __device__ static constexpr uint32_t scratch(int rows) { return 4 * rows * (DP * 4 + 8); }
    static constexpr int stages(int rows) {
        const uint32_t room = kSmemBudget - 1024 - kItemSlots * kQueryBytes - kTail - scratch(rows);
        const int n = static_cast<int>(room / kStageBytes);
        return n < kMaxStages ? n : kMaxStages;
    }
    static constexpr uint32_t bytes(int rows) {
        return stages(rows) * kStageBytes + kItemSlots * kQueryBytes + kTail + scratch(rows) + 1024;
    }
};
static_assert(DecodeCfg<128>::stages(16) >= 2 && DecodeCfg<64>::stages(16) >= 2, "ring");

// Units of an item that are tiles; kItemUnits more stand for its end, so that a CTA with many short items has fewer tiles
__device__ __forceinline__ int units_with_tiles(int keys, int chunk) {
    return max((keys + kKeys * chunk - 1) / (kKeys * chunk), 1);
}

struct DecodeItem {
    int32_t valid, seq, kv_head, row_block;
    int32_t keys;            // of the sequence
    int32_t tile0, tile1;    // this piece's tiles
    int32_t index;           // of the item
    int32_t in_pieces;       // other CTAs have tiles of it too
    int64_t first, last;     // the units of its tiles, in all of the call's
    int64_t per;             // units of a CTA
};
static_assert(sizeof(DecodeItem) <= 64, "item slots");

struct DecodeParams {
    AttnParams a;
    DecodePlan plan;
    DecodeWork w;
    int32_t group, tile_tokens, stages, negate, boxes, has_prefix, sms;
    float c;
};

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// byte offset of 16-byte chunk `chunk` of row `row` in a tile of 128-byte rows with the TMA's 128-byte swizzle
__device__ __forceinline__ uint32_t swizzled(int row, int chunk) { return row * 128 + ((chunk ^ (row & 7)) << 4); }
__device__ __forceinline__ void sync_consumers() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
// the same, and whether any of the 128 threads has gone wrong: they leave together, so none waits for one that left
__device__ __forceinline__ bool any_failed(bool ok) {
    int r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.s32 p, %1, 0;\n\t"
        "barrier.cta.red.or.pred q, 1, 128, p;\n\t"
        "selp.s32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"(ok ? 0 : 1)
        : "memory");
    return r != 0;
}

template <int DP>
__global__ void __launch_bounds__(kThreads, 2)
decode_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
              const __grid_constant__ CUtensorMap map_v, const __grid_constant__ DecodeParams p) {
    using C = DecodeCfg<DP>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = s32(sm);
    const int S = p.stages, rows = p.plan.rows;
    const uint32_t off_q = S * C::kStageBytes, off_scratch = off_q + kItemSlots * C::kQueryBytes,
                   off_bar = off_scratch + C::scratch(rows);
    const uint32_t full = sbase + off_bar, empty = full + 8 * C::kMaxStages, item_full = empty + 8 * C::kMaxStages,
                   item_empty = item_full + 8 * kItemSlots;
    uint8_t* item_mem = sm + off_bar + C::kBarBytes;
    auto item_slot = [&](uint32_t n) { return reinterpret_cast<DecodeItem*>(item_mem + 64 * (n % kItemSlots)); };
    volatile int32_t* abort = reinterpret_cast<volatile int32_t*>(item_mem + 64 * kItemSlots);
    volatile int32_t* last = abort + 1;
    unsigned* err = p.a.err;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (p.has_prefix) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the join, once all CTAs run
    if (warp == 0 && lane == 0)
        for (const CUtensorMap* m : {&map_q, &map_k, &map_v})
            asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory");
    if (warp == 1) prefetch_lengths(p.a, lane);
    if (threadIdx.x == 0) {
        auto init = [](uint32_t bar, int n) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(n)); };
        for (int s = 0; s < S; ++s) {
            init(full + 8 * s, 1);
            init(empty + 8 * s, 4);
        }
        for (int s = 0; s < kItemSlots; ++s) {
            init(item_full + 8 * s, 1);
            init(item_empty + 8 * s, 4);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        *abort = 0;
    }
    __syncthreads();

    if (warp == 0) {
        // ---------------- units and loads
        const AttnParams& a = p.a;
        const KvCacheDev& cache = a.cache;
        const int n_seqs = a.batch.n_seqs, shift = cache.page_shift;
        const int per_seq = cache.n_kv_heads * p.plan.row_blocks;   // items of a sequence
        auto keys_of = [&](int s) {
            return checked_len(__ldg(a.batch.kv_lens + s), a.batch.max_pages, shift, err, kErrKvLens);
        };
        // A unit is `chunk` tiles of an item (an item without keys has one, to be written).  Few items: as many tiles as
        // give every CTA one unit at most, so that none has the ends of two items; else one tile.
        int64_t per = 1, unit = 0, unit_end = 0, first = 0;   // `first`: the first unit of sequence `seq`
        int seq = 0, chunk = 1, end_units = 0;
        auto units_of = [&](int keys) { return units_with_tiles(keys, chunk) + end_units; };
        // Behind the prefixes the last CTAs come when the prefixes' are done, and have no units: they take that from the
        // CTAs before them rather than by a schedule of their own (64 sequences: 34.5 us, 36.2 without).
        int with_units = 0;
        if (p.has_prefix && lane == 0) with_units = *static_cast<volatile int32_t*>(p.w.prefix.counters + 2);
        with_units = __shfl_sync(0xffffffffu, with_units, 0);
        if (with_units == 0 || static_cast<int>(blockIdx.x) < with_units) {
            const int sum_tiles = own_tiles(a, lane);
            const int64_t total_tiles = static_cast<int64_t>(sum_tiles) * per_seq;
            int ctas = gridDim.x;
            if (p.has_prefix) {   // the prefixes' SMs are not there yet: the CTAs that come to them later have no units
                int64_t units = 0;
                for (int g = lane; g < a.prefix.n_groups; g += 32)
                    units += seq_units<true>(load_seq<true>(a, g), 2 * p.tile_tokens, cache.n_kv_heads);
                units = (static_cast<int64_t>(__reduce_add_sync(0xffffffffu, static_cast<int>(units >> 24))) << 24) +
                        __reduce_add_sync(0xffffffffu, static_cast<int>(units & 0xffffff));
                const int taken = prefix_ctas(a, units, sum_tiles, p.sms, lane);
                if (taken < p.sms) ctas = min(ctas, 2 * (p.sms - taken));
            }
            const int64_t spare = static_cast<int64_t>(ctas) - p.plan.items;
            chunk = 2 * spare >= ctas ? static_cast<int>(max(divide(total_tiles + spare - 1, spare), int64_t{1})) : 1;
            end_units = chunk == 1 ? kItemUnits : 0;
            int64_t total = total_tiles + p.plan.items * end_units;
            if (chunk > 1) {
                int sum = 0;
                for (int s = lane; s < n_seqs; s += 32) sum += units_of(keys_of(s));
                total = static_cast<int64_t>(__reduce_add_sync(0xffffffffu, sum)) * per_seq;
            }
            per = divide(total + ctas - 1, ctas);
            unit = min(per * blockIdx.x, total);
            unit_end = min(unit + per, total);
            if (p.has_prefix && blockIdx.x == 0 && lane == 0) {   // for the CTAs that come late, and the join
                *static_cast<volatile int32_t*>(p.w.prefix.counters + 2) = ctas;
                *p.w.units_per_cta = per;
                *p.w.chunk = chunk;
            }
            const bool all = p.has_prefix && blockIdx.x == 0;
            bool found = false;
            for (int s0 = 0; (all || (unit < unit_end && !found)) && s0 < n_seqs; s0 += 32) {
                const int s = s0 + lane;
                const int u = s < n_seqs ? units_of(keys_of(s)) : 0;   // of one item (a sequence's fit 25 bits)
                const int sum = warp_scan(u, lane);
                const int64_t end = first + static_cast<int64_t>(sum) * per_seq;
                if (all && s < n_seqs) p.w.unit_end[s] = end;
                const unsigned m = __ballot_sync(0xffffffffu, end > unit);
                if (m && !found) {
                    found = true;
                    const int at = __ffs(m) - 1;
                    seq = s0 + at;
                    // (CTA 0 begins with sequence 0)
                    if (!all) first += static_cast<int64_t>(__shfl_sync(0xffffffffu, sum - u, at)) * per_seq;
                }
                if (all || !found) first = __shfl_sync(0xffffffffu, end, 31);
            }
            if (all) first = 0;
        }
        const int box_rows = min(cache.page_size, kKeys);
        // a lane's box of a tile: page box, keys or values, half of the head
        const int box = lane / (2 * C::kHalves), is_v = (lane / C::kHalves) & 1, half = lane % C::kHalves;
        uint32_t n_items = 0, st = 0;
        bool stop = false;
        while (!stop) {
            DecodeItem it;
            for (it.valid = 0; unit < unit_end && !it.valid;) {
                int keys = keys_of(seq), units = units_of(keys);
                while (unit >= first + static_cast<int64_t>(units) * per_seq) {
                    first += static_cast<int64_t>(units) * per_seq;
                    keys = keys_of(++seq);
                    units = units_of(keys);
                }
                const int j = static_cast<int>(divide(unit - first, units));
                const int64_t item_first = first + static_cast<int64_t>(j) * units;
                const int tiles = max((keys + kKeys - 1) / kKeys, 1), real = units - end_units;
                const int u0 = static_cast<int>(unit - item_first);
                const int u1 = static_cast<int>(min(unit_end - item_first, static_cast<int64_t>(units)));
                unit = item_first + u1;
                if (u0 >= real) continue;   // the end of an item whose tiles are another CTA's
                it.valid = 1;
                it.seq = seq;
                it.kv_head = j / p.plan.row_blocks;
                it.row_block = j % p.plan.row_blocks;
                it.keys = keys;
                it.tile0 = u0 * chunk;
                it.tile1 = min(min(u1, real) * chunk, tiles);
                it.index = seq * per_seq + j;
                it.in_pieces = u0 > 0 || u1 < real;
                it.first = item_first;
                it.last = item_first + real - 1;
                it.per = per;
            }
            const uint32_t slot = n_items % kItemSlots;
            if (n_items >= kItemSlots && !wait_bounded(item_empty + 8 * slot, (n_items / kItemSlots - 1) & 1, abort, err))
                stop = true;
            if (__any_sync(0xffffffffu, stop)) break;
            if (lane == 0) {
                *item_slot(n_items) = it;
                if (it.valid) {
                    const uint32_t dst = sbase + off_q + slot * C::kQueryBytes;
                    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(item_full + 8 * slot),
                                 "r"(C::kHalves * rows * 128)
                                 : "memory");
                    for (int h = 0; h < C::kHalves; ++h)
                        tma_load_3d(dst + h * C::kQueryHalf, &map_q, 64 * h, it.kv_head * p.group + it.row_block * kMaxRows,
                                    it.seq, item_full + 8 * slot);
                } else {
                    arrive(item_full + 8 * slot);
                }
            }
            __syncwarp();
            ++n_items;
            if (!it.valid) break;
            const int32_t* table = a.batch.page_table + it.seq * a.batch.page_table_stride;
            auto page_of = [&](int t) {
                const int key = t * kKeys + box * box_rows;
                if (box >= p.boxes || key >= it.keys || t >= it.tile1) return -1;
                const int page = __ldg(table + (key >> shift));
                if (static_cast<unsigned>(page) >= static_cast<unsigned>(cache.n_pages)) {
                    atomicOr(err, kErrPageRange);
                    return cache.n_pages;   // past the map's end: zeros
                }
                return page;
            };
            int page = page_of(it.tile0);
            for (int t = it.tile0; t < it.tile1; ++t, ++st) {
                const int next = page_of(t + 1);
                const uint32_t s = st % S;
                if (st >= static_cast<uint32_t>(S) && !wait_bounded(empty + 8 * s, (st / S - 1) & 1, abort, err)) stop = true;
                if (__any_sync(0xffffffffu, stop)) {
                    stop = true;
                    break;
                }
                const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, page >= 0)) * box_rows * 128;
                if (lane == 0)
                    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(full + 8 * s), "r"(bytes)
                                 : "memory");
                __syncwarp();
                if (page >= 0)
                    tma_load_4d(sbase + s * C::kStageBytes + is_v * C::kTileBytes + half * C::kHalfBytes +
                                    box * box_rows * 128,
                                is_v ? &map_v : &map_k, 64 * half, (t * kKeys) & (cache.page_size - 1), it.kv_head, page,
                                full + 8 * s);
                page = next;
            }
        }
        // teardown: the copies in flight land before the CTA may exit
        if (lane == 0) {
            for (uint32_t j = st > static_cast<uint32_t>(S) ? st - S : 0; j < st; ++j) drain_wait(full + 8 * (j % S), (j / S) & 1);
            for (uint32_t j = n_items > kItemSlots ? n_items - kItemSlots : 0; j < n_items; ++j)
                drain_wait(item_full + 8 * (j % kItemSlots), (j / kItemSlots) & 1);
        }
        __syncwarp();
        if (p.has_prefix) asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }

    // ---------------- attention: warp w takes keys [16 w, 16 w + 16) of each tile
    const int w = warp - 1, key0 = 16 * w;
    const bool upper = rows > 8;   // rows 8-15 of the mma hold query heads
    float* scratch_o = reinterpret_cast<float*>(sm + off_scratch);                 // [4][rows][DP]
    float2* scratch_ml = reinterpret_cast<float2*>(scratch_o + 4 * rows * DP);     // [4][rows]
    uint32_t st = 0;
    for (uint32_t n = 0;; ++n) {
        const uint32_t slot = n % kItemSlots;
        bool ok = wait_bounded(item_full + 8 * slot, (n / kItemSlots) & 1, abort, err);
        if (any_failed(ok)) break;
        const DecodeItem it = *item_slot(n);
        if (!it.valid) break;
        uint32_t qf[DP / 16][4];
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
            ldmatrix4(sbase + off_q + slot * C::kQueryBytes + (k >> 2) * C::kQueryHalf +
                          swizzled(((lane >> 3) & 1) * 8 + (lane & 7), 2 * (k & 3) + (lane >> 4)),
                      qf[k]);
        __syncwarp();
        if (lane == 0) arrive(item_empty + 8 * slot);
        int c0 = 0, c1 = 0;   // CTAs that hold the item's pieces
        if (it.in_pieces && !p.has_prefix) {
            c0 = static_cast<int>(divide(it.first, it.per));
            c1 = static_cast<int>(divide(it.last, it.per));
        }

        float o[DP / 8][4];
#pragma unroll
        for (int i = 0; i < DP / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};   // rows lane / 4 and lane / 4 + 8
        for (int t = it.tile0; t < it.tile1; ++t, ++st) {
            const uint32_t s = st % S;
            ok = wait_bounded(full + 8 * s, (st / S) & 1, abort, err);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const int valid = it.keys - t * kKeys - key0;   // of this warp's 16 keys
            if (valid > 0) {
                const uint32_t k_base = sbase + s * C::kStageBytes, v_base = k_base + C::kTileBytes;
                if (valid < 16) {   // what lies past the last key may be anything: 0 * NaN would reach the sums
                    for (int i = lane; i < (16 - valid) * 8 * C::kHalves; i += 32) {
                        const int h = i / ((16 - valid) * 8), r = i % ((16 - valid) * 8);
                        *reinterpret_cast<uint4*>(sm + (v_base - sbase) + h * C::kHalfBytes + (key0 + valid) * 128 + 16 * r) =
                            make_uint4(0, 0, 0, 0);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // before the ring's next copy there
                    __syncwarp();
                }
                float sc[2][4] = {};
#pragma unroll
                for (int k = 0; k < DP / 16; ++k) {
                    uint32_t kf[4];
                    ldmatrix4(k_base + (k >> 2) * C::kHalfBytes +
                                  swizzled(key0 + (lane >> 4) * 8 + (lane & 7), 2 * (k & 3) + ((lane >> 3) & 1)),
                              kf);
                    mma_16x8x16(sc[0], qf[k], kf[0], kf[1]);
                    mma_16x8x16(sc[1], qf[k], kf[2], kf[3]);
                }
                uint32_t pf[4];   // P as the next product's left operand: [row half + 2 * key half]
                float f[2] = {1.0f, 1.0f};
                bool rise = false;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (h == 1 && !upper) {
                        pf[1] = pf[3] = 0;
                        break;
                    }
                    float x[4] = {sc[0][2 * h], sc[0][2 * h + 1], sc[1][2 * h], sc[1][2 * h + 1]};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (p.negate) x[i] = -x[i];
                        const int key = 2 * (lane & 3) + (i & 1) + 8 * (i >> 1);
                        if (key >= valid) x[i] = -INFINITY;
                    }
                    float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    if (m[h] == -INFINITY) {
                        m[h] = top;
                    } else if ((top - m[h]) * p.c > 8.0f) {
                        f[h] = exp2_fast((m[h] - top) * p.c);
                        m[h] = top;
                        rise = true;
                    }
                    const float mc = m[h] == -INFINITY ? 0.0f : m[h] * p.c;
                    float e[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) e[i] = exp2_fast(__fmaf_rn(x[i], p.c, -mc));
                    l[h] = __fmaf_rn(l[h], f[h], (e[0] + e[1]) + (e[2] + e[3]));
                    pf[h] = pack_bf16(e[0], e[1]);
                    pf[2 + h] = pack_bf16(e[2], e[3]);
                }
                if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
                    for (int i = 0; i < DP / 8; ++i) {
                        o[i][0] *= f[0];
                        o[i][1] *= f[0];
                        o[i][2] *= f[1];
                        o[i][3] *= f[1];
                    }
                }
#pragma unroll
                for (int d = 0; d < DP / 16; ++d) {
                    uint32_t vf[4];
                    ldmatrix4_t(v_base + (d >> 2) * C::kHalfBytes +
                                    swizzled(key0 + ((lane >> 3) & 1) * 8 + (lane & 7), 2 * (d & 3) + (lane >> 4)),
                                vf);
                    mma_16x8x16(o[2 * d], pf, vf[0], vf[1]);
                    mma_16x8x16(o[2 * d + 1], pf, vf[2], vf[3]);
                }
            }
            __syncwarp();
            if (lane == 0) arrive(empty + 8 * s);
        }

        // ---- the four warps' sums to shared memory, then a warp per row
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = (lane >> 2) + 8 * h;
            float sum = l[h];
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            if (r < rows) {
                float* dst = scratch_o + (w * rows + r) * DP + 2 * (lane & 3);
#pragma unroll
                for (int i = 0; i < DP / 8; ++i) *reinterpret_cast<float2*>(dst + 8 * i) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
                if ((lane & 3) == 0) scratch_ml[w * rows + r] = make_float2(m[h] == -INFINITY ? m[h] : m[h] * p.c, sum);
            }
        }
        if (any_failed(ok)) break;
        const int live_rows = min(rows, p.group - it.row_block * kMaxRows);
        const int head0 = it.kv_head * p.group + it.row_block * kMaxRows;
        const int64_t part0 = static_cast<int64_t>(it.index) * rows;   // piece c at + c * rows
        for (int i = threadIdx.x - 32; i < live_rows * (DP / 2); i += 128) {   // a thread: two dims of a row
            const int r = i / (DP / 2), d = 2 * (i % (DP / 2));
            float2 ml[4];
            float top = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                ml[k] = scratch_ml[k * rows + r];
                top = fmaxf(top, ml[k].x);
            }
            float2 x = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                // (no key: weight 0; a NaN reference or sum makes the row NaN)
                const float f = ml[k].x == -INFINITY ? 0.0f : exp2_fast(ml[k].x - top);
                const float2 y = *reinterpret_cast<const float2*>(scratch_o + (k * rows + r) * DP + d);
                sum = __fmaf_rn(f, ml[k].y, sum);
                x.x = __fmaf_rn(f, y.x, x.x);
                x.y = __fmaf_rn(f, y.y, x.y);
            }
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            const float lse = top + log2f(sum);   // no key: -inf
            if (!it.in_pieces && !p.has_prefix) {
                if (d < p.a.cache.head_dim)
                    *reinterpret_cast<__nv_bfloat162*>(p.a.rows.out + it.seq * p.a.rows.out_row +
                                                       (head0 + r) * p.a.rows.out_head + d) =
                        __floats2bfloat162_rn(x.x * inv, x.y * inv);
                if (d == 0 && p.a.rows.lse)
                    p.a.rows.lse[static_cast<int64_t>(it.seq) * p.a.rows.n_q_heads + head0 + r] = lse * kLn2;
            } else {
                const int64_t at = part0 + static_cast<int64_t>(blockIdx.x) * rows + r;
                *reinterpret_cast<float2*>(p.w.part_o + at * DP + d) = make_float2(x.x * inv, x.y * inv);
                if (d == 0) p.w.part_lse[at] = lse;
            }
        }
        if (it.in_pieces && !p.has_prefix) {   // the CTA that comes last joins them
            __threadfence();
            sync_consumers();
            if (threadIdx.x == 32) {
                const int before = atomicAdd(p.w.tickets + it.index, 1);
                *last = before == c1 - c0;
                if (*last) p.w.tickets[it.index] = 0;
                __threadfence();
            }
            sync_consumers();
            if (*last)
                for (int i = threadIdx.x - 32; i < live_rows * (DP / 4); i += 128) {
                    const int r = i / (DP / 4), d = 4 * (i % (DP / 4));
                    PartSum<DP> sum;
                    sum.add(p.w.part_lse, p.w.part_o, part0 + r, rows, c0, c1, d);
                    sum.write(p.a, it.seq, head0 + r, d);
                }
        }
    }   // (the next item's first barrier comes before its writes to the scratch)
    // the join that follows reads the prefixes' results too: this kernel does not end before theirs
    if (p.has_prefix) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// With prefixes: the rows' own pieces and those of their group's prefix, a block for each sequence and key head.
template <int DP>
__global__ void __launch_bounds__(256) decode_join_kernel(const __grid_constant__ DecodeParams p) {
    const AttnParams& a = p.a;
    const int lane = threadIdx.x & 31, kv_heads = a.cache.n_kv_heads;
    const int s = blockIdx.x / kv_heads, kv_head = blockIdx.x % kv_heads, head0 = kv_head * p.group;
    const int g = find_sequence(a.prefix.group_offsets, a.prefix.n_groups, s, lane);
    const int keys = checked_len(__ldg(a.batch.kv_lens + s), a.batch.max_pages, a.cache.page_shift, a.err, kErrKvLens);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (blockIdx.x == 0 && threadIdx.x == 0) p.w.prefix.counters[2] = 0;
    const int chunk = *p.w.chunk, real = units_with_tiles(keys, chunk), units = real + (chunk == 1 ? kItemUnits : 0);
    const int64_t per = *p.w.units_per_cta, first_of_seq = s > 0 ? p.w.unit_end[s - 1] : 0;
    PieceSpan at{0, 1, 0};
    if (g >= 0) at = piece_span<true>(a, p.w.prefix, g, s, head0, p.tile_tokens);
    for (int i = threadIdx.x; i < p.group * (DP / 4); i += blockDim.x) {
        const int r = i / (DP / 4), d = 4 * (i % (DP / 4));
        const int j = kv_head * p.plan.row_blocks + r / kMaxRows;
        const int64_t first = first_of_seq + static_cast<int64_t>(j) * units;
        const int64_t item = static_cast<int64_t>(s) * kv_heads * p.plan.row_blocks + j;
        PartSum<DP> sum;
        sum.add(p.w.part_lse, p.w.part_o, item * p.plan.rows + r % kMaxRows, p.plan.rows,
                static_cast<int>(divide(first, per)), static_cast<int>(divide(first + real - 1, per)), d);
        if (at.c0 <= at.c1) sum.add(p.w.prefix.part_lse, p.w.prefix.part_o, at.base + r, kPartRows, at.c0, at.c1, d);
        sum.write(a, s, head0 + r, d);
    }
}

template <int DP>
cudaError_t launch_dim(DecodeParams& p, cudaStream_t stream) {
    CUtensorMap q, k, v;
    if (!make_row_map(&q, p.a, 1, p.plan.rows) || !make_cache_map(&k, p.a.cache, p.a.cache.k, kKeys) ||
        !make_cache_map(&v, p.a.cache, p.a.cache.v, kKeys))
        return cudaErrorInvalidValue;
    p.stages = DecodeCfg<DP>::stages(p.plan.rows);
    const size_t smem = DecodeCfg<DP>::bytes(p.plan.rows);
    static std::atomic<uint64_t> attr_set{0};   // one bit per device ordinal whose attribute is set
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (!(attr_set.load(std::memory_order_acquire) & bit)) {
        e = cudaFuncSetAttribute(decode_kernel<DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBudget);
        if (e != cudaSuccess) return e;
        attr_set.fetch_or(bit, std::memory_order_acq_rel);
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(p.plan.grid);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // starts as the prefix kernel drains
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.has_prefix ? 1 : 0;
    e = cudaLaunchKernelEx(&cfg, decode_kernel<DP>, q, k, v, p);
    if (e != cudaSuccess || !p.has_prefix) return e;
    cfg.gridDim = dim3(static_cast<unsigned>(static_cast<int64_t>(p.a.batch.n_seqs) * p.a.cache.n_kv_heads));
    cfg.blockDim = dim3(join_threads(p.group, DP));
    cfg.dynamicSmemBytes = 0;
    return cudaLaunchKernelEx(&cfg, decode_join_kernel<DP>, p);
}

}  // namespace

DecodePlan plan_decode(const AttnParams& a, int sms) {
    const int group = a.rows.n_q_heads / a.cache.n_kv_heads;
    DecodePlan plan{};
    plan.sms = sms;
    plan.rows = std::min(group, kMaxRows);
    plan.row_blocks = (group + kMaxRows - 1) / kMaxRows;
    plan.dim = a.cache.head_dim <= 64 ? 64 : 128;
    plan.items = static_cast<int64_t>(a.batch.n_seqs) * a.cache.n_kv_heads * plan.row_blocks;
    const int64_t tiles = (static_cast<int64_t>(a.batch.max_pages) * a.cache.page_size + kKeys - 1) / kKeys;
    plan.grid = static_cast<int>(std::min<int64_t>(plan.items * tiles, 2 * sms));
    plan.part_rows = (plan.items + plan.grid) * plan.rows;
    return plan;
}

cudaError_t launch_decode_attention(const AttnParams& a, const DecodePlan& plan, const DecodeWork& w, cudaStream_t stream) {
    const Geometry g = geometry(a);
    DecodeParams p{a, plan, w, g.group, g.tile_tokens, 0, a.rows.scale < 0.0f,
                   a.cache.page_size >= kKeys ? 1 : kKeys / a.cache.page_size, a.prefix.n_groups > 0, plan.sms,
                   exp2_scale(a.rows.scale)};
    return plan.dim == 64 ? launch_dim<64>(p, stream) : launch_dim<128>(p, stream);
}

}  // namespace vw
